"""Register budgets of the kernels of ``nn`` over time, norms and lists (as tests/test_build_resources_nn.py)."""

import json
from pathlib import Path

import pytest

RESOURCES = Path(__file__).resolve().parents[1] / "open-pacho_amd" / "_build" / "resources.json"


@pytest.fixture(scope="module")
def resources():
    if not RESOURCES.exists():
        pytest.skip("library not built in this tree (open-pacho_amd/build.py)")
    return json.loads(RESOURCES.read_text())


# Lists of whole rows keep up to 17 values that do not change from row to row in memory, which the row's registers need.
# The scan's gradient in double precision takes a wave a SIMD, and accumulation registers beside the others.
@pytest.mark.parametrize("unit,waves,scratch", [("residual", 2, 0), ("conv", 2, 0), ("scan", 2, 0), ("scan_backward", 1, 0), ("distillation", 2, 64)])
def test_kernels_do_not_spill_and_keep_their_waves(resources, unit, waves, scratch):
    kernels = {name: r for name, r in resources.get(unit, {}).items() if "kernel" in name}
    assert kernels, unit
    for name, r in kernels.items():
        assert r.get("ScratchSize [bytes/lane]", 0) <= scratch, (name, r)
        assert r.get("Dynamic Stack") in (None, "False"), (name, r)
        assert r["Occupancy [waves/SIMD]"] >= waves, (name, r)


def test_float32_gradients_of_scans_keep_two_waves(resources):
    kernels = {n: r for n, r in resources["scan_backward"].items() if "backward_kernelIf" in n}
    assert kernels
    for name, r in kernels.items():
        assert r["Occupancy [waves/SIMD]"] >= 2 and r.get("AGPRs", 0) == 0, (name, r)
