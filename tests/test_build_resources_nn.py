"""Register budgets of the kernels of ``nn`` (as tests/test_build_resources.py):
no kernel spills a vector register to memory, and the ones that have to hide the
memory's latency keep their waves."""

import json
from pathlib import Path

import pytest

RESOURCES = Path(__file__).resolve().parents[1] / "open-pacho_amd" / "_build" / "resources.json"


@pytest.fixture(scope="module")
def resources():
    if not RESOURCES.exists():
        pytest.skip("library not built in this tree (open-pacho_amd/build.py)")
    return json.loads(RESOURCES.read_text())


@pytest.mark.parametrize("unit,waves", [("recurrence", 2), ("token_loss", 2), ("adamw", 8)])
def test_kernels_do_not_spill_and_keep_their_waves(resources, unit, waves):
    kernels = {name: r for name, r in resources.get(unit, {}).items() if "kernel" in name}
    assert kernels, unit
    for name, r in kernels.items():
        assert r.get("VGPRs Spill", 0) == 0 and r.get("ScratchSize [bytes/lane]", 0) == 0, (name, r)
        assert r.get("Dynamic Stack") in (None, "False"), (name, r)
        assert r["Occupancy [waves/SIMD]"] >= waves, (name, r)


def test_chained_tiles_leave_room_for_a_second_workgroup(resources):
    # Eight waves each: while one waits for the tiles before it, another loads.
    kernels = {n: r for n, r in resources["recurrence"].items() if "chained_kernel" in n}
    assert kernels
    for name, r in kernels.items():
        assert r["Occupancy [waves/SIMD]"] >= 4, (name, r)
