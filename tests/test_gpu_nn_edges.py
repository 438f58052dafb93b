"""Operators of ``nn`` on the device at the ends of what they take."""

import pytest

from test_nn_adamw import check_mixed_lists

pytestmark = pytest.mark.gpu


def test_mixed_lists(hip):
    check_mixed_lists(hip)
