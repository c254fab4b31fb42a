"""Rules and frequencies of the rotary operators, restated without the package's own functions (no GPU is needed)."""

import math

import pytest

from deca_b200.operators import Rotary, RotaryAppend


def test_no_rotated_elements_is_not_all_of_them():
    """rot_dim left out means the whole head; a rot_dim of 0 has no pair to turn and is refused."""
    assert Rotary(64).rot_dim == 64 and Rotary(64, rot_dim=32).rot_dim == 32
    for make in (lambda: Rotary(64, rot_dim=0), lambda: RotaryAppend(4, 2, 64, 16, rot_dim=0)):
        with pytest.raises(AssertionError):
            make()
