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


def frequencies(rot, base=10000.0, kind=None, factor=1.0, length=0, low=0.0, high=0.0):
    """Radians per position from the definitions: pair i turns at base^(-2 i / rot); "linear" divides by the factor; "base"
    raises the base so that the last pair is slowed by the factor and the first stays; "band" keeps what turns more than
    `high` times in `length` positions, divides what turns less than `low` times and mixes linearly in between."""
    out = []
    for i in range(rot // 2):
        f = math.exp(-2.0 * i / rot * math.log(base))
        if kind == "linear":
            f /= factor
        elif kind == "base":
            f *= math.exp(-2.0 * i / (rot - 2) * math.log(factor))  # (factor^(rot / (rot - 2)))^(-2 i / rot)
        elif kind == "band":
            turns = length * f / (2.0 * math.pi)
            if turns <= low:
                f /= factor
            elif turns < high:
                share = (turns - low) / (high - low)
                f = share * f + (1.0 - share) * f / factor
        out.append(f)
    return out


@pytest.mark.parametrize("D,rot", [(128, 128), (128, 64), (64, 16), (256, 256), (80, 20), (96, 4)])
@pytest.mark.parametrize("base", [10000.0, 500000.0, 1.0])
@pytest.mark.parametrize("scaling", [None, {"type": "linear", "factor": 4.0}, {"type": "base", "factor": 4.0}, {"type": "base", "factor": 1.0},
                                     {"type": "band", "factor": 8.0, "original_length": 4096, "low": 1.0, "high": 32.0},
                                     {"type": "band", "factor": 32.0, "original_length": 8192, "low": 1.0, "high": 4.0},
                                     {"type": "band", "factor": 4.0, "original_length": 300, "low": 0.25, "high": 40.0}])
def test_frequencies(scaling, base, D, rot):
    """Within a few roundings of 64 bits: exp and log of arguments up to 20 err by 20 2^-53 each."""
    s = scaling or {}
    want = frequencies(rot, base, s.get("type"), s.get("factor", 1.0), s.get("original_length", 0), s.get("low", 0.0), s.get("high", 0.0))
    for op in (Rotary(D, rot_dim=rot, base=base, scaling=scaling), RotaryAppend(4, 2, D, 16, rot_dim=rot, base=base, scaling=scaling)):
        got, amplitude = op.frequencies()
        assert len(got) == rot // 2
        for i, (a, b) in enumerate(zip(got, want)):
            assert abs(a - b) <= 1e-13 * b, f"pair {i}"
        assert amplitude == pytest.approx(0.1 * math.log(s["factor"]) + 1.0 if s.get("type") == "band" else 1.0, rel=1e-15)


def test_band_has_pairs_on_both_sides_and_between():
    """The case above is no empty statement: of 64 pairs some keep their frequency, some are divided, some are mixed."""
    plain = frequencies(128)
    band = frequencies(128, kind="band", factor=8.0, length=4096, low=1.0, high=32.0)
    kept = sum(a == b for a, b in zip(plain, band))
    divided = sum(b == a / 8.0 for a, b in zip(plain, band))
    assert kept > 10 and divided > 10 and 64 - kept - divided > 10


def test_ends_of_the_base_scaling():
    """The fastest pair stays, the slowest is slowed by the factor."""
    plain, slow = (Rotary(128, scaling=s).frequencies()[0] for s in (None, {"type": "base", "factor": 4.0}))
    assert slow[0] == plain[0] == 1.0 and slow[-1] == pytest.approx(plain[-1] / 4.0, rel=1e-12)


@pytest.mark.parametrize("given", [0.5, 1.0, 1.2])
def test_band_amplitude_may_be_given(given):
    scaling = {"type": "band", "factor": 8.0, "original_length": 4096, "low": 1.0, "high": 32.0, "amplitude": given}
    assert Rotary(128, scaling=scaling).frequencies()[1] == given
