"""Rotary positions (csrc/rotary.cu): frequencies, rules and binding to the native library.

The kernels take the frequencies as 64-bit fixed-point fractions of a turn per position (``turns``), so
that an angle is exact modulo a turn at any position.  Scaling for long contexts changes only the
frequencies and an amplitude, both computed here once per operator:

* ``{"type": "linear", "factor": s}``: every frequency divided by s (positions interpolated);
* ``{"type": "base", "factor": s}``: the base multiplied by s ** (rot_dim / (rot_dim - 2)), which leaves the
  fastest pair as it is and slows the slowest one down by s;
* ``{"type": "band", "factor": s, "original_length": L, "low": a, "high": b[, "amplitude": m]}``: pairs
  that turn more than b times within the L positions of training keep their frequency, those that turn
  less than a times are divided by s, the ones between are mixed linearly; the amplitude, a factor on cos
  and sin, is m, or 0.1 ln s + 1.
"""

from __future__ import annotations

import math
from fractions import Fraction

from .module import KernelModule, KernelSpec

LAYOUTS = ("half", "interleaved")
MAX_HEAD_DIM = 256
PI_BITS = int(Fraction("3.14159265358979323846264338327950288419716939937510") * 2**160)  # pi * 2^160


def rotary_frequencies(rot_dim: int, base: float = 10000.0, scaling: dict | None = None):
    """([radians per position of every pair], amplitude) in double precision."""
    if base < 1.0:
        raise ValueError("base: at least 1")
    kind = None if scaling is None else scaling.get("type")
    if kind not in (None, "linear", "base", "band"):
        raise ValueError(f"scaling: unknown type {kind!r}")
    allowed = {None: set(), "linear": {"type", "factor"}, "base": {"type", "factor"},
               "band": {"type", "factor", "original_length", "low", "high", "amplitude"}}[kind]
    unknown = set(scaling or ()) - allowed
    if unknown:
        raise ValueError(f"scaling: unknown entries {sorted(unknown)}")
    factor = 1.0 if kind is None else float(scaling["factor"])
    if not (1.0 <= factor < math.inf):
        raise ValueError("scaling: factor of at least 1")
    if kind == "base":
        if rot_dim <= 2:
            raise ValueError("scaling: the base of a single pair cannot be scaled")
        base = base * factor ** (rot_dim / (rot_dim - 2))
    freq = [base ** (-2.0 * i / rot_dim) for i in range(rot_dim // 2)]
    amplitude = 1.0
    if kind == "linear":
        freq = [f / factor for f in freq]
    if kind == "band":
        low, high, length = float(scaling["low"]), float(scaling["high"]), float(scaling["original_length"])
        if not high > low:
            raise ValueError("scaling: high must exceed low")
        keep = [min(max((length * f / (2 * math.pi) - low) / (high - low), 0.0), 1.0) for f in freq]
        freq = [f * k + f / factor * (1.0 - k) for f, k in zip(freq, keep)]
        amplitude = float(scaling.get("amplitude", 0.1 * math.log(factor) + 1.0))
    return freq, amplitude


def fixed_point_turns(freq):
    """Fractions of a turn per position as 64-bit integers (a turn is 2 ** 64), rounded down.  Whole-number
    arithmetic: a double quotient would be off by 4e-7 rad at position 2 ** 31."""
    ratios = (f.as_integer_ratio() for f in freq)
    return [(n << 223) // (d * PI_BITS) % 2**64 for n, d in ratios]


def check_rotary(D: int, rot_dim: int, layout: str, dtype: str) -> None:
    assert dtype in ("float16", "bfloat16")
    assert layout in LAYOUTS, f"layout is one of {LAYOUTS}"
    assert 2 <= D <= MAX_HEAD_DIM and D % 2 == 0, "head dim even, 2 to 256"
    assert 2 <= rot_dim <= D and rot_dim % 2 == 0, "rot_dim even, 2 to the head dim"


def make_rotary(D: int, rot_dim: int, base: float, layout: str, scaling, dtype: str) -> KernelSpec:
    check_rotary(D, rot_dim, layout, dtype)
    rotary_frequencies(rot_dim, base, scaling)
    return KernelSpec("rotary", (D,), dtype, {}, {"rot_dim": rot_dim, "base": base, "layout": layout, "scaling": scaling})


def make_rotary_append(H_q: int, H_kv: int, D: int, page_size: int, rot_dim: int, base: float, layout: str, scaling,
                       dtype: str) -> KernelSpec:
    check_rotary(D, rot_dim, layout, dtype)
    rotary_frequencies(rot_dim, base, scaling)
    assert H_q >= 1 and H_kv >= 1
    assert page_size >= 1 and page_size & (page_size - 1) == 0, "page size a power of two"
    return KernelSpec("rotary_append", (H_q, H_kv, D, page_size), dtype, {},
                      {"rot_dim": rot_dim, "base": base, "layout": layout, "scaling": scaling})


def build_rotary(mod: KernelSpec) -> KernelModule:
    return KernelModule(mod)


def _plan(launch, dtype: str, D: int, p: dict, H_q: int = 0, H_kv: int = 0, page_size: int = 0):
    from .. import native

    freq, amplitude = rotary_frequencies(p["rot_dim"], p["base"], p["scaling"])
    layout = native.ROT_HALF if p["layout"] == "half" else native.ROT_INTERLEAVED
    return launch.rotary_plan(native.DTYPE_CODE[dtype], D, p["rot_dim"], layout, H_q, H_kv, page_size, amplitude,
                              fixed_point_turns(freq))


def bind(spec: KernelSpec):
    """Returns main(x, positions[, y, inverse]) launching deca_rotary on torch's current stream; it returns y."""
    from functools import partial

    from .. import native

    launch = native.launch()
    return partial(launch.rotary, _plan(launch, spec.dtype, *spec.shape, spec.params))


def bind_append(spec: KernelSpec):
    """Returns main(q, k, v, positions, slots, k_cache, v_cache[, q_out]) launching deca_rotary_append on torch's
    current stream; it returns q_out."""
    from functools import partial

    from .. import native

    launch = native.launch()
    H_q, H_kv, D, page_size = spec.shape
    return partial(launch.rotary_append, _plan(launch, spec.dtype, D, spec.params, H_q, H_kv, page_size))
