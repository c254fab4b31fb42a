"""Residual addition + RMSNorm (csrc/add_rmsnorm.cu): rules and binding to the native library."""

from __future__ import annotations

from .module import KernelModule, KernelSpec

OUTPUTS = ("same", "e4m3")
GROUPS = (0, 32, 64, 128, 256)
E4M3_MAX = 448.0


def check_add_rmsnorm(M: int, N: int, dtype: str, out: str, group: int) -> None:
    assert M >= 0 and 0 < N <= 1 << 30
    assert dtype in ("float16", "bfloat16")
    assert out in OUTPUTS, f"out is one of {OUTPUTS}"
    assert group in GROUPS, f"group is one of {GROUPS} (0: one scale a row)"
    assert out == "e4m3" or group == 0, "groups belong to the 8-bit output"


def scale_columns(N: int, group: int) -> int:
    return -(-N // group) if group else 1


def make_add_rmsnorm(M: int, N: int, dtype: str, eps: float, out: str, group: int) -> KernelSpec:
    check_add_rmsnorm(M, N, dtype, out, group)
    return KernelSpec("add_rmsnorm", (M, N), dtype, {}, {"eps": float(eps), "out": out, "group": group})


def build_add_rmsnorm(mod: KernelSpec) -> KernelModule:
    return KernelModule(mod)


def bind(spec: KernelSpec):
    """Returns main(x, res, w[, h, y, scales]) launching deca_add_rmsnorm on torch's current stream; it returns
    (h, y) or (h, y, scales), made where they are not given."""
    from functools import partial

    from .. import native

    M, N = spec.shape
    out, group = spec.params["out"], spec.params["group"]
    check_add_rmsnorm(M, N, spec.dtype, out, group)
    launch = native.launch()
    plan = launch.add_rmsnorm_plan(native.DTYPE_CODE[spec.dtype], M, N, scale_columns(N, group), spec.params["eps"],
                                   native.OUT_E4M3 if out == "e4m3" else native.OUT_SAME, group)
    return partial(launch.add_rmsnorm, plan)
