"""Residual addition + RMSNorm (csrc/add_rmsnorm.cu): rules and binding to the native library."""

from __future__ import annotations

from .module import KernelModule, KernelSpec, _check_view, current_stream_ptr

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
    """Returns main(x, res, w, h, y[, scales]) launching deca_add_rmsnorm on torch's current stream."""
    import ctypes

    import torch

    from .. import native

    L = native.lib()
    M, N = spec.shape
    out, group = spec.params["out"], spec.params["group"]
    check_add_rmsnorm(M, N, spec.dtype, out, group)
    code, tdt = native.DTYPE_CODE[spec.dtype], getattr(torch, spec.dtype)
    eps = ctypes.c_float(spec.params["eps"])
    eight = out == "e4m3"
    out_code, out_dt = (native.OUT_E4M3, torch.float8_e4m3fn) if eight else (native.OUT_SAME, tdt)
    groups = scale_columns(N, group)

    def rows(t, dtype, name, written):
        _check_view(t, (M, N), dtype, name)
        if M > 1 and t.stride(0) < N:
            raise ValueError(f"{name}: rows overlap (row stride {t.stride(0)} for {N} columns)")
        return t.stride(0)

    def main(x, res, w, h, y, scales=None):
        sx, sr = rows(x, tdt, "x", False), rows(res, tdt, "res", False)
        sh, sy = rows(h, tdt, "h", True), rows(y, out_dt, "y", True)
        _check_view(w, (N,), tdt, "w")
        if eight:
            if scales is None:
                raise ValueError("scales: the e4m3 output needs a tensor for its scales")
            _check_view(scales, (M, groups), torch.float32, "scales")
            if not scales.is_contiguous():
                raise ValueError("scales: expected a contiguous tensor")
        native.check(
            L.deca_add_rmsnorm(code, x.data_ptr(), sx, res.data_ptr(), sr, w.data_ptr(), h.data_ptr(), sh, y.data_ptr(), sy,
                               scales.data_ptr() if eight else None, M, N, eps, out_code, group, current_stream_ptr()),
            "deca_add_rmsnorm")

    return main
