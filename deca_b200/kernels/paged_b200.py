"""Serving over a paged cache (csrc/paged_step.cu, csrc/paged_attn*.cu): rules and binding of the step's
bookkeeping and of the attention to the native library."""

from __future__ import annotations

import math

from .module import KernelModule, KernelSpec

MAX_REQUESTS = 8192  # the step's prefix sums live in one CTA's shared memory
PAGE_SIZES = (16, 32, 64, 128, 256)
MAX_GROUP = 128


def check_step(B: int, page_size: int, table_width: int, max_tokens: int) -> None:
    assert 1 <= B <= MAX_REQUESTS, f"1 to {MAX_REQUESTS} requests"
    assert page_size >= 1 and page_size & (page_size - 1) == 0, "page size a power of two"
    assert table_width >= 1 and table_width * page_size < 2**31
    assert 0 <= max_tokens < 2**31


def check_attn(B: int, H_q: int, H_kv: int, D: int, page_size: int, max_q: int, max_kv: int, dtype: str) -> None:
    assert dtype in ("float16", "bfloat16")
    assert B >= 1 and max_q >= 0 and max_kv >= 0
    assert D in (64, 128), "head dim 64 or 128"
    assert H_kv >= 1 and H_q >= 1 and H_q % H_kv == 0, "H_q a multiple of H_kv"
    assert H_q // H_kv <= MAX_GROUP, f"at most {MAX_GROUP} query heads share a key head"
    assert page_size in PAGE_SIZES, f"page size one of {PAGE_SIZES}"


def make_paged_step(B: int, page_size: int, table_width: int, max_tokens: int) -> KernelSpec:
    check_step(B, page_size, table_width, max_tokens)
    return KernelSpec("paged_step", (B, page_size, table_width, max_tokens), "int32", {}, {})


def make_paged_attn(B: int, H_q: int, H_kv: int, D: int, page_size: int, max_q: int, max_kv: int, dtype: str,
                    softmax_scale: float | None = None, causal: bool = True) -> KernelSpec:
    check_attn(B, H_q, H_kv, D, page_size, max_q, max_kv, dtype)
    scale = softmax_scale if softmax_scale is not None else 1.0 / math.sqrt(D)
    assert math.isfinite(scale)
    return KernelSpec("paged_attn", (B, H_q, H_kv, D, page_size, max_q, max_kv), dtype, {},
                      {"softmax_scale": float(scale), "causal": bool(causal)})


def build_paged(mod: KernelSpec) -> KernelModule:
    return KernelModule(mod)


def bind_step(spec: KernelSpec):
    """Returns main(ctx_lens, new_lens, block_table, free_pages, n_free[, cu_q, kv_lens, positions, slots, n_free_out,
    short]) launching deca_paged_step on torch's current stream; it returns the six outputs, made where they
    are not given."""
    from functools import partial

    from .. import native

    launch = native.launch()
    return partial(launch.paged_step, launch.paged_step_plan(*spec.shape))


def bind_attn(spec: KernelSpec):
    """Returns main(q, k_cache, v_cache, block_table, cu_q, kv_lens[, out]) launching deca_paged_attn on torch's
    current stream; it returns out.  The workspace is allocated per call."""
    from functools import partial

    from .. import native

    B, H_q, H_kv, D, page_size, max_q, max_kv = spec.shape
    check_attn(B, H_q, H_kv, D, page_size, max_q, max_kv, spec.dtype)
    launch = native.launch()
    plan = launch.paged_attn_plan(native.DTYPE_CODE[spec.dtype], B, H_q, H_kv, D, page_size, int(spec.params["causal"]),
                                  spec.params["softmax_scale"], max_q, max_kv)
    return partial(launch.paged_attn, plan)
