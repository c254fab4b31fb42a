"""Serving over a paged cache (csrc/paged_step.cu, csrc/paged_attn*.cu): rules and binding of the step's
bookkeeping and of the attention to the native library."""

from __future__ import annotations

import math

from .module import KernelModule, KernelSpec, _check_view, current_stream_ptr

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
    """Returns main(ctx_lens, new_lens, block_table, free_pages, n_free, cu_q, kv_lens, positions, slots,
    n_free_out, short) launching deca_paged_step on torch's current stream."""
    import torch

    from .. import native

    L = native.lib()
    B, page_size, W, T = spec.shape
    i32, i64 = torch.int32, torch.int64

    def main(ctx_lens, new_lens, block_table, free_pages, n_free, cu_q, kv_lens, positions, slots, n_free_out, short):
        _check_view(ctx_lens, (B,), i32, "ctx_lens")
        _check_view(new_lens, (B,), i32, "new_lens")
        _check_view(block_table, (B, W), i32, "block_table")
        _check_view(free_pages, (None,), i32, "free_pages")
        _check_view(n_free, (1,), i32, "n_free")
        _check_view(cu_q, (B + 1,), i32, "cu_q")
        _check_view(kv_lens, (B,), i32, "kv_lens")
        _check_view(positions, (T,), i32, "positions")
        _check_view(slots, (T,), i64, "slots")
        _check_view(n_free_out, (1,), i32, "n_free_out")
        _check_view(short, (1,), i32, "short")
        stride = block_table.stride(0) if B > 1 else W
        if stride < W:
            raise ValueError(f"block_table: rows overlap (row stride {stride} for {W} entries)")
        native.check(
            L.deca_paged_step(ctx_lens.data_ptr(), new_lens.data_ptr(), B, block_table.data_ptr(), stride, W,
                              free_pages.data_ptr(), free_pages.shape[0], n_free.data_ptr(), page_size, T, cu_q.data_ptr(),
                              kv_lens.data_ptr(), positions.data_ptr(), slots.data_ptr(), n_free_out.data_ptr(),
                              short.data_ptr(), current_stream_ptr()), "deca_paged_step")

    return main


def bind_attn(spec: KernelSpec):
    """Returns main(q, k_cache, v_cache, block_table, cu_q, kv_lens, out) launching deca_paged_attn on torch's
    current stream.  The workspace is allocated per call (torch's caching allocator), so calls that
    overlap, captured ones too, never share one."""
    import ctypes

    import torch

    from .. import native

    L = native.lib()
    B, H_q, H_kv, D, page_size, max_q, max_kv = spec.shape
    check_attn(B, H_q, H_kv, D, page_size, max_q, max_kv, spec.dtype)
    tdt, i32 = getattr(torch, spec.dtype), torch.int32
    a0 = native.PagedAttnArgs(dtype=native.DTYPE_CODE[spec.dtype], B=B, H_q=H_q, H_kv=H_kv, D=D, page_size=page_size,
                              causal=int(spec.params["causal"]), scale=spec.params["softmax_scale"], max_q=max_q,
                              max_kv=max_kv)
    template = bytes(a0)
    workspace_of = {}  # device -> bytes

    def workspace_bytes(device):
        n = ctypes.c_size_t()
        native.check(L.deca_paged_attn_workspace_bytes(ctypes.byref(a0), ctypes.byref(n)), "deca_paged_attn_workspace_bytes")
        workspace_of[device] = n.value
        return n.value

    def main(q, k_cache, v_cache, block_table, cu_q, kv_lens, out):
        _check_view(q, (None, H_q, D), tdt, "q")
        T = q.shape[0]
        _check_view(out, (T, H_q, D), tdt, "out")
        _check_view(k_cache, (None, page_size, H_kv, D), tdt, "k_cache")
        pages = k_cache.shape[0]
        _check_view(v_cache, (pages, page_size, H_kv, D), tdt, "v_cache")
        _check_view(block_table, (B, None), i32, "block_table")
        _check_view(cu_q, (B + 1,), i32, "cu_q")
        _check_view(kv_lens, (B,), i32, "kv_lens")
        if H_q > 1 and out.stride(1) < D or T > 1 and out.stride(0) < 1:
            raise ValueError(f"out: elements overlap (strides {tuple(out.stride())})")
        if T == 0:
            return
        dev = q.get_device()
        n = workspace_of.get(dev) or workspace_bytes(dev)
        ws = torch.empty(n, dtype=torch.uint8, device=q.device)
        a = native.PagedAttnArgs.from_buffer_copy(template)
        a.T, a.num_pages, a.table_width = T, pages, block_table.shape[1]
        a.table_stride = block_table.stride(0) if B > 1 else block_table.shape[1]
        t = a.Q
        t.data, t.token_stride, t.head_stride = q.data_ptr(), q.stride(0), q.stride(1)
        t = a.O
        t.data, t.token_stride, t.head_stride = out.data_ptr(), out.stride(0), out.stride(1)
        for c, x in ((a.K, k_cache), (a.V, v_cache)):
            c.data = x.data_ptr()
            c.page_stride, c.row_stride, c.head_stride, _ = x.stride()
        a.block_table, a.cu_q, a.kv_lens = block_table.data_ptr(), cu_q.data_ptr(), kv_lens.data_ptr()
        a.workspace, a.workspace_bytes = ws.data_ptr(), n
        native.check(L.deca_paged_attn(ctypes.byref(a), current_stream_ptr()), "deca_paged_attn")

    return main
