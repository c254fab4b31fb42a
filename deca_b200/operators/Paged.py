"""Serving over a paged cache: the bookkeeping of a step (``PagedStep``) and the attention of its new
tokens (``PagedAttention``)."""

import math
from collections import namedtuple

from ..kernels.module import BuiltInSchedule
from ..kernels.paged_b200 import make_paged_attn, make_paged_step
from .Op import Operator

PagedStepResult = namedtuple("PagedStepResult", "cu_q kv_lens positions slots n_free short")


class PagedStep(Operator):
    """From the cached and new lengths of B requests: prefix sums, pages, positions and slots, on the device
    and in one launch, so a step (captured in a graph, say) needs no lengths on the host.

    ``table_width``: entries of a request's block table; ``max_tokens``: token rows of the step (rows behind the
    last token get position 0 and slot -1).
    """

    def __init__(self, B: int, page_size: int, table_width: int, max_tokens: int, name: str = "PagedStep"):
        self.B, self.page_size, self.table_width, self.max_tokens = B, page_size, table_width, max_tokens
        self._mod = None
        super().__init__(name=name)
        self.build_mod()

    @property
    def shape(self):
        return (self.B, self.page_size, self.table_width, self.max_tokens)

    def default_config(self):
        return BuiltInSchedule()

    def is_valid(self, cfg) -> bool:
        return isinstance(cfg, BuiltInSchedule)

    def build_mod(self, cfg=None):
        return make_paged_step(*self.shape)

    def compile(self, mod):
        from ..kernels.paged_b200 import build_paged

        return build_paged(mod)

    def __call__(self, ctx_lens, new_lens, block_table, free_pages, n_free, out: PagedStepResult | None = None):
        """ctx_lens, new_lens [B], block_table [B, table_width], free_pages [F], n_free [1], all int32.

        Pages for the new tokens are taken from the end of ``free_pages[:n_free]`` in request order and written
        to ``block_table`` in place (-1 where the list has run out).  Returns cu_q [B + 1], kv_lens [B],
        positions and slots [max_tokens], n_free [1] and short [1] (pages that were missing; 0: none), in the
        tensors of ``out`` (the result of another call, say), which may not be the inputs' own."""
        if self._mod is None:
            self._mod = self.compile(self.build_mod())["main"]
        return PagedStepResult(*self._mod(ctx_lens, new_lens, block_table, free_pages, n_free, *(out or ())))

    def describe(self) -> str:
        return (f"{self.name}(B={self.B}, page_size={self.page_size}, table_width={self.table_width}, "
                f"max_tokens={self.max_tokens})")


class PagedAttention(Operator):
    """Attention of each request's newest tokens over its cached keys and values, which lie in pages.

    ``B`` requests; ``H_q`` query heads share ``H_kv`` key heads; D = 64 or 128; page sizes 16 to 256 (powers of
    two); fp16 or bf16 with fp32 scores, statistics and accumulators.  ``max_q`` and ``max_kv`` are the caller's
    bounds on a request's new and cached tokens: they choose the schedule, any value gives right
    results.  A capacity for ``max_kv`` costs a step of short contexts at most 3 us; a chunk's budget for ``max_q`` makes
    a step that only decodes up to twice as slow, so keep one operator for decoding (``max_q`` 1, or the length of a guess)
    and one for chunks.  ``causal``: a token sees the keys up to its own place (its request's new tokens are the last of
    its ``kv_lens`` keys); otherwise all of them.  A token that sees nothing gets zeros.
    """

    metric = "TFLOPS"

    def __init__(self, B: int, H_q: int, H_kv: int, D: int, page_size: int, max_q: int, max_kv: int,
                 dtype: str = "float16", softmax_scale: float | None = None, causal: bool = True,
                 name: str = "PagedAttention"):
        from ..kernels.rowwise_bench import canonical_dtype

        self.B, self.H_q, self.H_kv, self.D, self.page_size = B, H_q, H_kv, D, page_size
        self.max_q, self.max_kv = max_q, max_kv
        self.dtype = canonical_dtype(dtype)
        self.softmax_scale = softmax_scale if softmax_scale is not None else 1.0 / math.sqrt(D)
        self.causal = causal
        seen = max_q * max_kv - (max_q * (max_q - 1) // 2 if causal else 0)
        self.num_flops = 4 * B * H_q * D * max(seen, 0)  # of a batch of max_q new tokens behind max_kv - max_q
        self._mod = None
        super().__init__(name=name)
        self.build_mod()

    @property
    def shape(self):
        return (self.B, self.H_q, self.H_kv, self.D, self.page_size, self.max_q, self.max_kv)

    @property
    def tolerance(self):
        """(atol, rtol) against fp32 attention on values of order one: the output's rounding and that of the
        16-bit probabilities."""
        return (2e-3, 2e-3) if self.dtype == "float16" else (1.6e-2, 1.6e-2)

    def default_config(self):
        return BuiltInSchedule()

    def is_valid(self, cfg) -> bool:
        return isinstance(cfg, BuiltInSchedule)

    def build_mod(self, cfg=None):
        return make_paged_attn(*self.shape, dtype=self.dtype, softmax_scale=self.softmax_scale, causal=self.causal)

    def compile(self, mod):
        from ..kernels.paged_b200 import build_paged

        return build_paged(mod)

    def __call__(self, q, k_cache, v_cache, block_table, cu_q, kv_lens, out=None):
        """q [T, H_q, D]: request r owns rows cu_q[r] .. cu_q[r + 1] - 1; caches [pages, page_size, H_kv, D];
        block_table [B, width], cu_q [B + 1], kv_lens [B], int32 on the device.  Returns O [T, H_q, D] (``out`` may
        be ``q``, and is refused where it shares memory with a tensor of the call in any other way).  Rows that belong to no
        request are not written.

        Lengths are clipped to what q and the table hold, a table entry that names no page reads as zeros, and
        what a token does not see does not reach its output, whatever the cache holds there."""
        if self._mod is None:
            self._mod = self.compile(self.build_mod())["main"]
        return self._mod(q, k_cache, v_cache, block_table, cu_q, kv_lens, out)

    def make_inputs(self):
        """A full batch from one seeded generator: max_q new tokens behind max_kv - max_q, pages in random order."""
        import torch

        dt = getattr(torch, self.dtype)
        gen = torch.Generator(device="cuda").manual_seed(0)
        width = max(-(-self.max_kv // self.page_size), 1)
        pages = self.B * width
        q = torch.randn(self.B * self.max_q, self.H_q, self.D, device="cuda", dtype=dt, generator=gen)
        k, v = (torch.randn(pages, self.page_size, self.H_kv, self.D, device="cuda", dtype=dt, generator=gen) for _ in range(2))
        table = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32).view(self.B, width)
        cu = torch.arange(self.B + 1, device="cuda", dtype=torch.int32) * self.max_q
        return q, k, v, table, cu, torch.full((self.B,), self.max_kv, device="cuda", dtype=torch.int32)

    def make_output(self, inputs):
        import torch

        return torch.empty_like(inputs[0])

    def reference(self, inputs):
        """Eager fp32 attention, request by request and head by head."""
        import torch

        q, k_cache, v_cache, table, cu_q, kv_lens = inputs
        out = torch.zeros(q.shape, dtype=torch.float32, device=q.device)
        g = self.H_q // self.H_kv
        cu, kv = cu_q.tolist(), kv_lens.tolist()
        for r in range(self.B):
            n = cu[r + 1] - cu[r]
            if n == 0 or kv[r] == 0:
                continue
            k, v = (c[table[r].long()].flatten(0, 1)[: kv[r]].float() for c in (k_cache, v_cache))
            seen = torch.arange(kv[r], device=q.device) <= kv[r] - n + torch.arange(n, device=q.device)[:, None]
            for h in range(self.H_q):
                s = q[cu[r] : cu[r + 1], h].float() @ k[:, h // g].T * self.softmax_scale
                if self.causal:
                    s = s.masked_fill(~seen, -math.inf)
                out[cu[r] : cu[r + 1], h] = torch.softmax(s, -1).nan_to_num(0.0) @ v[:, h // g]
        return out.to(q.dtype)

    def kernel_args(self, inputs, out):
        """Tensors in the kernel's argument order: q, k_cache, v_cache, block_table, cu_q, kv_lens, out."""
        return (*inputs, out)

    def describe(self) -> str:
        return (f"{self.name}(B={self.B}, H_q={self.H_q}, H_kv={self.H_kv}, D={self.D}, page_size={self.page_size}, "
                f"max_q={self.max_q}, max_kv={self.max_kv}, {self.dtype}{', causal' if self.causal else ''})")
