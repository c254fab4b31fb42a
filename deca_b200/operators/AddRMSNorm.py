"""Residual addition + RMSNorm, the form RMSNorm takes between two layers of a model, with a 16-bit or
an 8-bit output."""

from ..kernels.add_rmsnorm_b200 import E4M3_MAX, check_add_rmsnorm, make_add_rmsnorm, scale_columns
from ..kernels.module import BuiltInSchedule
from .Op import Operator


class AddRMSNorm(Operator):
    """h = x + res; y = h * rsqrt(mean(h^2) + eps) * w over the rows of [M, N] tensors (fp32 arithmetic).

    ``out="same"``: y in the inputs' type.  ``out="e4m3"``: y / s in 8 bits with fp32 scales
    s = max|y| / 448, one a row (``group=0``) or one per ``group`` columns (32, 64, 128 or 256).

    Unlike ``RMSNorm``, which rounds x * rsqrt(..) to 16 bits before the weight as its reference does, y is
    rounded once; and h is normalised before it is rounded.  Rows may be strided, N is any length.
    """

    def __init__(self, M: int, N: int, dtype: str = "float16", eps: float = 1e-6, out: str = "same", group: int = 0,
                 name: str = "AddRMSNorm"):
        from ..kernels.rowwise_bench import canonical_dtype

        self.M, self.N = M, N
        self.dtype = canonical_dtype(dtype)
        self.eps, self.out, self.group = eps, out, group
        check_add_rmsnorm(M, N, self.dtype, out, group)
        scales = 4 * M * scale_columns(N, group) if out == "e4m3" else 0
        self.num_bytes = M * N * (6 + (2 if out == "same" else 1)) + 2 * N + scales
        self._mod = None
        super().__init__(name=name)

    @property
    def shape(self):
        return (self.M, self.N)

    @property
    def tolerance(self):
        """(atol, rtol) of y against the reference: a rounding (half a step) of either side, and the fp32
        sums' order, which can move a value over a rounding boundary."""
        if self.out == "e4m3":  # in steps of the scaled value: the largest is 448, the smallest step 2^-9
            return (2.0**-8, 2.0**-3)
        return (1e-6, 2.0**-10 if self.dtype == "float16" else 2.0**-7)

    def is_valid(self, cfg) -> bool:
        return isinstance(cfg, BuiltInSchedule)

    def default_config(self):
        return BuiltInSchedule()

    def build_mod(self, cfg=None):
        return make_add_rmsnorm(self.M, self.N, self.dtype, self.eps, self.out, self.group)

    def compile(self, mod):
        from ..kernels.add_rmsnorm_b200 import build_add_rmsnorm

        return build_add_rmsnorm(mod)

    def __call__(self, x, res, w, out=None, res_out=None, scales=None):
        """Runs the kernel; returns (y, h), or (q, scales, h) with ``out="e4m3"``.  ``res_out`` may be ``res``
        or ``x`` (updated in place), ``out`` the other of them where it is 16 bits wide; an output that shares memory with
        another tensor of the call in any other way is refused."""
        if self._mod is None:
            self._mod = self.compile(self.build_mod())["main"]
        if self.out == "same":
            h, y = self._mod(x, res, w, res_out, out)
            return y, h
        h, y, scales = self._mod(x, res, w, res_out, out, scales)
        return y, scales, h

    def _scales(self, x):
        import torch

        return torch.empty((self.M, scale_columns(self.N, self.group)), dtype=torch.float32, device=x.device)

    def make_inputs(self):
        """(x, res, w) on the GPU from one seeded generator: x, res ~ N(0, 1), w = 1 + 0.1 N(0, 1)."""
        import torch

        dt = getattr(torch, self.dtype)
        gen = torch.Generator(device="cuda").manual_seed(0)
        x, res = (torch.randn(self.M, self.N, device="cuda", dtype=dt, generator=gen) for _ in range(2))
        return x, res, torch.randn(self.N, device="cuda", generator=gen).mul_(0.1).add_(1.0).to(dt)

    def make_output(self, inputs):
        import torch

        dt = torch.float8_e4m3fn if self.out == "e4m3" else inputs[0].dtype
        return torch.empty((self.M, self.N), dtype=dt, device=inputs[0].device)

    def reference(self, inputs):
        """y (or the scaled 8-bit values) in eager torch."""
        import torch
        import torch.nn.functional as F

        x, res, w = inputs
        h = x.float() + res.float()
        y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + self.eps) * w.float()
        if self.out == "same":
            return y.to(x.dtype)
        n, group = scale_columns(self.N, self.group), self.group or self.N
        y = F.pad(y, (0, n * group - self.N)).view(self.M, n, group)
        s = y.abs().amax(-1, keepdim=True) / E4M3_MAX
        q = (y / s).nan_to_num(0.0).clamp(-E4M3_MAX, E4M3_MAX)
        return q.view(self.M, n * group)[:, : self.N].to(torch.float8_e4m3fn)

    def kernel_args(self, inputs, out):
        """Tensors in the kernel's argument order: x, res, w, h, y[, scales]."""
        import torch

        h = torch.empty((self.M, self.N), dtype=inputs[0].dtype, device=inputs[0].device)
        return (*inputs, h, out) + ((self._scales(inputs[0]),) if self.out == "e4m3" else ())

    def describe(self) -> str:
        form = "" if self.out == "same" else f", e4m3{f' per {self.group}' if self.group else ''}"
        return f"{self.name}(M={self.M}, N={self.N}, {self.dtype}{form})"
