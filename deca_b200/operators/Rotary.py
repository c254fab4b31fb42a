"""Rotary positions of attention heads, alone (``Rotary``) and together with the append of the new
keys and values to a paged cache (``RotaryAppend``)."""

from ..kernels.module import BuiltInSchedule
from ..kernels.rotary_b200 import make_rotary, make_rotary_append, rotary_frequencies
from .Op import Operator


class Rotary(Operator):
    """Turns pair i of a head's first ``rot_dim`` elements by position * frequency_i; the other elements are
    copied.  ``layout="half"`` pairs (i, i + rot_dim / 2), ``"interleaved"`` pairs (2i, 2i + 1).
    ``scaling`` adapts the frequencies to long contexts (see ``kernels/rotary_b200.py``).  D even, up to 256.

    Angles are exact modulo a turn at any int32 position.  ``inverse=True`` applies the transposed map:
    the gradient of the input is the inverse of the gradient of the output.
    """

    def __init__(self, D: int, rot_dim: int | None = None, base: float = 10000.0, layout: str = "half",
                 scaling: dict | None = None, dtype: str = "float16", name: str = "Rotary"):
        from ..kernels.rowwise_bench import canonical_dtype

        self.D, self.rot_dim = D, D if rot_dim is None else rot_dim
        self.base, self.layout, self.scaling = base, layout, scaling
        self.dtype = canonical_dtype(dtype)
        self._mod = None
        super().__init__(name=name)
        self.build_mod()  # refuses what the kernel does not take

    @property
    def shape(self):
        return (self.D,)

    def default_config(self):
        return BuiltInSchedule()

    def is_valid(self, cfg) -> bool:
        return isinstance(cfg, BuiltInSchedule)

    def build_mod(self, cfg=None):
        return make_rotary(self.D, self.rot_dim, self.base, self.layout, self.scaling, self.dtype)

    def compile(self, mod):
        from ..kernels.rotary_b200 import build_rotary

        return build_rotary(mod)

    def frequencies(self):
        """([radians per position of every pair], amplitude)."""
        return rotary_frequencies(self.rot_dim, self.base, self.scaling)

    def __call__(self, x, positions, out=None, inverse: bool = False):
        """Returns x [T, H, D] turned by ``positions`` [T] (int32); ``out`` may be ``x``, and is refused where it shares
        memory with x or the positions in any other way."""
        if self._mod is None:
            self._mod = self.compile(self.build_mod())["main"]
        return self._mod(x, positions, out, inverse)

    def describe(self) -> str:
        return f"{self.name}(D={self.D}, rot_dim={self.rot_dim}, {self.layout}, {self.dtype})"


class RotaryAppend(Rotary):
    """One launch between the q/k/v projection and the attention of a serving step: q turned into a tensor
    of its own; k turned and v copied into row ``slots[t] % page_size`` of page ``slots[t] // page_size`` of
    ``k_cache`` / ``v_cache`` [pages, page_size, H_kv, D].  Slots outside the cache (-1: padding) write nothing;
    no two tokens may share a slot."""

    def __init__(self, H_q: int, H_kv: int, D: int, page_size: int, rot_dim: int | None = None, base: float = 10000.0,
                 layout: str = "half", scaling: dict | None = None, dtype: str = "float16", name: str = "RotaryAppend"):
        self.H_q, self.H_kv, self.page_size = H_q, H_kv, page_size
        super().__init__(D, rot_dim, base, layout, scaling, dtype, name)

    @property
    def shape(self):
        return (self.H_q, self.H_kv, self.D, self.page_size)

    def build_mod(self, cfg=None):
        return make_rotary_append(self.H_q, self.H_kv, self.D, self.page_size, self.rot_dim, self.base, self.layout,
                                  self.scaling, self.dtype)

    def __call__(self, q, k, v, positions, slots, k_cache, v_cache, out=None):
        """q [T, H_q, D], k and v [T, H_kv, D] (views of one projection will do), positions [T] int32, slots [T]
        int64; returns the turned q (``out`` may be ``q``).  An output or a cache that shares memory with another tensor of
        the call in any other way is refused; views whose elements alternate in one buffer do not share any."""
        if self._mod is None:
            self._mod = self.compile(self.build_mod())["main"]
        return self._mod(q, k, v, positions, slots, k_cache, v_cache, out)

    def describe(self) -> str:
        return (f"{self.name}(H_q={self.H_q}, H_kv={self.H_kv}, D={self.D}, page_size={self.page_size}, "
                f"rot_dim={self.rot_dim}, {self.layout}, {self.dtype})")
