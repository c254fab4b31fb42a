"""Rules of the serving operators that need no GPU: refusals of the constructors and of the C entry points
(nothing is launched), records, and the fixed-point frequencies."""

import ctypes
import math
from fractions import Fraction

import pytest


@pytest.fixture(scope="module")
def native():
    from deca_b200 import build, native as n

    build.build()
    n.lib()
    return n


def test_constructors_refuse():
    from deca_b200.operators import AddRMSNorm, PagedAttention, PagedStep, Rotary, RotaryAppend

    for make in (lambda: AddRMSNorm(4, 0), lambda: AddRMSNorm(4, 64, out="int8"), lambda: AddRMSNorm(4, 64, group=64),
                 lambda: AddRMSNorm(4, 64, out="e4m3", group=48), lambda: PagedStep(0, 16, 4, 4), lambda: PagedStep(4, 20, 4, 4),
                 lambda: PagedAttention(1, 3, 2, 64, 16, 1, 1), lambda: PagedAttention(1, 4, 2, 96, 16, 1, 1),
                 lambda: PagedAttention(1, 4, 2, 64, 8, 1, 1), lambda: PagedAttention(1, 258, 2, 64, 16, 1, 1),
                 lambda: PagedAttention(1, 4, 2, 64, 16, 1, 1, softmax_scale=math.inf), lambda: Rotary(63), lambda: Rotary(258),
                 lambda: RotaryAppend(4, 2, 64, 24)):
        with pytest.raises(AssertionError):
            make()


def test_records():
    from deca_b200.kernels.module import KernelSpec
    from deca_b200.operators import AddRMSNorm, PagedAttention, PagedStep, RotaryAppend

    op = AddRMSNorm(16, 4096, "bf16", out="e4m3", group=128)
    assert op.num_bytes == 16 * 4096 * 7 + 2 * 4096 + 4 * 16 * 32
    assert AddRMSNorm(16, 4096).num_bytes == 16 * 4096 * 8 + 2 * 4096
    assert op.describe() == "AddRMSNorm(M=16, N=4096, bfloat16, e4m3 per 128)"
    at = PagedAttention(2, 8, 2, 128, 16, 3, 10)
    assert at.num_flops == 4 * 2 * 8 * 128 * (8 + 9 + 10)
    for o in (op, at, PagedStep(3, 16, 4, 5), RotaryAppend(4, 2, 64, 16, scaling={"type": "linear", "factor": 2.0})):
        spec = o.build_mod(o.default_config())
        assert KernelSpec.from_json(spec.to_json()) == spec and o.is_valid(o.default_config())


def test_fixed_point_turns():
    """2^64 times frequency / 2 pi: within one of the quotient with pi to 35 digits."""
    from deca_b200.kernels.rotary_b200 import fixed_point_turns, rotary_frequencies

    pi = Fraction(314159265358979323846264338327950288, 10**35)
    freq, _ = rotary_frequencies(128)
    for f, t in zip(freq, fixed_point_turns(freq)):
        assert 0 < t < 2**64
        assert abs(Fraction(t) - Fraction(f) * 2**63 / pi) <= 1


def test_add_rmsnorm_entry_refuses(native):
    L, p = native.lib(), 4096  # an aligned address that is never followed: every call here is refused first
    good = dict(dtype=0, x=p, xs=64, r=p, rs=64, w=p, h=p, hs=64, y=p, ys=64, s=p, M=2, N=64, eps=1e-6, out=1, group=32)

    def call(**kw):
        a = {**good, **kw}
        return L.deca_add_rmsnorm(a["dtype"], a["x"], a["xs"], a["r"], a["rs"], a["w"], a["h"], a["hs"], a["y"], a["ys"], a["s"],
                                  a["M"], a["N"], a["eps"], a["out"], a["group"], None)

    assert call(M=0) == 0
    for kw, code in (({"dtype": 2}, -5), ({"out": 2}, -5), ({"M": -1}, -2), ({"N": 0}, -2), ({"N": 2**31}, -2), ({"group": 16}, -4),
                     ({"out": 0}, -4), ({"x": None}, -1), ({"w": None}, -1), ({"s": None}, -1), ({"xs": 63}, -2), ({"ys": 1}, -2),
                     ({"x": p + 1}, -3), ({"s": p + 2}, -3)):
        assert call(**kw) == code, kw


def test_rotary_entries_refuse(native):
    L, p = native.lib(), 4096
    turns = (ctypes.c_uint64 * 32)()
    rot = dict(D=64, rot_dim=64, layout=0, inverse=0, amplitude=1.0, turns=turns)
    t, c = native.Tokens(p, 128, 64), native.Cache(p, 2048, 128, 64)

    def call(tokens=1, heads=2, x=t, pos=p, **kw):
        return L.deca_rotary(kw.pop("dtype", 0), x, t, pos, tokens, heads, native.Rotation(**{**rot, **kw}), None)

    def append(tokens=1, pages=2, page=16, slots=p, hkv=2, cache=c):
        return L.deca_rotary_append(0, t, t, t, t, cache, c, p, slots, tokens, 2, hkv, pages, page, native.Rotation(**rot), None)

    assert call(tokens=0) == 0 and append(tokens=0) == 0
    for kw, code in (({"dtype": 3}, -5), ({"layout": 2}, -5), ({"D": 65}, -2), ({"rot_dim": 66}, -2), ({"D": 258}, -2), ({"tokens": -1}, -2),
                     ({"heads": 0}, -2), ({"pos": None}, -1), ({"pos": p + 2}, -3), ({"x": None}, -1), ({"x": native.Tokens(None, 128, 64)}, -1)):
        assert call(**kw) == code, kw
    for kw, code in (({"pages": 0}, -2), ({"page": 12}, -2), ({"hkv": 0}, -2), ({"slots": None}, -1), ({"slots": p + 4}, -3), ({"cache": None}, -1)):
        assert append(**kw) == code, kw


def test_step_entry_refuses(native):
    L, p = native.lib(), 4096
    k = 1024
    good = dict(ctx=p, new=p + k, B=2, table=p + 2 * k, stride=4, W=4, free=p + 3 * k, cap=3, n_free=p + 4 * k, page=16, T=8, cu=p + 5 * k,
                kv=p + 6 * k, pos=p + 7 * k, slots=p + 8 * k, left=p + 9 * k, short=p + 10 * k)

    def call(**kw):
        return L.deca_paged_step(*{**good, **kw}.values(), None)

    for kw, code in (({"B": 0}, -2), ({"B": 8193}, -2), ({"W": 0}, -2), ({"T": -1}, -2), ({"cap": -1}, -2), ({"page": 24}, -2),
                     ({"stride": 3}, -2), ({"W": 2**27, "stride": 2**27}, -2), ({"ctx": None}, -1), ({"free": None}, -1), ({"slots": None}, -1),
                     ({"kv": p}, -5), ({"kv": p + 4}, -5), ({"left": p + 4 * k}, -5), ({"cu": p + k - 4}, -5), ({"pos": p + 2 * k + 16}, -5),
                     ({"slots": p + 7 * k + 28}, -5), ({"free": p + 2 * k + 28}, -5), ({"short": p + 9 * k}, -5), ({"slots": p + 8 * k + 4}, -3), ({"ctx": p + 2}, -3),
                     ({"pos": p + 7 * k + 1}, -3)):
        assert call(**kw) == code, kw


def test_attention_entry_refuses(native):
    L, p = native.lib(), 4096

    def args(**kw):
        a = native.PagedAttnArgs(dtype=0, B=2, H_q=4, H_kv=2, D=64, page_size=16, causal=1, scale=0.125, T=4, num_pages=3, table_stride=5,
                                 table_width=5, max_q=2, max_kv=70, Q=native.Tokens(p, 256, 64), O=native.Tokens(p, 256, 64),
                                 K=native.Cache(p, 2048, 128, 64), V=native.Cache(p, 2048, 128, 64), block_table=p, cu_q=p, kv_lens=p)
        for k, v in kw.items():
            setattr(a, k, v)
        return a

    assert L.deca_paged_attn_check(args()) == 0 and L.deca_paged_attn_check(None) == -1
    for kw, code in (({"dtype": 2}, -5), ({"D": 96}, -5), ({"B": 0}, -2), ({"H_q": 5}, -2), ({"H_q": 512}, -2), ({"T": -1}, -2),
                     ({"num_pages": 0}, -2), ({"page_size": 8}, -2), ({"page_size": 48}, -2), ({"table_stride": 4}, -2), ({"table_width": 2**28, "table_stride": 2**28}, -2),
                     ({"max_q": -1}, -2), ({"scale": math.nan}, -4), ({"scale": math.inf}, -4), ({"cu_q": None}, -1),
                     ({"Q": native.Tokens(p + 8, 256, 64)}, -3), ({"Q": native.Tokens(p, 252, 64)}, -3), ({"K": native.Cache(p, 2048, 130, 64)}, -3),
                     ({"block_table": p + 2}, -3)):
        assert L.deca_paged_attn_check(args(**kw)) == code, kw


def test_calls_refuse_what_is_not_on_a_gpu():
    import torch

    from deca_b200.operators import AddRMSNorm, PagedAttention, PagedStep, Rotary, RotaryAppend

    x, i = torch.ones(4, 64, dtype=torch.float16), torch.ones(4, dtype=torch.int32)
    for op, args in ((AddRMSNorm(4, 64), (x, x, x[0])), (Rotary(64), (x[:, None], i)), (RotaryAppend(1, 1, 64, 16), (x[:, None],) * 3 + (i,) * 2 + (x,) * 2),
                     (PagedStep(4, 16, 2, 4), (i,) * 5), (PagedAttention(4, 1, 1, 64, 16, 1, 1), (x[:, None],) * 3 + (i,) * 3)):
        with pytest.raises(ValueError, match="CUDA"):
            op(*args)
        with pytest.raises(TypeError):
            op(3, *args[1:])


def test_missing_extension_fails_loudly(native, monkeypatch):
    import sys

    from deca_b200.operators import AddRMSNorm

    monkeypatch.setitem(sys.modules, "deca_b200._launch", None)
    monkeypatch.delattr("deca_b200._launch", raising=False)
    with pytest.raises(RuntimeError, match="no fallback"):
        AddRMSNorm(4, 64)(None, None, None)
