"""Outputs over other buffers of a call: refused by the C entries before anything is launched (no GPU is needed), apart from
the places that are documented; regions whose columns alternate are apart.

Addresses are numbers that nothing follows: a call that is not refused ends at the launch, for want of a device, with
another code."""

import ctypes

import pytest

OVERLAP = -5


@pytest.fixture(scope="module")
def native():
    import torch

    from deca_b200 import build, native as n

    if torch.cuda.is_available():
        pytest.skip("the addresses of these calls are made up: on a GPU the accepted ones would run")
    build.build()
    n.lib()
    return n


K = 1 << 20  # distance of buffers that have nothing to do with each other


def norm(native, **kw):
    a = {**dict(dtype=0, x=K, xs=64, r=2 * K, rs=64, w=3 * K, h=4 * K, hs=64, y=5 * K, ys=64, s=None, M=8, N=64, eps=1e-6, out=0, group=0), **kw}
    return native.lib().deca_add_rmsnorm(*a.values(), None)


@pytest.mark.parametrize("kw", [
    {"h": K}, {"h": 2 * K}, {"y": K}, {"y": 2 * K}, {"h": K, "y": 2 * K}, {"h": 2 * K, "y": K},  # in place
    {"r": K},  # inputs may be one
    {"h": K + 128 * 8}, {"y": K - 128 * 8},  # side by side
    {"xs": 256, "hs": 256, "h": K + 128}, {"xs": 256, "rs": 256, "hs": 256, "ys": 256, "r": K + 128, "h": K + 256, "y": K + 384},  # columns of one buffer
    {"h": K, "M": 1, "xs": 64, "hs": 640},  # one row: its stride is no matter
    {"out": 1, "s": 6 * K}, {"out": 1, "s": 6 * K, "group": 32, "h": K}, {"out": 1, "s": K + 128 * 8}])
def test_add_rmsnorm_takes(native, kw):
    assert norm(native, **kw) not in (0, OVERLAP)


@pytest.mark.parametrize("kw", [
    {"h": 5 * K}, {"h": K, "y": K}, {"y": 4 * K + 128 * 7},  # h lost under y
    {"h": 3 * K}, {"y": 3 * K + 64}, {"w": 4 * K + 1022},
    {"h": K + 2}, {"h": K + 128}, {"y": 2 * K - 2}, {"h": K, "hs": 65}, {"h": K, "hs": 128},  # shifted, or at other strides
    {"xs": 96, "hs": 96, "h": K + 128},  # columns that meet
    {"out": 1, "s": K}, {"out": 1, "s": 4 * K + 4}, {"out": 1, "s": 5 * K}, {"out": 1, "s": 3 * K, "group": 32},
    {"out": 1, "s": 6 * K, "y": K}, {"out": 1, "s": 6 * K, "y": K + 64}])
def test_add_rmsnorm_refuses(native, kw):
    assert norm(native, **kw) == OVERLAP


def tokens(native, at, token=128, head=64):
    return native.Tokens(at, token, head)


def rotation(native):
    return native.Rotation(D=64, rot_dim=64, layout=0, inverse=0, amplitude=1.0, turns=(ctypes.c_uint64 * 32)())


def rotary(native, x, y, pos=9 * K, T=8, H=2):
    return native.lib().deca_rotary(0, tokens(native, *x), tokens(native, *y), pos, T, H, rotation(native), None)


# X and Y as (address, token stride, head stride)
@pytest.mark.parametrize("x,y", [((K,), (2 * K,)), ((K,), (K,)), ((K, 256), (K + 256, 256)), ((K, 64, 1024), (K + 128 * 8, 64, 1024)),
                                 ((K, 192, 64), (K, 192, 64)), ((K, 0, 0), (2 * K,)), ((K, 256, 128), (K + 128, 256, 128))])
def test_rotary_takes(native, x, y):
    assert rotary(native, x, y) not in (0, OVERLAP)


@pytest.mark.parametrize("x,y,pos", [((K,), (K + 16,), 9 * K), ((K,), (K + 128,), 9 * K), ((K,), (K, 64, 512), 9 * K), ((K, 192), (K + 128, 192), 9 * K),
                                     ((K, 0, 0), (K,), 9 * K), ((K,), (2 * K,), 2 * K + 4), ((K,), (K - 2032,), 9 * K)])
def test_rotary_refuses(native, x, y, pos):
    assert rotary(native, x, y, pos) == OVERLAP


def cache(native, at, page=2048, row=128, head=64):
    return native.Cache(at, page, row, head)


def append(native, **kw):
    """8 tokens of 4 + 2 x 2 heads of 64 into 3 pages of 16 rows."""
    a = {**dict(q=(K, 256), k=(2 * K,), v=(3 * K,), out=(4 * K, 256), kc=(5 * K,), vc=(6 * K,), pos=7 * K, slots=8 * K, pages=3), **kw}
    q, k, v, out = (tokens(native, *a[n]) for n in ("q", "k", "v", "out"))
    return native.lib().deca_rotary_append(0, q, k, v, out, cache(native, *a["kc"]), cache(native, *a["vc"]), a["pos"], a["slots"], 8, 4, 2,
                                           a["pages"], 16, rotation(native), None)


PROJECTION = {"q": (K, 512), "k": (K + 512, 512), "v": (K + 768, 512)}  # column blocks of one buffer


@pytest.mark.parametrize("kw", [
    {}, {"out": (K, 256)}, PROJECTION, {**PROJECTION, "out": (K, 512)}, {"k": (2 * K, 0, 0), "v": (2 * K, 0, 0)},
    {"kc": (5 * K, 4096), "vc": (5 * K + 4096, 4096)},  # pages of keys, then values
    {"kc": (5 * K, 4096, 256), "vc": (5 * K + 256, 4096, 256)},  # rows of keys, then values
    {"kc": (5 * K, 4096, 256, 128), "vc": (5 * K + 128, 4096, 256, 128)},  # heads of keys, then values
    {"kc": (5 * K, 4096, 64, 1024), "vc": (5 * K + 4096, 4096, 64, 1024)},  # head by head
    {"kc": (5 * K,), "vc": (5 * K + 3 * 4096,)}, {"kc": (5 * K, 1, 128), "vc": (5 * K + 4096, 7, 128), "pages": 1}])
def test_rotary_append_takes(native, kw):
    assert append(native, **kw) not in (0, OVERLAP)


@pytest.mark.parametrize("kw", [
    {**PROJECTION, "out": (K + 512, 512)}, {**PROJECTION, "out": (K + 128, 512)}, {"out": (K + 128, 256)}, {"out": (2 * K, 256)}, {"out": (3 * K - 128, 256)},
    {"kc": (6 * K,)}, {"kc": (6 * K + 128,)}, {"kc": (5 * K, 4096), "vc": (5 * K + 2048, 4096)}, {"kc": (5 * K, 4096, 256), "vc": (5 * K + 128, 4096, 256)},
    {"out": (5 * K, 256)}, {"out": (6 * K + 4096, 256)}, {"q": (5 * K, 256)}, {"k": (5 * K + 3 * 4096 - 2,)}, {"v": (6 * K,)}, {"k": (6 * K,)},
    {"pos": 5 * K}, {"slots": 6 * K + 16}, {"pos": 4 * K + 4}, {"slots": 4 * K + 2040}])
def test_rotary_append_refuses(native, kw):
    assert append(native, **kw) == OVERLAP


def attend(native, **kw):
    a = native.PagedAttnArgs(dtype=0, B=2, H_q=4, H_kv=2, D=64, page_size=16, causal=1, scale=0.125, T=8, num_pages=3, table_stride=5,
                             table_width=5, max_q=2, max_kv=70, Q=tokens(native, K, 256), O=tokens(native, 2 * K, 256),
                             K=cache(native, 3 * K), V=cache(native, 4 * K), block_table=5 * K, cu_q=6 * K, kv_lens=7 * K,
                             workspace=8 * K, workspace_bytes=1 << 16)
    for name, v in kw.items():
        setattr(a, name, {"Q": tokens, "O": tokens, "K": cache, "V": cache}[name](native, *v) if isinstance(v, tuple) else v)
    assert native.lib().deca_paged_attn_check(ctypes.byref(a)) == 0
    return native.lib().deca_paged_attn(ctypes.byref(a), None)


@pytest.mark.parametrize("kw", [
    {}, {"O": (K, 256)}, {"Q": (K, 512), "O": (K, 512)}, {"Q": (K, 512), "O": (K + 512, 512)}, {"Q": (K, 512, 128), "O": (K + 128, 512, 128)},
    {"V": (3 * K,)}, {"V": (3 * K + 128, 4096, 256, 128), "K": (3 * K, 4096, 256, 128)}, {"K": (3 * K, 1024, 64, 0)},
    {"Q": (K, 64, 512), "O": (K, 64, 512)}, {"O": (K + 4096, 256)}])
def test_paged_attention_takes(native, kw):
    assert attend(native, **kw) not in (0, OVERLAP)


@pytest.mark.parametrize("kw", [
    {"O": (K + 128, 256)}, {"O": (K + 16, 256)}, {"O": (K, 512)}, {"O": (K, 64, 512)}, {"Q": (K, 512), "O": (K + 256, 512)},
    {"O": (3 * K, 256)}, {"O": (4 * K + 3 * 4096 - 128, 256)}, {"block_table": 2 * K + 64}, {"cu_q": 2 * K + 4000}, {"kv_lens": 2 * K},
    {"workspace": K}, {"workspace": 2 * K}, {"workspace": 3 * K + 4096}, {"workspace": 4 * K}, {"workspace": 5 * K}, {"workspace": 6 * K}, {"workspace": 7 * K - 256}])
def test_paged_attention_refuses(native, kw):
    assert attend(native, **kw) == OVERLAP


@pytest.mark.parametrize("kw,code", [
    ({"kc": (5 * K, 4104, 256), "vc": (5 * K + 256, 4104, 256)}, 0),  # rows of keys, then values, in pages with a tail
    ({"kc": (5 * K, 4104, 256, 128), "vc": (5 * K + 128, 4104, 256, 128)}, 0),
    ({"kc": (5 * K, 4104, 264, 128), "vc": (5 * K + 128, 4104 + 120, 264, 128)}, OVERLAP),  # other pitches of pages
    ({"kc": (5 * K, 4352, 264, 128), "vc": (5 * K + 128, 4352, 264, 128)}, 0),  # a tail behind rows and behind pages
    ({"kc": (5 * K, 4352, 264, 128), "vc": (5 * K + 126, 4352, 264, 128)}, OVERLAP),
    ({"kc": (5 * K, 4104, 256), "vc": (5 * K + 254, 4104, 256)}, OVERLAP)])
def test_caches_with_tails(native, kw, code):
    got = append(native, **kw)
    assert got == code if code else got not in (0, OVERLAP)


def test_regions_against_enumeration(native):
    """Small layouts of two caches, byte by byte: what shares a byte is always refused; what is accepted shares none."""
    import random

    rng = random.Random(5)
    seen = {True: 0, False: 0}
    for _ in range(4000):
        def layout():
            dims = [64 * rng.choice([1, 2, 3, 4]) for _ in range(3)]
            rng.shuffle(dims)
            return 5 * K + 64 * rng.randrange(0, 24), tuple(d * rng.choice([1, 1, 2, 5, 16, 33]) for d in dims)

        (k_at, k_strides), (v_at, v_strides) = layout(), layout()
        if rng.random() < 0.6:
            v_strides = k_strides

        def bytes_of(at, strides):  # 2 pages x 16 rows x 2 heads, in units of a head's 128 bytes split in two
            return {at + 2 * (p * strides[0] + r * strides[1] + h * strides[2]) + half for p in range(2) for r in range(16) for h in range(2) for half in (0, 64)}

        def cover(at, strides):
            return {b // 64 for b in bytes_of(at, strides)}

        share = bool(cover(k_at, k_strides) & cover(v_at, v_strides))
        refused = append(native, kc=(k_at, *k_strides), vc=(v_at, *v_strides), pages=2) == OVERLAP
        assert refused or not share, (k_at, k_strides, v_at, v_strides)
        seen[refused] += 1
    assert seen[True] > 300 and seen[False] > 300
