"""Attention over the whole range of scores: keys that outscore all others by far, at every place of a group of
eight keys, on both schedules of PagedAttention and the schedules of FlashAttention; against softmax in 64 bits.

q is 8 everywhere, one key of each request delta / 64, the others zero, scale 8 / D: scores are delta (exact in fp32) and 0.
From delta = 85 on the weight of that key is 1 to 2^-110, so the bound of attention_bound holds without its score term."""

import math

import pytest

torch = pytest.importorskip("torch")

from serving_util import attention_bound, i32, make_paged  # noqa: E402

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16]


def formula(q, k, v, scale, shift=None):
    """(O, A) of q [n, D] over k, v [m, D] in 64 bits: key j is seen by row i where j <= shift + i (None: by all), and
    what is not seen does not enter; A: the same weights on |v|.  A row that sees nothing gives zeros."""
    s = q.double() @ k.double().T * scale
    if shift is None:
        seen = torch.ones_like(s, dtype=torch.bool)
    else:
        seen = torch.arange(len(k), device=q.device) <= shift + torch.arange(len(q), device=q.device)[:, None]
    p = torch.softmax(torch.where(seen, s, -math.inf), -1)
    p = torch.where(seen, p, 0.0)
    return p @ v.double(), p @ v.double().abs()


def set_key(cache, table, r, at, value, page, d=slice(None)):
    cache[table[r, at // page].long(), at % page, :, d] = value


def run_paged(data, page, max_q, max_kv, scale, causal=True):
    from deca_b200.operators import PagedAttention

    q, kc, vc, table, cu, kv = data
    op = PagedAttention(len(kv), q.shape[1], kc.shape[2], q.shape[2], page, max_q, max_kv, str(q.dtype).split(".")[1], scale, causal)
    return op(q, kc, vc, table, i32(cu), i32(kv))


def compare(got, data, scale, causal=True):
    q, kc, vc, table, cu, kv = data
    group = q.shape[1] // kc.shape[2]
    for r in range(len(kv)):
        n = cu[r + 1] - cu[r]
        k, v = (c[table[r].long()].flatten(0, 1)[: kv[r]] for c in (kc, vc))
        for h in range(q.shape[1]):
            want, mag = formula(q[cu[r] : cu[r + 1], h], k[:, h // group], v[:, h // group], scale, kv[r] - n if causal else None)
            have, nan = got[cu[r] : cu[r + 1], h].double(), torch.isnan(want)
            assert torch.equal(torch.isnan(have), nan), f"request {r}, head {h}"
            bad = ((have - want).abs() > attention_bound(want, mag, q.dtype)) & ~nan
            assert not bad.any(), f"request {r}, head {h}: {int(bad.sum())} values, rows {bad.any(-1).nonzero().flatten().tolist()[:9]}"


# (keys of a request, new tokens, base of the eight places): the first 32 keys, which start the maximum, the rest of the first
# tile, a later tile, tiles on the diagonal (the first one and a later one); 200 keys are one item taken whole by the
# tiles, more are cut
PLACES = [(200, 40, 8), (200, 40, 72), (200, 40, 176), (400, 40, 64), (400, 40, 200), (400, 40, 368), (90, 90, 40), (3000, 24, 2216)]
SCHEDULES = [(1, 1), (1, 100000), (1000, 1)]  # (max_q, max_kv): streamed whole, streamed and cut, tiles


@pytest.mark.parametrize("max_q,max_kv", SCHEDULES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("delta", [85, 90, 100, 1000])
def test_paged_one_key_far_above(delta, D, dtype, max_q, max_kv):
    for kv, new, base in PLACES:
        data = make_paged([kv] * 8, [new] * 8, 2, 1, D, 64, dtype, seed=base)
        q, kc, vc, table, _, _ = data
        q.fill_(8.0)
        kc.zero_()
        for r in range(8):
            set_key(kc, table, r, base + r, delta / 64, 64)
        compare(run_paged(data, 64, max_q, max_kv, 8.0 / D), data, 8.0 / D)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("D,S,persistent", [(64, 512, True), (128, 512, True), (64, 512, False), (64, 192, False)])
@pytest.mark.parametrize("delta", [85, 90, 100, 1000])
def test_dense_one_key_far_above(delta, D, S, persistent, causal):
    """Head h has its key at base + h, in a first and in a later tile."""
    from deca_b200.kernels.flash_attn_b200 import FAConfig
    from deca_b200.operators import FlashAttention

    op = FlashAttention(1, 8, S, S, D, softmax_scale=8.0 / D, causal=causal)
    cfg = None if persistent else FAConfig(Bc=64, stages=2, p_tmem=True) if S == 192 else FAConfig(Bc=128, stages=4, q_tiles=2, p_tmem=True)
    if S == 192:
        op = FlashAttention(1, 8, 128, S, D, softmax_scale=8.0 / D) if not causal else FlashAttention(1, 8, 128, 128, D, softmax_scale=8.0 / D, causal=True)
    g = torch.Generator().manual_seed(delta)
    for base in (40, 72) + ((336, 456) if S == 512 else ()):
        q = torch.full((1, 8, op.S_q, D), 8.0, dtype=torch.float16, device="cuda")
        k = torch.zeros(1, 8, op.S_kv, D, dtype=torch.float16, device="cuda")
        v = torch.randn(1, 8, op.S_kv, D, generator=g).half().cuda()
        for h in range(8):
            k[0, h, base + h] = delta / 64
        got = op(q, k, v, cfg=cfg)
        for h in range(8):
            want, mag = formula(q[0, h], k[0, h], v[0, h], 8.0 / D, 0 if causal else None)
            bad = ~((got[0, h].double() - want).abs() <= attention_bound(want, mag, q.dtype))
            assert not bad.any(), f"key {base + h}: rows {bad.any(-1).nonzero().flatten().tolist()[:9]}"


# ---------------------------------------------------------------------------- keys that are not finite
def special_keys(kv, new, base, value, D, dtype):
    """Requests of ordinary data; in request r one element of key base + r is `value`, where q is 1."""
    data = make_paged([kv] * 8, [new] * 8, 2, 1, D, 64, dtype, seed=base + 1)
    q, kc, vc, table, _, _ = data
    q[..., 5] = 1.0
    for r in range(8):
        set_key(kc, table, r, base + r, value, 64, 5)
    return data


@pytest.mark.parametrize("max_q,max_kv", SCHEDULES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_paged_key_that_is_not_finite(value, D, dtype, max_q, max_kv):
    """A visible key with a NaN or a score of +inf makes its rows NaN, as the formula does; a score of -inf has no
    weight; rows that do not see the key do not notice."""
    for kv, new, base in PLACES:
        data = special_keys(kv, new, base, value, D, dtype)
        compare(run_paged(data, 64, max_q, max_kv, D**-0.5), data, D**-0.5)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("D,persistent", [(64, True), (128, True), (64, False)])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_dense_key_that_is_not_finite(value, D, persistent, causal):
    from deca_b200.kernels.flash_attn_b200 import FAConfig
    from deca_b200.operators import FlashAttention

    op = FlashAttention(1, 8, 512, 512, D, causal=causal)
    cfg = None if persistent else FAConfig(Bc=128, stages=4, q_tiles=2, p_tmem=True)
    g = torch.Generator().manual_seed(7)
    for base in (40, 72, 336):
        q, k, v = (torch.randn(1, 8, 512, D, generator=g).half().cuda() for _ in range(3))
        q[..., 5] = 1.0
        for h in range(8):
            k[0, h, base + h, 5] = value
        got = op(q, k, v, cfg=cfg)
        for h in range(8):
            want, mag = formula(q[0, h], k[0, h], v[0, h], D**-0.5, 0 if causal else None)
            have, nan = got[0, h].double(), torch.isnan(want)
            assert torch.equal(torch.isnan(have), nan), f"key {base + h}"
            bad = ((have - want).abs() > attention_bound(want, mag, q.dtype)) & ~nan
            assert not bad.any(), f"key {base + h}: rows {bad.any(-1).nonzero().flatten().tolist()[:9]}"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("fill", [math.nan, math.inf, 300.0])
def test_rows_of_nobody_do_not_steer_their_neighbours(fill, D, dtype):
    """The rows of Q behind the last token (a padded batch) lie in a tile with live rows: the results do not
    depend on them, to the bit."""
    from deca_b200.operators import PagedAttention

    q, kc, vc, table, cu, kv = make_paged([600, 1500], [70, 40], 2, 2, D, 64, dtype)
    op = PagedAttention(2, 2, 2, D, 64, 128, 1500, str(dtype).split(".")[1])
    padded = torch.zeros(160, 2, D, dtype=dtype, device="cuda")
    padded[:110] = q
    want = op(padded, kc, vc, table, i32(cu), i32(kv))[:110].clone()
    padded[110:] = fill
    assert torch.equal(op(padded, kc, vc, table, i32(cu), i32(kv))[:110], want)


@pytest.mark.parametrize("max_q,max_kv", SCHEDULES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dead", [32, 40, 128, 200])
def test_paged_first_scores_minus_infinity(dead, D, dtype, max_q, max_kv):
    """The first `dead` visible keys score -inf and the others -200 and -199: the maximum starts at -inf there and
    the weights of the others are still theirs."""
    for kv, new in ((400, 40), (3000, 24)):
        data = make_paged([kv], [new], 2, 1, D, 64, dtype, seed=dead)
        q, kc, vc, table, _, _ = data
        q.fill_(8.0)
        kc.fill_(-200 / 64)
        for at in range(kv):
            if at < dead:
                set_key(kc, table, 0, at, 0.0, 64)
                set_key(kc, table, 0, at, -math.inf, 64, 5)
            elif at % 3 == 0:
                set_key(kc, table, 0, at, -199 / 64, 64)
        compare(run_paged(data, 64, max_q, max_kv, 8.0 / D), data, 8.0 / D)


@pytest.mark.parametrize("max_q,max_kv", SCHEDULES)
@pytest.mark.parametrize("D", [64, 128])
def test_paged_all_scores_minus_infinity(D, max_q, max_kv):
    """A row without a finite score gives zeros, like one that sees no key; the rows that see one more key do not."""
    data = make_paged([300], [40], 2, 1, D, 64, torch.float16)
    q, kc, vc, table, _, _ = data
    q.fill_(1.0)
    for at in range(280):
        set_key(kc, table, 0, at, -math.inf, 64, 5)
    got = run_paged(data, 64, max_q, max_kv, D**-0.5)
    assert (got[:20] == 0).all()  # tokens 260 .. 279
    first = vc[table[0, 280 // 64].long(), 280 % 64, 0]
    assert torch.equal(got[20], first.expand(2, D))  # one key of weight one
    assert torch.isfinite(got.float()).all()
