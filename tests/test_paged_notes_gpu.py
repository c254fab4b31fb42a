"""Values that are not finite in keys that only some rows of a tile see, in the states the schedules can be in: many
items a CTA (the tiles keep such values of two items at a time), items cut over several CTAs, both head dimensions and types.

A weight is positive wherever a key is seen, so a row's output is +inf or -inf where it sees infinities of one sign in
that column, NaN where it sees both or a NaN, and elsewhere the product with those values left out."""

import math

import pytest

torch = pytest.importorskip("torch")

from serving_util import attention_bound, i32, make_paged  # noqa: E402

pytestmark = pytest.mark.gpu

VALUES = [math.inf, -math.inf, math.nan]


def formula(q, k, v, scale):
    """(O, A) of the last len(q) tokens over k, v in 64 bits, not-finite values of v apart."""
    n, m = len(q), len(k)
    seen = torch.arange(m, device=q.device) <= m - n + torch.arange(n, device=q.device)[:, None]
    p = torch.softmax((q.double() @ k.double().T * scale).masked_fill(~seen, -math.inf), -1)
    v, seen = v.double(), seen.double()
    fine = torch.where(torch.isfinite(v), v, 0.0)
    out = p @ fine
    up, down, nan = (seen @ f.double() > 0 for f in (torch.isposinf(v), torch.isneginf(v), torch.isnan(v)))
    out[up], out[down] = math.inf, -math.inf
    out[nan | (up & down)] = math.nan
    return out, p @ fine.abs()


def run_and_compare(data, page, max_q, max_kv):
    from deca_b200.operators import PagedAttention

    q, kc, vc, table, cu, kv = data
    op = PagedAttention(len(kv), q.shape[1], kc.shape[2], q.shape[2], page, max_q, max_kv, str(q.dtype).split(".")[1])
    got = op(q, kc, vc, table, i32(cu), i32(kv))
    again = op(q, kc, vc, table, i32(cu), i32(kv))
    assert torch.equal(got.view(torch.int16), again.view(torch.int16))
    group = q.shape[1] // kc.shape[2]
    for r in range(len(kv)):
        k, v = (c[table[r].long()].flatten(0, 1)[: kv[r]] for c in (kc, vc))
        for h in range(q.shape[1]):
            want, mag = formula(q[cu[r] : cu[r + 1], h], k[:, h // group], v[:, h // group], q.shape[2] ** -0.5)
            have, fine = got[cu[r] : cu[r + 1], h].double(), torch.isfinite(want)
            same = (have == want) | (torch.isnan(have) & torch.isnan(want))
            near = (have - want).abs() <= attention_bound(want, mag, q.dtype)
            bad = ~torch.where(fine, near, same)
            assert not bad.any(), f"request {r} of {kv[r]} keys, head {h}: (row, column) {bad.nonzero().tolist()[:6]}"


def put(data, page, r, at, head, d, value):
    data[2][data[3][r, at // page].long(), at % page, head, d] = value


@pytest.mark.parametrize("max_q,max_kv", [(1000, 1), (1, 1), (1, 100000)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,H_q,H_kv", [(64, 8, 4), (128, 8, 4), (64, 6, 6), (128, 3, 3)])
@pytest.mark.parametrize("longest", [130, 700])
def test_many_items_a_cta(longest, D, H_q, H_kv, dtype, max_q, max_kv):
    """Some (request, head) pairs hold such values, the ones before and behind them none."""
    g = torch.Generator().manual_seed(longest + D)
    B = 200
    new = torch.randint(2, 40, (B,), generator=g).tolist()
    kv = [n + k for n, k in zip(new, torch.randint(0, longest - 40, (B,), generator=g).tolist())]
    data = make_paged(kv, new, H_q, H_kv, D, 32, dtype, seed=longest)
    for r in range(0, B, 2):
        for i in range(1 + r % 3):
            at = kv[r] - 1 - int(torch.randint(0, new[r], (1,), generator=g))
            put(data, 32, r, at, (r // 2 + i) % H_kv, int(torch.randint(0, D, (1,), generator=g)), VALUES[(r // 2 + i) % 3])
    run_and_compare(data, 32, max_q, max_kv)


@pytest.mark.parametrize("max_q,max_kv", [(1000, 1), (1, 100000)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,kv", [(1, 5000), (2, 300), (40, 2500)])
def test_noted_items_that_are_cut(B, kv, D, dtype, max_q, max_kv):
    """Infinities of both signs and a NaN in the chunk's own keys, in one column and in several, with the item's keys
    spread over several CTAs: few items (one part each) and many (cut anywhere)."""
    data = make_paged([kv] * B, [250] * B, 2, 2, D, 64, dtype, seed=kv)
    for r in range(B):
        if r % 3 == 1:
            continue  # nothing in this one
        put(data, 64, r, kv - 240, 0, 7, math.inf)
        put(data, 64, r, kv - 60, 0, 7, -math.inf)  # rows from here on see both
        put(data, 64, r, kv - 200 + r, 0, D - 1, -math.inf)
        put(data, 64, r, kv - 1, 0, 0, math.nan)  # the last row alone
        put(data, 64, r, kv - 249, 1, 33, math.nan)  # all rows but one
        put(data, 64, r, 3, 1, 34, math.inf)  # seen by all
    run_and_compare(data, 64, max_q, max_kv)
