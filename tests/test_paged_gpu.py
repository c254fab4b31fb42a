"""PagedStep against a plain loop, PagedAttention against 64-bit attention over the visible keys alone
(bounds in serving_util.attention_bound)."""

import pytest

torch = pytest.importorskip("torch")

from serving_util import attention64, attention_bound, i32, make_paged  # noqa: E402

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16]


# ------------------------------------------------------------------------------------------- step
def step_loop(ctx, new, table, free, n_free, page, W, T):
    cu, kv, pos, slots = [0], [], [0] * T, [-1] * T
    table = [list(r) for r in table]
    free = list(free[:n_free])
    short = 0
    for r, (c, n) in enumerate(zip(ctx, new)):
        c, n = max(c, 0), max(n, 0)
        total = min(c + n, W * page)
        held = min(-(-c // page), W)
        for e in range(held, -(-total // page)):
            if free:
                table[r][e] = free.pop()
            else:
                table[r][e] = -1
                short += 1
        for i in range(n):
            t, p = cu[-1] + i, c + i
            if t < T:
                pos[t] = p
                if p < W * page and table[r][p // page] >= 0:
                    slots[t] = table[r][p // page] * page + p % page
        cu.append(cu[-1] + n)
        kv.append(total)
    return cu, kv, table, pos, slots, len(free), short


@pytest.mark.parametrize("B,page,W,T,ctx_max,new_max,spare", [
    (1, 16, 1, 1, 0, 1, 0), (1, 16, 4, 64, 5, 50, 0), (8, 16, 64, 8, 900, 1, 3), (3, 1, 9, 20, 3, 5, 1), (33, 32, 20, 700, 300, 40, 2),
    (1000, 16, 30, 5000, 300, 9, 5), (1030, 64, 8, 9000, 200, 20, 5), (8192, 16, 4, 10000, 40, 3, 100), (5, 128, 6, 40, 500, 30, -3),
    (7, 16, 3, 90, 40, 30, 0)])
def test_step(B, page, W, T, ctx_max, new_max, spare):
    from deca_b200.operators import PagedStep

    g = torch.Generator().manual_seed(B + page)
    ctx = torch.randint(0, ctx_max + 1, (B,), generator=g).tolist()
    new = torch.randint(0, new_max + 1, (B,), generator=g).tolist()
    new[-1] = new_max
    need = sum(max(min(-(-(c + n) // page), W) - min(-(-c // page), W), 0) for c, n in zip(ctx, new))
    n_free = max(need + spare, 0)
    ids = torch.randperm(B * W + n_free + 10, generator=g).tolist()
    free = ids[: n_free + 10]
    table = [[ids[n_free + 10 + r * W + e] if e < -(-ctx[r] // page) else -7 for e in range(W)] for r in range(B)]
    wide = torch.full((B, W + 3), 99, dtype=torch.int32, device="cuda")
    wide[:, :W] = i32(table)
    out = PagedStep(B, page, W, T)(i32(ctx), i32(new), wide[:, :W], i32(free), i32([n_free]))
    cu, kv, want, pos, slots, left, short = step_loop(ctx, new, table, free, n_free, page, W, T)
    assert out.cu_q.tolist() == cu and out.kv_lens.tolist() == kv
    assert wide[:, :W].tolist() == want and (wide[:, W:] == 99).all()
    assert out.positions.tolist() == pos and out.slots.tolist() == slots
    assert out.n_free.tolist() == [left] and out.short.tolist() == [short]


def test_step_with_senseless_lengths():
    """Negative and huge lengths stay within the tables."""
    from deca_b200.operators import PagedStep

    table = torch.full((4, 8), -1, dtype=torch.int32, device="cuda")
    out = PagedStep(4, 16, 8, 50)(i32([-5, 2**31 - 1, 3, 0]), i32([4, 2**31 - 1, -9, 2**31 - 1]), table, i32([5, 6, 7]), i32([1000]))
    assert out.kv_lens.tolist() == [4, 128, 3, 128] and out.n_free.tolist() == [0]
    assert table[0].tolist() == [7] + [-1] * 7 and table[3].tolist() == [6, 5] + [-1] * 6 and out.short.tolist() == [6]
    assert out.slots[:4].tolist() == [112, 113, 114, 115] and (out.slots[4:] == -1).all()


def test_step_refusals():
    from deca_b200.operators import PagedStep

    op = PagedStep(2, 16, 4, 8)
    a, b, table, free, n = i32([1, 2]), i32([1, 1]), i32([[0] * 4] * 2), i32([3, 4]), i32([2])
    for bad in [(a.long(), b, table, free, n), (a, b[:1], table, free, n), (a, b, table[:, :3], free, n), (a, b, table, free, n[0])]:
        with pytest.raises(ValueError):
            op(*bad)
    out = op(a, b, table, free, n)
    with pytest.raises(RuntimeError):
        op(a, b, table, free, n, out=out._replace(kv_lens=a))
    for bad in ((0, 16, 4, 8), (8193, 16, 4, 8), (2, 24, 4, 8), (2, 16, 2**28, 8)):
        with pytest.raises(AssertionError):
            PagedStep(*bad)


# -------------------------------------------------------------------------------------- attention
def run(q, kc, vc, table, cu, kv, page, max_q=None, max_kv=None, causal=True, scale=None, out=None):
    from deca_b200.operators import PagedAttention

    B = len(kv)
    new = [b - a for a, b in zip(cu, cu[1:])]
    op = PagedAttention(B, q.shape[1], kc.shape[2], q.shape[2], page, max(new) if max_q is None else max_q,
                        max(kv) if max_kv is None else max_kv, str(q.dtype).split(".")[1], scale, causal)
    return op(q, kc, vc, table, i32(cu), i32(kv), out=out)


def check(got, q, kc, vc, table, cu, kv, causal=True, scale=None):
    want, mag = attention64(q, kc, vc, table, cu, kv, scale if scale is not None else q.shape[2] ** -0.5, causal)
    bound = attention_bound(want, mag, q.dtype)
    n = cu[-1]
    err = (got[:n].double() - want[:n]).abs()
    assert (err <= bound[:n]).all(), f"worst {(err / bound[:n]).max().item():.3f}"


BATCHES = [  # (kv_lens, new tokens)
    ([1], [1]), ([16], [1]), ([333], [1]), ([17, 64, 1, 0, 65, 300], [1] * 6), ([1000, 3, 70], [1, 1, 1]),
    ([5], [5]), ([40, 130], [3, 7]), ([100, 64], [64, 64]), ([129, 257, 500], [129, 1, 300]), ([700], [650]), ([30, 0, 4], [2, 0, 4]),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H_q,H_kv,D,page", [(2, 2, 64, 16), (8, 2, 128, 16), (6, 2, 64, 64), (5, 1, 128, 128), (16, 1, 64, 256), (7, 7, 128, 32)])
@pytest.mark.parametrize("batch", BATCHES)
def test_attention(batch, H_q, H_kv, D, page, dtype):
    data = make_paged(*batch, H_q, H_kv, D, page, dtype)
    check(run(*data, page), *data)


@pytest.mark.parametrize("max_q,max_kv", [(1, 1), (1, 100000), (1000, 1), (1000, 100000)])
def test_any_bounds_give_right_results(max_q, max_kv):
    data = make_paged([400, 37, 900], [300, 1, 17], 8, 2, 128, 32, torch.bfloat16)
    check(run(*data, 32, max_q, max_kv), *data)


@pytest.mark.parametrize("max_q", [1, 64])
@pytest.mark.parametrize("dtype", DTYPES)
def test_long_context_is_split_and_joined(dtype, max_q):
    """One request's keys over all CTAs, and requests of very different lengths; runs repeat to the bit."""
    for kv, new in (([20011], [1]), ([9000, 1, 128, 5000], [1, 1, 1, 2])):
        data = make_paged(kv, new, 8, 2, 128, 64, dtype)
        a, b = run(*data, 64, max_q=max_q), run(*data, 64, max_q=max_q)
        check(a, *data)
        assert torch.equal(a, b)


@pytest.mark.parametrize("max_q,max_kv", [(1, 90), (1, 100000), (1000, 90)])
def test_many_requests(max_q, max_kv):
    """More (request, key head) pairs than CTAs: taken whole, cut anywhere, and on tensor-core tiles."""
    g = torch.Generator().manual_seed(9)
    kv = torch.randint(0, 90, (700,), generator=g).tolist()
    data = make_paged(kv, [1] * 700, 4, 2, 64, 16, torch.float16)
    check(run(*data, 16, max_q=max_q, max_kv=max_kv), *data)


@pytest.mark.parametrize("max_q,max_kv", [(1, 1000000), (1000, 1)])
@pytest.mark.parametrize("B", [19, 37, 75, 110, 149, 200, 301, 600])
@pytest.mark.parametrize("longest", [1, 70, 3000])
def test_ranges_shorter_than_an_item_and_its_start(longest, B, max_q, max_kv):
    """A CTA's range may begin or end in what an item's start costs, or hold no key tile at all."""
    g = torch.Generator().manual_seed(B + longest)
    kv = torch.randint(0, 3, (B,), generator=g).tolist()
    kv[0], kv[B // 2], kv[-1] = longest, longest // 2 + 1, longest
    data = make_paged(kv, [min(k, 1) for k in kv], 4, 4, 64, 16, torch.float16)
    got = run(*data, 16, max_q=max_q, max_kv=max_kv)
    check(got, *data)
    assert torch.equal(got, run(*data, 16, max_q=max_q, max_kv=max_kv))


@pytest.mark.parametrize("max_q,max_kv", [(1, 1), (1, 1000000), (1000, 1)])
def test_more_requests_than_shared_memory_holds(max_q, max_kv):
    """Every request has one key: its output is that key's value, to the bit."""
    B = 17000
    g = torch.Generator().manual_seed(0)
    q = torch.randn(B, 2, 64, generator=g).half().cuda()
    kc, vc = (torch.randn(B, 16, 1, 64, generator=g).half().cuda() for _ in range(2))
    table = torch.randperm(B, generator=g).to(torch.int32).view(B, 1).cuda()
    got = run(q, kc, vc, table, list(range(B + 1)), [1] * B, 16, max_q=max_q, max_kv=max_kv)
    assert torch.equal(got, vc[table[:, 0].long(), 0].expand(B, 2, 64))


@pytest.mark.parametrize("new", [1, 3])
def test_long_ragged_batch_is_cut_between_requests(new):
    """Long contexts on more pairs than CTAs: a CTA's steps start and end inside items."""
    g = torch.Generator().manual_seed(3)
    kv = torch.randint(3, 2500, (40,), generator=g).tolist()
    data = make_paged(kv, [new] * 40, 8, 8, 128, 32, torch.bfloat16)
    a, b = (run(*data, 32, max_kv=20000) for _ in range(2))
    check(a, *data)
    assert torch.equal(a, b)


@pytest.mark.parametrize("B,H_kv,D,max_kv", [(3, 2, 128, 1500), (3, 2, 64, 1500), (3, 2, 128, 700), (160, 2, 128, 3000), (160, 2, 64, 3000), (160, 2, 128, 900)])
def test_short_guesses(B, H_kv, D, max_kv):
    """17 to 32 rows a key head: few long contexts, many, and shorter ones."""
    g = torch.Generator().manual_seed(B + D)
    new = torch.randint(1, 8, (B,), generator=g).tolist()
    new[0] = 7
    kv = [n + k for n, k in zip(new, torch.randint(0, min(max_kv, 1200) - 8, (B,), generator=g).tolist())]
    data = make_paged(kv, new, 4 * H_kv, H_kv, D, 16, torch.bfloat16)
    got = run(*data, 16, max_kv=max_kv)
    check(got, *data)
    assert torch.equal(got, run(*data, 16, max_kv=max_kv))


@pytest.mark.parametrize("H_q,H_kv,new", [(128, 1, 2), (200, 2, 3), (24, 1, 1), (40, 2, 70), (31, 1, 33)])
def test_wide_and_odd_groups(H_q, H_kv, new):
    data = make_paged([1500, 77], [new, 1], H_q, H_kv, 64, 64, torch.float16)
    check(run(*data, 64), *data)
    check(run(*data, 64, max_q=1, max_kv=100), *data)


@pytest.mark.parametrize("new,max_q", [([3, 40], None), ([3, 40], 1), ([1, 1], None)])
def test_rows_that_see_nothing(new, max_q):
    """More new tokens than keys: the first rows see no key and are zero; a request without keys is zero."""
    data = make_paged([2, 0], new, 4, 2, 64, 16, torch.float16)
    got = run(*data, 16, max_q=max_q)
    check(got, *data)
    assert (got[: max(new[0] - 2, 0)] == 0).all() and (got[new[0] :] == 0).all() and torch.isfinite(got.float()).all()


@pytest.mark.parametrize("max_q", [1, 1000])
def test_without_causal_mask(max_q):
    data = make_paged([65, 200, 0], [7, 150, 2], 6, 2, 128, 16, torch.float16)
    check(run(*data, 16, max_q=max_q, causal=False), *data, causal=False)


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
@pytest.mark.parametrize("max_q", [1, 1000])
def test_scales(scale, max_q):
    data = make_paged([300, 33], [40, 1], 4, 2, 64, 16, torch.float16)
    q = data[0] * 0.25  # scores of order one at a scale of two: the bound of the fp32 scores holds
    data = (q, *data[1:])
    check(run(*data, 16, max_q=max_q, scale=scale), *data, scale=scale)


@pytest.mark.parametrize("max_q", [1, 12, 1000])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_what_a_row_does_not_see_never_reaches_it(value, max_q):
    """A key of the chunk itself that is not finite: tokens before it are untouched, tokens from it on are
    what the formula gives."""
    data = make_paged([70, 150], [30, 9], 4, 2, 64, 16, torch.float16)
    q, kc, vc, table, cu, kv = data
    at = 55  # the first request's token 15
    vc[table[0, at // 16].long(), at % 16, 1, 3] = value
    got = run(*data, 16, max_q=max_q)
    want, mag = attention64(q, kc, vc, table, cu, kv, 0.125)
    fine = torch.isfinite(want)
    assert int((~fine).sum()) == 2 * 15
    bound = attention_bound(want, mag, q.dtype)
    assert ((got.double() - want).abs()[fine] <= bound[fine]).all()
    assert torch.equal(torch.isnan(got.double()), torch.isnan(want))
    assert torch.equal(got.double()[~fine].nan_to_num(9.0), want[~fine].nan_to_num(9.0))


@pytest.mark.parametrize("max_q", [1, 1000])
def test_strides_and_untouched_rows(max_q):
    """q and out as slices of wider tensors, the cache head by head with keys and values in one tensor; rows
    behind the last request stay."""
    q, kc, vc, table, cu, kv = make_paged([77, 130], [5, 40], 6, 2, 64, 16, torch.bfloat16, fill=0.0)
    pages = kc.shape[0]
    both = torch.zeros(pages, 2, 2, 16, 64, dtype=q.dtype, device="cuda")
    k2, v2 = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    k2.copy_(kc), v2.copy_(vc)
    wide = torch.zeros(60, 10 * 64, dtype=q.dtype, device="cuda")
    q2 = wide[:, 128 : 128 + 384].view(60, 6, 64)
    q2[:45] = q
    q2[45:] = float("nan")
    out = torch.full((60, 8, 64), 7.0, dtype=q.dtype, device="cuda")
    run(q2, k2, v2, table, cu, kv, 16, max_q=max_q, out=out[:, 1:7])
    check(out[:, 1:7], q, kc, vc, table, cu, kv)
    assert (out[45:] == 7).all() and (out[:, 0] == 7).all() and (out[:, 7] == 7).all()


@pytest.mark.parametrize("max_q,max_kv", [(1, 100), (1, 20000), (1000, 100)])
def test_out_may_be_q(max_q, max_kv):
    data = make_paged([3000, 70], [40, 1], 8, 2, 64, 32, torch.bfloat16, fill=0.0)
    want = run(*data, 32, max_q=max_q, max_kv=max_kv)
    q = data[0].clone()
    assert torch.equal(run(q, *data[1:], 32, max_q=max_q, max_kv=max_kv, out=q), want)


@pytest.mark.parametrize("max_q", [1, 1000])
def test_one_key_head_expanded(max_q):
    """A cache of one key head seen as four (a head stride of zero) is that head four times; query rows that do not
    advance are read as they lie; a cache whose rows do not advance is refused."""
    q, kc, vc, table, cu, kv = make_paged([300, 70], [40, 1], 8, 1, 64, 32, torch.bfloat16, fill=0.0)
    wide_k, wide_v = kc.expand(-1, -1, 4, -1), vc.expand(-1, -1, 4, -1)
    got = run(q, wide_k, wide_v, table, cu, kv, 32, max_q=max_q)
    check(got, q, wide_k, wide_v, table, cu, kv)
    same = q[:1].expand(41, 8, 64)
    check(run(same, kc, vc, table, cu, kv, 32, max_q=max_q), same, kc, vc, table, cu, kv)
    with pytest.raises(RuntimeError, match="aligned"):
        run(q, kc[:, :1].expand(-1, 32, -1, -1), vc, table, cu, kv, 32, max_q=max_q)


@pytest.mark.parametrize("max_q", [1, 1000])
def test_senseless_lengths_and_tables(max_q):
    """Lengths are clipped to what Q and the table hold and entries that name no page read as zeros."""
    q, kc, vc, table, cu, kv = make_paged([60, 40], [4, 20], 4, 2, 64, 16, torch.float16, fill=0.0)
    room = table.shape[1] * 16
    bad = table.clone()
    bad[1, 1], bad[1, 2] = -1, 10**9
    zeroed_k, zeroed_v = (torch.cat([c, torch.zeros_like(c[:1])]) for c in (kc, vc))
    plain = bad.clone()
    plain[1, 1:3] = kc.shape[0]
    got = run(q, kc, vc, bad, [0, 4, 10**6], [10**9, 40], 16, max_q=max_q)
    check(got, q, zeroed_k, zeroed_v, plain, [0, 4, 24], [room, 40])
    got = run(q, kc, vc, table, [0, -3, 24], [60, -5], 16, max_q=max_q)  # no rows, and rows without keys
    assert (got[:24] == 0).all()


@pytest.mark.parametrize("max_q", [1, 1000])
def test_large_scores_and_raised_maxima(max_q):
    """Scores that climb by far more than the lazy maximum's threshold from tile to tile."""
    q, kc, vc, table, cu, kv = make_paged([500], [30], 2, 1, 64, 16, torch.float16)
    q.fill_(1.0)
    for j in range(500):
        kc[table[0, j // 16].long(), j % 16] = j / 500.0 * 8  # scores 0 .. 64
    got = run(q, kc, vc, table, cu, kv, 16, max_q=max_q)
    want, mag = attention64(q, kc, vc, table, cu, kv, 0.125)
    # sums of 64 equal products below 512: fp32 errs by 64 * 2^-24 * 64 < 2^-12 in the scores
    assert ((got.double() - want).abs() <= attention_bound(want, mag, q.dtype) + 2.0**-11 * mag).all()


@pytest.mark.parametrize("new", [1, 60])
def test_graphs_streams_and_two_calls_at_once(new):
    """Two captured graphs replayed on two streams at the same time, each with work to join."""
    from deca_b200.operators import PagedAttention

    sets = [make_paged([9000, 500], [new, 1], 8, 2, 128, 64, torch.bfloat16, seed=s) for s in (1, 2)]
    op = PagedAttention(2, 8, 2, 128, 64, new, 9000, "bfloat16")
    args = [(q, kc, vc, t, i32(cu), i32(kv)) for q, kc, vc, t, cu, kv in sets]
    want = [op(*a) for a in args]
    outs = [torch.zeros_like(w) for w in want]
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in sets]
    for graph, a, o in zip(graphs, args, outs):
        with torch.cuda.graph(graph):
            op(*a, out=o)
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
                graph.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w)


def test_one_operator_in_two_threads():
    """Two host threads call one operator object on streams of their own."""
    import threading

    from deca_b200.operators import PagedAttention

    sets = [make_paged([9000, 500], [1, 1], 8, 2, 128, 64, torch.bfloat16, seed=s) for s in (5, 6)]
    op = PagedAttention(2, 8, 2, 128, 64, 1, 9000, "bfloat16")
    args = [(q, kc, vc, t, i32(cu), i32(kv)) for q, kc, vc, t, cu, kv in sets]
    want = [op(*a) for a in args]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(30):
                got = op(*args[i])
                torch.cuda.current_stream().synchronize()
                if not torch.equal(got, want[i]):
                    wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("max_q", [1, 1000])
def test_offsets_past_31_bits(max_q):
    """Pages whose first element lies behind 2^31 of a cache."""
    from deca_b200.operators import RotaryAppend

    q, kc, vc, table, cu, kv = make_paged([300, 40], [5, 7], 8, 8, 128, 256, torch.float16, fill=0.0)
    pages = 2**31 // (256 * 8 * 128) + 6  # of 262144 elements
    far_k, far_v = (torch.empty(pages, 256, 8, 128, dtype=q.dtype, device="cuda") for _ in range(2))
    shift = pages - kc.shape[0]
    far_k[shift:], far_v[shift:] = kc, vc
    got = run(q, far_k, far_v, table + shift, cu, kv, 256, max_q=max_q)
    check(got, q, kc, vc, table, cu, kv)
    slots = torch.tensor([(pages - 1) * 256 + 3], device="cuda")
    one = torch.ones(1, 8, 128, dtype=q.dtype, device="cuda")
    RotaryAppend(8, 8, 128, 256)(one, one, 2 * one, i32([0]), slots, far_k, far_v)
    assert (far_k[-1, 3] == 1).all() and (far_v[-1, 3] == 2).all() and (far_k[-1, 4] == kc[-1, 4]).all()


def test_attention_refusals():
    from deca_b200.operators import PagedAttention

    q, kc, vc, table, cu, kv = make_paged([60, 40], [4, 20], 4, 2, 64, 16, torch.float16)
    op = PagedAttention(2, 4, 2, 64, 16, 20, 60)
    ok = (q, kc, vc, table, i32(cu), i32(kv))
    for i, bad in [(0, q[:, :2]), (0, q.bfloat16()), (0, q.cpu()), (1, kc[:, :8]), (2, vc[:-1]), (3, table.long()), (3, table[:1]),
                   (4, i32(cu[:-1])), (5, i32(kv).long()), (0, q.clone().requires_grad_())]:
        with pytest.raises(ValueError):
            op(*ok[:i], bad, *ok[i + 1 :])
    with pytest.raises(ValueError):
        op(*ok, out=q[:1].expand(24, 4, 64)[:, :1].expand(24, 4, 64))
    shifted = torch.empty(q.numel() + 1, dtype=q.dtype, device="cuda")[1:].view(q.shape)
    with pytest.raises(RuntimeError, match="aligned"):
        op(shifted, *ok[1:])
    assert op(q[:0], *ok[1:]).shape == (0, 4, 64)
    op(*ok)
    torch.cuda.synchronize()
