"""One captured PagedAttention launch replayed while the lengths on the device change between replays: from long to empty
and back, one request or all, so that items are whole, cut into parts or gone, in any order."""

import pytest

torch = pytest.importorskip("torch")

from serving_util import attention64, attention_bound, i32, make_paged  # noqa: E402

pytestmark = pytest.mark.gpu

STEPS = [  # kv_lens of six requests, new tokens
    ([9000, 9000, 9000, 9000, 9000, 9000], [4] * 6), ([9000, 1, 0, 0, 0, 0], [4, 1, 0, 0, 0, 0]), ([0] * 6, [0] * 6), ([5] * 6, [1] * 6),
    ([1, 1, 1, 1, 1, 9000], [1, 1, 1, 1, 1, 4]), ([300, 8000, 64, 65, 0, 128], [4, 3, 2, 1, 4, 0]), ([9000, 9000, 9000, 9000, 9000, 9000], [4] * 6),
    ([0, 0, 0, 0, 0, 7777], [0, 0, 0, 0, 0, 1])]


@pytest.mark.parametrize("max_q,max_kv", [(1, 9000), (4, 9000), (1, 500), (400, 9000)])
@pytest.mark.parametrize("D,H_q,H_kv", [(128, 8, 2), (64, 4, 4)])
def test_lengths_change_between_replays(D, H_q, H_kv, max_q, max_kv):
    from deca_b200.operators import PagedAttention

    q, kc, vc, table, _, _ = make_paged([9000] * 6, [4] * 6, H_q, H_kv, D, 64, torch.bfloat16, fill=0.0)
    op = PagedAttention(6, H_q, H_kv, D, 64, max_q, max_kv, "bfloat16")
    cu, kv, out = i32([0] * 7), i32([0] * 6), torch.zeros_like(q)
    op(q, kc, vc, table, cu, kv, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        op(q, kc, vc, table, cu, kv, out=out)
    for lens, new in STEPS + STEPS[::-1]:
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        cu.copy_(i32(starts)), kv.copy_(i32(lens)), out.fill_(7.0)
        graph.replay()
        got = out.clone()
        out.fill_(7.0)
        graph.replay()
        assert torch.equal(got, out)
        assert torch.equal(got, op(q, kc, vc, table, cu, kv, out=torch.full_like(q, 7.0)))
        n = starts[-1]
        assert (got[n:] == 7).all()
        want, mag = attention64(q, kc, vc, table, starts, lens, D**-0.5)
        bound = attention_bound(want, mag, q.dtype)
        assert ((got[:n].double() - want[:n]).abs() <= bound[:n]).all()
