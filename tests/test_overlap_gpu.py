"""Outputs over other tensors of a call, through the operators: in place where that is documented, with the same bits as
tensors of their own, and refused elsewhere."""

import pytest

torch = pytest.importorskip("torch")

from serving_util import i32, make_paged  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,N", [(6, 1000), (6, 1001), (300, 513), (5, 40000), (5, 40001)])
def test_add_rmsnorm_over_its_inputs(M, N):
    from deca_b200.operators import AddRMSNorm

    g = torch.Generator().manual_seed(N)
    x, res = (torch.randn(M, N, generator=g).bfloat16().cuda() for _ in range(2))
    w = torch.randn(N, generator=g).bfloat16().cuda()
    op = AddRMSNorm(M, N, "bfloat16")
    y, h = op(x, res, w)
    for y_over, h_over in ((0, None), (1, None), (None, 0), (None, 1), (0, 1), (1, 0)):
        both = [x.clone(), res.clone()]
        got_y, got_h = op(*both, w, out=None if y_over is None else both[y_over], res_out=None if h_over is None else both[h_over])
        assert torch.equal(got_y, y) and torch.equal(got_h, h)
    wide = torch.cat([x, res, x, res], 1)  # columns of one buffer
    a, b, c, d = (wide[:, i * N : (i + 1) * N] for i in range(4))
    op(a, b, w, out=c, res_out=d)
    assert torch.equal(c, y) and torch.equal(d, h) and torch.equal(a, x) and torch.equal(b, res)


def test_add_rmsnorm_refuses_overlaps():
    from deca_b200.operators import AddRMSNorm

    big = torch.randn(20, 64, device="cuda").half()
    x, res, w = big[:8], big[8:16], big[16]
    before = big.clone()
    op, eight = AddRMSNorm(8, 64), AddRMSNorm(8, 64, out="e4m3")
    for call in (lambda: op(x, res, w, out=x, res_out=x), lambda: op(x, res, w, out=big[1:9]), lambda: op(x, res, w, res_out=big[4:12]),
                 lambda: op(x, res, w, out=big[10:18]), lambda: eight(x, res, w, out=x.view(torch.float8_e4m3fn)[:, :64]),
                 lambda: eight(x, res, w, scales=res.view(torch.float32).view(-1)[:8].view(8, 1))):
        with pytest.raises(RuntimeError, match="another buffer"):
            call()
    torch.cuda.synchronize()
    assert torch.equal(big, before)


def test_rotary_refuses_overlaps():
    from deca_b200.operators import Rotary

    g = torch.Generator().manual_seed(1)
    buffer = torch.randn(20 * 6 * 64, generator=g).half().cuda()
    before = buffer.clone()
    x = buffer[: 12 * 4 * 64].view(12, 4, 64)
    op, pos = Rotary(64), i32(list(range(12)))
    for out in (buffer[64 : 64 + x.numel()].view(12, 4, 64), buffer[2 : 2 + x.numel()].view(12, 4, 64), buffer.as_strided((12, 4, 64), (64, 12 * 64, 1)),
                buffer[32 * 64 :][: x.numel()].view(12, 4, 64)):
        with pytest.raises(RuntimeError, match="another buffer"):
            op(x, pos, out=out)
    torch.cuda.synchronize()
    assert torch.equal(buffer, before)
    halves = torch.zeros(12, 8, 64, dtype=torch.float16, device="cuda")
    halves[:, :4] = x
    op(halves[:, :4], pos, out=halves[:, 4:])
    assert torch.equal(halves[:, 4:], op(x, pos)) and torch.equal(halves[:, :4], x)


def test_rotary_append_refuses_overlaps():
    from deca_b200.operators import RotaryAppend

    g = torch.Generator().manual_seed(2)
    T, Hq, Hkv, D, page = 9, 4, 2, 64, 16
    qkv = torch.randn(T, (Hq + 2 * Hkv) * D, generator=g).half().cuda()
    q, k, v = (t.view(T, -1, D) for t in qkv.split([Hq * D, Hkv * D, Hkv * D], -1))
    both = torch.zeros(3, page, 2, Hkv, D, dtype=torch.float16, device="cuda")  # rows of keys, then values
    kc, vc = both[:, :, 0], both[:, :, 1]
    before, slots, pos = qkv.clone(), torch.arange(T, device="cuda"), i32(list(range(T)))
    op = RotaryAppend(Hq, Hkv, D, page)
    for out, caches in ((qkv[:, 2 * D : 6 * D].view(T, 4, D), (kc, vc)), (both.view(-1)[: T * Hq * D].view(T, Hq, D), (kc, vc)), (None, (kc, kc)),
                        (None, (both.view(3, 2, page, Hkv, D)[:, 0], vc))):
        with pytest.raises(RuntimeError, match="another buffer"):
            op(q, k, v, pos, slots, *caches, out=out)
    torch.cuda.synchronize()
    assert torch.equal(qkv, before) and not both.any()
    want_k, want_v = torch.zeros(2, 3, page, Hkv, D, dtype=torch.float16, device="cuda")
    want = op(q, k, v, pos, slots, want_k, want_v)
    assert op(q, k, v, pos, slots, kc, vc, out=q) is not None
    assert torch.equal(q, want) and torch.equal(kc, want_k) and torch.equal(vc, want_v) and torch.equal(v, before[:, 6 * D :].view(T, Hkv, D))


@pytest.mark.parametrize("max_q", [1, 1000])
def test_paged_attention_refuses_overlaps(max_q):
    from deca_b200.operators import PagedAttention

    q, kc, vc, table, cu, kv = make_paged([300, 70], [40, 1], 8, 2, 64, 32, torch.bfloat16, fill=0.0)
    buffer = torch.zeros(50 * 8 * 64, dtype=q.dtype, device="cuda")
    inside = buffer[: q.numel()].view(q.shape)
    inside.copy_(q)
    before, k_before = buffer.clone(), kc.clone()
    op = PagedAttention(2, 8, 2, 64, 32, max_q, 300, "bfloat16")
    for out in (buffer[512 : 512 + q.numel()].view(q.shape), buffer[8 : 8 + q.numel()].view(q.shape), kc.view(-1)[: q.numel()].view(q.shape),
                buffer.as_strided(q.shape, (64, 41 * 64, 1))):
        with pytest.raises(RuntimeError, match="another buffer"):
            op(inside, kc, vc, table, i32(cu), i32(kv), out=out)
    torch.cuda.synchronize()
    assert torch.equal(buffer, before) and torch.equal(kc, k_before)
    want = op(q, kc, vc, table, i32(cu), i32(kv))
    wide = torch.zeros(41, 16, 64, dtype=q.dtype, device="cuda")  # heads of q, then of the output
    wide[:, :8] = q
    op(wide[:, :8], kc, vc, table, i32(cu), i32(kv), out=wide[:, 8:])
    assert torch.equal(wide[:, 8:], want) and torch.equal(wide[:, :8], q)
