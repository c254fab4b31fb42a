"""AddRMSNorm against 64-bit arithmetic.

h: half a step of the type.  y: half a step plus 1e-5 relative for the fp32 arithmetic: a sum of squares of
positive terms errs by its longest chain (at most 8 chunks of 8, 10 exchange levels and 15 warps, or 260
iterations of 8 for the longest streamed row here: 2^-24 times 2100) halved by the root, 6.3e-5 there and below
3e-6 for a row in registers, plus a few 2^-24.  e4m3: half a step (2^-4 relative, 2^-10 of the scale among the
subnormals) around y / s, on top of y's own error."""

import pytest

torch = pytest.importorskip("torch")

from serving_util import HALF_STEP, TINY  # noqa: E402

pytestmark = pytest.mark.gpu

DT = {"float16": torch.float16, "bfloat16": torch.bfloat16}


def exact(x, res, w, eps):
    h = x.double() + res.double()
    return h, h / (h.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()


def inputs(M, N, dtype, seed=3):
    g = torch.Generator().manual_seed(seed)
    x, res = (torch.randn(M, N, generator=g).to(DT[dtype]).cuda() for _ in range(2))
    return x, res, (1 + 0.1 * torch.randn(N, generator=g)).to(DT[dtype]).cuda()


def check(got, want, dtype, fp32):
    u = HALF_STEP[got.dtype]
    err = (got.double() - want).abs()
    bound = u * want.abs() * (1 + 1e-6) + fp32 * want.abs() + TINY[got.dtype]
    assert (err <= bound).all(), f"worst {(err / bound).max().item():.3f}"


def check_e4m3(q, s, y, N, group, fp32=1e-5):
    size = group or N
    n = -(-N // size)
    pad = torch.nn.functional.pad(y, (0, n * size - N)).view(len(y), n, size)
    want_s = pad.abs().amax(-1) / 448.0
    assert ((s.double() - want_s).abs() <= fp32 * want_s).all()
    wide = s.double().repeat_interleave(size, -1)[:, :N]
    err = (q.double() * wide - y).abs()
    assert (err <= (2.0**-4 + 2 * fp32) * y.abs() + 2.0**-10 * wide * (1 + fp32)).all()


SHAPES = [(1, 1), (1, 7), (3, 8), (2, 63), (5, 64), (1, 4096), (300, 96), (297, 513), (17, 1000), (4, 8192), (301, 5000),
          (2, 20000), (3, 32768), (2, 32776), (1, 70001), (9, 65), (300, 66), (11, 255), (8, 249), (17, 4097), (5, 16389), (9, 40002)]


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("M,N", SHAPES)
def test_sixteen_bits(M, N, dtype):
    from deca_b200.operators import AddRMSNorm

    x, res, w = inputs(M, N, dtype)
    y, h = AddRMSNorm(M, N, dtype)(x, res, w)
    want_h, want_y = exact(x, res, w, 1e-6)
    check(h, want_h, dtype, 1e-7)
    check(y, want_y, dtype, 7e-5 if N > 32768 else 1e-5)


@pytest.mark.parametrize("group", [0, 32, 64, 128, 256])
@pytest.mark.parametrize("M,N", [(1, 1), (3, 100), (5, 256), (300, 513), (17, 4096), (301, 5000), (2, 33000), (2, 32769), (13, 1003), (9, 70), (300, 129)])
def test_eight_bits(M, N, group):
    from deca_b200.operators import AddRMSNorm

    x, res, w = inputs(M, N, "bfloat16", 5)
    q, s, h = AddRMSNorm(M, N, "bfloat16", out="e4m3", group=group)(x, res, w)
    want_h, want_y = exact(x, res, w, 1e-6)
    check(h, want_h, "bfloat16", 1e-7)
    check_e4m3(q, s, want_y, N, group, 7e-5 if N > 32768 else 1e-5)


@pytest.mark.parametrize("extra", [40, 37])
@pytest.mark.parametrize("N,offset", [(512, 0), (512, 1), (511, 0), (4096, 8), (1000, 4)])
def test_strides_and_alignment(N, offset, extra):
    """Rows that are slices of wider tensors, aligned for wide accesses and not; neighbours stay."""
    from deca_b200.operators import AddRMSNorm

    M, wide = 9, N + extra
    g = torch.Generator().manual_seed(1)
    big = [torch.randn(M, wide, generator=g).half().cuda() for _ in range(4)]
    x, res, h, y = (b[:, offset : offset + N] for b in big)
    before = [b.clone() for b in big]
    w = torch.randn(N, generator=g).half().cuda()
    want_h, want_y = exact(x, res, w, 1e-6)
    AddRMSNorm(M, N)(x, res, w, out=y, res_out=h)
    check(h, want_h, "float16", 1e-7)
    check(y, want_y, "float16", 1e-5)
    for b, was in zip(big, before):
        assert torch.equal(b[:, :offset], was[:, :offset]) and torch.equal(b[:, offset + N :], was[:, offset + N :])
    assert torch.equal(x, before[0][:, offset : offset + N]) and torch.equal(res, before[1][:, offset : offset + N])


@pytest.mark.parametrize("N", [1000, 1001, 40000, 40001])
def test_in_place(N):
    """The residual updated in place and y over x give the same bits as tensors of their own."""
    from deca_b200.operators import AddRMSNorm

    x, res, w = inputs(6, N, "bfloat16")
    op = AddRMSNorm(6, N, "bfloat16")
    y, h = op(x, res, w)
    x2, res2 = x.clone(), res.clone()
    op(x2, res2, w, out=x2, res_out=res2)
    assert torch.equal(y, x2) and torch.equal(h, res2)


def test_special_rows():
    """A row of zeros, one that cancels, one with an infinity and one with a NaN; the others do not notice."""
    from deca_b200.operators import AddRMSNorm

    x, res, w = inputs(6, 256, "float16")
    x[0] = 0
    res[0] = 0
    res[1] = -x[1]
    x[2, 5] = float("inf")
    x[3, 7] = float("nan")
    y, h = AddRMSNorm(6, 256)(x, res, w)
    q, s, h8 = AddRMSNorm(6, 256, out="e4m3", group=64)(x, res, w)
    want_h, want_y = exact(x, res, w, 1e-6)
    for r in (0, 1, 4, 5):
        check(y[r : r + 1], want_y[r : r + 1], "float16", 1e-5)
    check_e4m3(q[4:], s[4:], want_y[4:], 256, 64)
    assert (y[:2] == 0).all() and (q[:2].float() == 0).all() and (s[:2] == 0).all()
    assert torch.isnan(y[3]).all() and torch.isnan(q[3].float()).all() and torch.isnan(s[3]).all()
    assert torch.isnan(y[2, 5]) and (y[2, :5] == 0).all() and torch.isnan(s[2, 0]) and (s[2, 1:] == 0).all()
    assert torch.equal(torch.isinf(h), torch.isinf(want_h)) and torch.equal(torch.isnan(h8), torch.isnan(want_h))


def test_subnormal_scale_gives_zeros():
    from deca_b200.operators import AddRMSNorm

    x = torch.full((1, 64), 2.0**-120, dtype=torch.bfloat16, device="cuda")
    w = torch.full((64,), 2.0**-20, dtype=torch.bfloat16, device="cuda")
    q, s, _ = AddRMSNorm(1, 64, "bfloat16", out="e4m3")(x, torch.zeros_like(x), w)  # y = 2^-130: s = 2^-138.8
    assert (q.float() == 0).all() and s.item() < 2.0**-126


def test_graph_and_repeatability():
    from deca_b200.operators import AddRMSNorm

    x, res, w = inputs(33, 4096, "bfloat16")
    op = AddRMSNorm(33, 4096, "bfloat16", out="e4m3", group=128)
    want = op(x, res, w)
    q, s, h = (torch.empty_like(t) for t in want)
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        op(x, res, w, out=q, res_out=h, scales=s)
    for _ in range(2):
        for t in (q, s, h):
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((q, s, h), want):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_offsets_past_31_bits():
    from deca_b200.operators import AddRMSNorm

    M, N = 2**31 // 8192 + 3, 8192
    x, res = (torch.zeros(M, N, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    tail = inputs(3, N, "bfloat16")
    x[-3:], res[-3:] = tail[0], tail[1]
    y, h = AddRMSNorm(M, N, "bfloat16")(x, res, tail[2], res_out=res)
    want_h, want_y = exact(*tail, 1e-6)
    check(h[-3:], want_h, "bfloat16", 1e-7)
    check(y[-3:], want_y, "bfloat16", 1e-5)
    assert (y[-4] == 0).all()


def test_harness_and_command_line():
    """The tuning harness verifies and times the operator, and run_case prints its rate."""
    import subprocess
    import sys

    from deca_b200.arch.B200 import B200
    from deca_b200.operators import AddRMSNorm, PagedAttention
    from deca_b200.RuntimeMod import RuntimeMod

    for op in (AddRMSNorm(300, 1000, "bf16"), AddRMSNorm(300, 1000, "bf16", out="e4m3", group=128), PagedAttention(2, 8, 2, 64, 16, 40, 300),
               PagedAttention(2, 8, 2, 128, 16, 1, 300, "bf16")):
        rt = RuntimeMod(op, B200(), False, op.default_config())
        rt.build()
        rt.time_evaluator()
        assert rt.throughput > 0 and op.name in rt.record
    for args in ("--op add_rmsnorm --dtype bf16 --shape 64 4096 --out e4m3", "--op paged_attention --shape 2 8 2 128 16 1 500"):
        res = subprocess.run([sys.executable, "-m", "deca_b200.run_case", *args.split(), "--iters", "2"], capture_output=True, text=True)
        assert res.returncode == 0 and " ms, " in res.stdout, res.stderr[-500:]


def test_empty_batch():
    from deca_b200.operators import AddRMSNorm

    x = torch.empty(0, 64, dtype=torch.float16, device="cuda")
    y, h = AddRMSNorm(0, 64)(x, x, torch.ones(64, dtype=torch.float16, device="cuda"))
    assert y.shape == h.shape == (0, 64)


def test_refusals():
    from deca_b200.operators import AddRMSNorm

    x, res, w = inputs(4, 64, "float16")
    op = AddRMSNorm(4, 64)
    for bad in [(x.cpu(), res, w), (x[:3], res, w), (x.float(), res, w), (x, res, w[:32]), (x, res.expand(4, 64).t().contiguous().t(), w),
                (x[:1].expand(4, 64), res, w), (x.requires_grad_(), res, w)]:
        with pytest.raises(ValueError):
            op(*bad)
    with torch.no_grad():
        op(x, res, w)
    with pytest.raises(ValueError):
        AddRMSNorm(4, 64, out="e4m3")(x.detach(), res, w, out=torch.empty_like(res))
