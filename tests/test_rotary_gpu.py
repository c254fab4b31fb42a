"""Rotary positions against complex rotation in 64 bits.

Bound of an output: half a step of the type, and (|a| + |b|) 2^-20 times the amplitude for the fp32 arithmetic:
the angle in half turns rounds to 2^-24 (1.9e-7 rad), sincospi errs by two last bits of at most 1
(1.2e-7), and two products and a sum round (1.8e-7)."""

import math

import pytest

torch = pytest.importorskip("torch")

from serving_util import HALF_STEP, TINY, i32  # noqa: E402

pytestmark = pytest.mark.gpu

BAND = {"type": "band", "factor": 8.0, "original_length": 4096, "low": 1.0, "high": 32.0}


def pairs(x, rot, layout):
    head = x[..., :rot]
    return (head[..., : rot // 2], head[..., rot // 2 :]) if layout == "half" else (head[..., 0::2], head[..., 1::2])


def turn64(op, x, positions, inverse=False):
    freq, amplitude = op.frequencies()
    x = x.double()
    angle = positions.double()[:, None, None] * torch.tensor(freq, dtype=torch.float64, device=x.device)
    c, s = angle.cos() * amplitude, angle.sin() * (-amplitude if inverse else amplitude)
    a, b = pairs(x, op.rot_dim, op.layout)
    out, mag = x.clone(), torch.zeros_like(x)
    oa, ob = pairs(out, op.rot_dim, op.layout)
    ra, rb = a * c - b * s, a * s + b * c
    m = (a.abs() + b.abs()) * amplitude
    oa.copy_(ra), ob.copy_(rb)
    ma, mb = pairs(mag, op.rot_dim, op.layout)
    ma.copy_(m), mb.copy_(m)
    return out, mag


def check(got, want, mag):
    u = HALF_STEP[got.dtype]
    bound = u * want.abs() * (1 + 1e-6) + 2.0**-20 * mag + TINY[got.dtype]
    err = (got.double() - want).abs()
    assert (err <= bound).all(), f"worst {(err / bound).max().item():.3f}"


def data(T, H, D, dtype, seed=0, far=5000):
    g = torch.Generator().manual_seed(seed)
    pos = torch.randint(0, far, (T,), generator=g).to(torch.int32)
    pos[0] = 0
    return torch.randn(T, H, D, generator=g).to(dtype).cuda(), pos.cuda()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("T,H,D,rot", [(1, 1, 2, 2), (1, 32, 128, 128), (7, 3, 64, 64), (5, 5, 128, 32), (3, 2, 96, 48),
                                       (4, 3, 80, 20), (6, 1, 256, 256), (2, 7, 10, 6), (400, 9, 128, 64)])
def test_forward_and_inverse(T, H, D, rot, layout, dtype):
    from deca_b200.operators import Rotary

    x, pos = data(T, H, D, dtype)
    op = Rotary(D, rot_dim=rot, layout=layout, dtype=str(dtype).split(".")[1])
    for inverse in (False, True):
        check(op(x, pos, inverse=inverse), *turn64(op, x, pos, inverse))


@pytest.mark.parametrize("scaling", [None, {"type": "linear", "factor": 4.0}, {"type": "base", "factor": 4.0}, BAND,
                                     {**BAND, "amplitude": 1.0}])
def test_scaling_at_far_positions(scaling):
    from deca_b200.operators import Rotary

    x, pos = data(64, 4, 128, torch.float16, far=2**20)
    pos[1], pos[2], pos[3] = 2**31 - 1, 2**24 + 1, -5  # the 64-bit product of the check errs by 2^31 * 2^-53 there
    op = Rotary(128, scaling=scaling)
    check(op(x, pos), *turn64(op, x, pos))


def test_band_frequencies():
    """Fast pairs keep their frequency, slow ones are divided by the factor, those between lie between."""
    from deca_b200.operators import Rotary

    plain, one = Rotary(128).frequencies()
    band, amplitude = Rotary(128, scaling=BAND).frequencies()
    assert one == 1.0 and amplitude == pytest.approx(0.1 * math.log(8.0) + 1.0)
    for f, b in zip(plain, band):
        turns = 4096 * f / (2 * math.pi)
        assert b == (f if turns >= 32 else pytest.approx(f / 8) if turns <= 1 else pytest.approx(b))
        assert f / 8 * 0.999999 <= b <= f


def test_gradient_is_the_inverse():
    """<grad_y, R dx> = <R^-1-form grad_y, dx>: against the formula's transpose and against differences, on
    inputs where the 16-bit roundings are the only error (bound: their sum over the products)."""
    from deca_b200.operators import Rotary

    for layout in ("half", "interleaved"):
        op = Rotary(64, rot_dim=32, layout=layout, scaling=BAND)
        x, pos = data(11, 3, 64, torch.float16, 1)
        grad, _ = data(11, 3, 64, torch.float16, 2)
        leaf = x.double().requires_grad_()
        freq, amplitude = op.frequencies()
        angle = pos.double()[:, None, None] * torch.tensor(freq, dtype=torch.float64, device="cuda")
        a, b = pairs(leaf, 32, layout)
        c, s = angle.cos() * amplitude, angle.sin() * amplitude
        ra, rb = a * c - b * s, a * s + b * c
        ga, gb = pairs(grad.double(), 32, layout)
        tail = (leaf[..., 32:] * grad.double()[..., 32:]).sum()
        ((ra * ga).sum() + (rb * gb).sum() + tail).backward()
        got = op(grad, pos, inverse=True)
        _, mag = turn64(op, grad, pos, True)
        check(got, leaf.grad, mag)
        # differences of the forward kernel: <grad, R(x + d) - R(x)> = <grad_x, d> for the linear map R
        d, _ = data(11, 3, 64, torch.float16, 3)
        xd = (x.float() + d.float()).half()
        step = xd.double() - x.double()
        ends = [op(v, pos).double() for v in (xd, x)]
        left = (grad.double() * (ends[0] - ends[1])).sum().item()
        right = (got.double() * step).sum().item()
        slack = sum((grad.double().abs() * (2.0**-11 * e.abs() + 2.0**-19 * 8)).sum().item() for e in ends)
        slack += (step.abs() * (2.0**-11 * got.double().abs() + 2.0**-19 * 8)).sum().item()
        assert abs(left - right) <= slack


def test_strided_in_place_and_graph():
    from deca_b200.operators import Rotary

    g = torch.Generator().manual_seed(4)
    wide = torch.randn(13, 6 * 64 + 16, generator=g).half().cuda()
    x = wide[:, 16:].view(13, 6, 64)[:, 1::2]  # every other head
    pos = i32(list(range(13)))
    op = Rotary(64)
    want = turn64(op, x, pos)
    rest = wide.clone()
    check(op(x, pos), *want)
    graph = torch.cuda.CUDAGraph()
    copy = x.clone()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        op(x, pos, out=x)
    graph.replay()
    torch.cuda.synchronize()
    check(x, *want)
    assert torch.equal(wide[:, :16], rest[:, :16])
    assert torch.equal(wide[:, 16:].view(13, 6, 64)[:, 0::2], rest[:, 16:].view(13, 6, 64)[:, 0::2])
    assert torch.equal(op(copy, pos), x)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,Hq,Hkv,D,page,rot,layout", [(1, 4, 4, 64, 16, 64, "half"), (8, 32, 8, 128, 16, 128, "half"),
                                                         (37, 6, 2, 128, 64, 32, "interleaved"), (5, 3, 1, 10, 4, 6, "half"),
                                                         (3, 24, 24, 64, 1, 64, "interleaved"), (500, 5, 1, 64, 32, 64, "half")])
def test_append(T, Hq, Hkv, D, page, rot, layout, dtype):
    from deca_b200.operators import RotaryAppend

    g = torch.Generator().manual_seed(T)
    qkv = torch.randn(T, (Hq + 2 * Hkv) * D, generator=g).to(dtype).cuda()
    q, k, v = (t.view(T, -1, D) for t in qkv.split([Hq * D, Hkv * D, Hkv * D], -1))
    pages = -(-T // page) + 2
    slots = torch.randperm(pages * page, generator=g)[:T]
    if T > 2:
        slots[1], slots[2] = -1, pages * page  # padding, and a row behind the cache
    pos = torch.randint(0, 9000, (T,), generator=g).to(torch.int32).cuda()
    kc, vc = (torch.full((pages, page, Hkv, D), 7.0, dtype=dtype, device="cuda") for _ in range(2))
    op = RotaryAppend(Hq, Hkv, D, page, rot_dim=rot, layout=layout, dtype=str(dtype).split(".")[1])
    out = op(q, k, v, pos, slots.cuda(), kc, vc)
    check(out, *turn64(op, q, pos))
    want_k, mag_k = turn64(op, k, pos)
    live = [t for t in range(T) if 0 <= slots[t] < pages * page]
    rows_k, rows_v = kc.view(-1, Hkv, D), vc.view(-1, Hkv, D)
    at = slots[live].cuda()
    check(rows_k[at], want_k[live], mag_k[live])
    assert torch.equal(rows_v[at], v[live])
    other = torch.ones(pages * page, dtype=torch.bool, device="cuda")
    other[at] = False
    assert (rows_k[other] == 7).all() and (rows_v[other] == 7).all()


def test_append_to_strided_cache():
    """Pages that hold the rows head by head, keys and values in one tensor; q in place."""
    from deca_b200.operators import RotaryAppend

    g = torch.Generator().manual_seed(0)
    T, Hq, Hkv, D, page = 9, 4, 2, 64, 16
    both = torch.full((3, 2, Hkv, page, D), 7.0, device="cuda").half()
    kc, vc = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    q, k, v = (torch.randn(T, h, D, generator=g).half().cuda() for h in (Hq, Hkv, Hkv))
    slots = torch.tensor([47, 0, 16, 15, 31, 32, 20, 5, 6], device="cuda")
    pos = i32(list(range(100, 109)))
    op = RotaryAppend(Hq, Hkv, D, page)
    want_q, want_k = turn64(op, q, pos), turn64(op, k, pos)
    op(q, k, v, pos, slots, kc, vc, out=q)
    check(q, *want_q)
    check(kc[slots // page, slots % page], *want_k)
    assert torch.equal(vc[slots // page, slots % page], v)
    assert int((both == 7).sum()) == both.numel() - 2 * T * Hkv * D


def test_refusals():
    from deca_b200.operators import Rotary, RotaryAppend

    x, pos = data(4, 2, 64, torch.float16)
    op = Rotary(64)
    for bad in [(x, pos.long()), (x, pos[:3]), (x[..., :32], pos), (x.bfloat16(), pos), (x.cpu(), pos), (x.transpose(1, 2), pos)]:
        with pytest.raises(ValueError):
            op(*bad)
    with pytest.raises(ValueError):
        op(x, pos, out=x[:1].expand(4, 2, 64))
    for kw in ({"rot_dim": 63}, {"rot_dim": 66}, {"layout": "quarter"}, {"dtype": "float32"}):
        with pytest.raises((AssertionError, KeyError)):
            Rotary(64, **kw)
    for scaling in ({"type": "linear", "factor": 0.5}, {"type": "other", "factor": 2}, {"type": "linear", "factor": 2, "low": 1}):
        with pytest.raises(ValueError):
            Rotary(64, scaling=scaling)
    ra = RotaryAppend(2, 2, 64, 16)
    kc = torch.zeros(2, 16, 2, 64, device="cuda").half()
    slots = torch.zeros(4, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError):
        ra(x, x, x, pos, slots.int(), kc, kc.clone())
    with pytest.raises(ValueError):
        ra(x, x, x, pos, slots, kc[:, :8], kc)
    assert op(x[:0], pos[:0]).shape == (0, 2, 64)
