"""Calls that the serving operators cannot answer rightly are refused before anything is launched."""

import pytest

torch = pytest.importorskip("torch")

from serving_util import i32, make_paged  # noqa: E402

pytestmark = pytest.mark.gpu


def test_forward_mode_tangents_are_refused():
    """The operators record no gradient of either mode: a dual tensor would lose its tangent."""
    import torch.autograd.forward_ad as fwd

    from deca_b200.operators import AddRMSNorm, PagedAttention, Rotary, RotaryAppend

    x = torch.randn(4, 64, device="cuda").half()
    q, kc, vc, table, cu, kv = make_paged([60, 40], [4, 20], 4, 2, 64, 16, torch.float16)
    slots = torch.arange(4, device="cuda")
    with fwd.dual_level():
        d = fwd.make_dual(x, torch.ones_like(x))
        for call in (lambda t: AddRMSNorm(4, 64)(t, x, x[0]), lambda t: AddRMSNorm(4, 64)(x, t, x[0]), lambda t: AddRMSNorm(4, 64)(x, x, t[0]),
                     lambda t: Rotary(64)(t[:, None], i32([1, 2, 3, 4])),
                     lambda t: RotaryAppend(1, 2, 64, 16)(x[:, None], t[:, None].expand(4, 2, 64), x[:, None].expand(4, 2, 64), i32([0, 1, 2, 3]), slots, kc, vc)):
            with pytest.raises(ValueError, match="tangent"):
                call(d)
            call(x)
        op = PagedAttention(2, 4, 2, 64, 16, 20, 60)
        dq = fwd.make_dual(q, torch.ones_like(q))
        with pytest.raises(ValueError, match="tangent"):
            op(dq, kc, vc, table, i32(cu), i32(kv))
        op(fwd.unpack_dual(dq).primal, kc, vc, table, i32(cu), i32(kv))
    torch.cuda.synchronize()


def test_pending_negation_is_refused():
    """The imaginary part of a conjugated complex tensor is a view whose memory holds the values with the other sign."""
    from deca_b200.operators import AddRMSNorm, Rotary

    z = torch.complex(*torch.randn(2, 4, 64, device="cuda").half())
    x = torch._neg_view(z.imag.contiguous())
    assert x.is_neg()
    w = torch.ones(64, device="cuda").half()
    for call in (lambda t: AddRMSNorm(4, 64)(t, w.expand(4, 64).contiguous(), w), lambda t: Rotary(64)(t[:, None], i32([0, 1, 2, 3]))):
        with pytest.raises(ValueError, match="negation"):
            call(x)
        call(x.resolve_neg())
    torch.cuda.synchronize()


def test_more_heads_than_an_int_holds_are_refused():
    """2^32 + 2 heads (one, expanded) are not two."""
    from deca_b200.operators import Rotary

    x = torch.ones(1, 1, 2, device="cuda").half()
    for H in (2**32 + 2, 2**31 + 1, 65537):
        with pytest.raises(ValueError, match="heads"):
            Rotary(2)(x.expand(1, H, 2), i32([0]))
    assert Rotary(2)(x.expand(1, 65536, 2), i32([0])).shape == (1, 65536, 2)
    torch.cuda.synchronize()
