"""The serving operators together, as a decoder layer's attention block runs them over several steps: residual and
norm, q/k/v projection (GEMMTC), bookkeeping, rotation and append, attention over the paged cache, output
projection.  Each operator's result is held to 64-bit arithmetic on the tensors it was given, while pages and
slots are followed by a plain allocator and keys and values by dense copies per request."""

import pytest

torch = pytest.importorskip("torch")

from serving_util import HALF_STEP, TINY, attention64, attention_bound, i32  # noqa: E402

pytestmark = pytest.mark.gpu

H_Q, H_KV, D, PAGE, WIDTH, HIDDEN = 8, 2, 64, 16, 12, 256


def turn64(op, x, positions):
    freq, amplitude = op.frequencies()
    angle = positions.double()[:, None, None] * torch.tensor(freq, dtype=torch.float64, device=x.device)
    c, s = angle.cos() * amplitude, angle.sin() * amplitude
    a, b = x.double().chunk(2, -1)
    return torch.cat([a * c - b * s, a * s + b * c], -1), torch.cat([a.abs() + b.abs()] * 2, -1) * amplitude


def within(got, want, slack):
    bound = HALF_STEP[got.dtype] * want.abs() * (1 + 1e-6) + slack + TINY[got.dtype]
    assert ((got.double() - want).abs() <= bound).all()


class Layer:
    def __init__(self, dtype, tokens, requests, max_q):
        from deca_b200.operators import GEMMTC, AddRMSNorm, PagedAttention, PagedStep, RotaryAppend

        self.dtype = dtype
        name = str(dtype).split(".")[1]
        g = torch.Generator().manual_seed(0)
        self.w = (1 + 0.1 * torch.randn(HIDDEN, generator=g)).to(dtype).cuda()
        self.w_qkv = (torch.randn(HIDDEN, (H_Q + 2 * H_KV) * D, generator=g) / HIDDEN**0.5).to(dtype).cuda()
        self.w_out = (torch.randn(H_Q * D, HIDDEN, generator=g) / (H_Q * D) ** 0.5).to(dtype).cuda()
        self.norm = AddRMSNorm(tokens, HIDDEN, name)
        self.qkv = GEMMTC(tokens, (H_Q + 2 * H_KV) * D, HIDDEN, name)
        self.proj = GEMMTC(tokens, HIDDEN, H_Q * D, name)
        self.step = PagedStep(requests, PAGE, WIDTH, tokens)
        self.rope = RotaryAppend(H_Q, H_KV, D, PAGE, dtype=name)
        self.attn = PagedAttention(requests, H_Q, H_KV, D, PAGE, max_q, WIDTH * PAGE, name)

    def __call__(self, x, res, ctx, new, table, free, n_free, kc, vc):
        y, res = self.norm(x, res, self.w, res_out=res)
        qkv = self.qkv(y, self.w_qkv)
        q, k, v = (t.view(len(x), -1, D) for t in qkv.split([H_Q * D, H_KV * D, H_KV * D], -1))
        s = self.step(ctx, new, table, free, n_free)
        turned = self.rope(q, k, v, s.positions, s.slots, kc, vc)
        o = self.attn(turned, kc, vc, table, s.cu_q, s.kv_lens, out=torch.zeros_like(turned))
        return self.proj(o.view(len(x), -1), self.w_out), s, (q, k, v, turned, o)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_steps_of_a_layer(dtype):
    """Prompts arrive, are continued in chunks and decoded; a batch carries padding rows at its end."""
    steps = [[37, 5, 0], [9, 1, 20], [1, 1, 1], [1, 1, 33], [1, 1, 1]]  # new tokens of three requests
    tokens = 64
    g = torch.Generator().manual_seed(7)
    pages = 20
    kc, vc = (torch.full((pages, PAGE, H_KV, D), float("nan"), dtype=dtype, device="cuda") for _ in range(2))
    free = torch.randperm(pages, generator=g).to(torch.int32).cuda()
    left = free.tolist()
    n_free, ctx = i32([pages]), i32([0, 0, 0])
    table = torch.full((3, WIDTH), -1, dtype=torch.int32, device="cuda")
    dense_k, dense_v = [[] for _ in range(3)], [[] for _ in range(3)]
    layer = Layer(dtype, tokens, 3, 40)
    for new in steps:
        x, res = (torch.randn(tokens, HIDDEN, generator=g).to(dtype).cuda() for _ in range(2))
        out, s, (q, k, v, turned, o) = layer(x, res, ctx, i32(new), table, free, n_free, kc, vc)
        assert torch.isfinite(out.float()).all() and s.short.tolist() == [0]
        # pages and slots
        t, had = 0, ctx.tolist()
        for r, n in enumerate(new):
            for i in range(n):
                place = had[r] + i
                if place % PAGE == 0:
                    assert table[r, place // PAGE].item() == left.pop()
                assert s.positions[t].item() == place and s.slots[t].item() == table[r, place // PAGE].item() * PAGE + place % PAGE
                t += 1
        assert (s.slots[t:] == -1).all() and s.n_free.tolist() == [len(left)]
        # rotation and append
        want_q, mag = turn64(layer.rope, q, s.positions)
        within(turned, want_q, 2.0**-20 * mag)
        want_k, mag = turn64(layer.rope, k, s.positions)
        rows = s.slots[:t]
        within(kc.view(-1, H_KV, D)[rows], want_k[:t], 2.0**-20 * mag[:t])
        assert torch.equal(vc.view(-1, H_KV, D)[rows], v[:t])
        # attention over each request's dense history
        at = 0
        for r, n in enumerate(new):
            dense_k[r].append(kc.view(-1, H_KV, D)[rows[at : at + n]])
            dense_v[r].append(vc.view(-1, H_KV, D)[rows[at : at + n]])
            if n:
                hk, hv = torch.cat(dense_k[r]), torch.cat(dense_v[r])
                one = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
                want, mag = attention64(turned[at : at + n], hk[None], hv[None], one, [0, n], [len(hk)], D**-0.5)
                assert ((o[at : at + n].double() - want).abs() <= attention_bound(want, mag, dtype)).all()
            at += n
        assert (o[at:] == 0).all()
        ctx, n_free = s.kv_lens, s.n_free


def test_decoding_loop_in_a_graph():
    """One captured decoding step, replayed with the state it leaves, gives the bits of the same steps made eagerly."""
    tokens, steps = 3, 20
    g = torch.Generator().manual_seed(1)
    xs = torch.randn(steps, tokens, HIDDEN, generator=g).half().cuda()
    layer = Layer(torch.float16, tokens, 3, 1)

    def state():
        gen = torch.Generator().manual_seed(2)
        kc, vc = (torch.randn(30, PAGE, H_KV, D, generator=gen).half().cuda() for _ in range(2))
        table = torch.full((3, WIDTH), -1, dtype=torch.int32, device="cuda")
        table[0, :2], table[1, :1] = i32([3, 4]), i32([9])
        return {"x": xs[0].clone(), "res": torch.zeros(tokens, HIDDEN, dtype=torch.float16, device="cuda"), "ctx": i32([31, 7, 0]),
                "new": i32([1, 1, 1]), "table": table, "free": i32(list(range(10, 30))), "n_free": i32([20]), "kc": kc, "vc": vc}

    def advance(st):
        out, s, _ = layer(st["x"], st["res"], st["ctx"], st["new"], st["table"], st["free"], st["n_free"], st["kc"], st["vc"])
        st["ctx"].copy_(s.kv_lens)
        st["n_free"].copy_(s.n_free)
        return out

    eager, want = state(), []
    for i in range(steps):
        eager["x"].copy_(xs[i])
        want.append(advance(eager).clone())
    st = state()
    stream = torch.cuda.Stream()
    warm = state()
    with torch.cuda.stream(stream):
        advance(warm)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = advance(st)
    for i in range(steps):
        st["x"].copy_(xs[i])
        graph.replay()
        assert torch.equal(out, want[i]), i
    for name in ("ctx", "n_free", "table", "kc", "vc", "res"):
        assert torch.equal(st[name], eager[name]), name
