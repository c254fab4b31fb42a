"""The operators of a paged serving step, as a user's program calls them, with their plain forms.

Four operators run one after the other around the projections of an attention block: PagedStep turns
the lengths of a batch of requests into pages, slots and positions; AddRMSNorm adds the residual and
normalises; RotaryAppend rotates q and k and writes k and v to the cache; PagedAttention attends to the
cache.  ``own`` selects between elementary torch operations in 32 bits and the framework's kernels.
"""

import math

import torch

own = False

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}
E4M3_MAX = 448.0


# ------------------------------------------------------------------------------------------- cases
def norm_case(M, N, dtype, out="same", group=0):
    return {"op": "norm", "M": M, "N": N, "dtype": dtype, "out": out, "group": group}


def append_case(T, Hq, Hkv, D, page, dtype, rot=0, layout="half", scaling="none", far=4096):
    return {"op": "append", "T": T, "Hq": Hq, "Hkv": Hkv, "D": D, "page": page, "dtype": dtype, "rot": rot or D,
            "layout": layout, "scaling": scaling, "far": far}


def rotary_case(T, H, D, dtype, rot=0, layout="half", scaling="none", far=4096, inverse=False):
    return {"op": "rotary", "T": T, "H": H, "D": D, "dtype": dtype, "rot": rot or D, "layout": layout,
            "scaling": scaling, "far": far, "inverse": inverse}


def step_case(B, page, W, new_max, ctx_max):
    return {"op": "step", "B": B, "page": page, "W": W, "new_max": new_max, "ctx_max": ctx_max}


def attn_case(B, Hq, Hkv, D, page, q_min, q_max, ctx_min, ctx_max, dtype):
    return {"op": "attn", "B": B, "Hq": Hq, "Hkv": Hkv, "D": D, "page": page, "q_min": q_min, "q_max": q_max,
            "ctx_min": ctx_min, "ctx_max": ctx_max, "dtype": dtype}


def listed():
    return [
        # one token each of sixteen requests between two layers: launch latency
        {"name": "norm_16x4096", **norm_case(16, 4096, "float16")},
        # a ragged batch of tokens and a row length that is no multiple of a tile; one scale a token
        {"name": "norm_1021x5000_e4m3", **norm_case(1021, 5000, "bfloat16", "e4m3")},
        # a large prefill batch that feeds an 8-bit product with a scale per 128 columns
        {"name": "norm_16384x8192_e4m3_g128", **norm_case(16384, 8192, "bfloat16", "e4m3", 128)},
        # eight requests that decode one token each
        {"name": "append_8", **append_case(8, 32, 8, 128, 16, "bfloat16")},
        # a prefill batch; q, k, v are column blocks of one projection's output
        {"name": "append_8192", **append_case(8192, 32, 8, 128, 64, "float16")},
        # the gradient of a partial, interleaved rotation at far positions with frequency bands
        {"name": "rotary_4099_inverse",
         **rotary_case(4099, 24, 128, "bfloat16", 64, "interleaved", "band", 1000000, True)},
        # the step of a small decoding batch, and of a large one in which new prompts arrive
        {"name": "step_8", **step_case(8, 16, 64, 1, 900)},
        {"name": "step_512_mixed", **step_case(512, 16, 512, 150, 7000)},
        # a single request that decodes: one token, a short context, equal head counts
        {"name": "attn_decode_1", **attn_case(1, 16, 16, 64, 16, 1, 1, 333, 333, "float16")},
        # a decoding batch with contexts of every length up to 8192
        {"name": "attn_decode_64", **attn_case(64, 32, 8, 128, 16, 1, 1, 1000, 8191, "bfloat16")},
        # two chunks of 2048 prompt tokens behind 6144 cached ones
        {"name": "attn_chunk_2x2048", **attn_case(2, 32, 8, 128, 64, 2048, 2048, 6144, 6144, "float16")},
        # decodes and odd chunks mixed in one batch, three query heads to a key head
        {"name": "attn_mixed_9", **attn_case(9, 24, 8, 64, 32, 1, 700, 0, 4300, "bfloat16")},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng):
    """(Hq, Hkv): equal counts, small groups, odd groups and one key head for all."""
    Hkv = rng.choice([1, 2, 4, 5, 8, 16])
    return Hkv * rng.choice([g for g in (1, 2, 3, 4, 5, 7, 8) if Hkv * g <= 48]), Hkv


def draw(rng):
    op = rng.choice(["norm", "append", "rotary", "step", "attn", "attn"])
    dtype = rng.choice(["float16", "bfloat16"])
    if op == "norm":
        N = _log_int(rng, 64, 12000)
        M = _log_int(rng, 1, max(1, 16384 * 8192 // N // 2) if N > 4096 else 16384)
        out = rng.choice(["same", "e4m3"])
        return norm_case(M, N, dtype, out, rng.choice([0, 64, 128]) if out == "e4m3" else 0)
    if op in ("append", "rotary"):
        D = rng.choice([64, 128])
        rot = rng.choice([D, D, D // 2, D // 4])
        layout = rng.choice(["half", "interleaved"])
        scaling = rng.choice(["none", "linear", "base", "band"])
        far = _log_int(rng, 1000, 1000000)
        if op == "append":
            Hq, Hkv = _heads(rng)
            return append_case(_log_int(rng, 1, 8000), Hq, Hkv, D, rng.choice([16, 32, 64, 128]), dtype, rot, layout,
                               scaling, far)
        return rotary_case(_log_int(rng, 1, 8000), rng.randint(1, 40), D, dtype, rot, layout, scaling, far,
                           rng.choice([True, False]))
    if op == "step":
        page = rng.choice([16, 32, 64, 128])
        new_max, ctx_max = _log_int(rng, 1, 300), _log_int(rng, 1, 8000)
        return step_case(_log_int(rng, 1, 600), page, -(-(new_max + ctx_max) // page) + rng.randint(0, 9), new_max,
                         ctx_max)
    Hq, Hkv = _heads(rng)
    D, page = rng.choice([64, 128]), rng.choice([16, 32, 64, 128])
    if rng.random() < 0.5:  # decoding: one token a request, or the few of a verified guess
        q_max = rng.choice([1, 1, 1, 2, 4])
        ctx_max = _log_int(rng, 16, 16000)
        B = _log_int(rng, 1, max(1, min(96, 300000 // (ctx_max + q_max))))
        return attn_case(B, Hq, Hkv, D, page, rng.randint(1, q_max), q_max, rng.randint(0, ctx_max), ctx_max, dtype)
    q_max = _log_int(rng, 8, 2000)
    ctx_max = _log_int(rng, 16, 6000)
    B = _log_int(rng, 1, max(1, min(12, 1000000000 // (Hq * q_max * (ctx_max + q_max)))))
    return attn_case(B, Hq, Hkv, D, page, rng.randint(1, q_max), q_max, rng.randint(0, ctx_max), ctx_max, dtype)


# ------------------------------------------------------------------------------------------ inputs
def _spread(lo, hi, n, gen):
    """n whole numbers over lo..hi on the CPU, the largest among them."""
    v = torch.randint(lo, hi + 1, (n,), generator=gen)
    v[0] = hi
    return v


def _scaling(case):
    return {"none": None, "linear": {"type": "linear", "factor": 4.0}, "base": {"type": "base", "factor": 4.0},
            "band": {"type": "band", "factor": 8.0, "original_length": 8192, "low": 1.0, "high": 32.0}}[case["scaling"]]


def _frequencies(case):
    """(inverse frequencies in 64 bits, amplitude) of a rotation."""
    rot, s = case["rot"], _scaling(case)
    base = 10000.0
    if s and s["type"] == "base":
        base *= s["factor"] ** (rot / (rot - 2))
    f = base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    amplitude = 1.0
    if s and s["type"] == "linear":
        f = f / s["factor"]
    if s and s["type"] == "band":
        turns = s["original_length"] * f / (2 * math.pi)
        keep = ((turns - s["low"]) / (s["high"] - s["low"])).clamp(0, 1)
        f = f * keep + f / s["factor"] * (1 - keep)
        amplitude = 0.1 * math.log(s["factor"]) + 1.0
    return f, amplitude


def _lengths(case):
    """(context lengths, new tokens) of an attention case, a property of the case and not of the seed."""
    gen = torch.Generator().manual_seed(1000 * case["B"] + case["q_max"] + case["ctx_max"])
    return (_spread(case["ctx_min"], case["ctx_max"], case["B"], gen),
            _spread(case["q_min"], case["q_max"], case["B"], gen))


def _step_lengths(case, seed):
    gen = torch.Generator().manual_seed(seed)
    B = case["B"]
    ctx = _spread(0, case["ctx_max"], B, gen)
    new = torch.ones(B, dtype=torch.int64)
    if case["new_max"] > 1:  # a share of the requests brings a chunk, the others decode
        new = torch.where(torch.rand(B, generator=gen) < 0.5, _spread(1, case["new_max"], B, gen), new)
    return ctx, new


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    cpu = torch.Generator().manual_seed(seed)
    s = {"case": dict(case)}
    if case["op"] == "norm":
        dt, M, N = DTYPES[case["dtype"]], case["M"], case["N"]
        s["x"] = torch.randn(M, N, device="cuda", dtype=dt, generator=g)
        s["res"] = torch.randn(M, N, device="cuda", dtype=dt, generator=g)
        s["w"] = torch.randn(N, device="cuda", generator=g).mul_(0.1).add_(1.0).to(dt)
    elif case["op"] == "append":
        dt, T, Hq, Hkv, D, P = (DTYPES[case["dtype"]], case["T"], case["Hq"], case["Hkv"], case["D"], case["page"])
        qkv = torch.randn(T, (Hq + 2 * Hkv) * D, device="cuda", dtype=dt, generator=g)
        s["q"] = qkv[:, : Hq * D].view(T, Hq, D)
        s["k"] = qkv[:, Hq * D : (Hq + Hkv) * D].view(T, Hkv, D)
        s["v"] = qkv[:, (Hq + Hkv) * D :].view(T, Hkv, D)
        s["pos"] = torch.randint(0, case["far"], (T,), generator=cpu).to(torch.int32).cuda()
        pages = -(-T // P) + 3
        page_of = torch.randperm(pages, generator=cpu)
        t = torch.arange(T)
        s["slots"] = (page_of[t // P] * P + t % P).cuda()
        s["kc"] = torch.zeros(pages, P, Hkv, D, device="cuda", dtype=dt)
        s["vc"] = torch.zeros(pages, P, Hkv, D, device="cuda", dtype=dt)
        f, s["amplitude"] = _frequencies(case)
        s["freq"] = f.cuda()
    elif case["op"] == "rotary":
        dt, T = DTYPES[case["dtype"]], case["T"]
        s["x"] = torch.randn(T, case["H"], case["D"], device="cuda", dtype=dt, generator=g)
        s["pos"] = torch.randint(0, case["far"], (T,), generator=cpu).to(torch.int32).cuda()
        f, s["amplitude"] = _frequencies(case)
        s["freq"] = f.cuda()
    elif case["op"] == "step":
        B, P, W = case["B"], case["page"], case["W"]
        ctx, new = _step_lengths(case, seed)
        held = -(-ctx // P)
        wanted = int((-(-(ctx + new) // P) - held).sum())
        pages = torch.randperm(int(held.sum()) + wanted + 40, generator=cpu).to(torch.int32)
        e = torch.arange(W)
        rank = (held.cumsum(0) - held)[:, None] + e
        table = torch.where(e < held[:, None], pages[rank.clamp(max=len(pages) - 1)], torch.tensor(-1, dtype=torch.int32))
        s["ctx"], s["new"] = ctx.to(torch.int32).cuda(), new.to(torch.int32).cuda()
        s["table"] = table.to(torch.int32).cuda()
        s["free"] = pages[int(held.sum()) :].cuda()
        s["n_free"] = torch.tensor([wanted + 40], dtype=torch.int32, device="cuda")
        s["T"] = B * case["new_max"]  # the batch's token budget: rows behind the last token are padding
    else:
        dt, B, Hq, Hkv, D, P = (DTYPES[case["dtype"]], case["B"], case["Hq"], case["Hkv"], case["D"], case["page"])
        ctx, new = _lengths(case)
        kv = ctx + new
        W = -(-int(kv.max()) // P)
        used = -(-kv // P)
        pages = int(used.sum()) + 5
        order = torch.randperm(pages, generator=cpu).to(torch.int32)
        rank = (used.cumsum(0) - used)[:, None] + torch.arange(W)
        s["table"] = order[rank.clamp(max=pages - 1)].cuda()
        s["kc"] = torch.randn(pages, P, Hkv, D, device="cuda", dtype=dt, generator=g)
        s["vc"] = torch.randn(pages, P, Hkv, D, device="cuda", dtype=dt, generator=g)
        T = int(new.sum())
        s["q"] = torch.randn(T, Hq, D, device="cuda", dtype=dt, generator=g)
        s["cu"] = torch.cat([torch.zeros(1, dtype=torch.int64), new.cumsum(0)]).to(torch.int32).cuda()
        s["kv"] = kv.to(torch.int32).cuda()
        s["max_q"], s["max_kv"] = int(new.max()), int(kv.max())
    return s


# ------------------------------------------------------------------------------------- plain forms
def _plain_norm(s):
    case, dt = s["case"], s["x"].dtype
    h = s["x"].float() + s["res"].float()
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-6) * s["w"].float()
    if case["out"] == "same":
        return {"y": y.to(dt), "h": h.to(dt)}
    M, N = y.shape
    group = case["group"] or N
    n = -(-N // group)
    grouped = torch.nn.functional.pad(y, (0, n * group - N)).view(M, n, group)
    scale = grouped.abs().amax(-1) / E4M3_MAX
    inverse = torch.where(scale > 0, 1.0 / scale, torch.zeros_like(scale))
    q = (grouped * inverse[..., None]).clamp(-E4M3_MAX, E4M3_MAX).view(M, n * group)[:, :N]
    return {"q": q.to(torch.float8_e4m3fn), "scales": scale, "h": h.to(dt)}


def _plain_rotate(x, s, inverse=False):
    case, rot = s["case"], s["case"]["rot"]
    angle = s["pos"].double()[:, None] * s["freq"]
    c, sn = ((f(angle) * s["amplitude"]).float()[:, None, :] for f in (torch.cos, torch.sin))
    if inverse:
        sn = -sn
    x = x.float()
    if case["layout"] == "half":
        a, b = x[..., : rot // 2], x[..., rot // 2 : rot]
        turned = torch.cat([a * c - b * sn, a * sn + b * c], -1)
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * c - b * sn, a * sn + b * c], -1).flatten(-2)
    return torch.cat([turned, x[..., rot:]], -1)


def _plain_append(s):
    case, dt = s["case"], s["q"].dtype
    rows = (-1, case["Hkv"], case["D"])
    s["kc"].view(rows)[s["slots"]] = _plain_rotate(s["k"], s).to(dt)
    s["vc"].view(rows)[s["slots"]] = s["v"]
    return {"q": _plain_rotate(s["q"], s).to(dt), "k_cache": s["kc"], "v_cache": s["vc"]}


def _plain_step(s):
    case = s["case"]
    P, W, B, T = case["page"], case["W"], case["B"], s["T"]
    dev = s["ctx"].device
    ctx, new = s["ctx"].long(), s["new"].long()
    kv = (ctx + new).clamp(max=W * P)
    cu = torch.cat([torch.zeros(1, dtype=torch.long, device=dev), new.cumsum(0)])
    held, wanted = (ctx + P - 1) // P, (kv + P - 1) // P
    need = wanted - held
    e = torch.arange(W, device=dev)
    rank = (need.cumsum(0) - need)[:, None] + e - held[:, None]
    fresh = (e >= held[:, None]) & (e < wanted[:, None])
    page = torch.where(rank < s["n_free"], s["free"][(s["n_free"] - 1 - rank).clamp(0, len(s["free"]) - 1)], -1)
    table = torch.where(fresh, page.to(torch.int32), s["table"])
    t = torch.arange(T, device=dev)
    r = torch.searchsorted(cu[1:], t, right=True).clamp(max=B - 1)
    pos = ctx[r] + t - cu[r]
    at = table[r, (pos // P).clamp(max=W - 1)].long()
    live = (t < cu[-1]) & (pos < W * P) & (at >= 0)
    short = (need.sum() - s["n_free"]).clamp(min=0)
    return {"cu_q": cu.to(torch.int32), "kv_lens": kv.to(torch.int32), "table": table,
            "positions": torch.where(t < cu[-1], pos, 0).to(torch.int32),
            "slots": torch.where(live, at * P + pos % P, -1),
            "n_free": (s["n_free"] - need.sum()).clamp(min=0).to(torch.int32), "short": short.to(torch.int32)}


def _plain_attn(s):
    case, q = s["case"], s["q"]
    B, Hq, Hkv, D = case["B"], case["Hq"], case["Hkv"], case["D"]
    dev, g = q.device, Hq // Hkv
    cu, kv = s["cu"].long(), s["kv"].long()
    lens = cu[1:] - cu[:-1]
    t, j = torch.arange(s["max_q"], device=dev), torch.arange(s["table"].shape[1] * case["page"], device=dev)
    padded = q[(cu[:-1, None] + t).clamp(max=len(q) - 1)].float().view(B, s["max_q"], Hkv, g, D)
    keys, values = (c[s["table"].long()].flatten(1, 2).float().permute(0, 2, 1, 3) for c in (s["kc"], s["vc"]))
    rows = padded.permute(0, 2, 3, 1, 4).reshape(B, Hkv, g * s["max_q"], D)
    scores = (rows @ keys.transpose(-1, -2)).mul_(1.0 / math.sqrt(D)).view(B, Hkv, g, s["max_q"], len(j))
    seen = j <= (kv - lens)[:, None, None] + t[:, None]  # [B, max_q, keys]
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    values = values.masked_fill((j >= kv[:, None])[:, None, :, None], 0.0)
    out = (p.view(B, Hkv, g * s["max_q"], len(j)) @ values).view(B, Hkv, g, s["max_q"], D)
    out = torch.where(total > 0, out / total, torch.zeros_like(out)).permute(0, 3, 1, 2, 4).reshape(B, s["max_q"], Hq, D)
    token = torch.arange(len(q), device=dev)
    r = torch.searchsorted(cu[1:], token, right=True)
    return {"out": out[r, token - cu[r]].to(q.dtype)}


# ------------------------------------------------------------------------------- framework's calls
def _operator(case, s):
    """The operator object that a program makes once for a geometry and keeps."""
    from deca_b200 import operators as ops

    if case["op"] == "norm":
        return ops.AddRMSNorm(case["M"], case["N"], case["dtype"], eps=1e-6, out=case["out"], group=case["group"])
    if case["op"] == "append":
        return ops.RotaryAppend(case["Hq"], case["Hkv"], case["D"], case["page"], rot_dim=case["rot"],
                                layout=case["layout"], scaling=_scaling(case), dtype=case["dtype"])
    if case["op"] == "rotary":
        return ops.Rotary(case["D"], rot_dim=case["rot"], layout=case["layout"], scaling=_scaling(case),
                          dtype=case["dtype"])
    if case["op"] == "step":
        return ops.PagedStep(case["B"], case["page"], case["W"], s["T"])
    return ops.PagedAttention(case["B"], case["Hq"], case["Hkv"], case["D"], case["page"], max_q=s["max_q"],
                              max_kv=s["max_kv"], dtype=case["dtype"])


def run(s):
    case = s["case"]
    if not own:
        if case["op"] == "rotary":
            return {"y": _plain_rotate(s["x"], s, case["inverse"]).to(s["x"].dtype)}
        return {"norm": _plain_norm, "append": _plain_append, "step": _plain_step, "attn": _plain_attn}[case["op"]](s)
    if "operator" not in s:
        s["operator"] = _operator(case, s)
    op = s["operator"]
    if case["op"] == "norm":
        r = op(s["x"], s["res"], s["w"])
        return {"y": r[0], "h": r[1]} if case["out"] == "same" else {"q": r[0], "scales": r[1], "h": r[2]}
    if case["op"] == "append":
        q = op(s["q"], s["k"], s["v"], s["pos"], s["slots"], s["kc"], s["vc"])
        return {"q": q, "k_cache": s["kc"], "v_cache": s["vc"]}
    if case["op"] == "rotary":
        return {"y": op(s["x"], s["pos"], inverse=case["inverse"])}
    if case["op"] == "step":
        r = op(s["ctx"], s["new"], s["table"], s["free"], s["n_free"])
        return {"cu_q": r.cu_q, "kv_lens": r.kv_lens, "table": s["table"], "positions": r.positions, "slots": r.slots,
                "n_free": r.n_free, "short": r.short}
    return {"out": op(s["q"], s["kc"], s["vc"], s["table"], s["cu"], s["kv"])}


# ---------------------------------------------------------------------------------- work, 64 bits
def work(case):
    if case["op"] == "norm":
        M, N = case["M"], case["N"]
        scales = 4 * M * (-(-N // case["group"]) if case["group"] else 1) if case["out"] == "e4m3" else 0
        return {"bytes": M * N * (6 + (1 if scales else 2)) + 2 * N + scales, "flops": 8 * M * N}
    if case["op"] == "append":
        heads = case["Hq"] + 2 * case["Hkv"]
        return {"bytes": case["T"] * (4 * heads * case["D"] + 12),
                "flops": 3 * case["T"] * (case["Hq"] + case["Hkv"]) * case["rot"]}
    if case["op"] == "rotary":
        n = case["T"] * case["H"]
        return {"bytes": 4 * n * case["D"] + 4 * case["T"], "flops": 3 * n * case["rot"]}
    if case["op"] == "step":
        B, tokens = case["B"], case["B"] * case["new_max"]
        pages = B * (case["new_max"] // case["page"] + 1)
        return {"bytes": 16 * B + 12 * tokens + 8 * pages, "flops": 4 * (B + tokens)}
    ctx, new = _lengths(case)
    kv = ctx + new
    seen = int((new * ctx + new * (new + 1) // 2).sum())
    T = int(new.sum())
    return {"bytes": 4 * T * case["Hq"] * case["D"] + 4 * int(kv.sum()) * case["Hkv"] * case["D"] + 4 * int((kv // case["page"]).sum()),
            "flops": 4 * seen * case["Hq"] * case["D"]}


def _exact_turn(x, s):
    """Rotation as a product of complex numbers."""
    case, rot = s["case"], s["case"]["rot"]
    angle = s["pos"].double()[:, None] * s["freq"] * (-1.0 if case.get("inverse") else 1.0)
    turn = torch.polar(torch.full_like(angle, s["amplitude"]), angle)[:, None, :]
    head, tail = x.double()[..., :rot], x.double()[..., rot:]
    if case["layout"] == "half":
        pairs = head.unflatten(-1, (2, rot // 2)).transpose(-1, -2)
    else:
        pairs = head.unflatten(-1, (rot // 2, 2))
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    z = z.transpose(-1, -2) if case["layout"] == "half" else z
    return torch.cat([z.flatten(-2), tail], -1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        h = s["x"].double() + s["res"].double()
        y = h / (h.pow(2).sum(-1, keepdim=True) / case["N"] + 1e-6).sqrt() * s["w"].double()
        if case["out"] == "same":
            return {"y": y, "h": h}
        scales, q = [], []
        for block in y.split(case["group"] or case["N"], -1):
            scales.append(block.abs().max(-1).values / E4M3_MAX)
            q.append(torch.nan_to_num(block / scales[-1][:, None]))
        return {"q": torch.cat(q, -1), "scales": torch.stack(scales, -1), "h": h}
    if case["op"] == "rotary":
        return {"y": _exact_turn(s["x"], s)}
    if case["op"] == "append":
        kc, vc = s["kc"].double(), s["vc"].double()
        page, row = s["slots"] // case["page"], s["slots"] % case["page"]
        kc[page, row] = _exact_turn(s["k"], s)
        vc[page, row] = s["v"].double()
        return {"q": _exact_turn(s["q"], s), "k_cache": kc, "v_cache": vc}
    if case["op"] == "step":
        return None  # whole numbers
    g, cu, kv = case["Hq"] // case["Hkv"], s["cu"].tolist(), s["kv"].tolist()
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for r in range(case["B"]):
        n, pages = cu[r + 1] - cu[r], s["table"][r, : -(-kv[r] // case["page"])].long()
        k, v = (c[pages].flatten(0, 1)[: kv[r]].double() for c in (s["kc"], s["vc"]))
        last = kv[r] - n + torch.arange(n, device="cuda")
        hidden = torch.arange(kv[r], device="cuda") > last[:, None]
        for head in range(case["Hq"]):
            a = s["q"][cu[r] : cu[r + 1], head].double() @ k[:, head // g].T / math.sqrt(case["D"])
            out[cu[r] : cu[r + 1], head] = torch.softmax(a.masked_fill(hidden, -math.inf), -1) @ v[:, head // g]
    return {"out": out}
