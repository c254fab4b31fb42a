"""Plain 64-bit forms of the serving operators, and the relative rounding of the 16-bit types."""

import math

import torch

HALF_STEP = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
TINY = {torch.float16: 2.0**-25, torch.bfloat16: 2.0**-134}  # half a subnormal step


def attention64(q, k_cache, v_cache, table, cu, kv_lens, scale, causal=True):
    """(O, A): softmax(scale q K^T) V and the same weights on |V|, request by request, over visible keys only."""
    T, H, D = q.shape
    g = H // k_cache.shape[2]
    out = torch.zeros(T, H, D, dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    for r in range(len(kv_lens)):
        lo, hi, kv = cu[r], cu[r + 1], kv_lens[r]
        n = hi - lo
        if n == 0 or kv == 0:
            continue
        pages = table[r].long()
        k, v = (c[pages.clamp(0, c.shape[0] - 1)].flatten(0, 1)[:kv].double() for c in (k_cache, v_cache))
        for i in range(n) if n <= 4 or not torch.isfinite(v).all() else [None]:  # row by row where masked keys may hold anything
            if i is not None:
                seen = min(kv, kv - n + i + 1) if causal else kv
                if seen <= 0:
                    continue
                for h in range(H):
                    p = torch.softmax(q[lo + i, h].double() @ k[:seen, h // g].T * scale, -1)
                    out[lo + i, h] = p @ v[:seen, h // g]
                    mag[lo + i, h] = p @ v[:seen, h // g].abs()
            else:
                hide = torch.arange(kv, device=q.device) > kv - n + torch.arange(n, device=q.device)[:, None]
                for h in range(H):
                    s = q[lo:hi, h].double() @ k[:, h // g].T * scale
                    if causal:
                        s = s.masked_fill(hide, -math.inf)
                    p = torch.softmax(s, -1).nan_to_num(0.0)
                    out[lo:hi, h] = p @ v[:, h // g]
                    mag[lo:hi, h] = p @ v[:, h // g].abs()
    return out, mag


def attention_bound(out, mag, dtype):
    """Half a step for the output; half a step for each probability that enters the product (their sum is
    not rounded), weighted with |V|; and 2^-12 of the same for the fp32 scores: 128 products of the
    largest sums met here (110) times the scale err by 110 * 0.088 * 128 * 2^-24 < 2^-13.7, once in
    the numerator and once in the sum."""
    u = HALF_STEP[dtype]
    return u * out.abs() * 1.01 + (u * 1.01 + 2.0**-12) * mag + TINY[dtype]


def make_paged(kv_lens, new, H_q, H_kv, D, page, dtype, seed=0, spare=3, fill=float("nan")):
    """(q, k_cache, v_cache, table, cu, kv) of a batch whose pages are scattered and whose unused cache
    rows and pages hold `fill`; table entries behind a request's pages name page 0 (also filled)."""
    g = torch.Generator().manual_seed(seed)
    B = len(kv_lens)
    used = [-(-n // page) for n in kv_lens]
    width = max(max(used), 1) + 1
    n_pages = 1 + sum(used) + spare
    order = (torch.randperm(n_pages - 1, generator=g) + 1).tolist()
    table = torch.zeros(B, width, dtype=torch.int32)
    kc = torch.full((n_pages, page, H_kv, D), fill).to(dtype)
    vc = kc.clone()
    for r, n in enumerate(kv_lens):
        for e in range(used[r]):
            p = order.pop()
            table[r, e] = p
            rows = min(page, n - e * page)
            kc[p, :rows] = torch.randn(rows, H_kv, D, generator=g).to(dtype)
            vc[p, :rows] = torch.randn(rows, H_kv, D, generator=g).to(dtype)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    q = torch.randn(cu[-1], H_q, D, generator=g).to(dtype)
    return q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), cu, list(kv_lens)


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")
