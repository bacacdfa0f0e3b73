"""Plain implementations of the 4-bit cache's operators, the eviction and the norm with rotation for the tests, in 64 bits."""
import math

import torch

U = 2.0 ** -8     # half a step of bf16, relative
GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def new_cache(nb, bs, h, d, layout, device="cpu", fill=0):
    """uint8 K and V views [nb, bs, h, d / 2] of one interleaved buffer ("vllm") or two arrays ("apart")."""
    if layout == "vllm":
        kv = torch.full((nb, h, bs, d), fill, dtype=torch.uint8, device=device).permute(0, 2, 1, 3)
        return kv[..., :d // 2], kv[..., d // 2:]
    return tuple(torch.full((nb, bs, h, d // 2), fill, dtype=torch.uint8, device=device) for _ in range(2))


def new_scales(nb, bs, h, d, layout="side by side", device="cpu", fill=0):
    if layout == "side by side":
        s = torch.full((nb, h, 2, bs, d // 32), fill, dtype=torch.uint8, device=device)
        return {"k_scale": s[:, :, 0], "v_scale": s[:, :, 1]}
    return {n: torch.full((nb, h, bs, d // 32), fill, dtype=torch.uint8, device=device) for n in ("k_scale", "v_scale")}


def quantize(x):
    """(bytes [..., D / 2], exponent bytes [..., D / 32]) of bf16 rows [..., D]."""
    g = x.double().unflatten(-1, (-1, 32))
    g = torch.where(torch.isnan(g), 0.0, g)
    a = g.abs()
    top = torch.where(torch.isfinite(a), a, 0.0).amax(-1)
    e = torch.where(top > 0, torch.floor(torch.log2(top.clamp_min(1e-300))), -200.0) - 2
    e = torch.where(top * torch.exp2(-e) > 7, e + 1, e).clamp(-100, 125)
    y = (a * torch.exp2(-e)[..., None]).clamp_max(6.0)
    grid = torch.tensor(GRID, dtype=torch.float64, device=x.device)
    far = (y[..., None] - grid).abs()
    best = far.amin(-1, keepdim=True)
    near = far == best
    # of two as near, the even code
    code = (near * torch.where(torch.arange(8, device=x.device) % 2 == 0, 2, 1)).argmax(-1)
    code = code + 8 * torch.signbit(g)
    code = code.flatten(-2).to(torch.uint8)
    return code[..., 0::2] | code[..., 1::2] << 4, (e + 127).to(torch.uint8)


def decode(code, e):
    """float64 [..., D]."""
    c = torch.stack([code & 15, code >> 4], -1).flatten(-2).long()
    grid = torch.tensor(GRID + [-x for x in GRID], dtype=torch.float64, device=code.device)
    return grid[c] * torch.exp2(e.double() - 127).repeat_interleave(32, -1)


def write(x, cache, scale, slots):
    """Rows x [T, H, D] of one side, in place."""
    bs = cache.shape[1]
    code, e = quantize(x)
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < cache.shape[0] * bs:
            cache[s // bs, s % bs] = code[t].to(cache.device)
            scale[s // bs, :, s % bs] = e[t].to(cache.device)


def values(cache, scale, table_row, n):
    """float64 [H, n, D]: a request's first n keys."""
    ids = table_row[:-(-n // cache.shape[1])].long()
    return decode(cache[ids].flatten(0, 1)[:n], scale[ids].transpose(1, 2).flatten(0, 1)[:n]).transpose(0, 1).contiguous()


def _scores(x, k, softmax_scale):
    """[t, g, n] scores of query rows x [t, g, D] over one head's keys k [n, D], -inf where not seen."""
    t, n = x.shape[0], k.shape[0]
    w = (x.reshape(-1, x.shape[-1]) @ k.t().contiguous()).view(t, -1, n) * softmax_scale
    seen = torch.arange(n, device=x.device)[None] <= (n - t + torch.arange(t, device=x.device))[:, None]
    return w.masked_fill(~seen[:, None], -torch.inf)


def _score_error(x, k, softmax_scale):
    """[t, g, 1]: how far a score may be off: d exact products, summed in fp32 in any order, each sum off by a step at most."""
    size = (x.abs().reshape(-1, x.shape[-1]) @ k.abs().t().contiguous()).amax(-1).view(*x.shape[:2], 1)
    return softmax_scale * size * x.shape[-1] * 2.0 ** -23


def attention(q, kc, vc, scales, cu, lens, table, softmax_scale, short_q=8):
    """(out, bound [T, Hq, D], lse, bound [T, Hq]) of a batch; the bounds: the largest error of outputs whose arithmetic is
    the operators', see the terms below. Rows of the batch past cu[-1] are zero."""
    hq, d = q.shape[1:]
    hkv = kc.shape[2]
    g = hq // hkv
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
    lse_bound = torch.zeros_like(lse)
    for r in range(len(cu) - 1):
        a, b, n = int(cu[r]), int(cu[r + 1]), int(lens[r])
        if b == a or n <= 0:
            continue
        ks, vs = values(kc, scales["k_scale"], table[r], n), values(vc, scales["v_scale"], table[r], n)
        for h in range(hkv):
            k, v = ks[h], vs[h]
            x = q[a:b, h * g:(h + 1) * g].double()                                 # [t, g, D]
            w = _scores(x, k, softmax_scale)
            of = torch.logsumexp(w, -1)
            p = torch.softmax(w, -1).nan_to_num(0.0)
            shape = (b - a, g, d)
            o, mag = (p.view(-1, n) @ v).view(shape), (p.view(-1, n) @ v.abs()).view(shape)
            off = _score_error(x, k, softmax_scale)
            # a score's error once in the numerator and once in the denominator; the weights to bf16, of short requests to a
            # sum of two, both cut off (a step, 2^-7, of what is left, itself below 2^-7); fp32 sums; a weight is at
            # least 2^-40 of itself in fp32 (a maximum that lags by 8, and 32 more), so one below 2^(40 - 126) of the row's may
            # be lost, and all of them together
            err = torch.expm1(2 * off) * mag + (U if b - a > short_q else 2.0 ** -14) * mag + 1e-5 * mag + n * 2.0 ** -86 * v.abs().max()
            out[a:b, h * g:(h + 1) * g] = o
            bound[a:b, h * g:(h + 1) * g] = U * (o.abs() + err) + err + 1e-38
            lse[a:b, h * g:(h + 1) * g] = of
            # fp32: the scores, their maximum plus 32 and a logarithm of 2^-32 and more
            size = torch.where(of.isfinite(), of.abs(), 0.0) + 32
            lse_bound[a:b, h * g:(h + 1) * g] = off[..., 0] + size * 2.0 ** -21
    return out, bound, lse, lse_bound


def check(got, want, bound, what=""):
    err = (got.double() - want).abs()
    worst = float((err / bound.clamp_min(1e-300)).max()) if err.numel() else 0.0
    assert torch.isfinite(got.float()).all(), what
    assert bool((err <= bound).all()), (what, worst, float(err.max()))
    return worst


def check_lse(got, want, bound, what=""):
    fine = torch.isfinite(want)
    assert torch.equal(got.double()[~fine], want[~fine]), what
    check(got[fine], want[fine], bound[fine], what)


def key_weights(q, kc, scales, lse, shape, cu, lens, table, softmax_scale, short_q=8):
    """(what is added, bound) [B, H, cols] in 64 bits."""
    hq = q.shape[1]
    hkv = kc.shape[2]
    g = hq // hkv
    add = torch.zeros(shape, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(add)
    for r in range(len(cu) - 1):
        a, b, n = int(cu[r]), int(cu[r + 1]), int(lens[r])
        if b == a or b - a > short_q or n <= 0:
            continue
        ks = values(kc, scales["k_scale"], table[r], n)
        m = min(n, shape[2])
        for h in range(hkv):
            x = q[a:b, h * g:(h + 1) * g].double()
            w = _scores(x, ks[h], softmax_scale)
            of = lse[a:b, h * g:(h + 1) * g].double()[..., None]
            real = (w > -math.inf) & of.isfinite()
            p = torch.where(real, torch.exp(w - of), 0.0)
            # a score's error, the exponent's in fp32 (a product, a sum) and of its power of two
            off = _score_error(x, ks[h], softmax_scale) + torch.where(real, w.abs() + of.abs(), 0.0) * 2.0 ** -22 + 2.0 ** -21
            add[r, h, :m] = p.sum((0, 1))[:m]
            bound[r, h, :m] = (p * torch.expm1(off)).sum((0, 1))[:m] + p.sum((0, 1))[:m] * 2.0 ** -18 + 1e-37
    return add, bound


def evict(weights, n, keep, recent, cols):
    """Positions that one head keeps (ascending), of its running sums [cols] in any order-preserving type."""
    m = max(min(keep, n), 0)
    if n <= keep:
        return list(range(n))
    recent = min(recent, m)
    w = [float(weights[i]) if i < cols else 0.0 for i in range(n - recent)]
    order = sorted(range(n - recent), key=lambda i: (0 if math.isnan(w[i]) else 1, 0.0 if math.isnan(w[i]) else -w[i], i))
    return sorted(order[:m - recent]) + list(range(n - recent, n))


def norm_rope(x, positions, table, weight, eps, interleaved):
    """(y, bound) of rows x [T, H, D] in 64 bits; the bound: one rounding to bf16 of fp32 arithmetic (a sum of D squares, a
    reciprocal square root, two products; then two products and a sum)."""
    r = table.shape[1]
    y = x.double()
    if weight is not None:
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * weight.double()
    t = table.double()[positions.long().clamp(0, table.shape[0] - 1)][:, None]
    cos, sin = t[..., :r // 2], t[..., r // 2:]
    if interleaved:
        a, b = y[..., 0:r:2], y[..., 1:r:2]
    else:
        a, b = y[..., :r // 2], y[..., r // 2:r]
    turned = (a * cos - b * sin, b * cos + a * sin)
    size = ((a * cos).abs() + (b * sin).abs(), (b * cos).abs() + (a * sin).abs())
    out, mag = y.clone(), y.abs()
    for got, part in ((out, turned), (mag, size)):
        if interleaved:
            got[..., 0:r:2], got[..., 1:r:2] = part
        else:
            got[..., :r // 2], got[..., r // 2:r] = part
    err = 40 * 2.0 ** -24 * mag
    return out, U * (out.abs() + err) + err + 1e-38
