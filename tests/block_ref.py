"""Plain implementations of the block-scaled cache's operators for the tests: the write in the fp32 arithmetic that
defines it, the values and the attention in 64 bits."""
import torch

U = 2.0 ** -8     # half a step of bf16, relative


def new_cache(nb, bs, h, d, layout, device="cpu", fill=0):
    """int8 K and V views [nb, bs, h, d] of one interleaved buffer ("vllm") or two arrays ("apart")."""
    if layout == "vllm":
        kv = torch.full((nb, h, bs, 2 * d), fill, dtype=torch.int8, device=device).permute(0, 2, 1, 3)
        return kv[..., :d], kv[..., d:]
    return tuple(torch.full((nb, bs, h, d), fill, dtype=torch.int8, device=device) for _ in range(2))


def new_scales(nb, bs, h, group, layout="side by side", device="cpu", fill=0.0):
    if layout == "side by side":
        s = torch.full((nb, h, bs // group, 2), fill, device=device)
        return {"k_scale": s[..., 0], "v_scale": s[..., 1]}
    return {n: torch.full((nb, h, bs // group), fill, device=device) for n in ("k_scale", "v_scale")}


def write(x, cache, scale, cu, lens, table):
    """Rows x [T, H, D] of one side into cache [nb, bs, H, D] and scale [nb, H, blocks], in place, on the host."""
    bs = cache.shape[1]
    gr = bs // scale.shape[2]
    for r in range(len(cu) - 1):
        n, q = int(lens[r]), int(cu[r + 1]) - int(cu[r])
        p = max(n - q, 0)
        while p < n and q > 0:
            b0 = p // gr * gr
            stop = min(n, b0 + gr)
            page, s0, blk = int(table[r, b0 // bs]), b0 % bs, b0 % bs // gr
            rows = x[int(cu[r + 1]) - n + p:int(cu[r + 1]) - n + stop].float()
            if 0 <= page < cache.shape[0]:
                a = rows.abs()
                top = torch.where(torch.isfinite(a), a, torch.zeros_like(a)).amax((0, 2))
                old = scale[page, :, blk].clone() if p > b0 else torch.zeros(x.shape[1])
                s = torch.maximum(torch.maximum(top / 127.0, torch.tensor(1e-8)), old)
                if p > b0:
                    c = cache[page, s0:s0 + p - b0]
                    grown = torch.round(c.float() * (old / s)[None, :, None]).to(torch.int8)
                    c.copy_(torch.where((s > old)[None, :, None], grown, c))
                cache[page, s0 + p - b0:s0 + stop - b0] = torch.round(rows / s[None, :, None]).clamp(-127, 127).to(torch.int8)
                scale[page, :, blk] = s
            p = stop


def values(cache, scale, table_row, n):
    """(codes, scales) of a request's first n keys in 64 bits: [H, n, D] and [H, n]."""
    bs = cache.shape[1]
    gr = bs // scale.shape[2]
    ids = table_row[:-(-n // bs)].long()
    codes = cache[ids].flatten(0, 1)[:n].transpose(0, 1).double()
    s = scale[ids].transpose(1, 2).repeat_interleave(gr, 1).flatten(0, 1)[:n].t().double()
    return codes, s


def attention(q, kc, vc, scales, cu, lens, table, softmax_scale):
    """(out, bound) of a batch in 64 bits, [T, Hq, D]; bound: the largest error of a bf16 output whose arithmetic is the
    operators': see the terms below. Rows of the batch past cu[-1] are zero in both."""
    hq, d = q.shape[1:]
    hkv = kc.shape[2]
    g = hq // hkv
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    for r in range(len(cu) - 1):
        a, b, n = int(cu[r]), int(cu[r + 1]), int(lens[r])
        if b == a or n <= 0:
            continue
        kcode, ks = values(kc, scales["k_scale"], table[r], n)
        vcode, vs = values(vc, scales["v_scale"], table[r], n)
        tiles = -(-n // 32)
        for h in range(hkv):
            k, v = kcode[h] * ks[h][:, None], vcode[h] * vs[h][:, None]
            x = q[a:b, h * g:(h + 1) * g].double()                                 # [t, g, D]
            w = torch.einsum("tgd,nd->tgn", x, k) * softmax_scale
            seen = torch.arange(n, device=q.device)[None] <= (n - (b - a) + torch.arange(b - a, device=q.device))[:, None]
            w = w.masked_fill(~seen[:, None], -torch.inf)
            p = torch.softmax(w, -1).nan_to_num(0.0)
            o, mag = p @ v, p @ v.abs()
            # q as a multiple of max|q| / 16256, each channel half a step off at most: a score's error, and twice that
            # (numerator and denominator) in the weights; fp32 sums of d products beside it
            top = x.abs().amax(-1, keepdim=True)
            off = softmax_scale * (top / 32512 + 2.0 ** -24 * d * top) * k.abs().sum(-1).max()
            # the weights: bf16 (half a step of each), or multiples of 1 / 16256 of their 32-key tile's largest p vs
            pv = torch.zeros(*p.shape[:2], tiles * 32, dtype=torch.float64, device=q.device)
            pv[..., :n] = p * vs[h]
            step = pv.view(*p.shape[:2], tiles, 32).amax(-1) / 32512
            per_tile = torch.zeros(tiles * 32, d, dtype=torch.float64, device=q.device)
            per_tile[:n] = vcode[h].abs()
            fixed = step @ per_tile.view(tiles, 32, d).sum(1)
            err = torch.expm1(2 * off) * 2 * mag + torch.maximum(U * mag, fixed) + 1e-5 * mag
            out[a:b, h * g:(h + 1) * g] = o
            bound[a:b, h * g:(h + 1) * g] = U * (o.abs() + err) + err + 1e-30
    return out, bound


def check(got, want, bound, what=""):
    err = (got.double() - want).abs()
    worst = float((err / bound.clamp_min(1e-30)).max()) if err.numel() else 0.0
    assert torch.isfinite(got.float()).all(), what
    assert bool((err <= bound).all()), (what, worst, float(err.max()))
    norm = float(want.norm())
    if norm:
        rel = float((got.double() - want).norm()) / norm
        assert rel <= 5e-3, (what, rel)      # a bf16 output's rounding is 1.7e-3, bf16 weights add less than that again
    return worst
