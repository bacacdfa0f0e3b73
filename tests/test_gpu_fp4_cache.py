"""The 4-bit cache's operators on the GPU (kvq.fp4_cache) against plain implementations: codes, exponents, rows read back and
evicted keys bit for bit, attention and weights within the bounds that their roundings add up to (fp4_ref)."""
import numpy as np
import pytest
import torch
from conftest import nan_like, nan_segm

import fp4_ref as R
from kvq import cuda_kernels as ck
from kvq import fp4_cache as fc
from kvq import rope

pytestmark = pytest.mark.gpu
DEV = "cuda"
GEOM = [(4, 128, 16), (8, 128, 32), (2, 64, 64), (1, 128, 128), (3, 64, 16)]
HEADS = [(28, 4, 128), (32, 8, 128), (14, 2, 64), (16, 16, 64), (32, 1, 128), (6, 3, 64), (4, 4, 128)]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rows(n, h, d, seed, loud=1.0):
    g = gen(seed)
    gain = torch.exp(0.7 * torch.randn(h, d, generator=g))
    size = 1 + loud * torch.rand(n, 1, 1, generator=g)
    return [((torch.randn(n, h, d, generator=g) * gain + 0.3) * size).to(torch.bfloat16) for _ in range(2)]


def page_table(lens, bs, seed, spare=3):
    """Shuffled pages for `lens` positions each: int32 [B, width + 1] (unused entries -1) and the pages in all."""
    pages = [-(-n // bs) for n in lens]
    nb = sum(pages) + spare
    perm = torch.randperm(nb, generator=gen(seed))
    t = torch.full((len(lens), max(pages + [1]) + 1), -1, dtype=torch.int32)
    at = 0
    for r, p in enumerate(pages):
        t[r, :p] = perm[at:at + p]
        at += p
    return t, nb


def slots_of(table, lens, bs, first=None):
    """Slots of positions first[r] .. lens[r] - 1 of each request, one after the other."""
    out = []
    for r, n in enumerate(lens):
        p = torch.arange(0 if first is None else first[r], n)
        out.append(table[r][p // bs].long() * bs + p % bs)
    return torch.cat(out)


def i32(x):
    return torch.as_tensor(np.asarray(x, dtype=np.int32)).to(DEV)


def cumsum(x):
    return np.concatenate([[0], np.cumsum(x)]).tolist()


class Cache:
    def __init__(self, h, d, bs, nb, layout="vllm", fill=0xff, scale_fill=0xff):
        self.geom = (h, d, bs)
        self.kc, self.vc = R.new_cache(nb, bs, h, d, layout, DEV, fill)
        self.scales = R.new_scales(nb, bs, h, d, "side by side" if layout == "vllm" else "apart", DEV, scale_fill)

    def parts(self):
        return (self.kc, self.vc, self.scales["k_scale"], self.scales["v_scale"])


def filled(h, d, bs, lens, seed=0, layout="vllm", loud=1.0):
    """A cache whose requests hold `lens` keys; what lies outside them is poison: codes of -6 and exponent bytes of 255, which
    are no number."""
    table, nb = page_table(lens, bs, seed)
    c = Cache(h, d, bs, nb, layout)
    c.k, c.v = rows(sum(lens), h, d, seed + 1, loud)
    fc.quant_fp4_cache(c.k.to(DEV), c.v.to(DEV), c.kc, c.vc, c.scales, slots_of(table, lens, bs).to(DEV))
    c.host, c.table = table, table.to(DEV)
    return c


# ------------------------------------------------------------------------------------------------ write
def _same_write(c, k, v, slots, before):
    for x, cache, name, old, old_scale in ((k, c.kc, "k_scale", before[0], before[2]), (v, c.vc, "v_scale", before[1], before[3])):
        R.write(x, old, old_scale, slots)
        bad = (cache != old).any(-1)
        assert not bool(bad.any()), (name, int(bad.sum()))
        assert torch.equal(c.scales[name], old_scale), name


@pytest.mark.parametrize("h,d,bs", GEOM)
@pytest.mark.parametrize("layout", ["vllm", "apart"])
@pytest.mark.parametrize("n", [1, 3, 37, 700])
def test_write(h, d, bs, layout, n):
    """Every code and exponent of the whole cache, untouched ones too."""
    nb = -(-n // bs) + 5
    c = Cache(h, d, bs, nb, layout, 0x5a, 0x11)
    k, v = rows(n + 2, h, d, n)
    slots = torch.randperm(nb * bs, generator=gen(n))[:n]
    before = [t.clone() for t in c.parts()]
    fc.quant_fp4_cache(k.to(DEV), v.to(DEV), c.kc, c.vc, c.scales, slots.to(DEV))
    _same_write(c, k, v, slots, before)


@pytest.mark.parametrize("h,d,bs", GEOM[:3])
def test_write_skips_padding_and_slots_that_are_not_there(h, d, bs):
    c = Cache(h, d, bs, 6, "vllm", 0x5a, 0x11)
    k, v = rows(9, h, d, 1)
    slots = torch.tensor([-1, 6 * bs, 3, -(1 << 40), 1 << 40, 6 * bs - 1, 0, -1, 17])
    before = [t.clone() for t in c.parts()]
    fc.quant_fp4_cache(k.to(DEV), v.to(DEV), c.kc, c.vc, c.scales, slots.to(DEV))
    _same_write(c, k, v, slots, before)


@pytest.mark.parametrize("d", [64, 128])
def test_write_of_every_bf16(d):
    """All 65,536 patterns: alone in their group beside zeros, and in groups of what they are next to (NaN, infinities, ties,
    subnormals and the largest among them)."""
    x = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    alone = torch.zeros(1 << 16, 1, d, dtype=torch.bfloat16)
    alone[:, 0, 5] = x
    alone[:, 0, 37] = 1.0
    near = x.view(-1, 1, d)
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 6.5, 0.5, 4.0, 6.0]).repeat(6)[:64].repeat(d // 64)
    ties = torch.cat([ties * s for s in (1.0, -1.0, 2.0 ** -90, -2.0 ** 100)]).to(torch.bfloat16).view(-1, 1, d)
    k = torch.cat([alone, near, ties])
    n = k.shape[0]
    c = Cache(1, d, 16, -(-n // 16), "apart", 0x5a, 0x11)
    slots = torch.arange(n)
    fc.quant_fp4_cache(k.to(DEV), k.flip(0).contiguous().to(DEV), c.kc, c.vc, c.scales, slots.to(DEV))
    for x, cache, s in ((k, c.kc, c.scales["k_scale"]), (k.flip(0), c.vc, c.scales["v_scale"])):
        code, e = R.quantize(x)
        got, ge = cache.flatten(0, 1)[:n].cpu(), s.transpose(1, 2).flatten(0, 1)[:n].cpu()
        assert torch.equal(ge, e)
        # (a NaN is a zero of either sign)
        assert bool(((got == code) | (R.decode(got, ge) == R.decode(code, e))[..., 0::2] & (R.decode(got, ge) == R.decode(code, e))[..., 1::2]).all())


def test_write_takes_strided_rows():
    """K and V as slices of a packed projection."""
    h, d, bs, n = 4, 128, 16, 33
    g = gen(3)
    qkv = torch.randn(n, 44 * d, generator=g).to(torch.bfloat16).to(DEV)
    k, v = qkv[:, 28 * d:32 * d].view(n, h, d), qkv[:, 40 * d:].view(n, h, d)
    c = Cache(h, d, bs, 4, "vllm", 0, 0)
    before = [t.clone() for t in c.parts()]
    slots = torch.arange(n) + 7
    fc.quant_fp4_cache(k, v, c.kc, c.vc, c.scales, slots.to(DEV))
    _same_write(c, k.cpu(), v.cpu(), slots, before)


# ------------------------------------------------------------------------------------------------ read
@pytest.mark.parametrize("h,d,bs", GEOM)
def test_read_back(h, d, bs):
    lens = [1, 15, 16, 33, 300, bs, 2 * bs + 1]
    c = filled(h, d, bs, lens, layout="apart" if h == 1 else "vllm")
    first = [0, 3, 15, 0, 41, 1, bs]
    count = [n - f for n, f in zip(lens, first)]
    out = [torch.full((sum(count) + 5, h, d), 9.0, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    fc.read_fp4_cache(c.kc, c.vc, c.scales, i32(first), i32(cumsum(count)), c.table, *out)
    for got, cache, name in ((out[0], c.kc, "k_scale"), (out[1], c.vc, "v_scale")):
        want = torch.cat([R.values(cache, c.scales[name], c.table[r], n)[:, f:].transpose(0, 1)
                          for r, (f, n) in enumerate(zip(first, lens))])
        assert torch.equal(got[:-5].double(), want)
        assert bool((got[-5:] == 9.0).all())


def test_read_skips_and_replaces():
    """A request of no rows, a negative start; a page id that is not there reads page 0; bytes of 255 give finite values."""
    c = filled(2, 128, 16, [40, 40, 40])
    table = c.table.clone()
    table[2, 1] = 1 << 30
    c.table[2, 1] = 0
    out = [torch.full((60, 2, 128), 9.0, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    fc.read_fp4_cache(c.kc, c.vc, c.scales, i32([-5, 4, 0]), i32([0, 20, 20, 60]), table, *out)
    assert bool((out[0][:20] == 9.0).all())
    c.scales["k_scale"].clamp_(max=252)
    assert torch.equal(out[0][20:].double(), R.values(c.kc, c.scales["k_scale"], c.table[2], 40).transpose(0, 1))


def test_read_past_the_last_level_cache():
    """A read of more than 256 MiB (streaming loads and stores)."""
    h, d, bs, n = 8, 128, 64, 60000
    c = filled(h, d, bs, [n])
    out = [torch.empty(n, h, d, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    fc.read_fp4_cache(c.kc, c.vc, c.scales, i32([0]), i32([0, n]), c.table, *out)
    for got, cache, name in ((out[0], c.kc, "k_scale"), (out[1], c.vc, "v_scale")):
        assert torch.equal(got.double(), R.values(cache, c.scales[name], c.table[0], n).transpose(0, 1))


# ------------------------------------------------------------------------------------------------ attention
def attend(c, hq, q_lens, lens, segm=None, seed=3, scale=None, pad=2, q=None):
    h, d, bs = c.geom
    cu = cumsum(q_lens)
    if q is None:
        q = torch.randn(cu[-1] + pad, hq, d, generator=gen(seed)).to(torch.bfloat16).to(DEV)
    scale = d ** -0.5 if scale is None else scale
    out = torch.full_like(q, 7.0)
    lse = torch.full(q.shape[:2], 7.0, device=DEV)
    plan = ck.plan_long(cu, lens, bs)
    got = fc.fp4_paged_attention(q, c.kc, c.vc, out, i32(cu), i32(lens), c.table, max(q_lens), scale, c.scales, plan, segm, lse)
    assert got is out
    want, bound, of, of_bound = R.attention(q, c.kc, c.vc, c.scales, cu, lens, c.table, scale, ck.SHORT_Q)
    assert bool((out[cu[-1]:] == 7.0).all()) and bool((lse[cu[-1]:] == 7.0).all())
    R.check(out[:cu[-1]], want[:cu[-1]], bound[:cu[-1]], (q_lens, lens))
    for r, n in enumerate(q_lens):
        at = slice(cu[r], cu[r + 1])
        if n <= ck.SHORT_Q:
            R.check_lse(lse[at], of[at], of_bound[at], (r, n, lens[r]))
        else:
            assert bool((lse[at] == 7.0).all())
    return q, out, lse


@pytest.mark.parametrize("hq,h,d", HEADS)
@pytest.mark.parametrize("qlen", [1, 2, 5, 8])
@pytest.mark.parametrize("split", [False, True])
def test_short_queries(hq, h, d, qlen, split):
    lens = [0, 1, qlen, 15, 16, 17, 31, 32, 33, 64, 100, 257, 1000]
    q_lens = [qlen] * len(lens)
    c = filled(h, d, 16 if h != 2 else 64, lens, seed=qlen, layout="vllm" if qlen % 2 else "apart")
    attend(c, hq, q_lens, lens, nan_segm(sum(q_lens), hq, 16, d) if split else None)


@pytest.mark.parametrize("splits", [1, 2, 7, 64])
@pytest.mark.parametrize("hq,h,d", [(28, 4, 128), (14, 2, 64)])
def test_long_contexts_are_cut(splits, hq, h, d):
    lens = [5000, 17, 9001]
    c = filled(h, d, 32, lens)
    attend(c, hq, [1, 4, 2], lens, nan_segm(7, hq, splits, d))
    attend(c, hq, [8, 8, 8], lens, nan_segm(24, hq, splits, d))
    attend(c, hq, [1, 1, 1], lens, nan_segm(3, hq, splits, d))


def test_split_buffers_of_fewer_rows():
    lens = [3000, 2000, 100]
    c = filled(4, 128, 16, lens)
    attend(c, 28, [2, 3, 1], lens, nan_segm(4, 28, 8, 128))


@pytest.mark.parametrize("hq,h,d", HEADS)
@pytest.mark.parametrize("bs", [16, 64])
def test_long_queries(hq, h, d, bs):
    lens = [9, 40, 333, 700]
    c = filled(h, d, bs, lens)
    attend(c, hq, [9, 20, 333, 130], lens)


@pytest.mark.parametrize("hq,h,d", HEADS)
def test_long_queries_hold_their_weights_as_short_ones(hq, h, d):
    """A row's weights are a sum of two bf16 (2^-14 of each and less) whatever its request's number of tokens."""
    lens, q_lens = [9, 40, 333, 700, 5000], [9, 20, 333, 130, 10]
    c = filled(h, d, 32, lens)
    q, out, _ = attend(c, hq, q_lens, lens, pad=0)
    cu = cumsum(q_lens)
    want, bound, _, _ = R.attention(q, c.kc, c.vc, c.scales, cu, lens, c.table, d ** -0.5, short_q=max(q_lens))
    R.check(out, want, bound)


def test_mixed_batch_and_few_rows_over_many_keys():
    lens = [500, 20, 64, 2000, 9000]
    c = filled(4, 128, 32, lens)
    attend(c, 28, [1, 20, 8, 300, 12], lens)
    attend(c, 28, [1, 20, 8, 300, 12], lens, nan_segm(341, 28, 16, 128))


def test_long_query_without_keys():
    """A request of a warm-up: more query tokens than keys, none at all."""
    c = filled(4, 128, 16, [3, 50])
    c.table[0] = 0
    attend(c, 28, [20, 60], [0, 50])
    attend(c, 28, [20, 3], [0, 0])


def test_padded_requests_of_a_graph_batch():
    lens = [50, 700, 0, 0]
    c = filled(4, 128, 16, lens)
    c.table[2:] = 0
    attend(c, 28, [1, 1, 0, 0], lens)
    attend(c, 28, [1, 1, 0, 0], lens, nan_segm(4, 28, 16, 128))


@pytest.mark.parametrize("magnitude", [1e-3, 1.0, 30.0])
def test_peaked_and_flat_softmax(magnitude):
    lens = [300, 4000, 77]
    c = filled(4, 128, 16, lens)
    q = (magnitude * torch.randn(13, 28, 128, generator=gen(8))).to(torch.bfloat16).to(DEV)
    attend(c, 28, [1, 8, 4], lens, nan_segm(13, 28, 16, 128), q=q)
    attend(c, 28, [1, 1, 11], lens, q=q)


@pytest.mark.parametrize("scale", [1e-16, 1e-5, 3.0])
def test_softmax_scales(scale):
    lens = [300, 900, 40]
    c = filled(4, 128, 16, lens)
    attend(c, 28, [1, 8, 30], lens, scale=scale)


@pytest.mark.parametrize("up", [-90, -40, 40, 90])
def test_values_of_other_magnitudes(up):
    """V of 2^up and K of 2^-up under a softmax scale that brings the scores back."""
    lens = [100, 900, 200]
    table, nb = page_table(lens, 16, 1)
    c = Cache(4, 128, 16, nb)
    k, v = rows(sum(lens), 4, 128, 2)
    fc.quant_fp4_cache((k.double() * 2.0 ** -up / 4).to(torch.bfloat16).to(DEV), (v.double() * 2.0 ** up).to(torch.bfloat16).to(DEV),
                       c.kc, c.vc, c.scales, slots_of(table, lens, 16).to(DEV))
    c.table = table.to(DEV)
    q = (torch.randn(34, 28, 128, generator=gen(4)).double() * 2.0 ** up).to(torch.bfloat16).to(DEV)
    attend(c, 28, [1, 3, 30], lens, q=q, pad=0)


def test_largest_values_stay_finite():
    """V at the format's end, 6 2^125, under equal weights: the output is that value, which bf16 holds."""
    lens = [4000, 50]
    table, nb = page_table(lens, 16, 1)
    c = Cache(4, 128, 16, nb)
    n = sum(lens)
    k = torch.zeros(n, 4, 128, dtype=torch.bfloat16, device=DEV)
    v = torch.full((n, 4, 128), 6 * 2.0 ** 125, dtype=torch.bfloat16, device=DEV)
    fc.quant_fp4_cache(k, v, c.kc, c.vc, c.scales, slots_of(table, lens, 16).to(DEV))
    for q_lens in ([1, 1], [8, 3], [30, 20]):
        cu = cumsum(q_lens)
        q = torch.ones(cu[-1], 28, 128, dtype=torch.bfloat16, device=DEV)
        for segm in (None, nan_segm(cu[-1], 28, 16, 128)):
            out = torch.zeros_like(q)
            fc.fp4_paged_attention(q, c.kc, c.vc, out, i32(cu), i32(lens), table.to(DEV), max(q_lens), 0.1, c.scales,
                                   ck.plan_long(cu, lens, 16), segm)
            assert bool(((out.double() / 2.0 ** 125 - 6).abs() <= 6 * (2 * R.U + 1e-5)).all())


@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("sign", [-1, 1])
@pytest.mark.parametrize("hq,h,d,q_lens", [(28, 4, 128, [1, 1, 1]), (28, 4, 128, [8, 2, 3]), (14, 2, 64, [4, 1, 8]), (28, 4, 128, [30, 9, 200]),
                                           (16, 16, 64, [9, 40, 300])])
def test_scores_of_any_size(hq, h, d, q_lens, sign, split):
    """Scores of some +-1e36: a row is the mean of V over the keys of the larger score, of which every row sees some, its
    log-sum-exp that score and the logarithm of their number."""
    lens = [3000, 40, 700]
    table, nb = page_table(lens, 16, 1)
    c = Cache(h, d, 16, nb)
    n, cu = sum(lens), cumsum(q_lens)
    far = torch.cat([torch.arange(m) % 3 != 2 for m in lens])       # position 2, 5, .. have the larger score
    k = sign * 2.0 ** 57 * torch.where(far, 2.0 if sign < 0 else 1.0, 1.0 if sign < 0 else 2.0)[:, None, None].expand(n, h, d)
    v = rows(n, h, d, 3)[1]
    fc.quant_fp4_cache(k.to(torch.bfloat16).contiguous().to(DEV), v.to(DEV), c.kc, c.vc, c.scales, slots_of(table, lens, 16).to(DEV))
    c.table = table.to(DEV)
    q = torch.full((cu[-1], hq, d), 2.0 ** 57, dtype=torch.bfloat16, device=DEV)
    out, lse = torch.full_like(q, 7.0), torch.zeros(cu[-1], hq, device=DEV)
    segm = nan_segm(cu[-1], hq, 16, d) if split else None
    fc.fp4_paged_attention(q, c.kc, c.vc, out, i32(cu), i32(lens), c.table, max(q_lens), d ** -0.5, c.scales,
                           ck.plan_long(cu, lens, 16), segm, lse)
    top = sign * d ** 0.5 * 2.0 ** 114 * (1 if sign < 0 else 2)
    for r, m in enumerate(lens):
        vs = R.values(c.vc, c.scales["v_scale"], c.table[r], m)
        for t in range(cu[r], cu[r + 1]):
            at = vs[:, 2:m - cu[r + 1] + t + 1:3]
            if at.shape[1] == 0:
                continue
            want = at.mean(1).repeat_interleave(hq // h, 0)
            mag = at.abs().mean(1).repeat_interleave(hq // h, 0)
            # equal weights: their rounding (2^-14), fp32 sums, the output's half step
            err = (2.0 ** -14 + 1e-5) * mag
            R.check(out[t], want, R.U * (want.abs() + err) + err, (r, t))
            if q_lens[r] <= ck.SHORT_Q:
                assert bool(((lse[t].double() - top).abs() <= abs(top) * d * 2.0 ** -22).all()), (r, t)


@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("q_lens", [[1, 1, 1, 1], [8, 8, 3, 8], [40, 9, 300, 12]])
def test_rows_that_are_no_number_stay_their_own(q_lens, split):
    """A NaN or an infinity in one q row makes that row and its log-sum-exp NaN and no other's; rows of zeros average."""
    lens = [3000, 70, 400, 33]
    c = filled(4, 128, 32, lens)
    cu = cumsum(q_lens)
    q = torch.randn(cu[-1], 28, 128, generator=gen(1)).to(torch.bfloat16).to(DEV)
    q[cu[1]:cu[2], 3] = 0
    q[cu[3]:] = 0
    clean = q.clone()
    bad = [(0, 5, 17, "nan"), (cu[1] - 1, 27, 127, "inf"), (cu[2], 0, 0, "-inf")]
    for t, h, d, x in bad:
        q[t, h, d] = float(x)
    segm = nan_segm(cu[-1], 28, 16, 128) if split else None
    out, lse = torch.full_like(q, 7.0), torch.zeros(cu[-1], 28, device=DEV)
    fc.fp4_paged_attention(q, c.kc, c.vc, out, i32(cu), i32(lens), c.table, max(q_lens), 128 ** -0.5, c.scales,
                           ck.plan_long(cu, lens, 32), segm, lse)
    want, bound, of, of_bound = R.attention(clean, c.kc, c.vc, c.scales, cu, lens, c.table, 128 ** -0.5)
    short = max(q_lens) <= 8
    for t, h, _, _ in bad:
        assert bool(torch.isnan(out[t, h]).all()), (t, h)
        out[t, h] = want[t, h].to(out.dtype)
        if short:
            assert bool(torch.isnan(lse[t, h]))
            lse[t, h] = of[t, h]
    R.check(out, want, bound, q_lens)
    if short:
        R.check_lse(lse, of, of_bound)


@pytest.mark.parametrize("byte", [253, 254, 255])
@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("hq,h,d,q_lens", [(28, 4, 128, [8, 2, 5, 3]), (4, 4, 128, [8, 2, 5, 3]), (14, 2, 64, [4, 2, 3, 2]),
                                           (16, 16, 64, [7, 2, 8, 3]), (28, 4, 128, [20, 40, 9, 300])])
def test_exponent_bytes_that_no_write_makes(hq, h, d, q_lens, split, byte):
    """A byte above 252 at a request's last key, K's and V's: query rows that do not see that key, all but the request's last,
    are what they are over the clean cache."""
    lens = [3000, 33, 400, 301]
    c = filled(h, d, 16, lens)
    cu = cumsum(q_lens)
    q = torch.randn(cu[-1], hq, d, generator=gen(2)).to(torch.bfloat16).to(DEV)
    want, bound, of, of_bound = R.attention(q, c.kc, c.vc, c.scales, cu, lens, c.table, d ** -0.5)
    for r, n in enumerate(lens):
        for s in c.scales.values():
            s[int(c.host[r, (n - 1) // 16]), :, (n - 1) % 16] = byte
    segm = nan_segm(cu[-1], hq, 16, d) if split else None
    out, lse = torch.full_like(q, 7.0), torch.zeros(cu[-1], hq, device=DEV)
    fc.fp4_paged_attention(q, c.kc, c.vc, out, i32(cu), i32(lens), c.table, max(q_lens), d ** -0.5, c.scales,
                           ck.plan_long(cu, lens, 16), segm, lse)
    seen = torch.ones(cu[-1], dtype=torch.bool)
    seen[torch.tensor(cu[1:]) - 1] = False
    R.check(out[seen], want[seen], bound[seen], q_lens)
    if max(q_lens) <= ck.SHORT_Q:
        R.check_lse(lse[seen], of[seen], of_bound[seen])


@pytest.mark.parametrize("short_q", [1, 1_000_000])
def test_other_short_query_limits(short_q, monkeypatch):
    """KVQ_SHORT_Q's other uses: verification rows through the long path, whole prompts through the short one."""
    monkeypatch.setattr(ck, "SHORT_Q", short_q)
    lens = [90, 500, 33, 700]
    c = filled(4, 128, 16, lens)
    attend(c, 28, [1, 8, 3, 1], lens)
    attend(c, 28, [1, 300, 33, 20], lens)
    attend(c, 28, [1, 300, 33, 20], lens, nan_segm(354, 28, 16, 128))


def test_many_requests_and_bad_pages():
    """More requests than a wavefront's lanes hold; a table entry that is not there reads page 0."""
    r = np.random.RandomState(0)
    lens = [int(x) for x in r.randint(0, 300, 333)]
    c = filled(2, 64, 16, lens)
    q_lens = [int(x) for x in r.randint(0, 4, 333)]
    attend(c, 14, q_lens, lens, nan_segm(sum(q_lens) + 2, 14, 8, 64))
    fc.quant_fp4_cache(*[x.to(DEV) for x in rows(16, 2, 64, 3)], c.kc, c.vc, c.scales, torch.arange(16, device=DEV))
    c.table[:, 0] = 0
    want = attend(c, 14, q_lens, lens)[1]
    table = c.table
    c.table = torch.where(table == 0, torch.tensor(1 << 30, dtype=torch.int32, device=DEV), table)
    cu = cumsum(q_lens)
    q = torch.randn(cu[-1] + 2, 14, 64, generator=gen(3)).to(torch.bfloat16).to(DEV)
    out = torch.full_like(q, 7.0)
    fc.fp4_paged_attention(q, c.kc, c.vc, out, i32(cu), i32(lens), c.table, 3, 64 ** -0.5, c.scales)
    assert torch.equal(out, want)


@pytest.mark.parametrize("most", [1, 2, 100])
@pytest.mark.parametrize("split", [False, True])
def test_longest_query_is_a_hint(most, split):
    """max_query_len picks the launch; rows of longer requests are served all the same."""
    lens, q_lens = [700, 33, 5000, 8], [8, 1, 5, 8]
    c = filled(4, 128, 16, lens)
    cu = cumsum(q_lens)
    q = torch.randn(cu[-1], 28, 128, generator=gen(9)).to(torch.bfloat16).to(DEV)
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device=DEV)
    fc.fp4_decode_attention(q, c.kc, c.vc, out, i32(cu), i32(lens), c.table, 0.09, c.scales,
                            nan_segm(cu[-1], 28, 16, 128) if split else None, most, lse)
    want, bound, of, of_bound = R.attention(q, c.kc, c.vc, c.scales, cu, lens, c.table, 0.09)
    R.check(out, want, bound, most)
    R.check_lse(lse, of, of_bound, most)


@pytest.mark.parametrize("splits", ["1", "3", "5", "8"])
@pytest.mark.parametrize("hq,h,d", [(28, 4, 128), (14, 2, 64), (32, 1, 128)])
@pytest.mark.parametrize("qlen", [1, 4, 8])
def test_other_numbers_of_key_splits(splits, hq, h, d, qlen, monkeypatch):
    monkeypatch.setenv("KVQ_KSPLIT", splits)
    lens = [0, 9, 100, 33, 700, 2049]
    c = filled(h, d, 16, lens)
    q_lens = [qlen] * len(lens)
    attend(c, hq, q_lens, lens)
    attend(c, hq, q_lens, lens, nan_segm(sum(q_lens), hq, 8, d))


@pytest.mark.parametrize("hq,h,d", [(28, 4, 128), (14, 2, 64)])
@pytest.mark.parametrize("qlen", [3, 8])
def test_many_pairs_of_many_rows(hq, h, d, qlen):
    """More pairs of a request and a kv head than take a wavefront a row tile, cut and whole; some of fewer tokens."""
    r = np.random.RandomState(1)
    lens = [int(x) for x in r.randint(8, 600, 40)]
    q_lens = [int(x) for x in r.randint(0, qlen + 1, 40)]
    q_lens[0] = qlen
    c = filled(h, d, 32, lens)
    attend(c, hq, q_lens, lens)
    attend(c, hq, q_lens, lens, nan_segm(sum(q_lens) + 2, hq, 8, d))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("order", ["heads first", "V first", "padded rows", "slots first"])
def test_other_orders_of_a_cache(d, order):
    """Caches of other strides through every operator that reads them, against the same calls on the usual layout."""
    lens, q_lens, h, bs, hq = [300, 20, 0, 1000], [1, 8, 1, 3], 4, 32, 12
    ref = filled(h, d, bs, lens)
    nb = ref.kc.shape[0]
    full = lambda *shape: torch.full(shape, 0xff, dtype=torch.uint8, device=DEV)  # noqa: E731
    c = Cache(h, d, bs, nb)
    if order == "heads first":
        c.kc, c.vc = (full(nb, h, bs, d // 2).transpose(1, 2) for _ in range(2))
    elif order == "V first":
        kv = full(nb, bs, h, d)
        c.kc, c.vc = kv[..., d // 2:], kv[..., :d // 2]
    elif order == "padded rows":
        c.kc, c.vc = (full(nb + 1, bs + 3, h + 1, d // 2 + 16)[:nb, :bs, 1:, :d // 2] for _ in range(2))
    else:
        c.kc, c.vc = (full(bs, nb, h, d // 2).transpose(0, 1) for _ in range(2))
    fc.quant_fp4_cache(ref.k.to(DEV), ref.v.to(DEV), c.kc, c.vc, c.scales, slots_of(ref.host, lens, bs).to(DEV))
    for x, y in zip(c.parts(), ref.parts()):
        assert torch.equal(x, y)
    c.host, c.table = ref.host, ref.table
    segm = [nan_segm(sum(q_lens), hq, 8, d) for _ in range(2)]
    a, b = attend(c, hq, q_lens, lens, segm[0]), attend(ref, hq, q_lens, lens, segm[1])
    assert torch.equal(a[1], b[1]) and torch.equal(a[2], b[2])
    attend(c, hq, [1, 20, 1, 40], lens)
    w = [torch.zeros(len(lens), h, 1000, device=DEV) for _ in range(2)]
    kept = [torch.zeros(len(lens), h, 64, dtype=torch.int32, device=DEV) for _ in range(2)]
    for i, (x, of) in enumerate(((c, a), (ref, b))):
        fc.add_key_weights(of[0], x.kc, x.scales, of[2], w[i], i32(cumsum(q_lens)), i32(lens), x.table, d ** -0.5, 8)
        fc.evict_keys(x.kc, x.vc, x.scales, w[i], i32(lens), i32([64] * 4), 8, x.table, kept[i], i32([0] * 4))
    assert torch.equal(w[0], w[1]) and torch.equal(kept[0], kept[1])
    for x, y in zip(c.parts(), ref.parts()):
        assert torch.equal(x, y)


def test_two_graphs_share_buffers():
    """Graphs of two batches over one cache, with the same split buffers, replayed in turn with eager work between."""
    lens = [3000, 17, 0, 900]
    c = filled(4, 128, 16, lens)
    segm = nan_segm(32, 28, 16, 128)
    batches = []
    for q_lens, short in (([1, 1, 1, 1], lens), ([8, 3, 1, 8], [2000, 10, 0, 901 - 1])):
        cu = cumsum(q_lens)
        q = torch.randn(cu[-1], 28, 128, generator=gen(cu[-1])).to(torch.bfloat16).to(DEV)
        x = dict(q=q, out=torch.zeros_like(q), lse=torch.zeros(q.shape[:2], device=DEV), cu=i32(cu), lens=i32(short),
                 most=max(q_lens), w=torch.zeros(4, 4, 3000, device=DEV))
        batches.append(x)

    def run(x):
        fc.fp4_paged_attention(x["q"], c.kc, c.vc, x["out"], x["cu"], x["lens"], c.table, x["most"], 0.09, c.scales, None, segm,
                               x["lse"])
        x["w"].zero_()
        fc.add_key_weights(x["q"], c.kc, c.scales, x["lse"], x["w"], x["cu"], x["lens"], c.table, 0.09, x["most"])

    want, graphs = [], []
    for x in batches:
        run(x)
        torch.cuda.synchronize()
        want.append([x[n].clone() for n in ("out", "lse", "w")])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            run(x)
        graphs.append(g)
    for i in (0, 1, 1, 0, 1, 0):
        for n in ("out", "lse", "w"):
            batches[i][n].fill_(7.0)
        graphs[i].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(batches[i][n], y) for n, y in zip(("out", "lse", "w"), want[i])), i
        run(batches[1 - i])
        assert all(torch.equal(batches[1 - i][n], y) for n, y in zip(("out", "lse", "w"), want[1 - i])), i


# ------------------------------------------------------------------------------------------------ weights
def weigh(c, hq, q_lens, lens, cols, seed=5, lse=None, most=None, pad=1):
    h, d, bs = c.geom
    cu = cumsum(q_lens)
    q = torch.randn(cu[-1] + pad, hq, d, generator=gen(seed)).to(torch.bfloat16).to(DEV)
    if lse is None:
        lse = R.attention(q, c.kc, c.vc, c.scales, cu, lens, c.table, d ** -0.5)[2].float()
    start = torch.rand(len(lens) + 1, h, cols, generator=gen(seed + 1)).to(DEV)
    got = start.clone()
    args = (q, c.kc, c.scales, lse, got, i32(cu), i32(lens), c.table, d ** -0.5, max(q_lens) if most is None else most)
    assert fc.add_key_weights(*args) is got
    add, bound = R.key_weights(q, c.kc, c.scales, lse, start.shape, cu, lens, c.table, d ** -0.5, ck.SHORT_Q)
    want = start.double() + add
    R.check(got, want, bound + want * 2.0 ** -20, (q_lens, lens))     # (up to 16 additions of row tiles' sums)
    assert torch.equal(got[add == 0], start[add == 0])
    again = start.clone()
    fc.add_key_weights(*args[:4], again, *args[5:])
    assert torch.equal(got, again)
    return q, lse, got


@pytest.mark.parametrize("hq,h,d", HEADS)
@pytest.mark.parametrize("qlen", [1, 3, 8])
def test_key_weights(hq, h, d, qlen):
    lens = [0, 1, qlen, 15, 16, 17, 31, 32, 33, 64, 100, 257, 1000]
    c = filled(h, d, 16 if h != 2 else 64, lens, seed=qlen, layout="vllm" if qlen % 2 else "apart")
    weigh(c, hq, [qlen] * len(lens), lens, 1024)


def test_key_weights_of_other_batches():
    lens = [3000, 0, 700, 5, 40]
    c = filled(4, 128, 32, lens)
    weigh(c, 28, [1, 1, 8, 3, 0], lens, 3008, most=1)           # more rows than the caller says
    weigh(c, 28, [1, 0, 20, 3, 9], lens, 3008, most=20)         # long requests are skipped
    weigh(c, 28, [8, 8, 8, 2, 1], lens, 600)                    # keys behind the last column are not counted
    q_lens = [2, 1, 8, 3, 1]
    lse = torch.randn(17, 28, generator=gen(1)).to(DEV) + 8     # rows without a number add nothing
    lse[0, 3], lse[5, 27], lse[4, 0] = float("nan"), float("inf"), -float("inf")
    weigh(c, 28, q_lens, lens, 3008, lse=lse, pad=2)


def test_key_weights_sum_to_the_rows():
    """With the attention's own log-sum-exp, a request's sums add up to its rows' count (each row's weights to 1)."""
    lens = [2000, 90, 31]
    c = filled(4, 128, 16, lens)
    q, _, lse = attend(c, 28, [1, 8, 3], lens, nan_segm(12, 28, 16, 128), pad=0)
    w = torch.zeros(3, 4, 2000, device=DEV)
    fc.add_key_weights(q, c.kc, c.scales, lse, w, i32([0, 1, 9, 12]), i32(lens), c.table, 128 ** -0.5, 8)
    # (two uses of scores off by 2^-16 of 128 products of about 1.5, and sums of 2,000)
    assert bool(((w.double().sum(-1) / torch.tensor([[7.0], [56.0], [21.0]], device=DEV) - 1).abs() < 1e-3).all())


def test_key_weights_under_another_short_limit(monkeypatch):
    monkeypatch.setattr(ck, "SHORT_Q", 40)
    lens = [300, 90]
    c = filled(4, 128, 16, lens)
    weigh(c, 28, [40, 3], lens, 320)


# ------------------------------------------------------------------------------------------------ eviction
def evict(c, lens, keep, recent, w, most=None, table=None):
    h, d, bs = c.geom
    most = max(keep + [0]) if most is None else most
    before = [t.clone() for t in c.parts()]
    start = w.clone()
    kept = torch.full((len(lens), h, most), -7, dtype=torch.int32, device=DEV)
    new = torch.full((len(lens),), -7, dtype=torch.int32, device=DEV)
    got = fc.evict_keys(c.kc, c.vc, c.scales, w, i32(lens), i32(keep), recent, c.table if table is None else table, kept, new)
    assert got is new
    cols = w.shape[2]
    host, after, hw, hk = start.cpu(), w.cpu(), c.host.long(), kept.cpu()
    old, cur = [t.cpu() for t in before], [t.cpu() for t in c.parts()]
    want_w = host.clone()
    for r, n in enumerate(lens):
        budget = max(min(keep[r], most), 0)
        m = min(n, budget)
        assert int(new[r]) == m
        for g in range(h):
            at = R.evict(host[r, g].tolist(), n, budget, recent, cols)
            assert hk[r, g, :m].tolist() == at, (r, g)
            assert bool((hk[r, g, m:] == -7).all())
            src = torch.tensor(at, dtype=torch.long)
            dst = torch.arange(m)
            for i, x in enumerate(old):
                if i < 2:
                    x[hw[r][dst // bs], dst % bs, g] = x[hw[r][src // bs], src % bs, g].clone()
                else:
                    x[hw[r][dst // bs], g, dst % bs] = x[hw[r][src // bs], g, src % bs].clone()
            if n > budget:
                vals = torch.tensor([float(host[r, g, i]) if i < cols else 0.0 for i in at])
                want_w[r, g, :min(m, cols)] = vals[:cols]
                want_w[r, g, m:n] = 0
    for x, y in zip(old, cur):
        assert torch.equal(x, y)
    assert torch.equal(torch.nan_to_num(after, nan=-3.0), torch.nan_to_num(want_w, nan=-3.0))


@pytest.mark.parametrize("h,d,bs", GEOM)
@pytest.mark.parametrize("recent", [0, 1, 40, 1000])
def test_evict(h, d, bs, recent):
    lens = [0, 1, 16, 100, 300, 1000, 2500, 333]
    keep = [5, 5, 16, 17, 40, 64, 1500, 0]
    c = filled(h, d, bs, lens, layout="vllm" if h % 2 else "apart")
    w = torch.rand(len(lens), h, 2560, generator=gen(recent)).to(DEV)
    evict(c, lens, keep, recent, w)


def test_evict_ties_zeros_and_numbers_that_are_none():
    lens = [3000, 2000, 500, 500, 700]
    c = filled(4, 128, 16, lens)
    g = gen(3)
    w = torch.randint(0, 4, (5, 4, 3008), generator=g).float()
    w[1] = 0.0
    w[1, :, ::3] = -0.0
    w[2, :, 7::11] = float("nan")
    w[2, :, 8::13] = -float("nan")
    w[3, :, 3::5], w[3, :, 4::5] = float("inf"), -float("inf")
    w[4] = torch.randn(4, 3008, generator=g) * 1e-40            # negative ones and subnormals
    evict(c, lens, [700, 700, 100, 450, 300], 16, w.to(DEV))


def test_evict_long_contexts_and_odd_budgets():
    lens = [70001, 5, 40000]
    c = filled(2, 64, 64, lens)
    w = torch.exp(2 * torch.randn(3, 2, 70016, generator=gen(1))).to(DEV)
    evict(c, lens, [69999, 4, 1], 0, w)
    c = filled(2, 128, 64, lens)
    w = torch.exp(2 * torch.randn(3, 2, 70016, generator=gen(2))).to(DEV)
    evict(c, lens, [20001, 5, 39999], 7000, w)


def test_evict_bounds_of_its_arguments():
    """Budgets above kept's size and below 0, lengths past the table's width, sums for fewer keys, pages that are not there."""
    lens = [200, 300, 100, 50]
    c = filled(2, 128, 16, lens)
    w = torch.rand(4, 2, 150, generator=gen(1)).to(DEV)
    evict(c, lens, [120, 1 << 30, -5, 50], 20, w, most=100)
    lens = [96]
    c = filled(2, 128, 16, lens)
    kept, new = torch.zeros(1, 2, 40, dtype=torch.int32, device=DEV), i32([0])
    w = torch.rand(1, 2, 96, generator=gen(1)).to(DEV)
    w0 = w.clone()
    fc.evict_keys(c.kc, c.vc, c.scales, w, i32([1 << 30]), i32([40]), 8, c.table[:, :6].contiguous(), kept, new)
    assert kept.cpu()[0, 1].tolist() == R.evict(w0[0, 1].tolist(), 96, 40, 8, 96) and int(new) == 40
    before = [t.clone() for t in c.parts()]
    fc.evict_keys(c.kc, c.vc, c.scales, w, i32([90]), i32([20]), 8, torch.full((1, 6), -1, dtype=torch.int32, device=DEV), kept, new)
    assert all(torch.equal(a, b) for a, b in zip(before, c.parts())) and int(new) == 20


@pytest.mark.parametrize("where", ["seq_lens", "keep", "both", "beside"])
def test_evict_updates_lengths_in_place(where):
    """new_lens as seq_lens or keep themselves, or right behind them: every head's choice, rows and sums as with lengths of
    their own. More workgroups (60 requests of 16 heads) than run at once, so that some start after others have ended."""
    h, d, bs = 16, 64, 16
    lens = [200 + 3 * r if r % 5 else 40 for r in range(60)]
    keep = lens if where == "both" else [64 + r for r in range(60)]
    a, b = (filled(h, d, bs, lens) for _ in range(2))
    w = [torch.rand(60, h, 400, generator=gen(5)).to(DEV) for _ in range(2)]
    kept = [torch.full((60, h, 100), -7, dtype=torch.int32, device=DEV) for _ in range(2)]
    own = i32([-7] * 60)
    fc.evict_keys(a.kc, a.vc, a.scales, w[0], i32(lens), i32(keep), 16, a.table, kept[0], own)
    both = i32(lens + [-7] * 60)
    at, budget = both[:60], i32(keep)
    if where == "both":
        budget = at
    new = {"seq_lens": at, "keep": budget, "both": at, "beside": both[60:]}[where]
    for _ in range(2):   # (again: nothing is left to do, the lengths stay)
        got = fc.evict_keys(b.kc, b.vc, b.scales, w[1], at, budget, 16, b.table, kept[1], new)
        assert got is new and torch.equal(new, own)
        if where != "seq_lens":
            break
    assert new.cpu().tolist() == [min(n, k, 100) for n, k in zip(lens, keep)]
    assert torch.equal(*w)
    assert all(torch.equal(x, y) for x, y in zip(a.parts(), b.parts()))
    if where != "seq_lens":
        assert torch.equal(*kept)


def test_sums_in_other_orders():
    """weights and kept as views of heads-first buffers, requests side by side; expanded over heads they are refused."""
    lens, h = [300, 40, 700], 4
    a, b = (filled(h, 128, 16, lens) for _ in range(2))
    w = torch.rand(3, h, 704, generator=gen(1)).to(DEV)
    v = w.transpose(0, 1).contiguous().transpose(0, 1)
    q = torch.randn(3, 28, 128, generator=gen(2)).to(torch.bfloat16).to(DEV)
    lse = torch.full((3, 28), 5.0, device=DEV)
    kept = torch.full((3, h, 100), -7, dtype=torch.int32, device=DEV)
    kept2 = torch.full((h, 3, 100), -7, dtype=torch.int32, device=DEV).transpose(0, 1)
    new = [i32([0] * 3) for _ in range(2)]
    for c, x, k, n in ((a, w, kept, new[0]), (b, v, kept2, new[1])):
        fc.add_key_weights(q, c.kc, c.scales, lse, x, i32([0, 1, 2, 3]), i32(lens), c.table, 0.1)
        fc.evict_keys(c.kc, c.vc, c.scales, x, i32(lens), i32([100] * 3), 10, c.table, k, n)
    assert torch.equal(w, v) and torch.equal(kept, kept2) and torch.equal(*new)
    assert all(torch.equal(x, y) for x, y in zip(a.parts(), b.parts()))
    shared = torch.rand(3, 1, 704, device=DEV).expand(3, h, 704)
    with pytest.raises(RuntimeError, match="rows of weights overlap"):
        fc.evict_keys(a.kc, a.vc, a.scales, shared, i32(lens), i32([50] * 3), 10, a.table, kept, new[0])
    with pytest.raises(RuntimeError, match="rows of weights overlap"):
        fc.add_key_weights(q, a.kc, a.scales, lse, shared, i32([0, 1, 2, 3]), i32(lens), a.table, 0.1)
    with pytest.raises(RuntimeError, match="rows of kept overlap"):
        fc.evict_keys(a.kc, a.vc, a.scales, w, i32(lens), i32([50] * 3), 10, a.table, kept[:, :1].expand(3, h, 100), new[0])


# ------------------------------------------------------------------------------------------------ together
@pytest.mark.parametrize("hq,h,d,bs", [(28, 4, 128, 16), (14, 2, 64, 64)])
def test_generation_captured_and_replayed(hq, h, d, bs):
    """Prompts eagerly, then steps in one captured graph -- norm and rotation, write, attention, weights, eviction --
    with every replay equal to the same calls made eagerly on a twin cache, and the last steps' outputs to the plain ones."""
    prompts, budget, steps = [37, 5, 128, 300], 64, 24
    n = len(prompts)
    table, nb = page_table([max(p, budget) + 2 for p in prompts], bs, 3)
    dtab, cols = table.to(DEV), 320
    angle = torch.arange(400)[:, None] * 1000.0 ** (-torch.arange(0, d, 2) / d)
    cos_sin = torch.cat([angle.cos(), angle.sin()], -1).to(DEV)
    weight = [(1 + 0.1 * torch.randn(d, generator=gen(s))).to(DEV) for s in (1, 2)]
    cu = i32(range(n + 1))

    class Side:
        def __init__(self):
            self.c = Cache(h, d, bs, nb)
            self.lens, self.next = i32(prompts), i32(prompts)
            self.pos = torch.tensor(prompts, device=DEV)
            self.qkv = torch.zeros(n, (hq + 2 * h) * d, dtype=torch.bfloat16, device=DEV)
            self.w, self.lse = torch.zeros(n, h, cols, device=DEV), torch.zeros(n, hq, device=DEV)
            self.out = torch.zeros(n, hq, d, dtype=torch.bfloat16, device=DEV)
            self.segm = ck.split_buffers(n, hq, d, 16, DEV)
            self.keep, self.kept = i32([budget] * n), torch.zeros(n, h, budget, dtype=torch.int32, device=DEV)
            k, v = rows(sum(prompts), h, d, 4)
            fc.quant_fp4_cache(k.to(DEV), v.to(DEV), self.c.kc, self.c.vc, self.c.scales, slots_of(table, prompts, bs).to(DEV))

        def load(self, i):
            self.qkv.copy_(torch.randn(n, (hq + 2 * h) * d, generator=gen(100 + i)))

        def run(self):
            q = self.qkv[:, :hq * d].view(n, hq, d)
            k, v = (x.view(n, h, d) for x in self.qkv[:, hq * d:].chunk(2, -1))
            self.q, self.k = q, k
            rope.norm_rope(q, k, self.pos, cos_sin, *weight)
            slots = (dtab.gather(1, (self.lens // bs).long()[:, None])[:, 0] * bs + self.lens % bs).long()
            self.lens.add_(1)
            fc.quant_fp4_cache(k, v, self.c.kc, self.c.vc, self.c.scales, slots)
            fc.fp4_paged_attention(q, self.c.kc, self.c.vc, self.out, cu, self.lens, dtab, 1, d ** -0.5, self.c.scales, None,
                                   self.segm, self.lse)
            fc.add_key_weights(q, self.c.kc, self.c.scales, self.lse, self.w, cu, self.lens, dtab, d ** -0.5)
            self.seen = self.lens.clone()
            fc.evict_keys(self.c.kc, self.c.vc, self.c.scales, self.w, self.lens, self.keep, 8, dtab, self.kept, self.next)
            self.lens.copy_(self.next)
            self.pos.add_(1)

    a, b, warm = Side(), Side(), Side()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm.run()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.run()
    for i in range(steps):
        for s in (a, b):
            s.load(i)
        graph.replay()
        plain = Cache(h, d, bs, nb)
        b.run()
        torch.cuda.synchronize()
        for x, y in zip(a.c.parts() + (a.out, a.lse, a.w, a.kept, a.lens), b.c.parts() + (b.out, b.lse, b.w, b.kept, b.lens)):
            assert torch.equal(x, y), i
        del plain
    assert b.lens.cpu().tolist() == [min(p + steps, budget) for p in prompts]
    # attention over what is left, by position: rows of the eviction's choice
    lens = b.lens.cpu().tolist()
    b.c.table = dtab
    attend(b.c, hq, [1] * n, lens)


@pytest.mark.parametrize("hq,h,d,bs", [(28, 4, 128, 16), (14, 2, 64, 64)])
def test_steps_of_a_generation_against_plain_forms(hq, h, d, bs):
    """Norm and rotation, write, attention, key weights and eviction (lengths in place) in one captured graph: what each replay
    leaves against the plain forms of what it found."""
    prompts, budget, recent, cols = [37, 5, 128, 300], 64, 8, 320
    n = len(prompts)
    table, nb = page_table([max(p, budget) + 2 for p in prompts], bs, 3)
    dtab, cu = table.to(DEV), i32(range(n + 1))
    angle = torch.arange(400)[:, None] * 1000.0 ** (-torch.arange(0, d, 2) / d)
    cos_sin = torch.cat([angle.cos(), angle.sin()], -1).to(DEV)
    weight = [(1 + 0.1 * torch.randn(d, generator=gen(s))).to(DEV) for s in (1, 2)]
    c = Cache(h, d, bs, nb)
    k, v = rows(sum(prompts), h, d, 4)
    fc.quant_fp4_cache(k.to(DEV), v.to(DEV), c.kc, c.vc, c.scales, slots_of(table, prompts, bs).to(DEV))
    lens, pos = i32(prompts), torch.tensor(prompts, device=DEV)
    qkv = torch.zeros(n, (hq + 2 * h) * d, dtype=torch.bfloat16, device=DEV)
    q = qkv[:, :hq * d].view(n, hq, d)
    k, v = (x.view(n, h, d) for x in qkv[:, hq * d:].chunk(2, -1))
    w, lse, out = torch.zeros(n, h, cols, device=DEV), torch.zeros(n, hq, device=DEV), torch.zeros_like(q)
    segm = ck.split_buffers(n, hq, d, 16, DEV)
    keep, kept = i32([budget] * n), torch.zeros(n, h, budget, dtype=torch.int32, device=DEV)

    def step():
        rope.norm_rope(q, k, pos, cos_sin, *weight)
        slots = (dtab.gather(1, (lens // bs).long()[:, None])[:, 0] * bs + lens % bs).long()
        lens.add_(1)
        fc.quant_fp4_cache(k, v, c.kc, c.vc, c.scales, slots)
        fc.fp4_paged_attention(q, c.kc, c.vc, out, cu, lens, dtab, 1, d ** -0.5, c.scales, None, segm, lse)
        fc.add_key_weights(q, c.kc, c.scales, lse, w, cu, lens, dtab, d ** -0.5)
        fc.evict_keys(c.kc, c.vc, c.scales, w, lens, keep, recent, dtab, kept, lens)
        pos.add_(1)

    state = (*c.parts(), lens, pos, w)
    start = [t.clone() for t in state]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for t, x in zip(state, start):
        t.copy_(x)
    for i in range(6):
        qkv.copy_(torch.randn(qkv.shape, generator=gen(100 + i)))
        q0, k0 = q.clone(), k.clone()
        kc, vc, ks, vs, lens0, pos0, w0 = [t.clone() for t in state]
        graph.replay()
        torch.cuda.synchronize()
        for x, got, g in ((q0, q, weight[0]), (k0, k, weight[1])):
            R.check(got, *R.norm_rope(x, pos0, cos_sin, g, 1e-6, False), i)
        assert torch.equal(pos, pos0 + 1)
        slots = torch.tensor([int(table[r, m // bs]) * bs + m % bs for r, m in enumerate(lens0.tolist())])
        scales = {"k_scale": ks, "v_scale": vs}
        for x, cache, scale in ((k, kc, ks), (v, vc, vs)):
            R.write(x.cpu(), cache, scale, slots)
        now = [m + 1 for m in lens0.tolist()]
        want, bound, of, of_bound = R.attention(q, kc, vc, scales, cu.tolist(), now, dtab, d ** -0.5)
        R.check(out, want, bound, i)
        R.check_lse(lse, of, of_bound, i)
        add, off = R.key_weights(q, kc, scales, lse, w.shape, cu.tolist(), now, dtab, d ** -0.5)
        sums = (w0.double() + add).cpu()
        off = (off + sums.to(DEV) * 2.0 ** -23).cpu()
        old, new = [t.cpu() for t in (kc, vc, ks, vs)], [t.cpu() for t in c.parts()]
        at, got = kept.cpu().long(), w.cpu().double()
        assert lens.tolist() == [min(m, budget) for m in now]
        for r, m in enumerate(now):
            left = min(m, budget)
            for g in range(h):
                mine = at[r, g, :left]
                if m <= budget:
                    assert mine.tolist() == list(range(m))
                else:
                    # in order, the latest, and none of the rest that is surely below one that was left
                    assert bool((mine[1:] > mine[:-1]).all()) and mine[-recent:].tolist() == list(range(m - recent, m))
                    gone = torch.ones(m, dtype=torch.bool)
                    gone[mine] = False
                    least = (sums[r, g, mine] + off[r, g, mine])[:left - recent].min()
                    assert bool(((sums[r, g, :m] - off[r, g, :m])[gone] <= least).all()), (i, r, g)
                    assert bool((got[r, g, left:] == 0).all())
                assert bool(((got[r, g, :left] - sums[r, g, mine]).abs() <= off[r, g, mine]).all()), (i, r, g)
                dst, src = torch.arange(left), mine
                ids = table[r].long()
                for side_old, side_new in zip(old[:2], new[:2]):
                    assert torch.equal(side_new[ids[dst // bs], dst % bs, g], side_old[ids[src // bs], src % bs, g])
                for side_old, side_new in zip(old[2:], new[2:]):
                    assert torch.equal(side_new[ids[dst // bs], g, dst % bs], side_old[ids[src // bs], g, src % bs])


def test_caches_past_two_and_four_gib():
    """A cache of more than 4 GiB a side: the pages used lie at its ends and around 2 and 4 GiB."""
    h, d, bs = 8, 128, 64
    nb = (4 << 30) // (h * d // 2 * bs) + 40
    kc, vc = (torch.empty(nb, bs, h, d // 2, dtype=torch.uint8, device=DEV) for _ in range(2))
    scales = fc.fp4_scales(nb, bs, h, d, DEV)
    ids = [nb - 1, 0, nb // 2, nb // 2 - 1, nb - 40, nb - 41, 1, nb - 2]
    lens = [64 * 4 - 3, 64 * 4]
    table = torch.tensor(ids, dtype=torch.int32).view(2, 4)
    k, v = rows(sum(lens), h, d, 1)
    fc.quant_fp4_cache(k.to(DEV), v.to(DEV), kc, vc, scales, slots_of(table, lens, bs).to(DEV))
    at = torch.tensor(ids, device=DEV).long()
    c = Cache(h, d, bs, 8, "apart")
    c.kc, c.vc, c.scales = kc[at].contiguous(), vc[at].contiguous(), {x: s[at] for x, s in scales.items()}
    c.table = c.host = torch.arange(8, dtype=torch.int32).view(2, 4)
    c.table = c.table.to(DEV)
    want = R.quantize(k)[0]
    assert torch.equal(torch.cat([c.kc[:4].flatten(0, 1)[:lens[0]], c.kc[4:].flatten(0, 1)]).cpu(), want)
    out = [torch.zeros(sum(lens), h, d, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    fc.read_fp4_cache(kc, vc, scales, i32([0, 0]), i32(cumsum(lens)), table.to(DEV), *out)
    assert torch.equal(out[1][lens[0]:].double(), R.values(c.vc, c.scales["v_scale"], c.table[1], lens[1]).transpose(0, 1))
    for q_lens in ([1, 8], [30, 100]):
        q, o, lse = attend(c, 32, q_lens, lens, pad=0)
        big, big_lse, cu = torch.zeros_like(o), torch.full_like(lse, 7.0), cumsum(q_lens)
        fc.fp4_paged_attention(q, kc, vc, big, i32(cu), i32(lens), table.to(DEV), max(q_lens), d ** -0.5, scales,
                               ck.plan_long(cu, lens, bs), None, big_lse)
        assert torch.equal(big, o) and torch.equal(big_lse, lse)
    w = [torch.zeros(2, h, 256, device=DEV) for _ in range(2)]
    q, o, lse = attend(c, 32, [1, 8], lens, pad=0)
    fc.add_key_weights(q, kc, scales, lse, w[0], i32([0, 1, 9]), i32(lens), table.to(DEV), d ** -0.5, 8)
    fc.add_key_weights(q, c.kc, c.scales, lse, w[1], i32([0, 1, 9]), i32(lens), c.table, d ** -0.5, 8)
    assert torch.equal(*w)
    kept, new = torch.zeros(2, h, 90, dtype=torch.int32, device=DEV), i32([0, 0])
    fc.evict_keys(kc, vc, scales, w[0], i32(lens), i32([90, 90]), 16, table.to(DEV), kept, new)
    evict(c, lens, [90, 90], 16, w[1])
    assert torch.equal(kc[at], c.kc) and torch.equal(vc[at], c.vc) and torch.equal(*w)


def test_another_stream():
    """Calls go to the stream that is current, behind what it holds already."""
    lens = [300, 41]
    table, nb = page_table(lens, 16, 1)
    c = Cache(4, 128, 16, nb, "vllm", 0, 0)
    before = [t.clone() for t in c.parts()]
    k, v = rows(sum(lens), 4, 128, 2)
    kd, vd = torch.zeros_like(k, device=DEV), torch.zeros_like(v, device=DEV)
    ks, vs = k.pin_memory(), v.pin_memory()
    slots = slots_of(table, lens, 16)
    dslots = slots.to(DEV)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        torch.cuda._sleep(20_000_000)
        kd.copy_(ks, non_blocking=True)
        vd.copy_(vs, non_blocking=True)
        fc.quant_fp4_cache(kd, vd, c.kc, c.vc, c.scales, dslots)
    s.synchronize()
    _same_write(c, k, v, slots, before)


# ------------------------------------------------------------------------------------------------ native calls
def _call_all(c, x):
    """Every operator once on the GPU state `x`; the outputs, or what was raised."""
    got = []
    for f in (lambda: fc.quant_fp4_cache(x["k"], x["v"], c.kc, c.vc, x["scales"], x["slots"]),
              lambda: fc.read_fp4_cache(c.kc, c.vc, x["scales"], x["lens"] // 2, x["cu"], c.table, x["ko"], x["vo"]),
              lambda: fc.fp4_paged_attention(x["q"], c.kc, c.vc, x["out"], x["cu"], x["lens"], c.table, x["most"], x["scale"],
                                             x["scales"], x["plan"], x["segm"], x["lse"]),
              lambda: fc.add_key_weights(x["q"], c.kc, x["scales"], x["lse"], x["w"], x["cu"], x["lens"], c.table, x["scale"], 8),
              lambda: fc.evict_keys(c.kc, c.vc, x["scales"], x["w"], x["lens"], x["keep"], x["recent"], c.table, x["kept"], x["new"]),
              lambda: rope.norm_rope(x["q"], x["k"], x["pos"], x["table"], *x["norm"])):
        try:
            f()
            got.append("served")
        except Exception as e:  # noqa: BLE001 - compared with the other path's
            got.append((type(e), str(e)))
    return got, [t.clone() for t in (*c.parts(), x["ko"], x["vo"], x["out"], x["lse"], x["w"], x["kept"], x["new"], x["q"], x["k"])]


CHANGES = {
    "plain": lambda x: None,
    "split": lambda x: x.update(segm=nan_segm(x["q"].shape[0], 28, 16, 128)),
    "strided_split": lambda x: x.update(segm=tuple(t[:, :28] for t in nan_segm(x["q"].shape[0], 30, 8, 128))),
    "packed_q": lambda x: x.update(q=torch.cat([x["q"], x["q"]], 1)[:, :28]),
    "wide_lse": lambda x: x.update(lse=torch.zeros(x["q"].shape[0] + 3, 31, device=DEV)[:, :28]),
    "parameter_scales": lambda x: x.update(scales={n: torch.nn.Parameter(t, requires_grad=False) for n, t in x["scales"].items()}),
    "scale_int": lambda x: x.update(scale=1),
    "half": lambda x: x.update(q=x["q"].half(), k=x["k"].half(), ko=x["ko"].half(), w=x["w"].half(), kept=x["kept"].long()),
    "few": lambda x: x.update(out=x["out"][:3], vo=x["vo"][:-1], w=x["w"][:2], lse=x["lse"][:2], new=x["new"][:2], pos=x["pos"][:-1]),
    "long_lengths": lambda x: x.update(lens=x["lens"].long(), pos=x["pos"].int(), slots=x["slots"].int()),
    "odd_rows": lambda x: x.update(q=torch.zeros(x["q"].shape[0], 28, 132, dtype=torch.bfloat16, device=DEV)[..., :128],
                                   k=torch.zeros(*x["k"].shape[:2], 132, dtype=torch.bfloat16, device=DEV)[..., :128]),
    "no_norm": lambda x: x.update(norm=(None, None)),
    "recent": lambda x: x.update(recent=-1, norm=(x["norm"][0], None)),
    "cpu": lambda x: x.update(q=x["q"].cpu(), k=x["k"].cpu(), ko=x["ko"].cpu(), w=x["w"].cpu()),
}


@pytest.mark.parametrize("change", CHANGES)
def test_native_calls_and_the_python_path_agree(change, monkeypatch):
    assert ck.ext().calls is not None, "kvq._torch_calls is not built"
    lens, q_lens = [300, 20, 64, 2000], [1, 20, 8, 300]
    got = []
    for native in (True, False):
        c = filled(4, 128, 32, lens)
        n = sum(q_lens)
        k, v = rows(n, 4, 128, 50)
        first = [a - b for a, b in zip(lens, q_lens)]
        x = {"k": k.to(DEV), "v": v.to(DEV), "scales": c.scales, "cu": i32(cumsum(q_lens)), "lens": i32(lens),
             "slots": slots_of(c.host, lens, 32, first).to(DEV), "ko": torch.zeros(n, 4, 128, dtype=torch.bfloat16, device=DEV),
             "vo": torch.zeros(n, 4, 128, dtype=torch.bfloat16, device=DEV),
             "q": torch.randn(n, 28, 128, generator=gen(1)).to(torch.bfloat16).to(DEV), "most": max(q_lens), "scale": 0.088,
             "plan": ck.plan_long(cumsum(q_lens), lens, 32), "segm": None, "lse": torch.zeros(n, 28, device=DEV),
             "w": torch.rand(4, 4, 2048, generator=gen(2)).to(DEV), "keep": i32([100, 100, 20, 300]), "recent": 16,
             "kept": torch.zeros(4, 4, 300, dtype=torch.int32, device=DEV), "new": i32([0] * 4),
             "pos": torch.arange(n, device=DEV), "table": torch.randn(400, 64, generator=gen(3)).to(DEV),
             "norm": [torch.rand(128, generator=gen(s)).to(DEV) for s in (4, 5)]}
        x["out"] = torch.zeros_like(x["q"])
        CHANGES[change](x)
        with monkeypatch.context() as m:
            if not native:
                m.setattr(ck.ext(), "calls", None)
            got.append(_call_all(c, x))
    (a, ta), (b, tb) = got
    assert a == b
    assert all(torch.equal(torch.nan_to_num(s.float()), torch.nan_to_num(t.float())) for s, t in zip(ta, tb))


def test_debug_check(monkeypatch):
    """KVQ_DEBUG=1 reports a table entry outside the cache."""
    monkeypatch.setenv("KVQ_DEBUG", "1")
    lens = [50, 20]
    c = filled(4, 128, 16, lens)
    q = torch.zeros(2, 28, 128, dtype=torch.bfloat16, device=DEV)
    args = (q, c.kc, c.vc, q.clone(), i32([0, 1, 2]), i32(lens), c.table, 1, 0.1, c.scales)
    fc.fp4_paged_attention(*args)
    c.table[0, 1] = 999
    with pytest.raises(RuntimeError, match="outside"):
        fc.fp4_paged_attention(*args)
