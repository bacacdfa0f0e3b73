"""The block-scaled cache's attention where its arithmetic could give way: values of extreme sizes, rows whose attention
lies almost whole on one key, q rows that hold an infinity, scales of blocks never written. Against 64 bits.

A bf16 output is off by at most 2^-8 of each value; by 2^-8 sqrt(1/3) 0.736 = 1.66e-3 of a row's norm for values spread evenly
over a binade's logarithm (the mean of 1 / x^2 there is 0.541 = 0.736^2). bf16 weights add the same in quadrature: 2.35e-3.
What else is rounded is far below: q to 2^-15 of its row's largest (1e-4 of a weight for the rows here), sums in fp32."""
import pytest
import torch
from conftest import nan_like, nan_segm

import block_ref as R
from kvq import block_cache as bc
from kvq import cuda_kernels as ck
from test_gpu_block_cache import DEV, Cache, cumsum, gen, i32, page_table, rows, source  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu
SHORT = 2.0 ** -9      # of the rows' norm: short queries, a bf16 output's rounding (1.66e-3) and 17% of it
MANY = 3e-3            # many query rows: bf16 weights too (2.35e-3), and 28%


def written(k, v, lens, bs=16, group=16, scale_fill=0.0, seed=1):
    h, d = k.shape[1:]
    table, nb = page_table(lens, bs, seed)
    c = Cache(h, d, bs, group, nb, scale_fill=scale_fill)
    bc.quant_block_cache(k.to(torch.bfloat16).to(DEV), v.to(torch.bfloat16).to(DEV), c.kc, c.vc, c.scales, i32(cumsum(lens)),
                         i32(lens), table.to(DEV))
    c.table = table.to(DEV)
    return c


def call(c, q, q_lens, lens, segm=None):
    cu = cumsum(q_lens)
    out = nan_like(q)
    bc.block_paged_attention(q, c.kc, c.vc, out, i32(cu), i32(lens), c.table, max(q_lens), c.geom[1] ** -0.5, c.scales,
                             ck.plan_long(cu, lens, c.geom[2]), segm)
    return out


def off(got, want):
    """Largest error of a request's rows, of their norm (rows: [.., D]; the norm over all of them)."""
    assert torch.isfinite(got.float()).all()
    return float((got.double() - want).norm() / want.norm())


def exact(c, q, q_lens, lens):
    return R.attention(q, c.kc, c.vc, c.scales, cumsum(q_lens), lens, c.table, c.geom[1] ** -0.5)[0]


def check(c, q, q_lens, lens, limit, segm=None, what=()):
    """Each request's rows within `limit` of their norm."""
    got, want, cu = call(c, q, q_lens, lens, segm), exact(c, q, q_lens, lens), cumsum(q_lens)
    for r in range(len(q_lens)):
        e = off(got[cu[r]:cu[r + 1]], want[cu[r]:cu[r + 1]])
        assert e <= limit, (what, r, e)


# ------------------------------------------------------------------------------------------------ cut rows
@pytest.mark.parametrize("where,size", [(w, s) for w in ("all", "the last keys") for s in (1e4, 1e6, 1e9, 1e20)] + [("all", 1e36)])
@pytest.mark.parametrize("q_lens", [[1, 1], [2, 1], [8, 5]])
def test_cut_rows_of_large_values(where, size, q_lens):
    """Rows cut into pieces keep their denominators whatever the V scales are, the last piece's as every other's, and agree
    with the rows run whole."""
    lens = [6000, 2500]
    k, v = rows(sum(lens), 4, 128, 2)
    big = torch.full((sum(lens),), size) if where == "all" else torch.cat([
        torch.where(torch.arange(n) >= n - 900, size, 1.0) for n in lens])
    c = written(k.float(), v.float() * big[:, None, None], lens)
    q = torch.randn(sum(q_lens), 28, 128, generator=gen(3)).to(torch.bfloat16).to(DEV)
    limit = SHORT if max(q_lens) < 8 else MANY
    check(c, q, q_lens, lens, limit, None, "whole")
    check(c, q, q_lens, lens, limit, nan_segm(sum(q_lens), 28, 16, 128), "cut")


@pytest.mark.parametrize("q_lens", [[1], [8]])
def test_cut_rows_without_keys_in_their_last_pieces(q_lens):
    """Verification rows of contexts that end a few keys into a piece: a row that sees nothing of the last piece (its
    denominator there is 0) is still merged, and so is one whose request has one tile more than its pieces."""
    for n in (4097, 4098, 4128, 4101):
        k, v = rows(n, 4, 128, 5)
        c = written(k.float(), v.float() * 1e5, [n])
        q = torch.randn(sum(q_lens), 28, 128, generator=gen(4)).to(torch.bfloat16).to(DEV)
        for splits in (2, 16, 64):
            check(c, q, q_lens, [n], SHORT if q_lens == [1] else MANY, nan_segm(sum(q_lens), 28, splits, 128), (n, splits))


# ------------------------------------------------------------------------------------------------ dominating keys
def sink(n, hq, h, d, q_rows, share, own, seed):
    """K, V [n, h, d] and q [q_rows, hq, d]: keys 0 and 40 each take `share` of a row's attention beside the other keys, with V
    of `own` times theirs."""
    g = gen(seed)
    u = torch.nn.functional.normalize(torch.randn(h, d, generator=g), dim=-1)
    k, v = torch.randn(n, h, d, generator=g), torch.randn(n, h, d, generator=g)
    k -= (k * u).sum(-1, keepdim=True) * u
    q = torch.randn(q_rows, h, hq // h, d, generator=g)
    q += (8.0 - (q * u[:, None]).sum(-1, keepdim=True)) * u[:, None]                 # q . u = 8 for every row
    top = torch.log(torch.tensor(float(n))) + 0.5 + torch.log(torch.tensor(share / (1 - share)))   # beside scores of N(0, 1)
    for i in (0, 40):
        if i < n:
            k[i] = u * (top * d ** 0.5 / 8.0)
            v[i] *= own
    return k, v, q.reshape(q_rows, hq, d)


@pytest.mark.parametrize("share,own", [(0.5, 0.0), (0.9, 0.02), (0.9, 0.0), (0.99, 0.0), (0.9999, 0.0)])
@pytest.mark.parametrize("hq,h,d", [(28, 4, 128), (14, 2, 64), (9, 1, 128)])
@pytest.mark.parametrize("query", [1, 2, 8, 20])
@pytest.mark.parametrize("n", [300, 4096])
def test_a_key_that_takes_most_of_a_row(share, own, hq, h, d, query, n, source):
    """The keys beside a dominating one keep their weights' precision: what is left of the output where the dominating
    key's own V is small is theirs, in its tile as in others."""
    k, v, q = sink(n, hq, h, d, query, share, own, 7)
    c = written(k, v, [n])
    q = q.to(torch.bfloat16).to(DEV)
    limit = SHORT if query * hq // h <= 16 else MANY
    check(c, q, [query], [n], limit, None, "whole")
    check(c, q, [query], [n], limit, nan_segm(query, hq, 16, d), "cut")


@pytest.mark.parametrize("query", [1, 2, 8, 20])
def test_a_loud_block_beside_quiet_ones(query, source):
    """Blocks of a tile whose V scales differ by 1e5, where the loud block's keys hold no value in most channels."""
    n = 512
    k, v, q = sink(n, 28, 4, 128, query, 0.01, 1.0, 8)
    v[torch.arange(n) // 16 % 2 == 0, :, 1:] = 0
    v[torch.arange(n) // 16 % 2 == 0, :, 0] *= 1e5
    c = written(k, v, [n])
    q = q.to(torch.bfloat16).to(DEV)
    got, want = call(c, q, [query], [n]), exact(c, q, [query], [n])
    assert off(got[..., 1:], want[..., 1:]) <= (SHORT if query < 8 else MANY)
    assert off(got[..., :1], want[..., :1]) <= (SHORT if query < 8 else MANY)


# ------------------------------------------------------------------------------------------------ V scales far apart
@pytest.mark.parametrize("size", [1e20, 1e30, 1e33, 1e37])
@pytest.mark.parametrize("q_lens", [[1, 1], [2, 1], [8, 8], [40, 30]])
def test_blocks_of_zeros_beside_the_largest_values(size, q_lens, source):
    """A block of zeros has the smallest V scale, 1e-8, and its keys' weights count in the denominator whatever the scales of
    the others are: up to bf16's largest values beside it."""
    lens = [700, 1500]
    k, v = rows(sum(lens), 4, 128, 6)
    at = torch.cat([torch.arange(n) for n in lens])
    v = v.float() * torch.where(at // 16 % 3 == 1, size, 0.0)[:, None, None]
    c = written(k.float() * 0.2, v.clamp(-3e38, 3e38), lens)
    q = torch.randn(sum(q_lens), 28, 128, generator=gen(3)).to(torch.bfloat16).to(DEV)
    limit = SHORT if max(q_lens) < 8 else MANY
    check(c, q, q_lens, lens, limit, None, "whole")
    check(c, q, q_lens, lens, limit, nan_segm(sum(q_lens), 28, 16, 128), "cut")


@pytest.mark.parametrize("q_lens", [[1, 1], [2, 1], [8, 5], [40, 30]])
def test_the_largest_values_behind_ones_of_order_one(q_lens, source):
    """The last 900 keys' V around 1e36, the others' around 1, rows whole and cut."""
    lens = [6000, 2500]
    k, v = rows(sum(lens), 4, 128, 2)
    big = torch.cat([torch.where(torch.arange(n) >= n - 900, 1e36, 1.0) for n in lens])
    c = written(k.float(), v.float() * big[:, None, None], lens)
    q = torch.randn(sum(q_lens), 28, 128, generator=gen(3)).to(torch.bfloat16).to(DEV)
    limit = SHORT if max(q_lens) < 8 else MANY
    check(c, q, q_lens, lens, limit, None, "whole")
    check(c, q, q_lens, lens, limit, nan_segm(sum(q_lens), 28, 16, 128), "cut")


@pytest.mark.parametrize("q_lens", [[1, 1], [8, 8], [40, 30]])
def test_values_of_the_smallest_scale(q_lens, source):
    """V around 1e-7: every block's scale is the smallest."""
    lens = [700, 1500]
    k, v = rows(sum(lens), 4, 128, 6)
    c = written(k.float(), v.float() * 1e-7, lens)
    q = torch.randn(sum(q_lens), 28, 128, generator=gen(3)).to(torch.bfloat16).to(DEV)
    check(c, q, q_lens, lens, SHORT if max(q_lens) < 8 else MANY)


# ------------------------------------------------------------------------------------------------ rows that are no number
@pytest.mark.parametrize("value", ["inf", "-inf", "nan"])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("q_lens", [[1, 1], [2, 3], [8, 8], [40, 20]])
def test_an_infinity_over_keys_of_one_sign(value, sign, q_lens, source):
    """q holds an infinity in a channel whose cached K has one sign, so that every score may be -inf: the row is NaN, not
    zeros (which say that it saw no key), where it sees one key and where it sees all; its neighbours are as they were."""
    lens = [q_lens[0], 9000]                       # the first request from its start: its first row sees one key
    k, v = rows(sum(lens), 4, 128, 9)
    k = k.float()
    k[..., 5] = sign * (1.0 + k[..., 5].abs())
    c = written(k, v.float(), lens)
    cu = cumsum(q_lens)
    q = torch.randn(cu[-1], 28, 128, generator=gen(1)).to(torch.bfloat16).to(DEV)
    bad = [(0, 3), (0, 27), (cu[1] - 1, 9), (cu[1], 0), (cu[2] - 1, 14)]
    for segm in (None, nan_segm(cu[-1], 28, 16, 128)):
        want = call(c, q, q_lens, lens, segm)
        odd = q.clone()
        for t, h in bad:
            odd[t, h, 5] = float(value)
        got = call(c, odd, q_lens, lens, segm)
        for t, h in bad:
            assert bool(torch.isnan(got[t, h]).all()), (t, h)
            got[t, h] = want[t, h]
        assert off(got, want.double()) <= 2.0 ** -8     # (a tile done again may round otherwise)


@pytest.mark.parametrize("q_lens", [[1, 2], [8, 8], [40, 20]])
def test_a_row_without_keys_is_zero_whatever_its_q(q_lens, source):
    """Requests of fewer keys than query tokens (and of none): the rows that see nothing are zero, also where q holds a NaN."""
    lens = [0 if q_lens[0] == 1 else 5, q_lens[1] - 1]
    k, v = rows(sum(lens), 4, 128, 9)
    c = written(k.float(), v.float(), lens)
    cu = cumsum(q_lens)
    q = torch.randn(cu[-1], 28, 128, generator=gen(1)).to(torch.bfloat16).to(DEV)
    unseen = [(0, 3), (cu[1], 9)]
    for t, h in unseen:
        q[t, h, 7] = float("nan")
    for segm in (None, nan_segm(cu[-1], 28, 16, 128)):
        got = call(c, q, q_lens, lens, segm)
        for t, h in unseen:
            assert not bool(got[t, h].any()), (t, h)
        assert torch.isfinite(got.float()).all()


@pytest.mark.parametrize("fill", [float("inf"), float("nan"), -1.0, 3e38])
@pytest.mark.parametrize("q_lens", [[1, 2, 3, 2], [8, 8, 3, 8], [12, 30, 3, 140]])
def test_scales_of_unwritten_blocks_are_not_read(fill, q_lens, source):
    """Scale buffers that were never cleared: what lies in the blocks behind a request's last key changes nothing."""
    lens = [70, 38, 3, 200]
    k, v = rows(sum(lens), 4, 128, 9)
    q = torch.randn(sum(q_lens), 28, 128, generator=gen(1)).to(torch.bfloat16).to(DEV)
    got = [call(written(k.float(), v.float(), lens, 64, 16, scale_fill=x), q, q_lens, lens) for x in (0.0, fill)]
    assert torch.isfinite(got[0].float()).all() and torch.equal(got[0].view(torch.int16), got[1].view(torch.int16))


# ------------------------------------------------------------------------------------------------ captured without lists
@pytest.mark.parametrize("copies", [True, False])
def test_capture_after_the_plans_own_copies(copies, monkeypatch):
    """A program that made a plan's device copies itself (tiles, and the pages' lists or not) and then captures its first
    call: replays follow the inputs and agree with an eager call."""
    monkeypatch.delenv("KVQ_PREFILL_DIRECT", raising=False)
    n, d = 2000, 128
    k, v = rows(n, 4, d, 3)
    c = written(k.float(), v.float(), [n])
    q = torch.randn(1500, 28, d, generator=gen(1)).to(torch.bfloat16).to(DEV)
    cu, sl = i32([0, 1500]), i32([n])
    plan = ck.plan_long([0, 1500], [n], 16)
    plan.tiles(7, DEV)
    if copies:
        plan.gpu(DEV)
    out = nan_like(q)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        bc.block_long_attention(q, c.kc, c.vc, out, cu, sl, c.table, plan, d ** -0.5, c.scales)
    for i in range(3):
        q.normal_()
        out.fill_(float("nan"))
        graph.replay()
        want = bc.block_long_attention(q, c.kc, c.vc, nan_like(q), cu, sl, c.table, plan, d ** -0.5, c.scales)
        assert off(out, want.double()) <= MANY, i


# ------------------------------------------------------------------------------------------------ scales made elsewhere
@pytest.mark.parametrize("q_lens", [[1, 1], [2, 1], [8, 8], [40, 30]])
def test_scales_far_below_the_writes(q_lens, source):
    """Scales that another program made: V's of 1e-18 as any other; of 0 (a cache that was cleared, not written) the values
    are zero, to what the smallest scale that counts leaves of 127 codes."""
    lens = [700, 1500]
    k, v = rows(sum(lens), 4, 128, 6)
    c = written(k.float(), v.float(), lens)
    q = torch.randn(sum(q_lens), 28, 128, generator=gen(3)).to(torch.bfloat16).to(DEV)
    c.scales["v_scale"].fill_(1e-18)
    for segm in (None, nan_segm(sum(q_lens), 28, 16, 128)):
        check(c, q, q_lens, lens, SHORT if max(q_lens) < 8 else MANY, segm)
    c.scales["v_scale"].zero_()
    assert float(call(c, q, q_lens, lens).abs().max()) <= 128 * 2.0 ** -70


@pytest.mark.parametrize("bs,group", [(128, 128), (256, 128), (64, 64), (32, 16)])
@pytest.mark.parametrize("order", [(2, 1, 0), (1, 0, 2), (0, 2, 1)])
@pytest.mark.parametrize("q_lens", [[1, 1, 1], [8, 3, 8], [40, 200, 9]])
def test_scales_in_any_order(bs, group, order, q_lens, source):
    """Scales of another memory order than [pages, heads, blocks], with the largest blocks and pages: the outputs are those of
    scales side by side, bit for bit."""
    lens = [700, 257, 1300]
    k, v = rows(sum(lens), 4, 128, 6)
    c = written(k.float(), v.float(), lens, bs, group)
    q = torch.randn(sum(q_lens), 28, 128, generator=gen(3)).to(torch.bfloat16).to(DEV)
    back = [i for i, _ in sorted(enumerate(order), key=lambda x: x[1])]
    for segm in (None, nan_segm(sum(q_lens), 28, 16, 128)):
        want = call(c, q, q_lens, lens, segm)
        check(c, q, q_lens, lens, SHORT if max(q_lens) < 8 else MANY, segm)
        kept = c.scales
        c.scales = {n: s.permute(order).contiguous().permute(back) for n, s in kept.items()}
        assert c.scales["k_scale"].stride() != kept["k_scale"].stride()
        got = call(c, q, q_lens, lens, segm)
        c.scales = kept
        assert torch.equal(got.view(torch.int16), want.view(torch.int16))
