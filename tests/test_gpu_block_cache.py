"""The block-scaled cache's operators on the GPU (kvq.block_cache) against plain implementations: codes, scales and rows
read back bit for bit, attention within the bound that its roundings add up to (block_ref.attention)."""
import numpy as np
import pytest
import torch
from conftest import nan_like, nan_segm

import block_ref as R
from kvq import block_cache as bc
from kvq import cuda_kernels as ck

pytestmark = pytest.mark.gpu
DEV = "cuda"
GEOM = [(4, 128, 16, 16), (8, 128, 32, 16), (2, 64, 64, 32), (1, 128, 128, 64), (3, 64, 128, 128), (2, 128, 64, 64)]


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


@pytest.fixture(params=["0", "1"], ids=["copied", "direct"])
def source(request, monkeypatch):
    """What long queries read: a temporary bf16 cache of the codes, or the int8 pages themselves."""
    monkeypatch.setenv("KVQ_PREFILL_DIRECT", request.param)
    return request.param


class Cache:
    """A cache on the GPU and its plain twin on the host, filled step by step through both."""

    def __init__(self, h, d, bs, group, nb, layout="vllm", scales="side by side", fill=77, scale_fill=0.0):
        self.geom = (h, d, bs, group)
        self.kc, self.vc = R.new_cache(nb, bs, h, d, layout, DEV, fill)
        self.scales = R.new_scales(nb, bs, h, group, scales, DEV, scale_fill)
        self.k_host, self.v_host = R.new_cache(nb, bs, h, d, "apart", "cpu", fill)
        self.s_host = R.new_scales(nb, bs, h, group, "apart", "cpu", scale_fill)

    def write(self, k, v, cu, lens, table):
        bc.quant_block_cache(k.to(DEV), v.to(DEV), self.kc, self.vc, self.scales, i32(cu), i32(lens), table.to(DEV))
        R.write(k, self.k_host, self.s_host["k_scale"], cu, lens, table)
        R.write(v, self.v_host, self.s_host["v_scale"], cu, lens, table)

    def check(self, what=""):
        for nm, got, want in (("k", self.kc, self.k_host), ("v", self.vc, self.v_host),
                              ("k_scale", self.scales["k_scale"], self.s_host["k_scale"]),
                              ("v_scale", self.scales["v_scale"], self.s_host["v_scale"])):
            same = torch.eq(got.cpu(), want) | (got.cpu() != got.cpu()) & (want != want)
            assert bool(same.all()), (what, nm, int((~same).sum()), same.numel())


def i32(x):
    return torch.as_tensor(np.asarray(x, dtype=np.int32)).to(DEV)


def cumsum(x):
    return np.concatenate([[0], np.cumsum(x)]).tolist()


def filled(h, d, bs, group, lens, seed=0, layout="vllm", poison=True):
    """A cache whose requests hold `lens` keys, written in one call; what lies outside them is poison: codes of 77 and
    -- where no block was begun -- NaN scales."""
    table, nb = page_table(lens, bs, seed)
    c = Cache(h, d, bs, group, nb, layout, scale_fill=float("nan") if poison else 0.0)
    k, v = rows(sum(lens), h, d, seed + 1)
    bc.quant_block_cache(k.to(DEV), v.to(DEV), c.kc, c.vc, c.scales, i32(cumsum(lens)), i32(lens), table.to(DEV))
    c.table = table.to(DEV)
    return c


# ------------------------------------------------------------------------------------------------ write
@pytest.mark.parametrize("h,d,bs,group", GEOM)
@pytest.mark.parametrize("layout", ["vllm", "apart"])
def test_write_step_by_step(h, d, bs, group, layout):
    """Prompts of ragged lengths, then steps of 1, 1, .., 3, 20 and 150 tokens that end inside, at and past blocks: every
    code and scale of the whole cache (untouched ones too) equals the plain write's after each."""
    lens = [1, 15, 16, 17, group - 1, group, 2 * group + 5, 301]
    steps = [lens] + [[1] * len(lens)] * 4 + [[3, 0, 1, 20, 0, 2, 0, 150]] + [[1] * len(lens)] * 2
    final = np.sum(steps, axis=0).tolist()
    table, nb = page_table(final, bs, 5)
    c = Cache(h, d, bs, group, nb, layout, "side by side" if layout == "vllm" else "apart")
    held = np.zeros(len(lens), dtype=int)
    for i, q in enumerate(steps):
        held = held + q
        k, v = rows(sum(q), h, d, 10 + i, loud=1.0 + i)     # later tokens are louder: scales grow
        c.write(k, v, cumsum(q), held.tolist(), table)
        c.check(f"step {i}")


def test_write_rewrites_after_a_rollback():
    """Rejected speculative tokens: 4 written, 3 taken back and written again (same block, then across its end)."""
    table, nb = page_table([64], 16, 1)
    c = Cache(4, 128, 16, 16, nb)
    for i, (q, n) in enumerate([(10, 10), (4, 14), (4, 15), (4, 18), (4, 19), (4, 17)]):
        k, v = rows(q, 4, 128, 20 + i, loud=2.0)
        c.write(k, v, [0, q], [n], table)
        c.check(i)


@pytest.mark.parametrize("h,d,bs,group", [(4, 128, 16, 16), (2, 64, 64, 64)])
def test_write_zeros_infinities_and_tiny_values(h, d, bs, group):
    """All-zero blocks get the smallest scale; an infinity saturates and leaves its neighbours' scale alone."""
    n = 3 * group + 5
    table, nb = page_table([n], bs, 2)
    k, v = rows(n, h, d, 3)
    k[:group] = 0
    v[group + 1, 0, 3], v[group + 2, 1, 5], v[group + 3, 0, d - 1] = float("inf"), float("-inf"), 3e38
    k[2 * group:] *= 1e-9
    c = Cache(h, d, bs, group, nb)
    c.write(k, v, [0, n], [n], table)
    c.check()
    assert bool((c.scales["k_scale"][table[0, 0], :, 0] == 1e-8).all())


def test_write_skips_padding_bad_pages_and_negative_positions():
    """Rows past cu_seqlens_q's end, requests without new tokens, tokens at negative positions and pages outside the
    cache write nothing."""
    lens, q = [40, 3, 20, 33], [8, 5, 0, 33]
    table, nb = page_table(lens, 16, 4)
    table[3, 1] = nb                      # the middle page of the last request is bad
    c = Cache(4, 128, 16, 16, nb)
    first = [32, 0, 20, 0]
    k, v = rows(sum(first), 4, 128, 5)
    c.write(k, v, cumsum(first), first, table)
    k, v = rows(sum(q) + 9, 4, 128, 6)
    c.write(k, v, cumsum(q), lens, table)
    c.check()
    c.write(k[:4], v[:4], [0, 0, 0, 0, 0], lens, table)
    c.check("no tokens")


def test_write_takes_strided_rows():
    """key / value as views of one packed qkv tensor, as a model has them."""
    h, d, n = 4, 128, 45
    k, v = rows(n, h, d, 7)
    qkv = torch.zeros(n, 12 + 2 * h, d, dtype=torch.bfloat16)
    qkv[:, 12:12 + h], qkv[:, 12 + h:] = k, v
    qkv = qkv.to(DEV)
    table, nb = page_table([n], 32, 3)
    c = Cache(h, d, 32, 32, nb)
    bc.quant_block_cache(qkv[:, 12:12 + h], qkv[:, 12 + h:], c.kc, c.vc, c.scales, i32([0, n]), i32([n]), table.to(DEV))
    R.write(k, c.k_host, c.s_host["k_scale"], [0, n], [n], table)
    R.write(v, c.v_host, c.s_host["v_scale"], [0, n], [n], table)
    c.check()


def test_write_many_requests():
    """300 requests (more than one round of the search over them), some with no new token."""
    r = np.random.RandomState(0)
    q = r.choice([0, 1, 1, 1, 2, 17, 40], 300).tolist()
    q[0] = q[-1] = 0
    lens = [a + int(b) for a, b in zip(q, r.randint(0, 50, 300))]
    table, nb = page_table(lens, 16, 8)
    c = Cache(2, 64, 16, 16, nb)
    first = [n - a for n, a in zip(lens, q)]
    c.write(*rows(sum(first), 2, 64, 9), cumsum(first), first, table)
    c.write(*rows(sum(q), 2, 64, 10, loud=3.0), cumsum(q), lens, table)
    c.check()


# ------------------------------------------------------------------------------------------------ read
@pytest.mark.parametrize("h,d,bs,group", GEOM)
def test_read_back(h, d, bs, group):
    """Ranges that begin and end anywhere, empty ones among them: bf16(code * scale) bit for bit; rows behind the last
    range stay as they were."""
    lens = [1, 16, 17, 33, 200, 5, 2 * group]
    c = filled(h, d, bs, group, lens, layout="apart" if h == 2 else "vllm")
    start = [0, 3, 16, 31, 57, 2, 0]
    count = [1, 13, 1, 2, 141, 0, 2 * group]
    cu = cumsum(count)
    wide = torch.full((cu[-1] + 6, 2 * h, d), 5.0, dtype=torch.bfloat16, device=DEV)
    k, v = bc.read_block_cache(c.kc, c.vc, c.scales, i32(start), i32(cu), c.table, wide[:, :h], wide[:, h:])
    for got, cache, scale in ((k, c.kc, c.scales["k_scale"]), (v, c.vc, c.scales["v_scale"])):
        for r, (s, n) in enumerate(zip(start, count)):
            codes, sc = R.values(cache, scale, c.table[r], s + n)
            want = (codes.float() * sc.float()[..., None]).to(torch.bfloat16)[:, s:].transpose(0, 1)
            assert torch.equal(got[cu[r]:cu[r + 1]], want), r
        assert bool((got[cu[-1]:] == 5.0).all())


def test_read_back_past_the_last_level_cache():
    """A read of more than 256 MiB (streaming loads and stores)."""
    h, d, bs = 16, 64, 64
    n = (258 << 20) // (6 * h * d)
    lens = [n - 777, 777]
    table, nb = page_table(lens, bs, 1)
    g = torch.Generator(device=DEV).manual_seed(1)
    kc, vc = (torch.randint(-127, 128, (nb, bs, h, d), generator=g, device=DEV, dtype=torch.int8) for _ in range(2))
    scales = {x: torch.rand(nb, h, 2, generator=g, device=DEV) + 0.1 for x in ("k_scale", "v_scale")}
    k, v = (torch.zeros(n, h, d, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    bc.read_block_cache(kc, vc, scales, i32([0, 0]), i32(cumsum(lens)), table.to(DEV), k, v)
    for got, cache, scale in ((k, kc, scales["k_scale"]), (v, vc, scales["v_scale"])):
        at = 0
        for r, m in enumerate(lens):
            codes, s = R.values(cache, scale, table[r].to(DEV), m)
            want = (codes.float() * s.float()[..., None]).to(torch.bfloat16).transpose(0, 1)
            assert torch.equal(got[at:at + m], want), r
            at += m


# ------------------------------------------------------------------------------------------------ attention
HEADS = [(28, 4, 128), (32, 8, 128), (14, 2, 64), (16, 16, 64), (32, 1, 128), (8, 1, 64), (9, 1, 128), (34, 2, 64)]


def attend(c, hq, q_lens, lens, segm=None, seed=3, scale=None, pad=2):
    h, d = c.geom[:2]
    cu = cumsum(q_lens)
    q = torch.randn(cu[-1] + pad, hq, d, generator=gen(seed)).to(torch.bfloat16).to(DEV)
    out = nan_like(q)
    scale = d ** -0.5 if scale is None else scale
    plan = ck.plan_long(cu, lens, c.geom[2])
    bc.block_paged_attention(q, c.kc, c.vc, out, i32(cu), i32(lens), c.table, max(q_lens), scale, c.scales, plan, segm)
    want, bound = R.attention(q, c.kc, c.vc, c.scales, cu, lens, c.table, scale)
    n = cu[-1]
    assert bool(torch.isnan(out[n:]).all()), "rows behind the batch were written"
    return R.check(out[:n], want[:n], bound[:n], (c.geom, hq, q_lens, lens))


SHORT_LENS = [0, 1, 15, 16, 17, 31, 32, 33, 64, 65, 500, 1000, 2049]


@pytest.mark.parametrize("hq,h,d", HEADS)
@pytest.mark.parametrize("qlen", [1, 2, 5, 8])
@pytest.mark.parametrize("split", [False, True])
def test_short_queries(hq, h, d, qlen, split):
    """Decode and verification rows over contexts that end anywhere in a tile and page; requests without keys and with
    fewer keys than query tokens (rows that see nothing are zero)."""
    bs, group = {1: (16, 16), 2: (32, 16), 5: (64, 32), 8: (128, 64)}[qlen]
    c = filled(h, d, bs, group, SHORT_LENS, layout="vllm" if qlen != 5 else "apart")
    q = [qlen] * len(SHORT_LENS)
    attend(c, hq, q, SHORT_LENS, nan_segm(sum(q), hq, 16, d) if split else None)


@pytest.mark.parametrize("splits", [1, 2, 7, 64])
def test_long_contexts_are_cut(splits):
    """Few requests over long contexts, cut into up to `splits` pieces."""
    lens = [20000, 3, 7777]
    c = filled(4, 128, 16, 16, lens)
    attend(c, 28, [1, 1, 1], lens, nan_segm(3, 28, splits, 128))
    attend(c, 28, [4, 1, 3], lens, nan_segm(8, 28, splits, 128))


def test_split_buffers_of_fewer_rows():
    lens = [5000, 4000, 300]
    c = filled(2, 64, 32, 32, lens)
    attend(c, 14, [1, 3, 2], lens, nan_segm(4, 14, 16, 64))


def test_scales_that_differ_by_orders_of_magnitude(source):
    """Blocks whose V (and K) is a million times larger or smaller than their neighbours'."""
    lens = [333, 96, 40]
    table, nb = page_table(lens, 16, 1)
    c = Cache(4, 128, 16, 16, nb)
    k, v = rows(sum(lens), 4, 128, 2)
    size = torch.tensor([1.0, 1e-6, 1e-3, 1e6, 1.0])[torch.arange(sum(lens)) // 24 % 5]
    v = v * size[:, None, None]
    k = k * torch.tensor([1.0, 1e-5, 0.3])[torch.arange(sum(lens)) // 40 % 3][:, None, None]
    c.write(k.to(torch.bfloat16), v.to(torch.bfloat16), cumsum(lens), lens, table)
    c.table = table.to(DEV)
    for q_lens in ([1, 1, 1], [8, 3, 8], [100, 20, 40]):
        attend(c, 28, q_lens, lens)
        attend(c, 28, q_lens, lens, nan_segm(sum(q_lens), 28, 16, 128))


@pytest.mark.parametrize("magnitude", [1e-3, 1.0, 30.0])
def test_peaked_and_flat_softmax(magnitude, source):
    """Scores from nearly equal to hundreds apart (the running maximum jumps by far more than its slack)."""
    lens = [700, 257, 64]
    c = filled(4, 128, 32, 32, lens)
    q = torch.randn(sum([2, 1, 1]), 28, 128, generator=gen(1)) * magnitude
    for q_lens in ([2, 1, 1], [60, 9, 30]):
        cu = cumsum(q_lens)
        q = (torch.randn(cu[-1], 28, 128, generator=gen(1)) * magnitude).to(torch.bfloat16).to(DEV)
        out = nan_like(q)
        bc.block_paged_attention(q, c.kc, c.vc, out, i32(cu), i32(lens), c.table, max(q_lens), 128 ** -0.5, c.scales,
                                 ck.plan_long(cu, lens, 32))
        want, bound = R.attention(q, c.kc, c.vc, c.scales, cu, lens, c.table, 128 ** -0.5)
        R.check(out, want, bound, (magnitude, q_lens))


@pytest.mark.parametrize("hq,h,d", HEADS)
@pytest.mark.parametrize("bs,group", [(16, 16), (64, 32)])
def test_long_queries(hq, h, d, bs, group, source):
    """Prompts from their start and mid-way, ending anywhere in tiles, pages and row tiles."""
    lens = [9, 40, 129, 333, 700, 64]
    c = filled(h, d, bs, group, lens, layout="vllm" if bs == 16 else "apart")
    attend(c, hq, [9, 10, 129, 57, 300, 64], lens)


def test_long_query_few_rows_over_many_keys(source):
    """Rows cut into pieces of keys and merged."""
    lens = [9000, 2000]
    c = filled(4, 128, 16, 16, lens)
    plan = ck.plan_long([0, 20, 31], lens, 16)
    assert plan.work(7, 4, 128, torch.device(DEV)).merge is not None
    attend(c, 28, [20, 11], lens)


def test_mixed_batch(source):
    lens = [1, 100, 0, 5000, 700, 2500]
    c = filled(8, 128, 32, 32, lens)
    q = [1, 1, 1, 1, 700, 333]
    attend(c, 32, q, lens, nan_segm(4, 32, 16, 128))
    attend(c, 32, q, lens)


def test_softmax_scale_and_host_bounds(source):
    """Another softmax scale; a plan made from upper bounds of the lengths."""
    lens = [100, 90]
    c = filled(4, 128, 16, 16, lens)
    attend(c, 28, [1, 30], lens, scale=0.3)
    cu = [0, 1, 31]
    q = torch.randn(31, 28, 128, generator=gen(2)).to(torch.bfloat16).to(DEV)
    wide = torch.cat([c.table, torch.zeros(2, 8, dtype=torch.int32, device=DEV)], 1)
    out = nan_like(q)
    bc.block_paged_attention(q, c.kc, c.vc, out, i32(cu), i32(lens), wide, 30, 128 ** -0.5, c.scales,
                             ck.plan_long(cu, [120, 170], 16))
    want, bound = R.attention(q, c.kc, c.vc, c.scales, cu, lens, c.table, 128 ** -0.5)
    R.check(out, want, bound)


@pytest.mark.parametrize("poison", [False, True])
@pytest.mark.parametrize("scale", [1e-16, 1e-12, 0.09])
def test_unwritten_halves_of_a_tile_under_small_softmax_scales(scale, poison, source):
    """The last tile of most requests ends in a half whose block was never written (scales 0 or NaN): masked, no NaN from it."""
    lens = [70, 38, 3, 200]
    c = filled(4, 128, 64, 16, lens, poison=poison)
    attend(c, 28, [1, 2, 3, 2], lens, scale=scale)
    attend(c, 28, [12, 30, 3, 140], lens, scale=scale)


def test_padded_requests_of_a_graph_batch():
    """Requests beyond the batch's: no query tokens (cu repeats), length 0, rows of the table unset."""
    lens = [50, 700, 0, 0]
    c = filled(4, 128, 16, 16, lens)
    c.table[2:] = 0
    attend(c, 28, [1, 1, 0, 0], lens)
    attend(c, 28, [1, 1, 0, 0], lens, nan_segm(4, 28, 16, 128))


@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("q_lens", [[1, 1, 1, 1], [8, 8, 3, 8], [40, 9, 300, 12]])
def test_rows_that_are_no_number_stay_their_own(q_lens, split, source):
    """A NaN or an infinity in one q row makes that row NaN and no other; rows of zeros average what they see, over zero
    scales too (blocks never written, as in a warm-up) and where their tiles are masked."""
    lens = [3000, 70, 400, 33]
    c = filled(4, 128, 32, 16, lens)
    c.scales["k_scale"][c.table[3, :2].long()] = 0
    cu = cumsum(q_lens)
    q = torch.randn(cu[-1], 28, 128, generator=gen(1)).to(torch.bfloat16).to(DEV)
    q[cu[1]:cu[2], 3] = 0
    q[cu[3]:] = 0
    clean = q.clone()
    bad = [(0, 5, 17, "nan"), (cu[1] - 1, 27, 127, "inf"), (cu[2], 0, 0, "-inf")]
    for t, h, d, x in bad:
        q[t, h, d] = float(x)
    segm = nan_segm(cu[-1], 28, 16, 128) if split else None
    out = torch.full_like(q, 7.0)
    bc.block_paged_attention(q, c.kc, c.vc, out, i32(cu), i32(lens), c.table, max(q_lens), 128 ** -0.5, c.scales,
                             ck.plan_long(cu, lens, 32), segm)
    want, bound = R.attention(clean, c.kc, c.vc, c.scales, cu, lens, c.table, 128 ** -0.5)
    for t, h, _, _ in bad:
        assert bool(torch.isnan(out[t, h]).all()), (t, h)
        out[t, h] = want[t, h].to(out.dtype)
    R.check(out, want, bound, q_lens)


@pytest.mark.parametrize("short_q", [1, 1_000_000])
def test_other_short_query_limits(short_q, monkeypatch, source):
    """KVQ_SHORT_Q's other uses: verification rows through the long path, whole prompts through the short one."""
    monkeypatch.setattr(ck, "SHORT_Q", short_q)
    lens = [90, 500, 33, 700]
    c = filled(4, 128, 16, 16, lens)
    attend(c, 28, [1, 8, 3, 1], lens)
    attend(c, 28, [1, 300, 33, 20], lens)
    attend(c, 28, [1, 300, 33, 20], lens, nan_segm(354, 28, 16, 128))


# ------------------------------------------------------------------------------------------------ together
@pytest.mark.parametrize("hq,h,d,bs,group", [(28, 4, 128, 16, 16), (14, 2, 64, 64, 32)])
def test_generation_captured_and_replayed(hq, h, d, bs, group):
    """A prompt step eagerly, then decode steps in one captured graph (write, attention, read of the block written):
    every replay equals the same calls made eagerly on a twin cache, and the plain cache."""
    prompts = [37, 5, 128, 300]
    steps, n = 20, len(prompts)
    table, nb = page_table([p + steps for p in prompts], bs, 3)
    a, b = (Cache(h, d, bs, group, nb) for _ in range(2))
    k, v = rows(sum(prompts), h, d, 4)
    for c in (a, b):
        c.write(k, v, cumsum(prompts), prompts, table)
    dtab = table.to(DEV)
    cu, cu_k = i32(range(n + 1)), i32(cumsum([group] * n))

    class Step:
        def __init__(self, c):
            self.c, self.lens, self.start = c, i32(prompts), i32([0] * n)
            self.k, self.v = (torch.zeros(n, h, d, dtype=torch.bfloat16, device=DEV) for _ in range(2))
            self.q = torch.zeros(n, hq, d, dtype=torch.bfloat16, device=DEV)
            self.out = torch.zeros_like(self.q)
            self.back = [torch.zeros(n * group, h, d, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
            self.segm = ck.split_buffers(n, hq, d, 16, DEV)

        def load(self, i):
            k, v = rows(n, h, d, 100 + i, loud=i)
            self.k.copy_(k)
            self.v.copy_(v)
            self.q.copy_(torch.randn(n, hq, d, generator=gen(200 + i)))
            held = [p + i + 1 for p in prompts]
            self.lens.copy_(i32(held))
            self.start.copy_(i32([(x - 1) // group * group for x in held]))
            return k, v, held

        def run(self):
            c = self.c
            bc.quant_block_cache(self.k, self.v, c.kc, c.vc, c.scales, cu, self.lens, dtab)
            bc.block_paged_attention(self.q, c.kc, c.vc, self.out, cu, self.lens, dtab, 1, d ** -0.5, c.scales, None, self.segm)
            bc.read_block_cache(c.kc, c.vc, c.scales, self.start, cu_k, dtab, *self.back)

    sa, sb = Step(a), Step(b)
    for s in (sa, sb):
        s.load(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        sa.run()        # warm up: step 0's write, which the first replay makes again
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sa.run()
    for i in range(steps):
        sa.load(i)
        k, v, held = sb.load(i)
        graph.replay()
        sb.run()
        torch.cuda.synchronize()
        R.write(k, b.k_host, b.s_host["k_scale"], range(n + 1), held, table)
        R.write(v, b.v_host, b.s_host["v_scale"], range(n + 1), held, table)
        b.check(i)
        assert torch.equal(sa.out, sb.out) and all(torch.equal(x, y) for x, y in zip(sa.back, sb.back)), i
        assert torch.equal(a.kc, b.kc) and torch.equal(a.vc, b.vc), i
        want, bound = R.attention(sb.q, b.kc, b.vc, b.scales, list(range(n + 1)), held, dtab, d ** -0.5)
        R.check(sb.out, want, bound, i)


def test_pages_past_two_and_four_gib(source):
    """A cache of more than 4 GiB a side: the pages used lie at its ends and around 2 and 4 GiB."""
    h, d, bs = 8, 128, 64
    nb = (4 << 30) // (h * d * bs) + 40
    kc, vc = (torch.empty(nb, bs, h, d, dtype=torch.int8, device=DEV) for _ in range(2))
    scales = bc.block_scales(nb, bs, h, 32, DEV)
    ids = [nb - 1, 0, nb // 2, nb // 2 - 1, nb - 40, nb - 41, 1, nb - 2]
    lens = [64 * 4 - 3, 64 * 4]
    table = torch.tensor(ids, dtype=torch.int32).view(2, 4)
    k, v = rows(sum(lens), h, d, 1)
    cu = cumsum(lens)
    bc.quant_block_cache(k.to(DEV), v.to(DEV), kc, vc, scales, i32(cu), i32(lens), table.to(DEV))
    at = torch.tensor(ids, device=DEV).long()
    small = {"kc": kc[at].contiguous(), "vc": vc[at].contiguous()}
    ss = {n: scales[n][at] for n in scales}
    tiny = torch.arange(8, dtype=torch.int32).view(2, 4)
    kr, vr = R.new_cache(8, bs, h, d, "apart")
    sr = R.new_scales(8, bs, h, 32, "apart")
    R.write(k, kr, sr["k_scale"], cu, lens, tiny)
    live = torch.ones(8 * bs, dtype=torch.bool)
    live[lens[0]:256] = False
    assert torch.equal(small["kc"].cpu().flatten(0, 1)[live], kr.flatten(0, 1)[live])
    assert torch.equal(ss["k_scale"].cpu(), sr["k_scale"])
    out = [torch.zeros(sum(lens), h, d, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    bc.read_block_cache(kc, vc, scales, i32([0, 0]), i32(cu), table.to(DEV), *out)
    codes, sc = R.values(small["vc"], ss["v_scale"], tiny[1].to(DEV), lens[1])
    assert torch.equal(out[1][cu[1]:], (codes.float() * sc.float()[..., None]).to(torch.bfloat16).transpose(0, 1))
    for q_lens in ([1, 8], [30, 100]):
        cq = cumsum(q_lens)
        q = torch.randn(cq[-1], 32, d, generator=gen(2)).to(torch.bfloat16).to(DEV)
        o = nan_like(q)
        bc.block_paged_attention(q, kc, vc, o, i32(cq), i32(lens), table.to(DEV), max(q_lens), d ** -0.5, scales,
                                 ck.plan_long(cq, lens, bs))
        want, bound = R.attention(q, small["kc"], small["vc"], ss, cq, lens, tiny.to(DEV), d ** -0.5)
        R.check(o, want, bound, q_lens)


def test_another_stream():
    """Calls go to the stream that is current, behind what it holds already."""
    lens = [300, 41]
    table, nb = page_table(lens, 16, 1)
    c = Cache(4, 128, 16, 16, nb)
    k, v = rows(sum(lens), 4, 128, 2)
    kd, vd = torch.zeros_like(k, device=DEV), torch.zeros_like(v, device=DEV)
    ks, vs = k.pin_memory(), v.pin_memory()
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        torch.cuda._sleep(20_000_000)
        kd.copy_(ks, non_blocking=True)
        vd.copy_(vs, non_blocking=True)
        bc.quant_block_cache(kd, vd, c.kc, c.vc, c.scales, i32(cumsum(lens)), i32(lens), table.to(DEV))
    s.synchronize()
    R.write(k, c.k_host, c.s_host["k_scale"], cumsum(lens), lens, table)
    R.write(v, c.v_host, c.s_host["v_scale"], cumsum(lens), lens, table)
    c.check()


def test_debug_check(monkeypatch):
    """KVQ_DEBUG=1 reports a scale that is not finite among the keys a batch uses."""
    monkeypatch.setenv("KVQ_DEBUG", "1")
    lens = [50, 20]
    c = filled(4, 128, 16, 16, lens)
    c.table[c.table < 0] = 0
    q = torch.zeros(2, 28, 128, dtype=torch.bfloat16, device=DEV)
    args = (q, c.kc, c.vc, q.clone(), i32([0, 1, 2]), i32(lens), c.table, 1, 0.1, c.scales)
    bc.block_paged_attention(*args)
    c.scales["v_scale"][c.table[0, 3]] = float("inf")
    with pytest.raises(RuntimeError, match="req 0: v_scale not finite"):
        bc.block_paged_attention(*args)


# ------------------------------------------------------------------------------------------------ native calls
def _call_all(c, x):
    """Every operator once on the GPU state `x`; the outputs, or what was raised."""
    got = []
    for f in (lambda: bc.quant_block_cache(x["k"], x["v"], c.kc, c.vc, x["scales"], x["cu"], x["lens"], c.table),
              lambda: bc.read_block_cache(c.kc, c.vc, x["scales"], x["lens"] // 2, x["cu"], c.table, x["ko"], x["vo"]),
              lambda: bc.block_paged_attention(x["q"], c.kc, c.vc, x["out"], x["cu"], x["lens"], c.table, x["most"], x["scale"],
                                               x["scales"], x["plan"], x["segm"])):
        try:
            f()
            got.append("served")
        except Exception as e:  # noqa: BLE001 - compared with the other path's
            got.append((type(e), str(e)))
    return got, [t.clone() for t in (c.kc, c.vc, x["scales"]["k_scale"], x["ko"], x["vo"], x["out"])]


CHANGES = {
    "plain": lambda x: None,
    "split": lambda x: x.update(segm=nan_segm(x["q"].shape[0], 28, 16, 128)),
    "strided_split": lambda x: x.update(segm=tuple(t[:, :28] for t in nan_segm(x["q"].shape[0], 30, 8, 128))),
    "packed_q": lambda x: x.update(q=torch.cat([x["q"], x["q"]], 1)[:, :28]),
    "parameter_scales": lambda x: x.update(scales={n: torch.nn.Parameter(t, requires_grad=False) for n, t in x["scales"].items()}),
    "scale_int": lambda x: x.update(scale=1),
    "half": lambda x: x.update(q=x["q"].half(), k=x["k"].half(), ko=x["ko"].half()),
    "few_outputs": lambda x: x.update(out=x["out"][:3], vo=x["vo"][:-1]),
    "long_lengths": lambda x: x.update(lens=x["lens"].long()),
    "odd_rows": lambda x: x.update(q=torch.zeros(x["q"].shape[0], 28, 132, dtype=torch.bfloat16, device=DEV)[..., :128],
                                   k=torch.zeros(*x["k"].shape[:2], 132, dtype=torch.bfloat16, device=DEV)[..., :128]),
    "cpu": lambda x: x.update(q=x["q"].cpu(), k=x["k"].cpu(), ko=x["ko"].cpu()),
}


@pytest.mark.parametrize("change", CHANGES)
def test_native_calls_and_the_python_path_agree(change, monkeypatch):
    assert ck.ext().calls is not None, "kvq._torch_calls is not built"
    lens, q_lens = [300, 20, 64, 2000], [1, 20, 8, 300]
    got = []
    for native, direct in ((True, "0"), (False, "0"), (True, "1"), (False, "1")):
        monkeypatch.setenv("KVQ_PREFILL_DIRECT", direct)
        c = filled(4, 128, 32, 16, lens)
        n = sum(q_lens)
        k, v = rows(n, 4, 128, 50)
        x = {"k": k.to(DEV), "v": v.to(DEV), "scales": c.scales, "cu": i32(cumsum(q_lens)), "lens": i32(lens),
             "ko": torch.zeros(n, 4, 128, dtype=torch.bfloat16, device=DEV),
             "vo": torch.zeros(n, 4, 128, dtype=torch.bfloat16, device=DEV),
             "q": torch.randn(n, 28, 128, generator=gen(1)).to(torch.bfloat16).to(DEV), "most": max(q_lens), "scale": 0.088,
             "plan": ck.plan_long(cumsum(q_lens), lens, 32), "segm": None}
        x["out"] = torch.zeros_like(x["q"])
        CHANGES[change](x)
        with monkeypatch.context() as m:
            if not native:
                m.setattr(ck.ext(), "calls", None)
            got.append(_call_all(c, x))
    for (a, ta), (b, tb) in zip(got[::2], got[1::2]):
        assert a == b
        assert all(torch.equal(torch.nan_to_num(s.float()), torch.nan_to_num(t.float())) for s, t in zip(ta, tb))
