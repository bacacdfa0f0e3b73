"""Operators of the block-scaled INT8 cache: a KV cache in int8 without calibrated scales, beside the static one of
kvq.cuda_kernels (no counterpart in the reference).

Each (page, kv head, block of `group` consecutive positions) holds one fp32 scale for K and one for V, made from the
values as they are written; a cached value is code * scale. Pages, block tables, lengths, split buffers and the plan of
long requests are those of kvq.cuda_kernels, so a program switches a layer between the two by its scales alone:

    kc, vc                              int8 [num_blocks, block_size, kv heads, D] views, as the static cache's
    scales = block_scales(num_blocks, block_size, kv_heads, group, device)
    quant_block_cache(key, value, kc, vc, scales, cu_seqlens_q, seq_lens, block_table)      a step's new tokens
    block_paged_attention(q, kc, vc, out, cu_seqlens_q, seq_lens, block_table, max_query_len, softmax_scale, scales,
                          plan, segm)                                                       the step's attention
    read_block_cache(kc, vc, scales, starts, cu_seqlens_k, block_table, k_out, v_out)       keys back as bf16 rows

The write needs the requests' lengths and pages in place of a slot mapping: which blocks a step touches, and which of
them hold earlier positions whose scale may only grow, follows from the positions. It runs before the step's attention,
with the lengths that count the new tokens.

Everything is enqueued on the current torch stream of the tensors' device; no call synchronises the host except the
KVQ_DEBUG=1 input check, so fixed-shape calls can be captured in a HIP graph.
"""
import os
from typing import NamedTuple

import torch

from . import _native
from . import cuda_kernels as ck
from .cuda_kernels import _check, _check_cuda

GROUPS = (16, 32, 64, 128)     # positions per scale


def block_scales(num_blocks, block_size, num_kv_heads, group=16, device="cuda"):
    """{"k_scale", "v_scale"}: zeroed scales of a cache, float32 [num_blocks, kv heads, block_size // group] views of one
    buffer that holds each block's two scales side by side (one 8-byte read in the attention)."""
    _check_group(group, block_size)
    both = torch.zeros(num_blocks, num_kv_heads, block_size // group, 2, dtype=torch.float32, device=device)
    return {"k_scale": both[..., 0], "v_scale": both[..., 1]}


def _check_group(group, block_size):
    _check(group in GROUPS and block_size % group == 0,
           f"block-scaled cache: positions per scale must be one of {GROUPS} and divide the block size, got {group} "
           f"for blocks of {block_size}")


def _cache_args(name, kc, vc, scales):
    """The checked C arguments of a cache's geometry and scales: (K view, V view, [blocks, block size, H, D], scales)."""
    ks, vs = scales["k_scale"], scales["v_scale"]
    _check(kc.dim() == 4 and vc.shape == kc.shape and kc.dtype == torch.int8 and vc.dtype == torch.int8 and
           kc.stride(3) == 1 and vc.stride(3) == 1,
           f"{name}: caches must be int8 [num_blocks, block_size, kv_heads, D] views")
    nb, bs, h, d = kc.shape
    _check(bs >= 16 and (bs & (bs - 1)) == 0, f"{name}: block_size must be a power of two >= 16")
    _check(ks.dtype == torch.float32 and vs.dtype == torch.float32 and ks.dim() == 3 and ks.shape == vs.shape and
           ks.stride() == vs.stride() and ks.shape[0] == nb and ks.shape[1] == h and ks.shape[2] >= 1,
           f"{name}: scales must be float32 [num_blocks, kv_heads, blocks per page] of one layout, got {tuple(ks.shape)} "
           f"and {tuple(vs.shape)} for {nb} blocks of {h} kv heads")
    _check(bs % ks.shape[2] == 0, f"{name}: {ks.shape[2]} scales do not divide a page of {bs} positions")
    group = bs // ks.shape[2]
    _check_group(group, bs)
    return ((kc.data_ptr(), *kc.stride()[:3]), (vc.data_ptr(), *vc.stride()[:3]), (nb, bs, h, d),
            (ks.data_ptr(), vs.data_ptr(), *ks.stride(), group))


def _check_index(name, num_seqs, block_table, **vectors):
    for nm, t in vectors.items():
        _check(t.dtype == torch.int32 and t.dim() == 1 and t.is_contiguous(),
               f"{name}: {nm} must be a contiguous int32 vector")
        _check(t.shape[0] >= num_seqs, f"{name}: {nm} has fewer entries than requests")
    _check(block_table.dtype == torch.int32 and block_table.dim() == 2 and block_table.stride(1) == 1 and
           block_table.shape[0] >= num_seqs, f"{name}: block_table must be int32 [num_seqs, pages] with a contiguous last dim")


def _call(name, device, *args):
    """The C entry point on the current stream of `device` (the library sizes its grids for the current device)."""
    if device.index == torch.cuda.current_device():
        _native.call(name, *args, torch.cuda.current_stream(device).cuda_stream)
    else:
        with torch.cuda.device(device):
            _native.call(name, *args, torch.cuda.current_stream(device).cuda_stream)


def quant_block_cache(key, value, key_cache, value_cache, scales, cu_seqlens_q, seq_lens, block_table):
    """Quantize a step's new K / V rows (bf16 [T, kv heads, D]) into the cache, making the scales of the blocks they
    fall in. Request r's rows cu_seqlens_q[r] .. are its last positions, up to seq_lens[r] - 1 (seq_lens count the new
    tokens), in the pages of block_table[r]; rows past cu_seqlens_q[-1] are padding.

    A block that the step begins gets the scale max|x| / 127 of its new values; one that holds earlier positions of the
    request keeps its scale if that is larger, else takes the new one and its earlier codes are requantized to it. Scales
    never shrink while a block is being filled (positions written again after a rollback, too); they start anew when the
    block's first position is written. Infinities saturate and do not count for the scale. The pages written must belong
    to one request each."""
    name = "quant_block_cache"
    if ck._served(ck.ext(), name, key, value, key_cache, value_cache, scales["k_scale"], scales["v_scale"], cu_seqlens_q,
                  seq_lens, block_table):
        return
    n, num_seqs = key.shape[0], cu_seqlens_q.shape[0] - 1
    _check(key.dim() == 3 and key.shape == value.shape and key.stride(2) == 1 and value.stride(2) == 1 and
           key.dtype == torch.bfloat16 and value.dtype == torch.bfloat16,
           f"{name}: key / value must be bf16 [T, kv_heads, D] with a contiguous last dim")
    k, v, geom, sc = _cache_args(name, key_cache, value_cache, scales)
    _check(key.shape[1:] == key_cache.shape[2:], f"{name}: cache shapes disagree with key")
    _check_index(name, num_seqs, block_table, cu_seqlens_q=cu_seqlens_q, seq_lens=seq_lens)
    if n == 0 or num_seqs <= 0:
        return
    _check_cuda(name, key, value, key_cache, value_cache, scales["k_scale"], scales["v_scale"], cu_seqlens_q, seq_lens,
                block_table)
    _call("kvq_quant_block_cache", key.device, key.data_ptr(), key.stride(0), key.stride(1), value.data_ptr(),
          value.stride(0), value.stride(1), n, *k, *v, *geom, *sc, cu_seqlens_q.data_ptr(), seq_lens.data_ptr(),
          block_table.data_ptr(), block_table.stride(0), num_seqs)


def read_block_cache(key_cache, value_cache, scales, starts, cu_seqlens_k, block_table, key_out, value_out):
    """Read keys back: positions starts[r] .. of request r become rows cu_seqlens_k[r] .. cu_seqlens_k[r + 1] - 1 of
    key_out / value_out (bf16 [N, kv heads, D], N at least cu_seqlens_k[-1]; rows behind are left as they were).
    Returns (key_out, value_out)."""
    name = "read_block_cache"
    if ck._served(ck.ext(), name, key_cache, value_cache, scales["k_scale"], scales["v_scale"], starts, cu_seqlens_k,
                  block_table, key_out, value_out):
        return key_out, value_out
    num_seqs = cu_seqlens_k.shape[0] - 1
    k, v, geom, sc = _cache_args(name, key_cache, value_cache, scales)
    for t in (key_out, value_out):
        _check(t.dim() == 3 and t.dtype == torch.bfloat16 and t.stride(2) == 1 and t.shape[1:] == key_cache.shape[2:] and
               t.shape[0] == key_out.shape[0], f"{name}: outputs must be bf16 [rows, kv_heads, D] with a contiguous last dim")
    _check_index(name, num_seqs, block_table, cu_seqlens_k=cu_seqlens_k, starts=starts)
    if key_out.shape[0] == 0 or num_seqs <= 0:
        return key_out, value_out
    _check_cuda(name, key_cache, value_cache, scales["k_scale"], scales["v_scale"], starts, cu_seqlens_k, block_table, key_out,
                value_out)
    _call("kvq_read_block_cache", key_cache.device, *k, *v, *geom, *sc, starts.data_ptr(), cu_seqlens_k.data_ptr(),
          block_table.data_ptr(), block_table.stride(0), num_seqs, key_out.data_ptr(), key_out.stride(0), key_out.stride(1),
          value_out.data_ptr(), value_out.stride(0), value_out.stride(1), key_out.shape[0])
    return key_out, value_out


def _check_attention(name, q, kc, out, cu_seqlens_q, seq_lens, block_table):
    _check(q.dim() == 3 and q.dtype == torch.bfloat16 and out.dtype == torch.bfloat16 and q.stride(2) == 1 and
           out.dim() == 3 and out.stride(2) == 1 and out.shape[1:] == q.shape[1:] and out.shape[0] >= q.shape[0] and
           q.shape[2] == kc.shape[3], f"{name}: q / out must be bf16 [T, q_heads, D] with a contiguous last dim")
    _check(kc.shape[2] > 0 and q.shape[1] % kc.shape[2] == 0,
           f"{name}: {q.shape[1]} q heads not a multiple of {kc.shape[2]} kv heads")
    _check_index(name, cu_seqlens_q.shape[0] - 1, block_table, cu_seqlens_q=cu_seqlens_q, seq_lens=seq_lens)


def block_decode_attention(q, k_cache, v_cache, out, cu_seqlens_q, seq_lens, block_table, softmax_scale, scales, segm=None,
                           max_query_len=1):
    """Attention over a block-scaled cache for the requests with at most SHORT_Q query tokens (others are skipped), with
    decode_attention's arguments: out rows softmax(q k^T softmax_scale) v, bottom-right causal, of the cached values and
    the bf16 q. Rounded: each channel of q to a multiple of its row's largest / 16,256; the weights to 2^-14 of each for up to
    16 (token, q head) rows per kv head (32 where the call is not cut), to bf16 (2^-8) for more. A row that sees no key is
    zero, another with a NaN or an infinity in q NaN. segm: split buffers (cuda_kernels.split_buffers), which allow a
    (request, kv head) to be cut into pieces."""
    name = "block_decode_attention"
    so, sm, ss = segm if segm is not None else (None, None, None)
    if ck._served(ck.ext(), name, q, k_cache, v_cache, out, cu_seqlens_q, seq_lens, block_table, scales["k_scale"],
                  scales["v_scale"], softmax_scale, so, sm, ss, max_query_len, ck.SHORT_Q, ck.MAX_SPLITS):
        return out
    num_seqs = cu_seqlens_q.shape[0] - 1
    k, v, geom, sc = _cache_args(name, k_cache, v_cache, scales)
    _check_attention(name, q, k_cache, out, cu_seqlens_q, seq_lens, block_table)
    hq, d = q.shape[1:]
    split = (None, None, None, 0, 0, 1, 0)
    if sm is not None:
        S = sm.shape[2]
        _check(S <= ck.MAX_SPLITS, f"at most {ck.MAX_SPLITS} split-KV segments")
        for t in (so, sm, ss):
            _check(t is not None and t.dtype == torch.float32 and tuple(t.shape[:3]) == (sm.shape[0], hq, S),
                   f"{name}: split buffers must be float32 [rows, Hq, S(, D)]")
        _check(sm.stride(2) == 1 and ss.stride() == sm.stride() and so.shape[3] == d and so.stride(3) == 1 and
               so.stride(2) == d and so.stride(1) == sm.stride(1) * d and so.stride(0) == sm.stride(0) * d,
               f"{name}: segm_out must be laid out as segm_max x head_dim, segm_sum as segm_max")
        split = (so.data_ptr(), sm.data_ptr(), ss.data_ptr(), sm.stride(0), sm.stride(1), S, sm.shape[0])
    if q.shape[0] == 0 or num_seqs <= 0:
        return out
    _check_cuda(name, q, k_cache, v_cache, out, cu_seqlens_q, seq_lens, block_table, scales["k_scale"], scales["v_scale"],
                so, sm, ss)
    _call("kvq_block_decode_attention", q.device, q.data_ptr(), q.stride(0), q.stride(1), *k, *v, *geom, *sc,
          out.data_ptr(), out.stride(0), out.stride(1), cu_seqlens_q.data_ptr(), seq_lens.data_ptr(),
          block_table.data_ptr(), block_table.stride(0), num_seqs, hq, float(softmax_scale), *split, ck._target_waves(),
          int(max_query_len), ck.SHORT_Q)
    return out


class _DirectCost(NamedTuple):
    """us by which reading the int8 pages in the kernel differs from copying their codes first, at one head_dim: a
    least-squares fit of 240 drawn steps timed in graphs both ways."""
    alone: float    # more per key tile of the longest workgroup, at most one workgroup a CU
    shared: float   # the same with more
    launch: float   # the copy's launch, and its time per million K elements (with their V)
    pages: float


_DIRECT = {128: _DirectCost(0.034, 0.172, 1.55, 0.90), 64: _DirectCost(0.130, 0.143, 2.17, 1.42)}


def direct_pays(longest, workgroups, d, fill, elems):
    """Whether the prefill of a block-scaled cache reads the int8 pages itself (block_prefill_kernel) instead of a copy of
    `elems` K (and as many V) codes as bf16. Over the 240 fitted steps the source taken is within 1.1 of the faster and
    0.2% off on average, over 240 others within 1.08 and 0.3%. Graph, us, copied and direct: 16 tokens of 16,384 keys (28 / 4 heads) 38.9 and 28.4, 776 of 1,390
    (32 / 8) 51.4 and 46.4; 1,302 of 1,490 with 274 of 5,979 (28 / 4) 81 and 93, 512 of 8,192 93 and 103."""
    c = _DIRECT.get(d, _DIRECT[128])
    return (c.shared if workgroups > fill else c.alone) * longest < c.launch + c.pages * elems / 1e6


def block_long_attention(q, k_cache, v_cache, out, cu_seqlens_q, seq_lens, block_table, plan, softmax_scale, scales):
    """Attention over a block-scaled cache for the plan's long requests (cuda_kernels.plan_long; the others' rows are left
    as they were): the formula of block_decode_attention, the codes exact, their scales applied in fp32, the softmax's
    weights rounded to bf16 (and q as there, where the int8 pages are read). KVQ_PREFILL_DIRECT as long_attention's: 1 (or fold) reads the int8 pages
    themselves, 0 a temporary bf16 cache of the plan's pages' codes; unset: whichever is faster (direct_pays)."""
    name, e = "block_long_attention", ck.ext()
    bs, h, d = k_cache.shape[1:]
    _check(bs == plan.block_size, f"block size {bs} != plan block size {plan.block_size}")
    work = plan.work(q.shape[1] // h, h, d, q.device)
    direct = os.environ.get("KVQ_PREFILL_DIRECT")
    _check(direct in (None, "0", "1", "fold"), f"KVQ_PREFILL_DIRECT must be 0, 1 or fold, got {direct!r}")
    if direct is None:
        if work.direct_block is None:
            work.direct_block = direct_pays(work.longest, work.tile_req.shape[0] * h, d, ck.one_pass_fill(q.device),
                                            plan.src_req.shape[0] * bs * h * d)
        # (a capture that finds the pages' lists missing reads the pages themselves: nothing can be copied inside it)
        direct = "1" if work.direct_block or (plan._gpu is None and ck._capturing(q.device)) else "0"
    src = plan.gpu(q.device) if direct == "0" else (None, None, None)
    if ck._served(e, name, q, k_cache, v_cache, out, cu_seqlens_q, seq_lens, block_table, scales["k_scale"],
                  scales["v_scale"], softmax_scale, e.prefill_rows, work.tile_req, work.tile_row, work.tile_piece,
                  work.tile_slot, work.merge, work.slots, *src):
        return out
    k, v, geom, sc = _cache_args(name, k_cache, v_cache, scales)
    _check_attention(name, q, k_cache, out, cu_seqlens_q, seq_lens, block_table)
    _check_cuda(name, q, k_cache, v_cache, out, cu_seqlens_q, seq_lens, block_table, scales["k_scale"], scales["v_scale"])
    n = work.tile_req.shape[0]
    split = work.split(h, e.prefill_rows, d)
    codes = (None, None, None, 0, None, 0)
    if src[0] is not None:
        src_req, src_j, bt_tmp = src
        kt = torch.empty((src_req.shape[0], bs, h, d), dtype=q.dtype, device=q.device)
        vt = torch.empty_like(kt)
        st = torch.empty((h, kt.shape[0] * (bs // 16), 4), dtype=torch.float32, device=q.device)
        _call("kvq_block_codes", q.device, *k, *v, *geom, *sc, kt.data_ptr(), vt.data_ptr(), st.data_ptr(),
              block_table.data_ptr(), block_table.stride(0), src_req.data_ptr(), src_j.data_ptr(), src_req.shape[0])
        codes = (kt.data_ptr(), vt.data_ptr(), st.data_ptr(), kt.shape[0], bt_tmp.data_ptr(), bt_tmp.stride(0))
    _call("kvq_block_prefill_attention", q.device, q.data_ptr(), q.stride(0), q.stride(1), *k, *v, *geom, *sc,
          out.data_ptr(), out.stride(0), out.stride(1), cu_seqlens_q.data_ptr(), seq_lens.data_ptr(),
          block_table.data_ptr(), block_table.stride(0), q.shape[1], work.tile_req.data_ptr(), work.tile_row.data_ptr(),
          n, e.prefill_rows, float(softmax_scale),
          *((None, None, None, 0, None, None) if split is None else e._split_args(split, n, h, d)), *codes)
    return out


def check_scales(k_cache, cu_seqlens_q, seq_lens, block_table, scales):
    """KVQ_DEBUG=1: every scale that a batch's keys use is finite and not negative (syncs the GPU; skipped while a graph is
    being captured)."""
    if k_cache.is_cuda and torch.cuda.is_current_stream_capturing():
        return
    bs, blocks = k_cache.shape[1], scales["k_scale"].shape[2]
    bt, errs = block_table.cpu().long(), []
    for r, n in enumerate(seq_lens.cpu().tolist()[:cu_seqlens_q.shape[0] - 1]):
        used = -(-n * blocks // bs)
        ids = bt[r, :-(-n // bs)].clamp(0, k_cache.shape[0] - 1)
        for nm in ("k_scale", "v_scale"):
            s = scales[nm][ids.to(k_cache.device)].transpose(1, 2).reshape(-1, k_cache.shape[2])[:used]
            if not bool((torch.isfinite(s) & (s >= 0)).all()):
                errs.append(f"req {r}: {nm} not finite or negative")
    if errs:
        raise RuntimeError("kvq scale check: " + "; ".join(errs[:8]))


def block_paged_attention(q, k_cache, v_cache, out, cu_seqlens_q, seq_lens, block_table, max_query_len, softmax_scale, scales,
                          plan=None, segm=None):
    """Attention of one batch over a block-scaled cache, with paged_attention's arguments (plan from plan_long, None if
    all requests are short)."""
    if os.environ.get("KVQ_DEBUG") == "1":
        ck.check_inputs(q, k_cache, cu_seqlens_q, seq_lens, block_table, plan)
        check_scales(k_cache, cu_seqlens_q, seq_lens, block_table, scales)
    if plan is not None:
        block_long_attention(q, k_cache, v_cache, out, cu_seqlens_q, seq_lens, block_table, plan, softmax_scale, scales)
    if plan is None or plan.has_short:
        if plan is not None and plan.short_qlen:
            max_query_len = min(max_query_len, plan.short_qlen)   # the short requests' own longest picks the kernel
        block_decode_attention(q, k_cache, v_cache, out, cu_seqlens_q, seq_lens, block_table, softmax_scale, scales, segm,
                               max_query_len)
    return out
