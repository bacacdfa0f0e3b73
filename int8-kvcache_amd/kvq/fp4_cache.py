"""Operators of the 4-bit cache: a KV cache of e2m1 codes with one exponent byte for each 32 channels of a row, beside the
INT8 caches of kvq.cuda_kernels and kvq.block_cache, and the eviction of keys that little attention goes to (no
counterpart in the reference).

A cached value is one of 0, 1/2, 1, 3/2, 2, 3, 4, 6 or their negatives times a power of two; head_dim 128 takes 136 bytes for a
key's K and V (256 in int8, 512 in bf16). Pages, block tables, lengths, slot
mappings, split buffers and the plan of long requests are those of kvq.cuda_kernels:

    kc, vc                              uint8 [num_blocks, block_size, kv heads, D / 2] views, strides multiples of 16
    scales = fp4_scales(num_blocks, block_size, kv_heads, head_dim, device)
    quant_fp4_cache(key, value, kc, vc, scales, slot_mapping)                               a step's new tokens
    fp4_paged_attention(q, kc, vc, out, cu_seqlens_q, seq_lens, block_table, max_query_len, softmax_scale, scales, plan,
                        segm, lse)                                                          the step's attention
    read_fp4_cache(kc, vc, scales, starts, cu_seqlens_k, block_table, k_out, v_out)         keys back as bf16 rows

A row's scales are its own, so rows may be written in any order and moved. Eviction keeps a cache within a budget of keys
per request:

    add_key_weights(q, kc, scales, lse, weights, cu_seqlens_q, seq_lens, block_table, softmax_scale, max_query_len)
    evict_keys(kc, vc, scales, weights, seq_lens, keep, recent, block_table, kept, new_lens)

Everything is enqueued on the current torch stream of the tensors' device; no call synchronises the host except the
KVQ_DEBUG=1 input check, so fixed-shape calls can be captured in a HIP graph.
"""
import os

import torch

from . import cuda_kernels as ck
from .block_cache import _call, _check_index
from .cuda_kernels import _check, _check_cuda

GROUP = 32     # channels per exponent byte


def fp4_scales(num_blocks, block_size, num_kv_heads, head_dim, device="cuda"):
    """{"k_scale", "v_scale"}: zeroed exponent bytes of a cache, uint8 [num_blocks, kv heads, block_size, head_dim // 32] views
    of one buffer that holds K's and V's of a page and head side by side."""
    both = torch.zeros(num_blocks, num_kv_heads, 2, block_size, head_dim // GROUP, dtype=torch.uint8, device=device)
    return {"k_scale": both[:, :, 0], "v_scale": both[:, :, 1]}


def _cache_args(name, kc, vc, scales):
    """The checked C arguments of a cache's geometry and scales: (K view, V view, [blocks, block size, H, D], scales)."""
    ks, vs = scales["k_scale"], scales["v_scale"]
    _check(kc.dim() == 4 and vc.shape == kc.shape and kc.dtype == torch.uint8 and vc.dtype == torch.uint8 and
           kc.stride(3) == 1 and vc.stride(3) == 1,
           f"{name}: caches must be uint8 [num_blocks, block_size, kv_heads, D / 2] views")
    nb, bs, h, d = *kc.shape[:3], 2 * kc.shape[3]
    _check(bs >= 16 and (bs & (bs - 1)) == 0, f"{name}: block_size must be a power of two >= 16")
    for s in (ks, vs):
        _check(s.dtype == torch.uint8 and tuple(s.shape) == (nb, h, bs, d // GROUP) and s.stride(3) == 1 and
               s.stride(2) == d // GROUP and s.stride() == ks.stride(),
               f"{name}: scales must be uint8 {(nb, h, bs, d // GROUP)} of one layout with contiguous pages of a head, got "
               f"{tuple(ks.shape)} and {tuple(vs.shape)}")
    return ((kc.data_ptr(), *kc.stride()[:3]), (vc.data_ptr(), *vc.stride()[:3]), (nb, bs, h, d),
            (ks.data_ptr(), vs.data_ptr(), *ks.stride()[:2]))


def quant_fp4_cache(key, value, key_cache, value_cache, scales, slot_mapping):
    """Quantize a step's new K / V rows (bf16 [T, kv heads, D]) into the slots of slot_mapping (int64 [n], n at most T; rows
    behind are padding, and so is a slot that the cache does not have, -1 for one). A group of 32 channels takes the exponent
    that brings its largest |x| into (3.5, 7], and the nearest codes (ties to even) at it: 6 for what is above it, infinities
    too, 0 for NaN. A slot may occur once in a call."""
    name = "quant_fp4_cache"
    if ck._served(ck.ext(), name, key, value, key_cache, value_cache, scales["k_scale"], scales["v_scale"], slot_mapping):
        return
    _check(key.dim() == 3 and key.shape == value.shape and key.stride(2) == 1 and value.stride(2) == 1 and
           key.dtype == torch.bfloat16 and value.dtype == torch.bfloat16,
           f"{name}: key / value must be bf16 [T, kv_heads, D] with a contiguous last dim")
    k, v, geom, sc = _cache_args(name, key_cache, value_cache, scales)
    _check(tuple(key.shape[1:]) == geom[2:], f"{name}: cache shapes disagree with key")
    _check(slot_mapping.dtype == torch.int64 and slot_mapping.dim() == 1 and slot_mapping.is_contiguous(),
           f"{name}: slot_mapping must be a contiguous int64 vector")
    n = slot_mapping.shape[0]
    _check(key.shape[0] >= n, f"{name}: {n} slots for {key.shape[0]} rows")
    if n == 0:
        return
    _check_cuda(name, key, value, key_cache, value_cache, scales["k_scale"], scales["v_scale"], slot_mapping)
    _call("kvq_quant_fp4_cache", key.device, key.data_ptr(), key.stride(0), key.stride(1), value.data_ptr(), value.stride(0),
          value.stride(1), *k, *v, *geom, *sc, slot_mapping.data_ptr(), n)


def read_fp4_cache(key_cache, value_cache, scales, starts, cu_seqlens_k, block_table, key_out, value_out):
    """Read keys back, exactly: positions starts[r] .. of request r become rows cu_seqlens_k[r] .. cu_seqlens_k[r + 1] - 1 of
    key_out / value_out (bf16 [N, kv heads, D], N at least cu_seqlens_k[-1]; rows behind are left as they were).
    Returns (key_out, value_out)."""
    name = "read_fp4_cache"
    if ck._served(ck.ext(), name, key_cache, value_cache, scales["k_scale"], scales["v_scale"], starts, cu_seqlens_k,
                  block_table, key_out, value_out):
        return key_out, value_out
    num_seqs = cu_seqlens_k.shape[0] - 1
    k, v, geom, sc = _cache_args(name, key_cache, value_cache, scales)
    for t in (key_out, value_out):
        _check(t.dim() == 3 and t.dtype == torch.bfloat16 and t.stride(2) == 1 and tuple(t.shape[1:]) == geom[2:] and
               t.shape[0] == key_out.shape[0], f"{name}: outputs must be bf16 [rows, kv_heads, D] with a contiguous last dim")
    _check_index(name, num_seqs, block_table, cu_seqlens_k=cu_seqlens_k, starts=starts)
    if key_out.shape[0] == 0 or num_seqs <= 0:
        return key_out, value_out
    _check_cuda(name, key_cache, value_cache, scales["k_scale"], scales["v_scale"], starts, cu_seqlens_k, block_table, key_out,
                value_out)
    _call("kvq_read_fp4_cache", key_cache.device, *k, *v, *geom, *sc, starts.data_ptr(), cu_seqlens_k.data_ptr(),
          block_table.data_ptr(), block_table.stride(0), num_seqs, key_out.data_ptr(), key_out.stride(0), key_out.stride(1),
          value_out.data_ptr(), value_out.stride(0), value_out.stride(1), key_out.shape[0])
    return key_out, value_out


def _check_rows(name, q, geom, cu_seqlens_q, seq_lens, block_table):
    _check(q.dim() == 3 and q.dtype == torch.bfloat16 and q.stride(2) == 1 and q.shape[2] == geom[3],
           f"{name}: q must be bf16 [T, q_heads, {geom[3]}] with a contiguous last dim")
    _check(geom[2] > 0 and q.shape[1] % geom[2] == 0, f"{name}: {q.shape[1]} q heads not a multiple of {geom[2]} kv heads")
    _check_index(name, cu_seqlens_q.shape[0] - 1, block_table, cu_seqlens_q=cu_seqlens_q, seq_lens=seq_lens)


def _check_out(name, q, out):
    _check(out.dim() == 3 and out.dtype == torch.bfloat16 and out.stride(2) == 1 and out.shape[1:] == q.shape[1:] and
           out.shape[0] >= q.shape[0], f"{name}: out must be bf16 [T, q_heads, D] with a contiguous last dim")


def _check_lse(name, q, lse):
    _check(lse.dtype == torch.float32 and lse.dim() == 2 and lse.stride(1) == 1 and lse.shape[0] >= q.shape[0] and
           lse.shape[1] == q.shape[1], f"{name}: lse must be float32 [T, q_heads] with a contiguous last dim")


def fp4_decode_attention(q, k_cache, v_cache, out, cu_seqlens_q, seq_lens, block_table, softmax_scale, scales, segm=None,
                         max_query_len=1, lse=None):
    """Attention over a 4-bit cache for the requests with at most SHORT_Q query tokens (others are skipped), with
    decode_attention's arguments: out rows softmax(q k^T softmax_scale) v, bottom-right causal, of the cached values and the
    bf16 q. Rounded: the weights, to a sum of two bf16 (2^-14 of each). A row that sees no key is zero, another with a
    NaN or an infinity in q NaN. The caches have the same page and slot strides. segm: split buffers
    (cuda_kernels.split_buffers), which allow a (request, kv head) to be cut into pieces. lse (float32 [T, q heads]): filled
    with the rows' natural log-sum-exp, -inf for a row that sees no key."""
    name = "fp4_decode_attention"
    so, sm, ss = segm if segm is not None else (None, None, None)
    if ck._served(ck.ext(), name, q, k_cache, v_cache, out, cu_seqlens_q, seq_lens, block_table, scales["k_scale"],
                  scales["v_scale"], softmax_scale, so, sm, ss, max_query_len, ck.SHORT_Q, ck.MAX_SPLITS, lse):
        return out
    num_seqs = cu_seqlens_q.shape[0] - 1
    k, v, geom, sc = _cache_args(name, k_cache, v_cache, scales)
    _check_rows(name, q, geom, cu_seqlens_q, seq_lens, block_table)
    _check_out(name, q, out)
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
    if lse is not None:
        _check_lse(name, q, lse)
    if q.shape[0] == 0 or num_seqs <= 0:
        return out
    _check_cuda(name, q, k_cache, v_cache, out, cu_seqlens_q, seq_lens, block_table, scales["k_scale"], scales["v_scale"],
                so, sm, ss, lse)
    _call("kvq_fp4_decode_attention", q.device, q.data_ptr(), q.stride(0), q.stride(1), *k, *v, *geom, *sc,
          out.data_ptr(), out.stride(0), out.stride(1), cu_seqlens_q.data_ptr(), seq_lens.data_ptr(),
          block_table.data_ptr(), block_table.stride(0), num_seqs, hq, float(softmax_scale), *split,
          None if lse is None else lse.data_ptr(), 0 if lse is None else lse.stride(0), ck._target_waves(),
          int(max_query_len), ck.SHORT_Q)
    return out


def fp4_long_attention(q, k_cache, v_cache, out, cu_seqlens_q, seq_lens, block_table, plan, softmax_scale, scales):
    """Attention over a 4-bit cache for the plan's long requests (cuda_kernels.plan_long; the others' rows are left as they
    were): fp4_decode_attention's formula and roundings, over a temporary bf16 copy of their pages (exact, 4 bytes per key,
    channel and kv head). Inside a graph capture the plan's lists must be on the GPU already
    (plan.gpu, plan.work: an earlier call with the plan made them)."""
    name, e = "fp4_long_attention", ck.ext()
    bs, h, d = *k_cache.shape[1:3], 2 * k_cache.shape[3]
    _check(bs == plan.block_size, f"block size {bs} != plan block size {plan.block_size}")
    work = plan.work(q.shape[1] // h, h, d, q.device)
    src_req, src_j, bt_tmp = plan.gpu(q.device)
    if ck._served(e, name, q, k_cache, v_cache, out, cu_seqlens_q, seq_lens, block_table, scales["k_scale"],
                  scales["v_scale"], softmax_scale, e.prefill_rows, work.tile_req, work.tile_row, work.tile_piece,
                  work.tile_slot, work.merge, work.slots, src_req, src_j, bt_tmp):
        return out
    k, v, geom, sc = _cache_args(name, k_cache, v_cache, scales)
    _check_rows(name, q, geom, cu_seqlens_q, seq_lens, block_table)
    _check_out(name, q, out)
    _check_cuda(name, q, k_cache, v_cache, out, cu_seqlens_q, seq_lens, block_table, scales["k_scale"], scales["v_scale"])
    pages, n = src_req.shape[0], work.tile_req.shape[0]
    kt = torch.empty((max(pages, 1), bs, h, d), dtype=q.dtype, device=q.device)
    vt = torch.empty_like(kt)
    st = torch.empty((h, kt.shape[0] * (bs // 16), 4), dtype=torch.float32, device=q.device)
    _call("kvq_fp4_pages", q.device, *k, *v, *geom, *sc, kt.data_ptr(), vt.data_ptr(), st.data_ptr(), block_table.data_ptr(),
          block_table.stride(0), src_req.data_ptr(), src_j.data_ptr(), pages)
    split = work.split(h, e.prefill_rows, d)
    _call("kvq_fp4_prefill_attention", q.device, q.data_ptr(), q.stride(0), q.stride(1), kt.data_ptr(), vt.data_ptr(),
          st.data_ptr(), kt.shape[0], bs, h, d, out.data_ptr(), out.stride(0), out.stride(1), cu_seqlens_q.data_ptr(),
          seq_lens.data_ptr(), bt_tmp.data_ptr(), bt_tmp.stride(0), q.shape[1], work.tile_req.data_ptr(),
          work.tile_row.data_ptr(), n, e.prefill_rows, float(softmax_scale),
          *((None, None, None, 0, None, None) if split is None else e._split_args(split, n, h, d)))
    return out


def fp4_paged_attention(q, k_cache, v_cache, out, cu_seqlens_q, seq_lens, block_table, max_query_len, softmax_scale, scales,
                        plan=None, segm=None, lse=None):
    """Attention of one batch over a 4-bit cache, with paged_attention's arguments (plan from plan_long, None if all requests
    are short). lse as fp4_decode_attention's: of the short requests' rows."""
    if os.environ.get("KVQ_DEBUG") == "1":
        ck.check_inputs(q, k_cache, cu_seqlens_q, seq_lens, block_table, plan)
    if plan is not None:
        fp4_long_attention(q, k_cache, v_cache, out, cu_seqlens_q, seq_lens, block_table, plan, softmax_scale, scales)
    if plan is None or plan.has_short:
        if plan is not None and plan.short_qlen:
            max_query_len = min(max_query_len, plan.short_qlen)   # the short requests' own longest picks the kernel
        fp4_decode_attention(q, k_cache, v_cache, out, cu_seqlens_q, seq_lens, block_table, softmax_scale, scales, segm,
                             max_query_len, lse)
    return out


def add_key_weights(q, k_cache, scales, lse, weights, cu_seqlens_q, seq_lens, block_table, softmax_scale, max_query_len=1):
    """Add the attention that each cached key gets of a step's rows to its running sum, weights (float32 [requests, kv heads,
    keys], the last dim contiguous, no rows in common; row r is request r's alone): the softmax's weights, summed over the request's query tokens
    and the kv head's q heads. For the requests with at most SHORT_Q query tokens; keys behind weights' last column are not
    counted. q, lse: fp4_decode_attention's of the same rows (rows whose lse is not finite add nothing). A prompt's keys are
    judged by its last tokens: attend with those rows of q as a short request over all of its keys, then call this with them.
    Returns weights."""
    name = "add_key_weights"
    if ck._served(ck.ext(), name, q, k_cache, scales["k_scale"], lse, weights, cu_seqlens_q, seq_lens, block_table,
                  softmax_scale, max_query_len, ck.SHORT_Q):
        return weights
    num_seqs = cu_seqlens_q.shape[0] - 1
    k, _, geom, sc = _cache_args(name, k_cache, k_cache, scales)
    _check_rows(name, q, geom, cu_seqlens_q, seq_lens, block_table)
    _check_lse(name, q, lse)
    _check_weights(name, weights, num_seqs, geom[2])
    if q.shape[0] == 0 or num_seqs <= 0 or weights.shape[2] == 0:
        return weights
    _check_cuda(name, q, k_cache, scales["k_scale"], lse, weights, cu_seqlens_q, seq_lens, block_table)
    _call("kvq_fp4_key_weights", q.device, q.data_ptr(), q.stride(0), q.stride(1), *k, *geom, sc[0], *sc[2:], lse.data_ptr(),
          lse.stride(0), weights.data_ptr(), weights.stride(0), weights.stride(1), weights.shape[2], cu_seqlens_q.data_ptr(),
          seq_lens.data_ptr(), block_table.data_ptr(), block_table.stride(0), num_seqs, q.shape[1], float(softmax_scale),
          int(max_query_len), ck.SHORT_Q)
    return weights


def _check_weights(name, weights, num_seqs, heads):
    _check(weights.dtype == torch.float32 and weights.dim() == 3 and weights.stride(2) == 1 and
           weights.shape[0] >= num_seqs and weights.shape[1] == heads,
           f"{name}: weights must be float32 [requests, kv_heads, keys] with a contiguous last dim")


def evict_keys(k_cache, v_cache, scales, weights, seq_lens, keep, recent, block_table, kept, new_lens):
    """Shorten the requests with more than keep[r] (int32 [requests]) of their seq_lens[r] keys to that many, in place. Each kv
    head keeps the last `recent` (all of keep[r] if that is less) and, of those before, the ones of the largest weights
    (add_key_weights; ties to the lowest position, a NaN counts as the largest); their rows move to the request's first positions
    in their order, their weights with them, and the weights behind become 0. kept (int32 [requests, kv heads, most that a
    request may keep]): filled with the position that each row held; new_lens (int32 [requests]): min(seq_lens, keep), the
    lengths from now on: the next token's slot is the one behind, while its position for the rotation goes on counting. new_lens
    may be seq_lens (or keep) itself, which is then updated in place, by a launch more; it overlaps them in no other way. keep
    counts as at most kept.shape[2] and as at least 0. A request within its budget is left as it is. The pages of the
    requests must be theirs alone, a prefix that two requests share is not evicted from. A table has at most 2^28 slots.
    Rows of weights, or of kept, have nothing in common (sums that a request's heads share are copied for each head). Returns
    new_lens."""
    name = "evict_keys"
    if ck._served(ck.ext(), name, k_cache, v_cache, scales["k_scale"], scales["v_scale"], weights, seq_lens, keep, recent,
                  block_table, kept, new_lens):
        return new_lens
    num_seqs = seq_lens.shape[0]
    k, v, geom, sc = _cache_args(name, k_cache, v_cache, scales)
    _check_index(name, num_seqs, block_table, seq_lens=seq_lens, keep=keep, new_lens=new_lens)
    _check_weights(name, weights, num_seqs, geom[2])
    _check(kept.dtype == torch.int32 and kept.dim() == 3 and kept.stride(2) == 1 and kept.shape[0] >= num_seqs and
           kept.shape[1] == geom[2], f"{name}: kept must be int32 [requests, kv_heads, keys] with a contiguous last dim")
    _check(int(recent) >= 0, f"{name}: recent must not be negative, got {recent}")
    if num_seqs == 0:
        return new_lens
    _check_cuda(name, k_cache, v_cache, scales["k_scale"], scales["v_scale"], weights, seq_lens, keep, block_table, kept, new_lens)
    _call("kvq_fp4_evict", k_cache.device, *k, *v, *geom, *sc, weights.data_ptr(), weights.stride(0), weights.stride(1),
          weights.shape[2], seq_lens.data_ptr(), keep.data_ptr(), int(recent), block_table.data_ptr(), block_table.stride(0),
          block_table.shape[1], num_seqs, kept.data_ptr(), kept.stride(0), kept.stride(1), kept.shape[2], new_lens.data_ptr())
    return new_lens
