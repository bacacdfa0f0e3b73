"""The operators around a KV cache held in 4 bits (kvq.fp4_cache, kvq.rope) and their plain forms: what their speed and
outputs are measured on. One layer's share of serving steps, from the projected q and k to the attention, and the
eviction of keys that little attention goes to. A cached value is an e2m1 code times a power of two, one exponent byte
for each 32 channels of a row, K and V apart.

Kinds:
  norm    RMS norm of each head's query and key rows and their rotation by position
  write   quantize a step's new K / V rows into the paged cache by slot, then read the step's rows back
  short   attention of decode (1 query token) and verification (2..8 tokens) requests, with the rows' log-sum-exp
  step    one attention call of a step with long-query requests (prefill, chunked prefill) beside decode requests
  weigh   add the attention weight that each cached key gets from a step's query rows to its running sum
  evict   keep each request's and kv head's latest keys and those of the largest sums, moved to the front of the
          request's pages, then read the kept rows back

Request lengths follow from the case alone (`lens_seed`), tensors from the seed. Caches hold model-like K (log-normal
channel gains and a mean) and normal V, in shuffled pages, laid out as vLLM lays them out ([num_blocks, H, block, D]
bytes, K and V interleaved) or as two [num_blocks, block, H, D / 2] arrays; scales beside them, K's and V's of a page
and head side by side.
"""
import math
import os
import random
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "int8-kvcache_amd"))

own = False     # the plain forms; True: kvq.fp4_cache, kvq.rope

DEV = "cuda"
CHUNK = 1 << 25     # elements drawn at a time
FAR = 1 << 17       # mixes a case's seeds apart
SHORT = 8           # requests with at most this many query tokens are short
PIECES = 16         # pieces of the split buffers a serving program keeps
GROUP = 32          # channels per exponent byte
EPS = 1e-6
POSITIONS = 40960   # rows of the rotation's table


def _case(name, kind, **kw):
    c = dict(name=name, kind=kind, hq=28, hkv=4, d=128, block=16, vllm=True,
             requests=0, query=1, lo=1, hi=1, lens_seed=1,      # requests of `query` tokens, keys log-uniform in [lo, hi]
             empty=0,                                           # that many of them hold no keys at all (padded rows)
             chunks="",                                         # long requests: "query:keys query:keys ..."
             tokens=0, rotary=0, interleaved=False, bf16_table=False,
             keep=0, recent=0)
    c.update(kw)
    return c


def listed():
    return [
        # queries and keys of a decode step, 32 requests' one token each: launch latency
        _case("norm_step_32", "norm", tokens=32, rotary=128),
        # those of a prefill step of 16,384 tokens: bound by memory bandwidth
        _case("norm_prefill_16384", "norm", hq=32, hkv=8, tokens=16384, rotary=128),
        # the cache write of a decode step: 32 requests' one new token each
        _case("write_step_32", "write", requests=32, lo=20, hi=4000),
        # the cache write of a prefill step: four prompts of 4,096 tokens
        _case("write_prefill_16384", "write", chunks="4096:4096 4096:4096 4096:4096 4096:4096"),
        # one user's decode at a moderate context: the smallest attention call
        _case("decode_1x4096", "short", requests=1, lo=4096, hi=4096),
        # 128 requests of 32k keys, bound by memory bandwidth
        _case("decode_128x32768", "short", requests=128, lo=32768, hi=32768),
        # speculative decoding: 64 requests of unequal contexts verify 8 tokens each (56 query rows per kv head)
        _case("verify_64x8", "short", requests=64, query=8, lo=512, hi=8192, lens_seed=7),
        # a mixed step: two prompts being read (one from its start, one mid-way) beside 48 decoding requests
        _case("mixed_48_decode_2_prompts", "step", hq=32, hkv=8, requests=48, lo=16, hi=8192, lens_seed=3,
              block=32, chunks="700:700 333:2500"),
        # the weights of one decode step of a small ragged batch, padded with rows that hold no keys
        _case("weigh_24_ragged", "weigh", requests=24, lo=1, hi=4000, lens_seed=5, empty=2),
        # a prompt's last 8 tokens decide about its keys (an observation window), 16 requests of 16k keys
        _case("weigh_16x8_of_16384", "weigh", hq=32, hkv=8, query=8, requests=16, lo=16384, hi=16384, block=32),
        # one user's context cut from 4,096 keys to 1,024, the latest 128 among them
        _case("evict_1x4096", "evict", requests=1, lo=4096, hi=4096, keep=1024, recent=128),
        # a batch's contexts cut to 2,048 keys each: some are shorter and stay as they are
        _case("evict_64_to_2048", "evict", hq=32, hkv=8, requests=64, lo=1024, hi=32768, lens_seed=11, keep=2048, recent=256),
    ]


HEADS = [(28, 4, 128), (32, 8, 128), (14, 2, 64), (12, 2, 128), (16, 16, 64), (32, 1, 128)]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    hq, hkv, d = rng.choice(HEADS)
    block = rng.choice([16, 16, 32, 64])
    base = dict(hq=hq, hkv=hkv, d=d, block=block, vllm=rng.random() < 0.7, lens_seed=rng.randrange(1000))
    kind = rng.choice(["norm", "norm", "write", "short", "short", "short", "step", "weigh", "weigh", "evict", "evict"])
    if kind == "norm":
        c = _case("", kind, tokens=_log(rng, 1, 16384), rotary=rng.choice([d, d, d // 2, 32]),
                  interleaved=rng.random() < 0.3, bf16_table=rng.random() < 0.3, **base)
    elif kind == "write":
        chunks, left = [], _log(rng, 1, 16384)
        for _ in range(rng.choice([0, 1, 1, 3])):
            q = min(left, _log(rng, 9, 8192))
            left -= q
            if q > 0:
                chunks.append("%d:%d" % (q, q + rng.choice([0, _log(rng, 1, 4000)])))
        query = rng.choice([1, 1, 4])
        c = _case("", kind, query=query, requests=_log(rng, 1, 128), lo=query, hi=4000, chunks=" ".join(chunks), **base)
    elif kind in ("short", "weigh"):
        query = rng.choice([1, 1, 1, 2, 3, 5, 8])
        requests = _log(rng, 1, 128)
        most = 2 ** 21 if kind == "short" else 2 ** 18
        hi = max(64, min(32768, int(most / requests), int(most / (requests * hkv / 4))))
        lo = rng.choice([1, max(1, hi // 16), hi])
        c = _case("", kind, query=query, requests=requests, lo=max(lo, query), hi=max(hi, query),
                  empty=rng.choice([0, 0, requests // 8]), **base)
    elif kind == "evict":
        requests = _log(rng, 1, 64)
        hi = max(64, min(32768, (1 << 19) // requests * 4 // hkv))
        keep = _log(rng, 16, max(17, hi // 2))
        c = _case("", kind, requests=requests, lo=rng.choice([1, max(1, hi // 16), hi]), hi=hi, keep=keep,
                  recent=rng.choice([0, 1, keep // 8, keep]), empty=rng.choice([0, 0, requests // 8]), **base)
    else:
        chunks = []
        for _ in range(rng.choice([1, 1, 2])):
            q = _log(rng, 9, 2048)
            chunks.append("%d:%d" % (q, q + rng.choice([0, _log(rng, 1, 8192)])))
        c = _case("", kind, requests=rng.choice([0, _log(rng, 1, 64)]), lo=1, hi=8192, chunks=" ".join(chunks), **base)
    del c["name"]
    return c


# ------------------------------------------------------------------------------------------------ shapes
def _lens(c):
    """(query lengths, key counts) of the requests, short-query ones first."""
    r = random.Random(c["lens_seed"])
    keys = [min(c["hi"], max(c["lo"], _log(r, c["lo"], c["hi"]))) for _ in range(c["requests"])]
    for i in range(c["empty"]):
        keys[(7 * i + 3) % len(keys)] = 0
    q = [c["query"]] * c["requests"]
    for part in c["chunks"].split():
        a, b = part.split(":")
        q.append(int(a))
        keys.append(int(b))
    return q, keys


def _gen(seed, what):
    return torch.Generator(device=DEV).manual_seed(int(seed) * FAR + what)


def _views(c, kv):
    """K and V as the operators take them, bytes [num_blocks, block, H, D / 2]."""
    if c["vllm"]:
        by_slot = kv.permute(0, 2, 1, 3)
        return by_slot[..., :c["d"] // 2], by_slot[..., c["d"] // 2:]
    return kv[0], kv[1]


def _channels(c, seed):
    g = _gen(seed, 1)
    return (torch.exp(0.5 * torch.randn(c["hkv"], c["d"], generator=g, device=DEV)),
            0.5 * torch.randn(c["hkv"], c["d"], generator=g, device=DEV))


def _quantize(x):
    """(bytes [..., D / 2], exponent bytes [..., D / 32]) of fp32 rows [..., D]. A group's exponent brings its largest
    |x| into (3.5, 7]; codes are its values' nearest of 0, 1/2, 1, 3/2, 2, 3, 4, 6 (ties to the even code), at most 6."""
    g = x.unflatten(-1, (-1, GROUP))
    top = g.abs().amax(-1).view(torch.int32)
    e = (((top + 0x1fffff) >> 23) - 2).clamp_(27, 252)
    y = g * torch.exp2((127 - e).float())[..., None]
    a = y.abs()
    code = torch.zeros_like(a, dtype=torch.uint8)
    for edge, up in ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        code += (a >= edge) if up else (a > edge)
    code += torch.signbit(y).to(torch.uint8) << 3
    code = code.flatten(-2)
    return code[..., 0::2] | code[..., 1::2] << 4, e.to(torch.uint8)


def _cache(c, blocks, seed):
    """Every slot filled with a token's K and V, quantized."""
    hkv, d, bs = c["hkv"], c["d"], c["block"]
    kv = torch.empty((blocks, hkv, bs, d) if c["vllm"] else (2, blocks, bs, hkv, d // 2), dtype=torch.uint8, device=DEV)
    caches = _views(c, kv)
    scales = torch.empty(blocks, hkv, 2, bs, d // GROUP, dtype=torch.uint8, device=DEV)
    gain, mean = _channels(c, seed)
    g = _gen(seed, 7)
    step = max(1, CHUNK // (bs * hkv * d))
    for at in range(0, blocks, step):
        n = min(step, blocks - at)
        for side in (0, 1):
            x = torch.randn(n, bs, hkv, d, generator=g, device=DEV)
            if side == 0:
                x = x * gain + mean
            code, e = _quantize(x)
            caches[side][at:at + n] = code
            scales[at:at + n, :, side] = e.transpose(1, 2)
    return kv, caches[0], caches[1], {"k_scale": scales[:, :, 0], "v_scale": scales[:, :, 1]}


def _table(c, keys, seed):
    """Block table [requests, pages] with shuffled pages, and the pages of the cache."""
    pages = [-(-k // c["block"]) for k in keys]
    blocks = sum(pages) + 8
    perm = torch.randperm(blocks, generator=_gen(seed, 2), device=DEV).to(torch.int32)
    rows = np.zeros((len(keys), max(max(pages), 1)), dtype=np.int64)
    at = 0
    for i, p in enumerate(pages):
        rows[i, :p] = np.arange(at, at + p)
        at += p
    return perm[torch.from_numpy(rows).to(DEV)].contiguous(), blocks


def _int32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


# ------------------------------------------------------------------------------------------------ one case
def prepare(case, seed):
    c = dict(case)
    s = _prepare_norm(c, seed) if c["kind"] == "norm" else _prepare_cache(c, seed)
    if own:
        from kvq import cuda_kernels, fp4_cache, rope
        s["rope"], s["ops"] = rope, fp4_cache
        if c["kind"] in ("short", "step"):   # what a serving program keeps: split buffers, and the step's plan
            q_lens, keys = s["q_lens"], s["keys"]
            s["plan"] = cuda_kernels.plan_long(s["cu_host"], torch.tensor(keys), c["block"])
            short = [q for q in q_lens if q <= SHORT]
            s["segm"] = None
            if short and cuda_kernels.split_pays(np.asarray(q_lens), np.asarray(keys), c["hkv"], cuda_kernels.one_pass_fill(DEV)):
                s["segm"] = cuda_kernels.split_buffers(sum(short), c["hq"], c["d"], PIECES, DEV)
    return s


def _prepare_norm(c, seed):
    n, hq, hkv, d, r = c["tokens"], c["hq"], c["hkv"], c["d"], c["rotary"]
    g = _gen(seed, 5)
    # q, k and v of a packed projection
    qkv = torch.randn(n, (hq + 2 * hkv) * d, generator=g, device=DEV, dtype=torch.bfloat16)
    qkv *= torch.exp(0.3 * torch.randn(n, 1, generator=g, device=DEV)).to(torch.bfloat16)
    w = (1 + 0.2 * torch.randn(2, d, generator=g, device=DEV)).to(torch.bfloat16)
    angle = torch.arange(POSITIONS, device=DEV, dtype=torch.float64)[:, None] * (
        10000.0 ** (-torch.arange(0, r, 2, device=DEV, dtype=torch.float64) / r))
    table = torch.cat([angle.cos(), angle.sin()], -1).to(torch.bfloat16 if c["bf16_table"] else torch.float32)
    return {"case": c, "qkv": qkv, "q": qkv[:, :hq * d].view(n, hq, d), "k": qkv[:, hq * d:(hq + hkv) * d].view(n, hkv, d),
            "q_weight": w[0], "k_weight": w[1], "table": table,
            "positions": torch.randint(0, POSITIONS, (n,), generator=g, device=DEV),
            "q_out": torch.empty(n, hq, d, device=DEV, dtype=torch.bfloat16),
            "k_out": torch.empty(n, hkv, d, device=DEV, dtype=torch.bfloat16)}


def _prepare_cache(c, seed):
    kind, hkv, hq, d = c["kind"], c["hkv"], c["hq"], c["d"]
    q_lens, keys = _lens(c)
    table, blocks = _table(c, keys, seed)
    cu = np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32)
    kv, kc, vc, scales = _cache(c, blocks, seed)
    s = {"case": c, "q_lens": q_lens, "keys": keys, "cu_host": torch.from_numpy(cu), "cu": _int32(cu), "lens": _int32(keys),
         "most": max(q_lens), "table": table, "kv": kv, "kc": kc, "vc": vc, "scales": scales, "scale": d ** -0.5}
    if kind == "write":
        gain, mean = _channels(c, seed)
        n, g = int(cu[-1]), _gen(seed, 6)
        loud = 1 + torch.rand(n, hkv, 1, generator=g, device=DEV)
        s["key"] = ((torch.randn(n, hkv, d, generator=g, device=DEV) * gain + mean) * loud).to(torch.bfloat16)
        s["value"] = (torch.randn(n, hkv, d, generator=g, device=DEV) * loud).to(torch.bfloat16)
        r, pos = _token_positions(s)
        s["slots"] = table[r, pos // c["block"]].long() * c["block"] + pos % c["block"]
        s["first"], s["cu_k"] = (s["lens"] - (s["cu"][1:] - s["cu"][:-1])).contiguous(), s["cu"]
    if kind in ("short", "step", "weigh"):
        s["q"] = torch.randn(int(cu[-1]), hq, d, generator=_gen(seed, 3), device=DEV, dtype=torch.bfloat16)
    if kind in ("short", "step"):
        s["out"] = torch.zeros_like(s["q"])
        s["lse"] = torch.zeros(int(cu[-1]), hq, device=DEV) if kind == "short" else None
    if kind in ("weigh", "evict"):
        # sums of earlier steps: few keys hold most of them, some were never looked at
        g = _gen(seed, 8)
        most = table.shape[1] * c["block"]
        w = torch.exp(1.5 * torch.randn(len(keys), hkv, most, generator=g, device=DEV))
        w *= torch.rand(w.shape, generator=g, device=DEV) > 0.1
        w *= torch.arange(most, device=DEV) < s["lens"][:, None, None]
        s["weights"] = w
    if kind == "weigh":
        s["lse"] = _plain_requests(s, None, 0, len(keys))   # (the attention call's, before this one)
    if kind == "evict":
        s["keep"], s["recent"] = _int32([c["keep"]] * len(keys)), c["recent"]
        s["kept"] = torch.full((len(keys), hkv, c["keep"]), -1, dtype=torch.int32, device=DEV)
        s["new_lens"] = torch.zeros_like(s["lens"])
        kept = [min(k, c["keep"]) for k in keys]
        s["first"], s["cu_k"] = torch.zeros_like(s["lens"]), _int32(np.concatenate([[0], np.cumsum(kept)]))
    if kind in ("write", "evict"):
        s["rows"] = int(s["cu_k"][-1])
        s["k_out"] = torch.empty(s["rows"], hkv, d, dtype=torch.bfloat16, device=DEV)
        s["v_out"] = torch.empty_like(s["k_out"])
    return s


def _token_positions(s):
    """Request and position of each of the step's tokens: a request's new tokens are its last positions."""
    cu = s["cu"].long()
    t = torch.arange(int(s["cu_host"][-1]), device=DEV)
    r = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    return r, s["lens"].long()[r] - cu[r + 1] + t


def run(state):
    s = state
    kind = s["case"]["kind"]
    if own:
        ops = s["ops"]
        if kind == "norm":
            q, k = s["rope"].norm_rope(s["q"], s["k"], s["positions"], s["table"], s["q_weight"], s["k_weight"], EPS,
                                       s["case"]["interleaved"], s["q_out"], s["k_out"])
            return {"q": q, "k": k}
        if kind in ("short", "step"):
            out = ops.fp4_paged_attention(s["q"], s["kc"], s["vc"], s["out"], s["cu"], s["lens"], s["table"], s["most"],
                                          s["scale"], s["scales"], s["plan"], s["segm"], s["lse"])
            return {"out": out, "lse": s["lse"]} if kind == "short" else out
        if kind == "weigh":
            return ops.add_key_weights(s["q"], s["kc"], s["scales"], s["lse"], s["weights"], s["cu"], s["lens"], s["table"],
                                       s["scale"], s["most"])
        if kind == "write":
            ops.quant_fp4_cache(s["key"], s["value"], s["kc"], s["vc"], s["scales"], s["slots"])
        else:
            ops.evict_keys(s["kc"], s["vc"], s["scales"], s["weights"], s["lens"], s["keep"], s["recent"], s["table"],
                           s["kept"], s["new_lens"])
        ops.read_fp4_cache(s["kc"], s["vc"], s["scales"], s["first"], s["cu_k"], s["table"], s["k_out"], s["v_out"])
        k, v = s["k_out"], s["v_out"]
    else:
        if kind == "norm":
            return {"q": _plain_norm(s, s["q"], s["q_weight"]), "k": _plain_norm(s, s["k"], s["k_weight"])}
        if kind in ("short", "step"):
            return _plain_attention(s)
        if kind == "weigh":
            s["weights"] += _plain_requests(s, None, 0, len(s["keys"]), s["lse"])
            return s["weights"]
        if kind == "write":
            _plain_write(s, s["key"], s["kc"], s["scales"]["k_scale"])
            _plain_write(s, s["value"], s["vc"], s["scales"]["v_scale"])
        else:
            _plain_evict(s)
        k = _plain_read(s, s["kc"], s["scales"]["k_scale"])
        v = _plain_read(s, s["vc"], s["scales"]["v_scale"])
    if kind == "write":
        return {"k": k, "v": v, **s["scales"]}
    return {"k": k, "v": v, "weights": s["weights"], "kept": s["kept"], "new_lens": s["new_lens"]}


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_norm(s, x, weight):
    r = s["case"]["rotary"]
    y = x.float()
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * weight.float()
    cos, sin = s["table"][s["positions"]].float()[:, None].chunk(2, -1)
    turn = y[..., :r].unflatten(-1, (-1, 2)).movedim(-1, -2) if s["case"]["interleaved"] else y[..., :r].unflatten(-1, (2, -1))
    a, b = turn[..., 0, :], turn[..., 1, :]
    turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1 if s["case"]["interleaved"] else -2).flatten(-2)
    return torch.cat([turned, y[..., r:]], -1).to(x.dtype)


def _plain_write(s, x, cache, scale):
    """New rows into the cache in place. x [T, H, D], cache [num_blocks, block, H, D / 2], scale [num_blocks, H, block, D / 32]."""
    page, at = s["slots"] // s["case"]["block"], s["slots"] % s["case"]["block"]
    code, e = _quantize(x.float())
    cache[page, at] = code
    scale.transpose(1, 2)[page, at] = e


_PAIRS = {}


def _pairs(device):
    """[256, 2]: the values of a byte's two codes, the even channel's in the low half."""
    if device not in _PAIRS:
        v = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
        v = torch.cat([v, -v])
        _PAIRS[device] = torch.stack([v.repeat(16), v.repeat_interleave(16)], -1).to(device)
    return _PAIRS[device]


def _decode(code, e):
    """fp32 [..., D] of bytes [..., D / 2] and exponent bytes [..., D / 32]."""
    x = _pairs(code.device)[code.int()].flatten(-2)
    return x.unflatten(-1, (-1, GROUP)).mul_(torch.exp2(e.float() - 127)[..., None]).flatten(-2)


def _plain_read(s, cache, scale):
    bs = s["case"]["block"]
    cu = s["cu_k"].long()
    t = torch.arange(s["rows"], device=cache.device)
    r = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    pos = s["first"].long()[r] + t - cu[r]
    page = s["table"][r, pos // bs].long()
    return _decode(cache[page, pos % bs], scale.transpose(1, 2)[page, pos % bs]).to(torch.bfloat16)


def _plain_attention(s):
    out = torch.zeros_like(s["q"])
    lse = torch.full(out.shape[:2], -math.inf, device=out.device)
    short = sum(q <= SHORT for q in s["q_lens"])
    for a, b in ((0, short), (short, len(s["q_lens"]))):
        if b > a:
            at = s["cu_host"][a], s["cu_host"][b]
            lse[at[0]:at[1]] = _plain_requests(s, out, a, b)
    return {"out": out, "lse": lse} if s["case"]["kind"] == "short" else out


def _plain_requests(s, out, a, b, lse=None):
    """Requests a .. b - 1, padded to their longest query and context: their rows of `out`, where there is one, and the
    log-sum-exp of those rows; with `lse`, the weights that their keys get, [B, H, columns of the running sums]."""
    c = s["case"]
    bs, hkv, d = c["block"], c["hkv"], c["d"]
    q_lens, keys = s["q_lens"][a:b], s["keys"][a:b]
    lq, lk, g = max(q_lens), max(max(keys), 1), c["hq"] // hkv
    cu, lens = s["cu"].long()[a:b + 1], s["lens"].long()[a:b]
    ql = cu[1:] - cu[:-1]
    i = torch.arange(lq, device=DEV)
    row = (cu[:-1, None] + torch.minimum(i[None], ql[:, None] - 1))                       # [B, lq]
    real = i[None] < ql[:, None]
    j = torch.arange(lk, device=DEV)
    page = s["table"][a:b].long().gather(1, (j // bs)[None].expand(b - a, lk))             # [B, lk]
    k = _decode(s["kc"][page, j % bs], s["scales"]["k_scale"].transpose(1, 2)[page, j % bs])
    k = k.permute(0, 2, 3, 1).contiguous()                                                # [B, H, D, lk]
    q = s["q"][row].float().view(b - a, lq, hkv, g, d).permute(0, 2, 1, 3, 4).reshape(b - a, hkv, lq * g, d)
    w = torch.matmul(q, k).mul_(s["scale"]).view(b - a, hkv, lq, g, lk)
    del k
    seen = j[None, None] <= (lens - ql)[:, None, None] + i[None, :, None]                 # [B, lq, lk]
    w.masked_fill_(~(seen & real[..., None])[:, None, :, None], -math.inf)
    if lse is not None:
        of = lse[row].view(b - a, lq, hkv, g).permute(0, 2, 1, 3)[..., None]
        added = torch.zeros_like(s["weights"][a:b])
        added[..., :lk] = w.sub_(of.clamp_min(-1e30)).exp_().sum((2, 3))
        return added
    top = w.amax(-1, keepdim=True).clamp_min(-1e30)
    w.sub_(top).exp_()                                                                    # a row that sees nothing: zeros
    total = w.sum(-1, keepdim=True)
    of = torch.log(total).add_(top)[..., 0].permute(0, 2, 1, 3).reshape(b - a, lq, c["hq"])[real]
    if out is None:
        return of
    v = _decode(s["vc"][page, j % bs], s["scales"]["v_scale"].transpose(1, 2)[page, j % bs])
    o = torch.matmul(w.view(b - a, hkv, lq * g, lk), v.permute(0, 2, 1, 3).contiguous())
    o = (o.view(b - a, hkv, lq, g, d) / total.clamp_min(1e-30)).permute(0, 2, 1, 3, 4).reshape(b - a, lq, c["hq"], d)
    out[row[real]] = o[real].to(out.dtype)
    return of


def _plain_evict(s):
    bs, hkv = s["case"]["block"], s["case"]["hkv"]
    w, lens = s["weights"], s["lens"].long()
    pos = torch.arange(w.shape[2], device=DEV)
    n, keep = lens[:, None, None], s["keep"].long()[:, None, None]
    # the latest keys first, then by weight, ties by position; what there is none of last
    rank = torch.where(pos >= n - torch.clamp_max(keep, s["recent"]), math.inf, w).masked_fill_(pos >= n, -math.inf)
    most = s["kept"].shape[2]
    kept = torch.zeros(*w.shape[:2], most, dtype=torch.long, device=DEV)
    first = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :most]
    i = torch.arange(most, device=DEV)
    real = (i < torch.minimum(n, keep)).expand_as(kept)
    kept[..., :first.shape[2]] = first
    kept = kept.masked_fill_(~real, w.shape[2]).sort(-1).values
    s["kept"][real] = kept[real].int()
    s["new_lens"].copy_(torch.minimum(lens, s["keep"].long()))
    r, h, to = real.nonzero(as_tuple=True)
    source = kept[real]
    src, dst = ((s["table"][r, p // bs].long(), p % bs, h) for p in (source, to))
    for cache in (s["kc"], s["vc"], s["scales"]["k_scale"].transpose(1, 2), s["scales"]["v_scale"].transpose(1, 2)):
        cache[dst] = cache[src]
    held = w[r, h, source]
    w.zero_()
    w[r, h, to] = held


# ------------------------------------------------------------------------------------------------ work
def work(case):
    c = case
    hq, hkv, d = c["hq"], c["hkv"], c["d"]
    if c["kind"] == "norm":
        rows = c["tokens"] * (hq + hkv)
        return {"bytes": rows * d * 4 + c["tokens"] * (8 + c["rotary"] * (2 if c["bf16_table"] else 4)), "flops": rows * d * 9}
    q_lens, keys = _lens(c)
    key = d // 2 + d // GROUP                    # a row of K or V in the cache
    if c["kind"] == "write":                     # rows in, cache rows out; those in again, rows out
        n = sum(q_lens) * hkv
        return {"bytes": n * (2 * (4 * d + 2 * key)) + 8 * sum(q_lens), "flops": 0}
    pages = 4 * sum(-(-k // c["block"]) for k in keys)
    if c["kind"] == "evict":
        kept = sum(min(k, c["keep"]) for k in keys) * hkv
        moved = sum(c["keep"] for k in keys if k > c["keep"]) * hkv
        held = sum(keys) * hkv                   # sums read, the kept ones written, the rest cleared
        return {"bytes": 8 * held + 4 * kept + moved * 4 * key + kept * (2 * key + 4 * d) + pages, "flops": 0}
    pairs = sum(q * (k - q) + q * (q + 1) // 2 if k >= q else 0 for q, k in zip(q_lens, keys))
    if c["kind"] == "weigh":
        return {"bytes": sum(keys) * hkv * (key + 8) + pages + sum(q_lens) * hq * (2 * d + 4), "flops": 2 * d * hq * pairs}
    return {"bytes": sum(keys) * hkv * 2 * key + pages + sum(q_lens) * hq * (4 * d + 4), "flops": 4 * d * hq * pairs}


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    c = dict(case)
    s = _prepare_norm(c, seed) if c["kind"] == "norm" else _prepare_cache(c, seed)
    if c["kind"] == "norm":
        return {"q": _exact_norm(c, s, s["q"], s["q_weight"]), "k": _exact_norm(c, s, s["k"], s["k_weight"])}
    if c["kind"] == "write":
        (k, ke), (v, ve) = _exact_code(s["key"]), _exact_code(s["value"])
        scales = {n: x.clone() for n, x in s["scales"].items()}
        for name, e in (("k_scale", ke), ("v_scale", ve)):
            scales[name].permute(0, 2, 1, 3)[s["slots"] // c["block"], s["slots"] % c["block"]] = e
        return {"k": k, "v": v, **scales}
    if c["kind"] == "evict":
        return _exact_evict(c, s)
    if c["kind"] == "weigh":
        total = s["weights"].double()
        at = 0
        for r, (ql, n) in enumerate(zip(s["q_lens"], s["keys"])):
            w = _exact_scores(c, s["q"][at:at + ql], _values(c, s, s["kc"], s["scales"]["k_scale"], r, n), s["scale"])
            of = s["lse"][at:at + ql].double().view(ql, c["hkv"], -1).transpose(0, 1)[..., None]
            total[r, :, :n] += torch.where(w > -math.inf, torch.exp(w - of), 0.0).sum((1, 2))
            at += ql
        return total
    out, lse, at = [], [], 0
    for r, (ql, n) in enumerate(zip(s["q_lens"], s["keys"])):
        o, e = _exact_attention(c, s["q"][at:at + ql], _values(c, s, s["kc"], s["scales"]["k_scale"], r, n),
                                _values(c, s, s["vc"], s["scales"]["v_scale"], r, n), s["scale"])
        out.append(o)
        lse.append(e)
        at += ql
    return {"out": torch.cat(out), "lse": torch.cat(lse)} if c["kind"] == "short" else torch.cat(out)


def _exact_norm(c, s, x, weight):
    d, r = c["d"], c["rotary"]
    y = x.double()
    y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / d + EPS) * weight.double()
    t = s["table"].double()[s["positions"]]
    turn = torch.complex(t[:, :r // 2], t[:, r // 2:])[:, None]
    z = torch.complex(y[..., 0:r:2], y[..., 1:r:2]) if c["interleaved"] else torch.complex(y[..., :r // 2], y[..., r // 2:r])
    z = z * turn
    if c["interleaved"]:
        y[..., 0:r:2], y[..., 1:r:2] = z.real, z.imag
    else:
        y[..., :r // 2], y[..., r // 2:r] = z.real, z.imag
    return y


def _exact_code(x):
    """The values of quantized rows, and their exponent bytes."""
    g = x.double().unflatten(-1, (-1, GROUP))
    top = g.abs().amax(-1)
    mant, e = torch.frexp(top)                          # top = mant 2^e, mant in [1/2, 1)
    e = e - 3 + (mant > 7 / 8).to(e.dtype)
    e = torch.where(top > 0, e, -100).clamp(-100, 125)
    y = g * torch.exp2(-e.double())[..., None]
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    a = y.abs().clamp_max(6.0)
    up = torch.searchsorted(grid, a).clamp_max(7)       # the first grid value at or above a
    down = (up - 1).clamp_min(0)
    far_up, far_down = grid[up] - a, a - grid[down]
    take_up = (far_up < far_down) | ((far_up == far_down) & (up % 2 == 0))
    value = torch.where(take_up, grid[up], grid[down]) * y.sign()
    return (value * torch.exp2(e.double())[..., None]).flatten(-2), (e + 127).to(torch.uint8)


def _values(c, s, cache, scale, r, n):
    """float64 [H, n, D]: a request's first n keys."""
    ids = s["table"][r, :-(-n // c["block"])].long()
    code = cache[ids].flatten(0, 1)[:n].permute(1, 0, 2).contiguous()              # [H, n, D / 2]
    code = torch.stack([code & 15, code >> 4], -1).flatten(-2)
    low = code & 7
    value = torch.where(low < 2, 0.5 * low, (1 + 0.5 * (low & 1)) * torch.exp2((low >> 1).double() - 1))
    value = torch.where(code > 7, -value, value)
    e = scale[ids].permute(1, 0, 2, 3).flatten(1, 2)[:, :n].double() - 127         # [H, n, D / 32]
    return value * torch.exp2(e).repeat_interleave(GROUP, -1)


def _exact_scores(c, q, k, scale):
    """[H, t, G, n] scores of one request in 64 bits, bottom-right causal, -inf where nothing is seen."""
    t, hq, d = q.shape
    h, n = k.shape[:2]
    w = torch.matmul(q.double().view(t, h, hq // h, d).transpose(0, 1).reshape(h, -1, d), k.transpose(1, 2).contiguous())
    w = (w * scale).view(h, t, hq // h, n)
    lim = n - t + 1 + torch.arange(t, device=q.device)
    return w.masked_fill_((torch.arange(n, device=q.device)[None] >= lim[:, None])[:, None], -math.inf)


def _exact_attention(c, q, k, v, scale):
    """One request in 64 bits: out [t, Hq, D] and log-sum-exp [t, Hq]; k and v [H, n, D]."""
    t, hq, d = q.shape
    h, n = k.shape[:2]
    out = torch.zeros(t, hq, d, dtype=torch.float64, device=q.device)
    lse = torch.full((t, hq), -math.inf, dtype=torch.float64, device=q.device)
    if n == 0:
        return out, lse
    step = max(1, (1 << 27) // (n * hq))
    for a in range(0, t, step):
        b = min(t, a + step)
        m = n - t + b                           # keys that the last row of these sees
        if m <= 0:
            continue
        w = _exact_scores(c, q[a:b], k[:, :m], scale)
        e = torch.logsumexp(w, -1)
        w = torch.where(w > -math.inf, torch.exp(w - e[..., None]), 0.0)
        o = torch.matmul(w.view(h, -1, m), v[:, :m].contiguous()).view(h, b - a, hq // h, d)
        out[a:b] = o.transpose(0, 1).reshape(b - a, hq, d)
        lse[a:b] = e.transpose(0, 1).reshape(b - a, hq)
    return out, lse


def _exact_evict(c, s):
    weights, kept, rows = torch.zeros_like(s["weights"], dtype=torch.float64), s["kept"].clone(), ([], [])
    lens = []
    for r, n in enumerate(s["keys"]):
        m = min(n, c["keep"])
        lens.append(m)
        if not m:
            continue
        recent = min(c["recent"], m)
        w = s["weights"][r, :, :n - recent].cpu().double().numpy()
        # numpy's order of (-weight, position)
        chosen = np.sort(np.argsort(-w, axis=-1, kind="stable")[:, :m - recent], axis=-1)
        last = np.broadcast_to(np.arange(n - recent, n), (w.shape[0], recent))
        at = torch.from_numpy(np.concatenate([chosen, last], -1)).to(DEV)
        kept[r, :, :m] = at.int()
        weights[r, :, :m] = s["weights"][r].double().gather(1, at)
        for out, name, cache in ((rows[0], "k_scale", s["kc"]), (rows[1], "v_scale", s["vc"])):
            x = _values(c, s, cache, s["scales"][name], r, n)
            out.append(x.gather(1, at[..., None].expand(-1, -1, x.shape[2])).transpose(0, 1))
    k, v = (torch.cat(x) if x else torch.zeros(0, c["hkv"], c["d"], device=DEV) for x in rows)
    return {"k": k, "v": v, "weights": weights, "kept": kept, "new_lens": _int32(lens)}
