"""kvq.fp4_cache and kvq.rope without a GPU: refusals before any launch, empty calls, and the tests' plain forms."""
import pytest
import torch

import fp4_ref as R
from kvq import _native
from kvq import cuda_kernels as ck
from kvq import fp4_cache as fc
from kvq import rope


def _batch(h=4, d=128, bs=32):
    kc, vc = R.new_cache(8, bs, h, d, "vllm")
    return {"kc": kc, "vc": vc, "scales": fc.fp4_scales(8, bs, h, d, "cpu"), "slots": torch.arange(5),
            "key": torch.zeros(5, h, d, dtype=torch.bfloat16), "q": torch.zeros(5, 7 * h, d, dtype=torch.bfloat16),
            "cu": torch.tensor([0, 2, 5], dtype=torch.int32), "lens": torch.tensor([2, 9], dtype=torch.int32),
            "bt": torch.zeros(2, 3, dtype=torch.int32), "lse": torch.zeros(5, 7 * h), "w": torch.zeros(2, h, 96),
            "keep": torch.tensor([4, 4], dtype=torch.int32), "kept": torch.zeros(2, h, 4, dtype=torch.int32),
            "new": torch.zeros(2, dtype=torch.int32)}


def _write(b):
    fc.quant_fp4_cache(b["key"], b["key"], b["kc"], b["vc"], b["scales"], b["slots"])


def _read(b):
    out = torch.zeros(11, *b["key"].shape[1:], dtype=torch.bfloat16)
    fc.read_fp4_cache(b["kc"], b["vc"], b["scales"], b["lens"], b["cu"], b["bt"], out, out.clone())


def _decode(b, segm=None):
    fc.fp4_decode_attention(b["q"], b["kc"], b["vc"], b["q"].clone(), b["cu"], b["lens"], b["bt"], 0.1, b["scales"], segm,
                            lse=b["lse"])


def _prefill(b):
    plan = ck.plan_long([0, 20], [40], b["kc"].shape[1])
    fc.fp4_long_attention(b["q"], b["kc"], b["vc"], b["q"].clone(), b["cu"], b["lens"], b["bt"], plan, 0.1, b["scales"])


def _weigh(b):
    fc.add_key_weights(b["q"], b["kc"], b["scales"], b["lse"], b["w"], b["cu"], b["lens"], b["bt"], 0.1, 3)


def _evict(b, recent=2):
    fc.evict_keys(b["kc"], b["vc"], b["scales"], b["w"], b["lens"], b["keep"], recent, b["bt"], b["kept"], b["new"])


CALLS = [_write, _read, _decode, _prefill, _weigh, _evict]


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("change,msg,but", [
    (lambda b: b.update(kc=b["kc"].to(torch.int8)), "caches must be uint8", ()),
    (lambda b: b.update(vc=b["vc"][:4]), "caches must be uint8", (_weigh,)),
    (lambda b: b["scales"].update(k_scale=b["scales"]["k_scale"].half()), "scales must be uint8", ()),
    (lambda b: b["scales"].update(v_scale=b["scales"]["v_scale"].clone()), "of one layout", (_weigh,)),
    (lambda b: b.update(scales=fc.fp4_scales(7, 32, 4, 128, "cpu")), "scales must be uint8", ()),
    (lambda b: b.update(scales={n: s.transpose(1, 2).contiguous().transpose(1, 2) for n, s in b["scales"].items()}),
     "contiguous pages of a head", ()),
    (lambda b: b.update(cu=b["cu"].long()), "contiguous int32 vector", (_write, _evict)),
    (lambda b: b.update(lens=b["lens"].long()), "contiguous int32 vector", (_write,)),
    (lambda b: b.update(lens=b["lens"][:1]), "fewer entries than requests", (_write, _evict)),
    (lambda b: b.update(bt=b["bt"].t().contiguous().t()), "contiguous last dim", (_write,)),
    (lambda b: b.update(bt=b["bt"][:1]), "block_table must be int32", (_write,)),
    (lambda b: b.update(key=b["key"].float(), q=b["q"].half()), "must be bf16", (_read, _evict)),
    (lambda b: b.update(key=b["key"][..., :64], q=b["q"][..., :64]), "disagree|must be bf16", (_evict,)),
    (lambda b: b.update(lse=b["lse"].double()), "lse must be float32", (_write, _read, _prefill, _evict)),
    (lambda b: b.update(lse=b["lse"][:4]), "lse must be float32", (_write, _read, _prefill, _evict)),
    (lambda b: b.update(w=b["w"].half()), "weights must be float32", (_write, _read, _decode, _prefill)),
    (lambda b: b.update(w=b["w"][:1]), "weights must be float32", (_write, _read, _decode, _prefill)),
    (lambda b: b.update(w=b["w"].transpose(1, 2)), "weights must be float32", (_write, _read, _decode, _prefill)),
    (lambda b: None, "on the GPU", ()),
])
def test_refusals(call, change, msg, but):
    if call in but:
        pytest.skip("takes no such argument")
    b = _batch()
    change(b)
    with pytest.raises(RuntimeError, match=msg):
        call(b)


def test_refusals_of_one_operator():
    b = _batch()
    with pytest.raises(RuntimeError, match="cache shapes disagree with key"):
        _write({**b, "key": b["key"][:, :2]})
    with pytest.raises(RuntimeError, match="5 slots for 3 rows"):
        _write({**b, "key": b["key"][:3]})
    with pytest.raises(RuntimeError, match="slot_mapping must be a contiguous int64"):
        _write({**b, "slots": b["slots"].int()})
    for call in (_decode, _weigh):
        with pytest.raises(RuntimeError, match="q heads not a multiple of 4 kv heads"):
            call({**b, "q": b["q"][:, :27]})
    sm = torch.zeros(5, 28, 65)
    with pytest.raises(RuntimeError, match="at most 64 split-KV segments"):
        _decode(b, (torch.zeros(5, 28, 65, 128), sm, sm))
    with pytest.raises(RuntimeError, match="laid out as segm_max"):
        _decode(b, (torch.zeros(5, 28, 128, 4).transpose(2, 3), torch.zeros(5, 28, 4), torch.zeros(5, 28, 4)))
    with pytest.raises(RuntimeError, match="split buffers must be float32"):
        _decode(b, (None, torch.zeros(5, 28, 4), torch.zeros(5, 28, 4)))
    with pytest.raises(RuntimeError, match="block size 32 != plan block size 16"):
        fc.fp4_long_attention(b["q"], b["kc"], b["vc"], b["q"].clone(), b["cu"], b["lens"], b["bt"],
                              ck.plan_long([0, 20], [40], 16), 0.1, b["scales"])
    with pytest.raises(RuntimeError, match="recent must not be negative"):
        _evict(b, -1)
    with pytest.raises(RuntimeError, match="kept must be int32"):
        _evict({**b, "kept": b["kept"].long()})
    with pytest.raises(RuntimeError, match="fewer entries than requests"):
        _evict({**b, "keep": b["keep"][:1]})
    with pytest.raises(RuntimeError, match="power of two"):
        _write({**b, "kc": torch.zeros(8, 24, 4, 64, dtype=torch.uint8), "vc": torch.zeros(8, 24, 4, 64, dtype=torch.uint8)})


def test_empty_calls_return_early():
    b = _batch()
    none = torch.zeros(1, dtype=torch.int32)
    _write({**b, "slots": b["slots"][:0]})
    _decode({**b, "cu": none, "q": b["q"][:0]})
    _weigh({**b, "cu": none, "q": b["q"][:0]})
    _weigh({**b, "w": b["w"][..., :0]})
    _evict({**b, "lens": b["lens"][:0]})
    out = torch.zeros(0, 4, 128, dtype=torch.bfloat16)
    assert fc.read_fp4_cache(b["kc"], b["vc"], b["scales"], b["lens"], b["cu"], b["bt"], out, out)[0] is out
    x = torch.zeros(0, 4, 128, dtype=torch.bfloat16)
    assert rope.norm_rope(x, x, torch.zeros(0, dtype=torch.int64), torch.zeros(3, 64))[0] is x


CACHE, GEOM, SCALES = [16, 2048, 64, 512], [8, 32, 4, 128], [16, 16, 512, 128]
C_ARGS = {
    "quant_fp4_cache": [16, 512, 128, 16, 512, 128, *CACHE, *CACHE, *GEOM, *SCALES, 16, 5, None],
    "read_fp4_cache": [*CACHE, *CACHE, *GEOM, *SCALES, 16, 16, 16, 3, 2, 16, 512, 128, 16, 512, 128, 5, None],
    "fp4_pages": [*CACHE, *CACHE, *GEOM, *SCALES, 16, 16, 16, 16, 3, 16, 16, 2, None],
    "fp4_decode_attention": [16, 3584, 128, *CACHE, *CACHE, *GEOM, *SCALES, 16, 3584, 128, 16, 16, 16, 3, 2, 28, 0.1, None, None,
                             None, 0, 0, 1, 0, None, 0, 0, 1, 8, None],
    "fp4_key_weights": [16, 3584, 128, *CACHE, *GEOM, 16, 512, 128, 16, 28, 16, 384, 96, 96, 16, 16, 16, 3, 2, 28, 0.1, 1, 8, None],
    "fp4_evict": [*CACHE, *CACHE, *GEOM, *SCALES, 16, 384, 96, 96, 16, 16, 2, 16, 3, 3, 2, 16, 16, 4, 4, 16, None],
    "fp4_prefill_attention": [16, 3584, 128, 16, 16, 16, 8, 32, 4, 128, 16, 3584, 128, 16, 16, 16, 3, 28, 16, 16, 1, 128, 0.1, None,
                              None, None, 0, None, None, None],
}
# where each argument stands (the pointers are never read: every call here is refused)
AT = {
    "quant_fp4_cache": dict(q=0, q_st=1, kc=6, k_sn=8, geom=14, scales=18),
    "read_fp4_cache": dict(q=21, q_st=22, kc=0, k_sn=2, geom=8, scales=12),
    "fp4_pages": dict(q=16, kc=0, k_sn=2, geom=8, scales=12),
    "fp4_decode_attention": dict(q=0, q_st=1, kc=3, k_sn=5, geom=11, scales=15, hq=27, scale=28, splits=34),
    "fp4_key_weights": dict(q=0, q_st=1, kc=3, k_sn=5, geom=7, scales=11, hq=25, scale=26),
    "fp4_evict": dict(kc=0, k_sn=2, geom=8, scales=12),
    "fp4_prefill_attention": dict(q=0, q_st=1, kc=3, geom=6, scales=5, hq=17, scale=22),
}


def _c(name, *changes):
    args = list(C_ARGS[name])
    assert len(args) == len(_native.SIGNATURES["kvq_" + name])
    for at, val in changes:
        args[at] = val
    lib = _native.load()
    return getattr(lib, "kvq_" + name)(*args), lib.kvq_last_error().decode()


@pytest.mark.parametrize("name", C_ARGS)
def test_c_entry_refusals(name):
    at = AT[name]
    geom = at["geom"]
    cases = [([(geom + 3, 96)], "head_dim must be 64 or 128"), ([(geom + 1, 24)], "block_size must be a power of two"),
             ([(geom + 1, 8)], "block_size must be a power of two"), ([(geom + 2, 0)], "bad sizes"),
             ([(geom + 2, 65536)], "bad sizes"), ([(geom, 0)], "bad sizes"), ([(geom, 1 << 31)], "bad sizes"),
             ([(at["kc"], None)], "null pointer"), ([(at["kc"], 24)], "16-byte aligned"),
             ([(at["scales"], None)], "null pointer"), ([(at["scales"], 8)], "16-byte aligned")]
    if "k_sn" in at:
        cases += [([(at["k_sn"], 40)], "16-byte aligned"), ([(at["k_sn"], 1 << 27)], "32-bit lane offsets"),
                  ([(at["k_sn"], -64)], "32-bit lane offsets")]
    if "q" in at:
        cases += [([(at["q"], None)], "null pointer"), ([(at["q"], 24)], "16-byte aligned")]
    if "q_st" in at:
        cases += [([(at["q_st"], 516)], "16-byte aligned")]
    if "hq" in at:
        cases += [([(at["hq"], 30)], "bad head counts"), ([(at["hq"], 0)], "bad head counts"),
                  ([(at["hq"], 65540)], "bad head counts")]
        for bad in (0.0, -1.0, 1e-17, 1e17, float("inf"), float("nan")):
            cases.append(([(at["scale"], bad)], "softmax_scale must be positive"))
    if "splits" in at:
        cases += [([(at["splits"], 65)], "at most 64"), ([(at["splits"], 4), (at["splits"] + 1, 5)], "split buffers missing")]
    for change, msg in cases:
        rc, err = _c(name, *change)
        assert rc == 1 and msg in err, (change, rc, err)


def test_c_entry_sizes():
    assert _c("quant_fp4_cache", (23, -1)) == (1, "quant_fp4_cache: bad sizes")
    assert _c("quant_fp4_cache", (23, 0)) == (0, "")
    assert _c("read_fp4_cache", (27, 1 << 31)) == (1, "read_fp4_cache: bad sizes")
    assert _c("fp4_pages", (23, 0)) == (0, "")
    assert _c("fp4_pages", (9, 1 << 24), (2, 64), (6, 64))[1] == "fp4_pages: page too large for 32-bit lane offsets"
    assert _c("fp4_evict", (22, -1)) == (1, "fp4_evict: bad sizes")
    assert _c("fp4_evict", (20, None)) == (1, "fp4_evict: null pointer")
    assert _c("fp4_evict", (26, 1 << 30)) == (1, "fp4_evict: too many requests and heads for one call")
    assert _c("fp4_key_weights", (28, 0)) == (1, "fp4_key_weights: bad sizes")
    assert _c("fp4_key_weights", (25, 65528), (28, 1 << 30)) == (1, "fp4_key_weights: too many rows for one kv head")
    assert _c("fp4_prefill_attention", (21, 64)) == (1, "fp4_prefill_attention: work list tiles must be 128 rows")


def test_c_entry_layouts():
    """The strides that the kernels' 32-bit offsets, or one address for a key's K and V, leave out."""
    for name, at in (("quant_fp4_cache", 7), ("quant_fp4_cache", 20), ("read_fp4_cache", 5), ("fp4_pages", 1),
                     ("fp4_decode_attention", 4), ("fp4_key_weights", 4), ("fp4_evict", 14), ("fp4_evict", 5)):
        for far in (1 << 32, -2048):
            assert _c(name, (at, far)) == (1, f"{name}: pages 4 GiB apart or more"), (name, at)
    same = "fp4_decode_attention: K and V caches must have the same page and slot strides"
    assert _c("fp4_decode_attention", (8, 4096)) == (1, same)
    assert _c("fp4_decode_attention", (9, 128)) == (1, same)
    assert _c("fp4_evict", (25, (1 << 23) + 1)) == (1, "fp4_evict: tables of more than 2^28 slots")


@pytest.mark.parametrize("seq_lens,keep,new_lens", [(64, 80, 68), (64, 80, 60), (80, 64, 68), (80, 64, 60), (64, 64, 68),
                                                    (64, 68, 64), (68, 64, 64)])
def test_new_lengths_that_overlap_others(seq_lens, keep, new_lens):
    """The workgroups of a request's heads read seq_lens and keep while new_lens is written: two requests' lengths (8 bytes)
    that are neither one of the others' nor apart from them."""
    assert _c("fp4_evict", (20, seq_lens), (21, keep), (31, new_lens)) == (
        1, "fp4_evict: new_lens may be seq_lens or keep, but not overlap them otherwise")


def test_rows_that_overlap():
    """Sums that requests or heads share (an expanded tensor's strides of 0) would be updated by several workgroups; rows apart in
    any order are taken (and these calls refused for what is looked at next)."""
    for sr, sh in ((384, 96), (96, 192), (1000, 97), (97, 1000)):
        assert _c("fp4_key_weights", (17, sr), (18, sh), (25, 65528), (28, 1 << 30))[1] == "fp4_key_weights: too many rows for one kv head"
        assert "new_lens may be" in _c("fp4_evict", (17, sr), (18, sh), (20, 64), (31, 68))[1]
    assert "new_lens may be" in _c("fp4_evict", (28, 4), (29, 8), (20, 64), (31, 68))[1]
    for name in ("fp4_key_weights", "fp4_evict"):
        for sr, sh in ((0, 96), (384, 0), (0, 0), (384, 95), (383, 96), (95, 190), (96, 191)):
            assert _c(name, (17, sr), (18, sh)) == (1, f"{name}: rows of weights overlap"), (name, sr, sh)
    for sr, sh in ((0, 4), (16, 0), (16, 3), (15, 4)):
        assert _c("fp4_evict", (28, sr), (29, sh)) == (1, "fp4_evict: rows of kept overlap"), (sr, sh)


ROPE = [16, 3584, 128, 16, 512, 128, 16, 3584, 128, 16, 512, 128, 5, 28, 4, 128, 16, 64, 16, 64, 100, 64, 0, 16, 16, 1, 1e-6, 0, None]


@pytest.mark.parametrize("change,msg", [
    ([(15, 96)], "head_dim must be 64 or 128"), ([(12, -1)], "bad sizes"), ([(13, 65535)], "bad sizes"), ([(21, 24)], "rotary_dim"),
    ([(21, 144)], "rotary_dim"), ([(21, -16)], "rotary_dim"), ([(17, 16)], "32 or 64 bits"), ([(26, -1.0)], "eps"),
    ([(26, float("nan"))], "eps"), ([(0, None)], "null pointer"), ([(9, None)], "null pointer"), ([(16, None)], "null pointer"),
    ([(18, None)], "null pointer"), ([(23, None)], "both weights or none"), ([(0, 24)], "16-byte aligned"), ([(4, 516)], "16-byte aligned"),
    ([(18, 8)], "table's rows and the weights"), ([(19, 68)], "table's rows and the weights"), ([(24, 40)], "table's rows and the weights"),
    ([(12, 1 << 31)], "bad sizes"), ([(12, 2 ** 31 - 1)], "too many tokens")])
def test_norm_rope_c_refusals(change, msg):
    args = list(ROPE)
    assert len(args) == len(_native.SIGNATURES["kvq_norm_rope"])
    for at, val in change:
        args[at] = val
    lib = _native.load()
    assert lib.kvq_norm_rope(*args) == 1 and msg in lib.kvq_last_error().decode()


@pytest.mark.parametrize("change,msg", [
    (dict(q=torch.zeros(3, 8, 128)), "must be bf16"), (dict(k=torch.zeros(2, 2, 128, dtype=torch.bfloat16)), "must be bf16"),
    (dict(k=torch.zeros(3, 2, 64, dtype=torch.bfloat16)), "must be bf16"),
    (dict(q_out=torch.zeros(3, 8, 64, dtype=torch.bfloat16)), "must be bf16"),
    (dict(positions=torch.zeros(2, dtype=torch.int64)), "positions must be"),
    (dict(positions=torch.zeros(3, dtype=torch.int16)), "positions must be"),
    (dict(cos_sin=torch.zeros(9, 64, dtype=torch.float16)), "cos_sin must be"), (dict(cos_sin=torch.zeros(64)), "cos_sin must be"),
    (dict(q_weight=torch.zeros(128)), "or neither"), (dict(q_weight=torch.zeros(64), k_weight=torch.zeros(64)), "weights must be"),
    (dict(q_weight=torch.zeros(128), k_weight=torch.zeros(128, dtype=torch.bfloat16)), "weights must be"), ({}, "on the GPU")])
def test_norm_rope_refusals(change, msg):
    a = dict(q=torch.zeros(3, 8, 128, dtype=torch.bfloat16), k=torch.zeros(3, 2, 128, dtype=torch.bfloat16),
             positions=torch.zeros(3, dtype=torch.int64), cos_sin=torch.zeros(9, 64))
    with pytest.raises(RuntimeError, match=msg):
        rope.norm_rope(**{**a, **change})


def test_plain_quantization_is_within_half_a_step():
    """Every finite bf16 whose group's largest is its own, up to 7 2^125 (the largest exponent is 125; 6 2^125 stands for what
    lies above): off by at most half the step it falls in, 2^-100 at the least."""
    bits = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16)
    x = bits.view(torch.bfloat16)
    x = x[x.abs().double() <= 7 * 2.0 ** 125][:, None].expand(-1, 32).contiguous()
    code, e = R.quantize(x)
    got, a = R.decode(code, e), x.double().abs()
    scale = torch.exp2(e.double() - 127)
    assert bool(((got - x.double()).abs() <= scale).all())                  # half the step from 4 to 6, and from 6 to 7
    assert bool((((got - x.double()).abs() <= a / 4) | (a < 2.0 ** -100)).all())
    big = a[:, 0] > 2.0 ** -98
    ratio = (a[:, 0] / scale[:, 0])[big]
    assert bool((ratio > 3.5).all()) and bool((ratio <= 7).all())
    top = torch.tensor([[7.5 * 2.0 ** 125, float("inf"), -float("inf"), float("nan")] + [1.0] * 28]).to(torch.bfloat16)
    assert R.decode(*R.quantize(top))[0, :4].tolist() == [6 * 2.0 ** 125, 6 * 2.0 ** 125, -6 * 2.0 ** 125, 0.0]


def test_plain_eviction():
    assert R.evict([5, 1, 3, 9, 3, 0, 0], 7, 4, 1, 7) == [0, 2, 3, 6]
    assert R.evict([5, float("nan"), 3, 9], 4, 2, 0, 4) == [1, 3]
    assert R.evict([1, 1, 1, 1], 4, 2, 0, 4) == [0, 1]
    assert R.evict([1, 2], 6, 3, 1, 2) == [0, 1, 5]
    assert R.evict([1, 2], 2, 3, 1, 2) == [0, 1] and R.evict([1, 2], 2, 0, 1, 2) == []
