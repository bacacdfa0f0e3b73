"""kvq.block_cache without a GPU: refusals before any launch, empty batches, and the tests' plain write."""
import pytest
import torch

import block_ref as R
from kvq import _native
from kvq import block_cache as bc
from kvq import cuda_kernels as ck


def _batch(h=4, d=128, bs=32, group=16):
    kc, vc = R.new_cache(8, bs, h, d, "vllm")
    return {"kc": kc, "vc": vc, "scales": bc.block_scales(8, bs, h, group, "cpu"),
            "key": torch.zeros(5, h, d, dtype=torch.bfloat16), "q": torch.zeros(5, 7 * h, d, dtype=torch.bfloat16),
            "cu": torch.tensor([0, 2, 5], dtype=torch.int32), "lens": torch.tensor([2, 9], dtype=torch.int32),
            "bt": torch.zeros(2, 3, dtype=torch.int32)}


def _write(b):
    bc.quant_block_cache(b["key"], b["key"], b["kc"], b["vc"], b["scales"], b["cu"], b["lens"], b["bt"])


def _read(b):
    out = torch.zeros(11, *b["key"].shape[1:], dtype=torch.bfloat16)
    bc.read_block_cache(b["kc"], b["vc"], b["scales"], b["lens"], b["cu"], b["bt"], out, out.clone())


def _decode(b, segm=None):
    bc.block_decode_attention(b["q"], b["kc"], b["vc"], b["q"].clone(), b["cu"], b["lens"], b["bt"], 0.1, b["scales"], segm)


def _prefill(b):
    plan = ck.plan_long([0, 20], [40], b["kc"].shape[1])
    bc.block_long_attention(b["q"], b["kc"], b["vc"], b["q"].clone(), b["cu"], b["lens"], b["bt"], plan, 0.1, b["scales"])


CALLS = [_write, _read, _decode, _prefill]


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("change,msg", [
    (lambda b: b.update(kc=b["kc"].float()), "caches must be int8"),
    (lambda b: b.update(vc=b["vc"][:4]), "caches must be int8"),
    (lambda b: b["scales"].update(k_scale=b["scales"]["k_scale"].half()), "scales must be float32"),
    (lambda b: b["scales"].update(v_scale=b["scales"]["v_scale"].clone()), "of one layout"),
    (lambda b: b.update(scales=bc.block_scales(7, 32, 4, 16, "cpu")), "for 8 blocks of 4 kv heads"),
    (lambda b: b.update(scales=R.new_scales(8, 32, 4, 8)), "positions per scale must be one of"),
    (lambda b: b.update(scales={n: torch.zeros(8, 4, 3) for n in ("k_scale", "v_scale")}), "do not divide a page"),
    (lambda b: b.update(cu=b["cu"].long()), "contiguous int32 vector"),
    (lambda b: b.update(lens=b["lens"][:1]), "fewer entries than requests"),
    (lambda b: b.update(bt=b["bt"].t().contiguous().t()), "contiguous last dim"),
    (lambda b: b.update(bt=b["bt"][:1]), "block_table must be int32"),
    (lambda b: b.update(key=b["key"].float(), q=b["q"].half()), "must be bf16|disagree|outputs must be"),
    (lambda b: None, "on the GPU"),
])
def test_refusals(call, change, msg):
    b = _batch()
    change(b)
    if call is _read and msg.startswith("must be bf16"):
        pytest.skip("reads no bf16 rows")
    with pytest.raises(RuntimeError, match=msg):
        call(b)


def test_refusals_of_one_operator():
    b = _batch()
    with pytest.raises(RuntimeError, match="cache shapes disagree with key"):
        _write({**b, "key": b["key"][:, :2]})
    with pytest.raises(RuntimeError, match="q heads not a multiple of 4 kv heads"):
        _decode({**b, "q": b["q"][:, :27]})
    sm = torch.zeros(5, 28, 65)
    with pytest.raises(RuntimeError, match="at most 64 split-KV segments"):
        _decode(b, (torch.zeros(5, 28, 65, 128), sm, sm))
    with pytest.raises(RuntimeError, match="laid out as segm_max"):
        _decode(b, (torch.zeros(5, 28, 128, 4).transpose(2, 3), torch.zeros(5, 28, 4), torch.zeros(5, 28, 4)))
    with pytest.raises(RuntimeError, match="split buffers must be float32"):
        _decode(b, (None, torch.zeros(5, 28, 4), torch.zeros(5, 28, 4)))
    with pytest.raises(RuntimeError, match="block size 32 != plan block size 16"):
        bc.block_long_attention(b["q"], b["kc"], b["vc"], b["q"].clone(), b["cu"], b["lens"], b["bt"],
                                ck.plan_long([0, 20], [40], 16), 0.1, b["scales"])
    for group, bs in ((8, 32), (64, 32), (24, 48), (256, 256)):
        with pytest.raises(RuntimeError, match="positions per scale"):
            bc.block_scales(4, bs, 2, group, "cpu")


def test_empty_calls_return_early():
    b = _batch()
    none = torch.zeros(1, dtype=torch.int32)
    _write({**b, "key": b["key"][:0]})
    _write({**b, "cu": none})
    _decode({**b, "cu": none, "q": b["q"][:0]})
    out = torch.zeros(0, 4, 128, dtype=torch.bfloat16)
    assert bc.read_block_cache(b["kc"], b["vc"], b["scales"], b["lens"], b["cu"], b["bt"], out, out)[0] is out


def _c(name, **change):
    """A call of an entry point with valid sizes and null data, one argument changed by its place."""
    geom = [8, 32, 4, 128]
    sc = [None, None, 16, 4, 1, 16]
    cache = [16, 4096, 128, 256]       # (never read: refused before)
    k = v = cache
    args = {"quant_block_cache": [None, 512, 128, None, 512, 128, 5, *k, *v, *geom, *sc, None, None, None, 3, 2, None],
            "read_block_cache": [*k, *v, *geom, *sc, None, None, None, 3, 2, None, 512, 128, None, 512, 128, 5, None],
            "block_decode_attention": [None, 3584, 128, *k, *v, *geom, *sc, None, 3584, 128, None, None, None, 3, 2, 28, 0.1,
                                       None, None, None, 0, 0, 1, 0, 0, 1, 8, None],
            "block_prefill_attention": [None, 3584, 128, *k, *v, *geom, *sc, None, 3584, 128, None, None, None, 3, 28, 16, 16,
                                        1, 128, 0.1, None, None, None, 0, None, None, None, None, None, 0, None, 0, None]}[name]
    at = {"quant_block_cache": 15, "read_block_cache": 8, "block_decode_attention": 11, "block_prefill_attention": 11}[name]
    places = {"num_blocks": at, "block_size": at + 1, "heads": at + 2, "d": at + 3, "group": at + 9, "k_cache": at - 8,
              "k_sn": at - 6, "num_seqs": len(args) - 2, "splits": 36, "rows_per_tile": 32, "scale": 30 if name == "block_decode_attention" else 33}
    for key, val in change.items():
        args[places[key]] = val
    lib = _native.load()
    return getattr(lib, "kvq_" + name)(*args), lib.kvq_last_error().decode()


@pytest.mark.parametrize("name", ["quant_block_cache", "read_block_cache", "block_decode_attention",
                                  "block_prefill_attention"])
def test_c_entry_refusals(name):
    for change, msg in (({"d": 96}, "head_dim must be 64 or 128"), ({"block_size": 24}, "block_size must be a power of two"),
                        ({"block_size": 8}, "block_size must be a power of two"), ({"group": 8}, "positions per scale"),
                        ({"group": 64}, "positions per scale"), ({"group": 48}, "positions per scale"),
                        ({"heads": 0}, "bad sizes"), ({"num_blocks": 0}, "bad sizes"), ({"num_blocks": 1 << 31}, "bad sizes"),
                        ({"k_cache": None}, "16-byte aligned"), ({"k_cache": 24}, "16-byte aligned"),
                        ({"k_sn": 120}, "16-byte aligned"), ({}, "null pointer")):
        rc, err = _c(name, **change)
        assert rc == 1 and msg in err, (change, rc, err)


def test_c_entry_refusals_of_the_attention():
    assert _c("block_decode_attention", splits=65) == (1, "block_decode_attention: at most 64 split-KV segments")
    rc, err = _c("block_prefill_attention", rows_per_tile=64)
    assert rc == 1 and "work list tiles must be 128 rows" in err
    rc, err = _c("block_decode_attention", heads=3)
    assert rc == 1 and "bad head counts" in err
    for name in ("block_decode_attention", "block_prefill_attention"):
        for scale in (0.0, -0.1, float("nan"), float("inf")):
            rc, err = _c(name, scale=scale)
            assert rc == 1 and "softmax_scale must be positive and finite" in err
        for scale in (9e-17, 1.1e16, 1e-300, 1e300):
            rc, err = _c(name, scale=scale)
            assert rc == 1 and "from 1e-16 to 1e+16" in err


def _codes_prefill(**change):
    """kvq_block_prefill_attention over a temporary cache, valid but for `change` (refused before any pointer is used)."""
    a = dict(kc=16, codes_k=16, codes_v=16, code_scales=16, pages=8, codes_table=16, block=32, heads=4)
    a.update(change)
    geom, cache, sc = [8, a["block"], a["heads"], 128], [16, 4096, 128, 256], [16, 16, 16, 4, 1, 16]
    lib = _native.load()
    rc = lib.kvq_block_prefill_attention(16, 3584, 128, *cache, *cache, *geom, *sc, 16, 3584, 128, 16, 16, 16, 3, 28, 16, 16, 1,
                                         128, 0.1, None, None, None, 0, None, None, a["codes_k"], a["codes_v"],
                                         a["code_scales"], a["pages"], a["codes_table"], 3, None)
    return rc, lib.kvq_last_error().decode()


@pytest.mark.parametrize("change", [{"codes_v": None}, {"code_scales": None}, {"codes_table": None}, {"codes_k": 24},
                                    {"codes_v": 24}, {"code_scales": 20}, {"pages": 0}, {"pages": -1}, {"pages": 1 << 31}])
def test_c_entry_refusals_of_a_temporary_cache(change):
    rc, err = _codes_prefill(**change)
    assert rc == 1 and "bad temporary cache" in err


def test_c_entry_refuses_a_temporary_cache_of_huge_pages():
    rc, err = _codes_prefill(block=1 << 22)    # 2 * 2^22 * 4 * 128 bytes a page
    assert rc == 1 and "page / slot offsets" in err


@pytest.mark.parametrize("place,val,msg", [
    (11, 96, "head_dim must be 64 or 128"), (9, 24, "block_size must be a power of two"), (17, 48, "positions per scale"),
    (17, 64, "positions per scale"), (10, 0, "bad sizes"), (8, 0, "bad sizes"), (0, None, "16-byte aligned"),
    (0, 24, "16-byte aligned"), (2, 120, "16-byte aligned"), (12, None, "null pointer"), (13, None, "null pointer"),
    (18, None, "null pointer"), (19, None, "null pointer"), (20, None, "null pointer"), (21, None, "null pointer"),
    (23, None, "null pointer"), (24, None, "null pointer"), (18, 24, "rows must be 16-byte aligned"),
    (19, 24, "rows must be 16-byte aligned"), (20, 24, "rows must be 16-byte aligned"), (25, -1, "bad sizes"),
    (25, 1 << 31, "bad sizes")])
def test_c_entry_refusals_of_block_codes(place, val, msg):
    args = [16, 4096, 128, 256, 16, 4096, 128, 256, 8, 32, 4, 128, 16, 16, 16, 4, 1, 16, 16, 16, 16, 16, 3, 16, 16, 2, None]
    args[place] = val
    lib = _native.load()
    rc = lib.kvq_block_codes(*args)
    assert rc == 1 and msg in lib.kvq_last_error().decode()


def test_plain_write_keeps_scales_and_grows_them():
    """The reference of the GPU tests, by hand: 3 positions, then one of twice the size, then a small one."""
    kc, _ = R.new_cache(2, 16, 1, 64, "apart")
    sc = torch.zeros(2, 1, 1)
    table = torch.tensor([[1]])
    x = torch.full((3, 1, 64), 1.0)
    x[1] = -0.5
    R.write(x.to(torch.bfloat16), kc, sc, [0, 3], [3], table)
    assert sc[1, 0, 0] == torch.tensor(1.0) / 127 and sc[0, 0, 0] == 0
    assert kc[1, :4, 0, 0].tolist() == [127, -64, 127, 0]          # -63.5 rounds to even
    R.write(torch.full((1, 1, 64), 2.0).to(torch.bfloat16), kc, sc, [0, 1], [4], table)
    assert sc[1, 0, 0] == torch.tensor(2.0) / 127 and kc[1, :4, 0, 0].tolist() == [64, -32, 64, 127]
    R.write(torch.full((1, 1, 64), 0.25).to(torch.bfloat16), kc, sc, [0, 1], [5], table)
    assert sc[1, 0, 0] == torch.tensor(2.0) / 127 and kc[1, :5, 0, 0].tolist() == [64, -32, 64, 127, 16]


def test_source_of_long_queries():
    """Few rows over many keys read the int8 pages, many rows a copy of the codes (the measured sides of the rule)."""
    elems = lambda keys, h, d=128: keys * h * d  # noqa: E731
    assert bc.direct_pays(8, 256, 128, 256, elems(16384, 4))        # 16 tokens of 16,384 keys, cut
    assert bc.direct_pays(44, 200, 128, 256, elems(1390, 8))        # 776 of 1,390, whole
    assert not bc.direct_pays(55, 500, 128, 256, elems(8192, 4))    # 512 of 8,192, cut
    assert not bc.direct_pays(512, 8192, 128, 256, 4 * elems(16384, 8))
