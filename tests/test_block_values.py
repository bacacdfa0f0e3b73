"""Host-side proofs for the block-scaled cache: what its kernels compute that also compiles for the host, and what the
write leaves of a value."""
import pytest
import torch

import block_ref as R
from kvq import block_cache as bc
from kvq import cuda_kernels as ck
from test_arith import _run_c


def test_a_last_pieces_denominator_comes_back_whole(tmp_path):
    """piece_sum.h: the mark of a cut row's last piece takes nothing from its denominator, however small."""
    rc, out = _run_c(tmp_path, "piece_sum_check")
    assert rc == 0 and out.endswith("mismatched 0"), out


@pytest.mark.parametrize("copies", [True, False])
@pytest.mark.parametrize("query,keys,copied", [(1500, 2000, True), (16384, 16384, True), (16, 300, False)])
def test_source_of_a_capture_without_a_work_list(query, keys, copied, copies, monkeypatch):
    """A program that made a plan's device copies itself and then captures its first call: the source follows from the rows'
    key tiles, as in any call (a copy of the codes for many rows), where the pages' lists are there."""
    class Library:
        prefill_rows, prefill_max_parts = 128, 64

    ran = []
    monkeypatch.setattr(ck, "_EXT", Library())
    monkeypatch.setattr(ck, "_served", lambda e, name, *a: ran.append(a[17:]) or True)
    monkeypatch.delenv("KVQ_PREFILL_DIRECT", raising=False)
    plan = ck.plan_long([0, query], [keys], 16)
    plan.tiles(7, "cpu")
    if copies:
        plan.gpu("cpu")
    monkeypatch.setattr(ck, "_capturing", lambda device: True)
    monkeypatch.setattr(ck, "_to_device", lambda *a: pytest.fail("a copy inside the capture"))
    kc, vc = R.new_cache(4, 16, 4, 128, "vllm")
    q = torch.zeros(1, 28, 128, dtype=torch.bfloat16).expand(query, 28, 128)
    cu, lens = torch.tensor([0, query], dtype=torch.int32), torch.tensor([keys], dtype=torch.int32)
    bc.block_long_attention(q, kc, vc, q, cu, lens, torch.zeros(1, 4, dtype=torch.int32), plan, 0.1, bc.block_scales(4, 16, 4, 16, "cpu"))
    (src,) = ran
    assert len(src) == 3 and (src[0] is not None) == (copied and copies)


@pytest.mark.parametrize("group", [16, 64])
@pytest.mark.parametrize("step", [1, 3, 64])
def test_a_cached_value_and_the_row_that_went_in(group, step):
    """However a prompt is cut into steps, a cached value is off its bf16 row by at most half a step of the scale it was
    quantized with and half a step of each larger one its block took since."""
    n, h, d, bs = 150, 2, 64, 64
    g = torch.Generator().manual_seed(step)
    x = (torch.randn(n, h, d, generator=g) * (0.2 + 3 * torch.rand(n, 1, 1, generator=g))).to(torch.bfloat16)
    cache, _ = R.new_cache(4, bs, h, d, "apart")
    scale, table = torch.zeros(4, h, bs // group), torch.tensor([[2, 0, 3]])
    off, held = torch.zeros(n, h), 0
    while held < n:
        m = min(step, n - held)
        _, before = R.values(cache, scale, table[0], n)
        R.write(x[held:held + m], cache, scale, [0, m], [held + m], table)
        held += m
        codes, s = R.values(cache, scale, table[0], n)
        grew = (s != before).t()                                    # [n, H]: new rows, and those behind whom a scale grew
        grew[held - m:held] = True
        off += torch.where(grew, s.t() / 2, torch.zeros_like(off)).float()
        off[held:] = 0
    got = (codes * s[..., None]).transpose(0, 1)
    assert bool(((got - x.double()).abs() <= off.double()[..., None] * (1 + 1e-4)).all())
