"""Host-side proofs for the block-scaled cache: what its kernels compute that also compiles for the host, and what the
write leaves of a value."""
from test_arith import _run_c


def test_a_last_pieces_denominator_comes_back_whole(tmp_path):
    """piece_sum.h: the mark of a cut row's last piece takes nothing from its denominator, however small."""
    rc, out = _run_c(tmp_path, "piece_sum_check")
    assert rc == 0 and out.endswith("mismatched 0"), out
