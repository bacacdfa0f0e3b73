"""What a step does with its queries and keys before the cache write: the RMS norm of each head's row and its rotation by
position, in one pass (no counterpart in the reference). The results go to any of the package's caches
(cuda_kernels.quant_reshape_and_cache, block_cache.quant_block_cache, fp4_cache.quant_fp4_cache) and attentions.

Enqueued on the current torch stream of the tensors' device, without synchronising the host; capturable in a HIP graph.
"""
import torch

from . import cuda_kernels as ck
from .block_cache import _call
from .cuda_kernels import _check, _check_cuda


def norm_rope(q, k, positions, cos_sin, q_weight=None, k_weight=None, eps=1e-6, interleaved=False, q_out=None, k_out=None):
    """For each token t and head, of q and k (bf16 [T, heads, D], D 64 or 128, strided views as a packed projection leaves them):

        y = x / sqrt(mean(x^2) + eps) * weight              (weights [D], bf16 or float32; both None: y = x)
        (a, b) -> (a cos - b sin, b cos + a sin)            for the pairs of y's first R channels

    cos_sin (float32 or bf16 [positions, R], R a multiple of 16 up to D): row p holds position p's R / 2 cosines, then its sines.
    A pair is (i, i + R / 2), or (2 i, 2 i + 1) where interleaved. positions: int32 or int64 [T]; the rows of a token whose
    position the table does not have are left as they are. float32 throughout, the sum of a row's squares too (so for values
    within 2^-60 .. 2^60, smaller ones where eps is not 0), one rounding. q_out, k_out: where the results go,
    q and k themselves by default (no other overlap). Returns (q_out, k_out)."""
    name = "norm_rope"
    q_out, k_out = q if q_out is None else q_out, k if k_out is None else k_out
    if ck._served(ck.ext(), name, q, k, positions, cos_sin, q_weight, k_weight, eps, interleaved, q_out, k_out):
        return q_out, k_out
    for t, o in ((q, q_out), (k, k_out)):
        _check(t.dim() == 3 and t.dtype == torch.bfloat16 and t.stride(2) == 1 and o.dtype == torch.bfloat16 and
               o.shape == t.shape and o.stride(2) == 1 and t.shape[0] == q.shape[0] and t.shape[2] == q.shape[2],
               f"{name}: q, k and their outputs must be bf16 [T, heads, D] with a contiguous last dim")
    _check(positions.dim() == 1 and positions.dtype in (torch.int32, torch.int64) and positions.is_contiguous() and
           positions.shape[0] == q.shape[0], f"{name}: positions must be a contiguous int32 or int64 vector, one per token")
    _check(cos_sin.dim() == 2 and cos_sin.dtype in (torch.float32, torch.bfloat16) and cos_sin.stride(1) == 1,
           f"{name}: cos_sin must be float32 or bf16 [positions, R] with a contiguous last dim")
    _check((q_weight is None) == (k_weight is None), f"{name}: q_weight and k_weight, or neither")
    for w in (q_weight, k_weight):
        _check(w is None or (tuple(w.shape) == (q.shape[2],) and w.dtype in (torch.float32, torch.bfloat16) and
                             w.dtype == q_weight.dtype and w.is_contiguous()),
               f"{name}: weights must be contiguous [{q.shape[2]}], both float32 or both bf16")
    if q.shape[0] == 0:
        return q_out, k_out
    _check_cuda(name, q, k, positions, cos_sin, q_weight, k_weight, q_out, k_out)
    _call("kvq_norm_rope", q.device, q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1),
          q_out.data_ptr(), q_out.stride(0), q_out.stride(1), k_out.data_ptr(), k_out.stride(0), k_out.stride(1), q.shape[0],
          q.shape[1], k.shape[1], q.shape[2], positions.data_ptr(), 8 * positions.element_size(), cos_sin.data_ptr(),
          cos_sin.stride(0), cos_sin.shape[0], cos_sin.shape[1], int(cos_sin.dtype == torch.bfloat16),
          None if q_weight is None else q_weight.data_ptr(), None if k_weight is None else k_weight.data_ptr(),
          int(q_weight is not None and q_weight.dtype == torch.bfloat16), float(eps), int(bool(interleaved)))
    return q_out, k_out
