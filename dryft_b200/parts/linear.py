"""``y = x @ W.T`` for the weights of the parts (all ``[out, in]``, no bias — ``OPTIMIZATION_GUIDE.md:117``;
``engine/dryft_qwen3/config.py:138``).

Which product runs:
  * 32-bit activations (the 32-bit path): the hand-written CUDA-core product, true fp32;
  * bfloat16, few rows (decode): the hand-written weight-streaming tensor-core products -- through registers into
    mma.sync up to ``small_m_max`` rows, by TMA into tcgen05.mma up to ``stream_m_max`` (64);
  * bfloat16, many rows (prefill): cuBLAS through ``torch.mm``, 32-bit accumulation — the library
    product the reference itself uses (``F.linear``, ``engine/dryft_qwen3/model.py:153,179,180``);
  * bfloat16 activations with a weight the checkpoint stores in 32-bit: the weight stays 32-bit,
    the activations are widened, the 32-bit product runs and its result is rounded once;
  * weights held in 4 bits (``ops.kernels.Weight4``): up to 256 rows of bfloat16 (64 of float32) the kernels that
    read the codes, above that the weights are taken out of their 4 bits for the products above;
  * weights in microscaled 4-bit floating point (``ops.kernels.Fp4``): the activations' rows are rounded to it too, and
    tcgen05.mma multiplies both as they are held, whatever their number.
"""

from __future__ import annotations

from typing import Optional

import torch

from ..ops import kernels as K
from .base import Runtime, fused_rms


def linear(x: torch.Tensor, w: torch.Tensor, rt: Runtime, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    out_dtype = out_dtype or x.dtype
    m, k = x.shape
    n = w.shape[0]
    if w.shape[1] != k:
        raise ValueError(f"linear: activations have width {k}, weight is {tuple(w.shape)}")
    if isinstance(w, K.Weight4):
        return _linear4(x, w, rt, out_dtype)
    if isinstance(w, K.Fp4):
        return K.linear_fp4(x, w, pdl=rt.pdl, out_dtype=out_dtype)
    if x.dtype == torch.float32:
        if w.dtype != torch.float32:
            raise ValueError(f"linear: 32-bit activations need a 32-bit weight, got {w.dtype}")
        out = torch.empty((m, n), dtype=torch.float32, device=x.device)
        K.gemm_nt_f32(x, w, out, pdl=rt.pdl)
        return out if out_dtype == torch.float32 else out.to(out_dtype)
    if x.dtype != torch.bfloat16:
        raise ValueError(f"linear: activations are float32 or bfloat16, got {x.dtype}")
    if w.dtype == torch.float32:
        out = torch.empty((m, n), dtype=torch.float32, device=x.device)
        K.gemm_nt_f32(x.to(torch.float32), w, out)
        return out if out_dtype == torch.float32 else out.to(out_dtype)
    if w.dtype != torch.bfloat16:
        raise ValueError(f"linear: weight dtype {w.dtype} is not supported")
    if K.fused_rows_supported(m, k, rt.small_m_max, 0, normed=True):   # above 8 rows: the narrow widths only
        out = torch.empty((m, n), dtype=out_dtype, device=x.device)
        # A programmatic dependent: its blocks start, and request their first weights, once every block of the launch before it
        # runs (the kernels that stand in front of products say so at their start).  A decode step of the 2,048-wide Vobusun shape
        # has 51 such products of about 6 us: a prompt of 1,300 tokens and 16 steps take 16.3 ms instead of 17.6.
        K.gemm_small_m(x, w, out, pdl=rt.pdl)
        return out
    if m <= min(rt.stream_m_max, K.STREAM_M_LIMIT) and K.gemm_stream_supported(m, k) and rt.tcgen05:
        out = torch.empty((m, n), dtype=out_dtype, device=x.device)
        K.gemm_stream(x, w, out)
        return out
    if out_dtype == torch.bfloat16:
        return torch.mm(x, w.t())
    return torch.mm(x, w.t(), out_dtype=out_dtype)


def held(w: torch.Tensor, rt: Runtime):
    """A part's matrix as the engine holds it: as loaded, or in 4 bits, as whole numbers or as microscaled floating point."""
    if rt.weight_bits != 4:
        return w
    return K.fp4_quantise(w, rt.weight_format) if rt.weight_format in K.FP4_KINDS else K.pack_weight4(w, K.bits4_group(w.shape[1], rt.bits_group))


def four_bits_fuse(n_rows: int, norm, rt: Runtime, *weights) -> bool:
    """Whether the norm before a step's products with 4-bit weights (the first one's inputs are the normed rows), and the sums behind them, are the products' own work."""
    return (rt.fuse_decode and rt.is_bf16 and n_rows <= K.LINEAR4_NORM_ROWS and n_rows * weights[0].k <= K.LINEAR4_NORM_NUMBERS and fused_rms(norm) is not None
            and all(K.linear4_fuses(n_rows, w) for w in weights))


EXPAND_BYTES = 256 << 20   # of weights at a time that a product of many rows takes out of their 4 bits (which bounds what that holds)


# Inputs that a product of many rows with a 32-bit result sums on the tensor cores at a time, which cut sums off, not round them, always towards zero (300 rows, 12,288
# inputs: off by 14 millionths of the whole in one piece, 1 in twelve, 32-bit multiply-adds in order 2).  777 rows, 24,576 outputs of 4,096 inputs: 436 us (379 in one piece);
# 300 rows, 151,936 of 2,560: 1,034 (1,014).
SUMMED = 1024


def _linear4(x: torch.Tensor, w: K.Weight4, rt: Runtime, out_dtype: torch.dtype) -> torch.Tensor:
    """Up to ``K.LINEAR4_ROWS`` rows the kernels read the codes; more rows take the weights out of their 4 bits, for the product that such rows run on
    otherwise.  For 32-bit results from bfloat16 activations the weights are taken out as two bfloat16 numbers whose sum they are, with a product each."""
    if x.dtype == torch.float32 and out_dtype != torch.float32:   # as other weights: the 32-bit product, rounded once
        return _linear4(x, w, rt, torch.float32).to(out_dtype)
    m = x.shape[0]
    if m <= (K.LINEAR4_ROWS if x.dtype == torch.bfloat16 else K.LINEAR4_ROWS_F32):
        return K.linear4(x, w, pdl=rt.pdl, out_dtype=out_dtype)
    n, k = w.shape
    out = torch.empty((m, n), dtype=out_dtype, device=x.device)
    step = max(16, EXPAND_BYTES // (k * x.element_size()) // 16 * 16)
    buf = torch.empty(((min(step, n) + 15) // 16 * 16, k), dtype=x.dtype, device=x.device)
    # Rows of results that begin anywhere send the library to a product that cuts the sums over the inputs and adds the parts up in bfloat16 (685 rows, 439 outputs of
    # 8,496 inputs: off by 0.0044 of the whole instead of 0.0017, and 108 us instead of 13).  It is given whole tiles of 16 outputs then, and what they are copied.
    whole = x.dtype == torch.float32 or n % 8 == 0
    # (an infinity's product with a weight's rest may be the opposite of its product with the weight, or NaN: the rests take their part in finite numbers only)
    finite = torch.nan_to_num(x, nan=0.0, posinf=0.0, neginf=0.0) if out_dtype == torch.float32 and x.dtype == torch.bfloat16 else x
    for first in range(0, n, step):
        end = min(n, first + step)
        rows, at = w if end - first == n else w.rows(first, end), out[:, first:end]
        part = buf[:end - first]
        K.weight4_expand(rows, part)
        if x.dtype == torch.float32:
            y = at if end - first == n else torch.empty((m, end - first), dtype=torch.float32, device=x.device)
            K.gemm_nt_f32(x, part, y)
            if y is not at:
                at.copy_(y)
            continue
        wide = part if whole else buf[:(end - first + 15) // 16 * 16]
        if out_dtype == torch.bfloat16 and whole:
            torch.mm(x, wide.t(), out=at)
        elif out_dtype == torch.bfloat16:
            at.copy_(torch.mm(x, wide.t())[:, :end - first])
        else:
            y = at if whole else torch.empty((m, wide.shape[0]), dtype=out_dtype, device=x.device)
            torch.mm(x[:, :SUMMED], wide[:, :SUMMED].t(), out_dtype=out_dtype, out=y)
            for at_k in range(SUMMED, k, SUMMED):
                torch.addmm(y, x[:, at_k:at_k + SUMMED], wide[:, at_k:at_k + SUMMED].t(), out_dtype=out_dtype, out=y)
            K.weight4_expand(rows, part, rest=True)
            torch.addmm(y, finite, wide.t(), out_dtype=out_dtype, out=y)
            if not whole:
                at.copy_(y[:, :end - first])
    return out


def fusable_rows(n_rows: int, k: int, rt: Runtime, normed: bool = False) -> bool:
    """Whether the fused decode products take ``n_rows`` rows over ``k`` inputs (``normed``: with a norm on the way in)."""
    return K.fused_rows_supported(n_rows, k, rt.small_m_max, rt.stream_m_max if rt.tcgen05 else 0, normed)


def weighted_for(next_norm, width: int, k_in: int, rt: Runtime, n_rows: int = 1) -> bool:
    """Whether a fused decode product of ``k_in`` inputs that updates a stream of ``width`` should also leave
    the stream weighted for ``next_norm`` (an RMS norm over ``width``): both it and the product behind that
    norm must be of the form compiled per inner size (which takes up to ``small_m_max`` rows)."""
    rms = fused_rms(next_norm) if next_norm is not None else None
    return (rms is not None and rt.norm_ahead and rt.is_bf16 and rms[0].numel() == width
            and n_rows <= min(rt.small_m_max, K.SMALL_M_LIMIT)
            and K.weighted_ahead_supported(width) and K.weighted_ahead_supported(k_in))
