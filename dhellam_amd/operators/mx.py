"""Microscaled floating point: quantisation to 8 and 4 bits with a power of two a block of 32, and products of such operands.

The reference has no low precision; these operators follow its wrapper convention (``stream=None`` means the current stream,
trailing elapsed-ms return; the product returns its result alone, as ``operators.moe.grouped_gemm_nt`` does).  A projection Y = X W^T in low precision is three products of the one form ``mx_gemm_nt``, each with
both operands quantised along its reduction:

    forward          y  = mx_gemm_nt(x, w)                                        x along its rows, w [out, in] along its rows
    data gradient    dx = mx_gemm_nt(dy, wt)                                      wt = the weight along its columns
    weight gradient  mx_gemm_nt(dy_t, x_t, out=main_grad, accumulate=True)        dy and x along their columns (tokens)

``mx_quantise(..., along="both")`` makes the two copies of a tensor in one pass over it, ``operators.layernorm.pyrmsnorm_mx_fwd`` writes a
norm's result in 8 bits directly.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from .. import _host, _lib
from ._util import issue

FORMATS = {"e4m3": 0, "e2m1": 1}
ALONG = {"rows": 1, "columns": 2, "both": 3}
SCALE_RULES = {"floor": False, "cover": True}


@dataclass
class MXTensor:
    """A rows x cols matrix in microscaled floating point, blocks of 32 along the columns (the OCP MX formats).  Every row is
    filled up to whole groups of 128 columns with zeros.  ``mx_quantise`` and ``pyrmsnorm_mx_fwd`` make codes and scales as two views of one
    allocation: what saves a tensor's whole storage, or refuses tensors that share one, wants ``clone()`` of each."""
    codes: torch.Tensor       # uint8 [rows, kp] (e4m3) or [rows, kp / 2] (e2m1: the even column in the low half), kp = cols rounded up to 128
    scales: torch.Tensor      # uint8 [kp / 128, rows / 4 rounded up, 4, 4]: [c, r // 4, i, r % 4] is the exponent code (2^(e - 127), 255: NaN) of
                              # columns 128 c + 32 i and on of row r; zeros for what is not there
    rows: int
    cols: int
    format: str               # "e4m3" or "e2m1"


def _one_of(what, value, known):
    try:
        return known[value]
    except KeyError:
        raise RuntimeError(f"{what} {value!r} is none of {', '.join(known)}") from None


def mx_quantise(x, format="e4m3", along="rows", scale_rule="floor", stream=None, profiling=False):
    """x [..., cols] (fp32, bf16, fp16; leading dimensions are rows) -> (MXTensor, ms).  ``along="rows"``: blocks of 32 columns of a row;
    ``"columns"``: blocks of 32 rows of a column, the MXTensor being that of the transpose [cols, rows]; ``"both"``: ((of x, of the
    transpose), ms).  ``scale_rule``: "floor" is the rule of the format's specification, the power of two of the largest magnitude
    less that of the format's largest element, under which a block's largest elements may saturate; "cover" the smallest power of two at which
    none does.  Elements are rounded to the nearest, ties to even.  A block that holds anything not finite becomes NaN as a whole."""
    form, way, cover = _one_of("format", format, FORMATS), _one_of("along", along, ALONG), _one_of("scale_rule", scale_rule, SCALE_RULES)
    (c, s, ct, st), ms = issue(_host.mx_quantise, stream, profiling, x, form, way, cover)
    rows, cols = x.shape[:-1].numel(), x.shape[-1]
    q = MXTensor(c, s, rows, cols, format) if c is not None else None
    if ct is None:
        return q, ms
    qt = MXTensor(ct, st, cols, rows, format)
    return (qt if q is None else (q, qt)), ms


def mx_gemm_nt(a, b, out=None, out_dtype=torch.bfloat16, accumulate=False, stream=None):
    """c [m, n] (+)= a @ b.T of two MXTensors, a [m, k] and b [n, k], in either format each.  ``out``: fp32, bf16 or fp16 with unit inner
    stride, added to with ``accumulate`` (one rounding); without it a new tensor of ``out_dtype``.  A NaN block makes its own row (of a) or
    column (of b) NaN.

    Sums are held in fp32.  For 16-bit results the matrix instructions add 8-bit products 16 at a time and drop what lies 2^-13 below the
    largest of them: 2e-5 of the result on normal data, far below its rounding, but not bounded by the result where large products cancel.  fp32 results
    of 8-bit operands are formed from the elements in bf16 instead, to fp32's own accuracy at a third of the speed (elements times their scale below
    2^-126 lose bits there, count as zero below 2^-133 and as infinite from 2^128 on); products of two 4-bit operands are exact either way."""
    if a.cols != b.cols:
        raise RuntimeError(f"mx_gemm_nt: {a.cols} and {b.cols} columns")
    if out is not None:
        _lib.mark_written(out)
    return _host.mx_gemm_nt(a.codes, a.scales, a.rows, _one_of("format", a.format, FORMATS), b.codes, b.scales, b.rows,
                            _one_of("format", b.format, FORMATS), a.cols, out, out_dtype, accumulate, stream)
