"""Token sampling from logits (``vx_sample`` of the C ABI), where ``MiniCpmModel.greedy`` picks
the largest."""
from __future__ import annotations

from ._lib import VX_ERR_ARG, VX_ERR_SHAPE, VxError, check, lib
from .minicpm4 import Context, _torch, raw_stream


def sample(ctx: Context, logits, u, temperature=None, top_k=None, top_p=None, min_p=None, return_logprob=False):
    """One id of each row of ``logits`` f32 ``[rows, vocab]`` (rows may be strided or
    one row expanded) drawn with the
    random numbers ``u`` f32 ``[rows]`` in ``[0, 1)``.  ``temperature``, ``top_p``, ``min_p`` (f32)
    and ``top_k`` (int32) are CUDA tensors of ``rows``, or None for off; they apply in the order
    temperature, top-k, top-p, min-p.  Temperature 0 is the greedy pick.  Returns int32 ids (-1
    for a row without a token to draw), with the log-probability of each under what was left
    when ``return_logprob``."""
    torch = _torch()
    f32, dev = torch.float32, logits.device
    if logits.dtype is not f32 or logits.get_device() != ctx.device:
        raise VxError(VX_ERR_ARG, f"logits: f32 on cuda:{ctx.device} is needed, got {logits.dtype} on {dev}")
    if logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise VxError(VX_ERR_SHAPE, f"logits: dense rows [rows, vocab] are needed, got {tuple(logits.shape)}")
    rows, vocab = logits.shape
    if u is None:
        raise VxError(VX_ERR_ARG, "u: a random number for each row is needed")

    def values(t, what, dt=f32):
        if t is None:
            return None
        if t.dtype is not dt or t.get_device() != ctx.device or not t.is_contiguous():
            raise VxError(VX_ERR_ARG, f"{what}: a contiguous {dt} tensor on {dev} is needed, got {t.dtype} on {t.device}")
        if t.shape != (rows,):
            raise VxError(VX_ERR_SHAPE, f"{what}: one value for each of {rows} rows is needed, got {tuple(t.shape)}")
        return t.data_ptr()

    ptrs = (values(u, "u"), values(temperature, "temperature"), values(top_k, "top_k", torch.int32),
            values(top_p, "top_p"), values(min_p, "min_p"))
    ids = logits.new_empty(rows, dtype=torch.int32)
    lp = logits.new_empty(rows) if return_logprob else None
    if rows:
        rc = lib().vx_sample(ctx.h, logits.data_ptr(), logits.stride(0) if rows > 1 else vocab, rows, vocab, *ptrs,
                             ids.data_ptr(), None if lp is None else lp.data_ptr(), raw_stream(ctx.device))
        if rc:
            check(rc, ctx.h)
    return (ids, lp) if return_logprob else ids
