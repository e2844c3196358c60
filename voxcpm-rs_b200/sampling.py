"""Token sampling from logits (``vx_sample`` of the C ABI), where ``MiniCpmModel.greedy`` picks
the largest."""
from __future__ import annotations

from ._lib import VX_ERR_ARG, VX_ERR_SHAPE, VxError, check, lib
from .minicpm4 import Context, _stream_of, _torch


def sample(ctx: Context, logits, u, temperature=None, top_k=None, top_p=None, min_p=None, return_logprob=False):
    """One id of each row of ``logits`` f32 ``[rows, vocab]`` (rows may be strided) drawn with the
    random numbers ``u`` f32 ``[rows]`` in ``[0, 1)``.  ``temperature``, ``top_p``, ``min_p`` (f32)
    and ``top_k`` (int32) are CUDA tensors of ``rows``, or None for off; they apply in the order
    temperature, top-k, top-p, min-p.  Temperature 0 is the greedy pick.  Returns int32 ids (-1
    for a row without a token to draw), with the log-probability of each under what was left
    when ``return_logprob``."""
    torch = _torch()
    if logits.dtype != torch.float32 or logits.device != torch.device("cuda", ctx.device):
        raise VxError(VX_ERR_ARG, f"logits: f32 on cuda:{ctx.device} is needed, got {logits.dtype} on {logits.device}")
    if logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise VxError(VX_ERR_SHAPE, f"logits: dense rows [rows, vocab] are needed, got {tuple(logits.shape)}")
    rows, vocab = logits.shape
    ptrs = []
    for t, what, dt in ((u, "u", torch.float32), (temperature, "temperature", torch.float32),
                        (top_k, "top_k", torch.int32), (top_p, "top_p", torch.float32),
                        (min_p, "min_p", torch.float32)):
        if t is None and what != "u":
            ptrs.append(None)
            continue
        if t is None or t.dtype != dt or t.device != logits.device or not t.is_contiguous():
            raise VxError(VX_ERR_ARG, f"{what}: a contiguous {dt} tensor on {logits.device} is needed")
        if tuple(t.shape) != (rows,):
            raise VxError(VX_ERR_SHAPE, f"{what}: one value for each of {rows} rows is needed, got {tuple(t.shape)}")
        ptrs.append(t.data_ptr())
    ids = torch.empty(rows, device=logits.device, dtype=torch.int32)
    lp = torch.empty(rows, device=logits.device) if return_logprob else None
    if rows:
        check(lib().vx_sample(ctx.h, logits.data_ptr(), logits.stride(0) if rows > 1 else vocab, rows, vocab, *ptrs,
                              ids.data_ptr(), None if lp is None else lp.data_ptr(), _stream_of(logits)), ctx.h)
    return (ids, lp) if return_logprob else ids
