"""The 4-bit KV cache: rows held as e2m1 codes with an e4m3 scale for each 16 dims
(``vx_kv4_*`` of the C ABI), beside the f32 ``StaticKvCache`` of ``MiniCpmModel``
(``src/minicpm4/cache.rs``) and ``attention_decode``.

Buffers are torch CUDA tensors; calls run on the current stream of the cache's device and
allocate their outputs and workspace there, so they can be captured into a CUDA graph.
"""
from __future__ import annotations

import ctypes as C

from . import _lib
from ._lib import VX_ERR_ARG, VX_ERR_SHAPE, VxError, check, lib
from .minicpm4 import Context, _torch


def _refuse(code, msg):
    raise VxError(code, msg)


def _need(t, what, dtype, shape, index):
    """`t` is a contiguous tensor of this type and shape on cuda:`index`, else the call is refused."""
    if t.dtype is not dtype or t.get_device() != index or not t.is_contiguous():
        _refuse(VX_ERR_ARG, f"{what}: a contiguous {dtype} tensor on cuda:{index} is needed, "
                            f"got {t.dtype} on {t.device}{'' if t.is_contiguous() else ', strided'}")
    if t.shape != shape:
        _refuse(VX_ERR_SHAPE, f"{what}: shape {tuple(shape)} is needed, got {tuple(t.shape)}")


class Kv4Cache:
    """A 4-bit cache of ``batch`` sequences: ``n_kv_heads`` heads of ``capacity`` rows (rounded up
    to a multiple of 32) of ``head_dim`` (64 or 128).  The filled lengths are the caller's: int32
    CUDA tensors of ``batch``, given to each call.  ``weights`` (the attention that each row has
    received) and ``positions`` (int64) are kept with ``track=True``; ``evict`` needs them.  A length
    outside its range leaves its sequence as it was (``attend``: NaN, ``read``: zeros), and the
    context's next ``synchronize`` raises."""

    def __init__(self, ctx: Context, batch, n_kv_heads, capacity, head_dim, track=True):
        torch = _torch()
        dev = torch.device("cuda", ctx.device)
        cap = -(-capacity // 32) * 32
        lead = (batch, n_kv_heads, cap)
        codes = [torch.zeros(*lead, head_dim // 2, device=dev, dtype=torch.uint8) for _ in range(2)]
        scales = [torch.zeros(*lead, head_dim // 16, device=dev, dtype=torch.uint8).view(torch.float8_e4m3fn)
                  for _ in range(2)]
        self._hold(ctx, codes[0], scales[0], codes[1], scales[1],
                   torch.zeros(lead, device=dev, dtype=torch.float32) if track else None,
                   torch.zeros(lead, device=dev, dtype=torch.int64) if track else None)

    @classmethod
    def from_buffers(cls, ctx: Context, k_codes, k_scales, v_codes, v_scales, weights=None, positions=None):
        """A cache over buffers that the caller holds: codes uint8 ``[B, nkv, capacity, d/2]``,
        scales float8_e4m3fn ``[B, nkv, capacity, d/16]``."""
        self = cls.__new__(cls)
        self._hold(ctx, k_codes, k_scales, v_codes, v_scales, weights, positions)
        return self

    def _hold(self, ctx, k_codes, k_scales, v_codes, v_scales, weights, positions):
        torch = _torch()
        if k_codes.dim() != 4:
            _refuse(VX_ERR_SHAPE, "k_codes: [batch, n_kv_heads, capacity, head_dim / 2] is needed")
        b, nkv, cap, half = k_codes.shape
        for t, what in ((k_codes, "k_codes"), (v_codes, "v_codes")):
            _need(t, what, torch.uint8, (b, nkv, cap, half), ctx.device)
        for t, what in ((k_scales, "k_scales"), (v_scales, "v_scales")):
            _need(t, what, torch.float8_e4m3fn, (b, nkv, cap, half // 8), ctx.device)
        for t, what, dt in ((weights, "weights", torch.float32), (positions, "positions", torch.int64)):
            if t is not None:
                _need(t, what, dt, (b, nkv, cap), ctx.device)
        self.ctx, self.device, self._index = ctx, torch.device("cuda", ctx.device), ctx.device
        self.k_codes, self.k_scales, self.v_codes, self.v_scales = k_codes, k_scales, v_codes, v_scales
        self.weights, self.positions = weights, positions
        self.batch, self.n_kv_heads, self.capacity, self.head_dim = b, nkv, cap, 2 * half
        p = [None if t is None else t.data_ptr() for t in (k_codes, k_scales, v_codes, v_scales, weights, positions)]
        self._c = _lib.Kv4C(*p, b, nkv, cap, 2 * half)
        self._ref = C.addressof(self._c)
        self._lens_shape = torch.Size((b,))
        self._plans = {}
        # what every call needs, looked up once: a call of a decode loop is a few microseconds of host time
        self._f32, self._i32 = torch.float32, torch.int32
        # (its new_empty is quicker than torch.empty(device=..))
        self._rows = torch.empty(0, device=k_codes.device, dtype=torch.float32)
        self._L, self._raw_stream = lib(), torch._C._cuda_getCurrentRawStream

    def _ints(self, t, what):
        if t is None:
            return None
        if (t.dtype is not self._i32 or t.get_device() != self._index or t.shape != self._lens_shape
                or not t.is_contiguous()):
            _need(t, what, self._i32, self._lens_shape, self._index)
        return t.data_ptr()

    def append(self, k, v, start, counts=None, first_position=None):
        """Quantise the rows of new tokens into the cache: ``k``, ``v`` f32 ``[B, S, nkv, d]``, the
        last two dims dense (views into a fused projection will do), token ``i < counts[b]`` into
        slot ``start[b] + i``.  Their weights become 0 and their positions
        ``first_position[b] + i`` (the slot without it)."""
        f32 = self._f32
        s = k.shape[1] if k.dim() == 4 else -1
        for t, what in ((k, "k"), (v, "v")):
            if t.shape != (self.batch, s, self.n_kv_heads, self.head_dim):
                _refuse(VX_ERR_SHAPE, f"{what}: [{self.batch}, S, {self.n_kv_heads}, {self.head_dim}] is needed, "
                                      f"got {tuple(t.shape)}")
            if t.dtype is not f32 or t.get_device() != self._index:
                _refuse(VX_ERR_ARG, f"{what}: f32 on {self.device} is needed, got {t.dtype} on {t.device}")
        if s == 0:
            return
        st, sv, many = k.stride(), v.stride(), self.batch > 1
        b_st, t_st = st[0] if many else 0, st[1] if s > 1 else 0  # of one alone the stride may be anything
        alike = st == sv or (sv[3] == 1 and (sv[2] == st[2] or self.n_kv_heads == 1) and (sv[0] == b_st or not many)
                             and (sv[1] == t_st or s == 1))
        if not alike or st[3] != 1 or (st[2] != self.head_dim and self.n_kv_heads != 1):
            _refuse(VX_ERR_ARG, "k and v: dense heads and the same strides are needed")
        rc = self._L.vx_kv4_append(self.ctx.h, self._ref, k.data_ptr(), v.data_ptr(), b_st, t_st, s,
                                   self._ints(start, "start"), self._ints(counts, "counts"),
                                   self._ints(first_position, "first_position"), self._raw_stream(self._index))
        if rc:
            check(rc, self.ctx.h)

    def read(self, n, start=None, counts=None):
        """The values of rows ``start[b] + i`` (``i < counts[b] <= n``; zeros behind them) as
        ``k, v`` f32 ``[B, nkv, n, d]``."""
        if n < 0:
            _refuse(VX_ERR_SHAPE, f"read: {n} rows")
        k, v = self._rows.new_empty((2, self.batch, self.n_kv_heads, n, self.head_dim)).unbind(0)
        if n:
            rc = self._L.vx_kv4_read(self.ctx.h, self._ref, n, self._ints(start, "start"), self._ints(counts, "counts"),
                                     k.data_ptr(), v.data_ptr(), self._raw_stream(self._index))
            if rc:
                check(rc, self.ctx.h)
        return k, v

    def attend(self, q, lens, max_len=None, track=False, scale=None):
        """Attention of one query token of each sequence (``q`` f32 ``[B, nh * d]``, rows may be
        strided) over its first ``lens[b]`` rows; ``lens[b] <= max_len`` (default the capacity; the
        work is split for that length).  Returns ``[B, nh * d]``.  With ``track`` the rows'
        ``weights`` grow by the probabilities that they received."""
        if q.dtype is not self._f32 or q.get_device() != self._index:
            _refuse(VX_ERR_ARG, f"q: f32 on {self.device} is needed, got {q.dtype} on {q.device}")
        batch, d = self.batch, self.head_dim
        if q.dim() != 2 or q.shape[0] != batch or q.shape[1] % d or q.stride(1) != 1:
            _refuse(VX_ERR_SHAPE, f"q: dense rows [{batch}, nh * {d}] are needed, got {tuple(q.shape)}")
        width = q.shape[1]
        n = self.capacity if max_len is None else max_len
        key = (width // d, n, bool(track))
        need = self._plans.get(key)
        if need is None:
            if len(self._plans) >= 1024:  # a max_len that grows with every token
                self._plans.clear()
            need = self._plans[key] = self._L.vx_kv4_attend_workspace(self._ref, *key)
        out = q.new_empty((batch, width))
        ws = self.k_codes.new_empty(need) if need else None
        rc = self._L.vx_kv4_attend(self.ctx.h, self._ref, q.data_ptr(), q.stride(0) if batch > 1 else width, width // d,
                                   self._ints(lens, "lens"), n, d ** -0.5 if scale is None else scale, track,
                                   out.data_ptr(), width, None if ws is None else ws.data_ptr(), need,
                                   self._raw_stream(self._index))
        if rc:
            check(rc, self.ctx.h)
        return out

    def evict(self, lens, seen, keep, sink=0, recent=0, max_len=None, weights_out=None, positions_out=None):
        """Keep the ``keep`` rows of largest weight of each sequence and KV head (rows of a position
        below ``sink`` or not below ``seen[b] - recent`` before all others; ties to the lowest
        slots) and return the new lengths ``min(lens, keep)``.  Kept rows behind slot ``keep`` move
        into the slots that became free; the rows' weights and positions go to ``weights_out`` and
        ``positions_out`` (default: the cache's own)."""
        torch = _torch()
        if self.weights is None or self.positions is None:
            _refuse(VX_ERR_ARG, "evict: the cache keeps no weights and positions")
        wo = self.weights if weights_out is None else weights_out
        po = self.positions if positions_out is None else positions_out
        _need(wo, "weights_out", torch.float32, self.weights.shape, self._index)
        _need(po, "positions_out", torch.int64, self.positions.shape, self._index)
        out = torch.empty(self._lens_shape, device=self.device, dtype=torch.int32)
        rc = self._L.vx_kv4_evict(self.ctx.h, self._ref, self._ints(lens, "lens"), self._ints(seen, "seen"),
                                  self.capacity if max_len is None else max_len, keep, sink, recent, wo.data_ptr(),
                                  po.data_ptr(), out.data_ptr(), self._raw_stream(self._index))
        if rc:
            check(rc, self.ctx.h)
        return out
