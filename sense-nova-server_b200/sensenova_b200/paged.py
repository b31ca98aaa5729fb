"""The paged key/value cache (snl_paged_* of include/snl_b200.h) for hosts that serve many
sequences at once: new rows enter the pages, attend over their sequence, the attention
weight of each slot is added up, and sequences over a budget keep their heaviest slots.

Arguments are device tensors: anything with data_ptr(), shape, stride() and dtype, as
torch.Tensor has. The caller owns every tensor; calls enqueue on `stream` (a CUDA stream
handle; 0 is the default stream) and return, and the tensors have to live until that work
is done. SnlError says what a call refuses; snl_device_error() what only the device saw.
"""
from __future__ import annotations

import ctypes as C
import struct
from typing import Any

from . import ffi
from .ffi import PagedBatchC, PagedCacheC, PagedEvictP, SnlError

ONE, SECTIONS, INTERLEAVED = 0, 1, 2  # which axis of a position turns which pair
HALVES, ADJACENT = 0, 1  # which elements form a pair
_TYPES = {"float32": ffi.SNL_T_F32, "float16": ffi.SNL_T_F16, "bfloat16": ffi.SNL_T_BF16}
_type_of: dict[Any, int] = {}
_is_int: dict[Any, bool] = {}
# snl_paged_append_p and snl_paged_attn_p, packed anew for each call: 0.15 us where a ctypes
# structure of as many fields takes 1.4 us to make, most of what a small call costs here.
_APPEND = struct.Struct("@9If8Q").pack
_ATTN = struct.Struct("@3Q2I2f2I6Q").pack
# snl_paged_batch and snl_paged_evict_p: a ctypes field would take a number's low 32 bits.
_BATCH = struct.Struct("@3Q4I").pack
_EVICT = struct.Struct("@4I").pack


def _type(t) -> int:
    """SNL_T_* of a tensor."""
    code = _type_of.get(t.dtype)
    if code is None:
        name = str(t.dtype).rsplit(".", 1)[-1]
        if name not in _TYPES:
            raise SnlError(ffi.SNL_E_UNSUPPORTED, f"paged cache: tensors of {name}")
        code = _type_of[t.dtype] = _TYPES[name]
    return code


def _fail(what: str):
    raise SnlError(ffi.SNL_E_INVALID, "paged cache: " + what)


def _need(ok: bool, what: str) -> None:
    if not ok:
        _fail(what)


def _ints(t, what: str, *shape: int) -> int:
    """The address of a contiguous tensor of 32-bit integers of that shape."""
    kind = t.dtype
    if kind not in _is_int:
        _is_int[kind] = str(kind).endswith("int32")
    if not (_is_int[kind] and t.shape == shape and t.is_contiguous()):
        _fail(f"{what} must be contiguous 32-bit integers of shape {shape}")
    return t.data_ptr()


def _floats(t, what: str, *shape: int) -> int | None:
    if t is None:
        return None
    if _type(t) != 0 or t.shape != shape or not t.is_contiguous():
        _fail(f"{what} must be contiguous float32 of shape {shape}")
    return t.data_ptr()


class PagedBatch:
    """One step's rows: rows start[b] .. start[b + 1] - 1 are the newest tokens of sequence
    b, whose slots lie in the pages table[b] and number lens[b] with them. table [seqs,
    pages], start [seqs + 1] and lens [seqs] are int32 on the device and may change between
    calls; n_rows and max_len (at least every length) are the host's."""

    def __init__(self, table, start, lens, n_rows: int, max_len: int):
        seqs, width = table.shape
        self.tensors = (table, start, lens)
        self.n_seqs, self.n_rows, self.max_len = seqs, n_rows, max_len
        try:
            self.c = PagedBatchC.from_buffer_copy(_BATCH(_ints(table, "table", seqs, width), _ints(start, "start", seqs + 1),
                                                         _ints(lens, "lens", seqs), seqs, n_rows, width, max_len))
        except struct.error as e:
            _fail(f"the batch's numbers: {e}")
        self.ref = C.byref(self.c)


class PagedCache:
    """Pages of keys and values [pages, kv heads, slots, head_dim] in f16 or bf16, as views of
    either layout, and their accumulated attention weights [pages, kv heads, slots] in f32."""

    def __init__(self, k, v, weight=None):
        self.lib = ffi.load()
        pages, n_kv, slots, d = k.shape
        _need(tuple(v.shape) == tuple(k.shape) and v.stride() == k.stride() and v.dtype == k.dtype,
              "k and v must have the same shape, strides and type")
        _need(k.stride(3) == 1, "the last dimension must be contiguous")
        self.type, self.n_kv, self.head_dim, self.page_size = _type(k), n_kv, d, slots
        self.tensors = (k, v, weight)
        self.c = PagedCacheC(k.data_ptr(), v.data_ptr(), _floats(weight, "weight", pages, n_kv, slots), k.stride(0),
                             k.stride(1), k.stride(2), self.type, pages, slots, n_kv, d, 0)
        self.ref = C.byref(self.c)

    def _rows(self, t, what: str, batch: PagedBatch, heads: int) -> tuple[int, int, int]:
        """Address and row and head strides of [rows, heads, head_dim]."""
        if t.shape == (batch.n_rows, heads, self.head_dim):
            row, head, one = t.stride()
        else:
            one = 0
        if one != 1:
            _fail(f"{what} must be [{batch.n_rows}, {heads}, {self.head_dim}] with a contiguous last dimension")
        return t.data_ptr(), row, head

    def append(self, batch: PagedBatch, q, k, v, q_out, pos=None, rope=None, *, axes: int = ONE, pairs: int = HALVES,
               sections=(0, 0, 0), q_norm=None, k_norm=None, eps: float = 1e-6, stream: int = 0) -> None:
        """New rows enter the cache (snl_paged_append). q [rows, heads, d] or None, k and v
        [rows, kv heads, d] in f32 or the cache's type, any row and head strides; q_out like
        q in the cache's type. pos [rows, 4] 32-bit integers (time, height, width, 0) and
        rope [positions, rot / 2, 2] turn the first rot elements; None turns nothing."""
        d = self.head_dim
        kp, k_row, k_head = self._rows(k, "k", batch, self.n_kv)
        vp, v_row, v_head = self._rows(v, "v", batch, self.n_kv)
        kind = k.dtype
        if v.dtype != kind or (q is not None and q.dtype != kind):
            _fail("q, k and v must have one type")
        qp = op = tp = rp = None
        heads = q_row = q_head = out_row = out_head = rot = n_pos = 0
        if q is not None:
            heads = q.shape[1]
            qp, q_row, q_head = self._rows(q, "q", batch, heads)
            op, out_row, out_head = self._rows(q_out, "q_out", batch, heads)
            _need(_type(q_out) == self.type, "q_out must have the cache's type")
        if rope is not None:
            n_pos, half, two = rope.shape
            _need(two == 2 and pos is not None, "rope must be [positions, rot / 2, 2] and pos be given")
            rot = 2 * half
            rp, tp = _floats(rope, "rope", n_pos, half, 2), _ints(pos, "pos", batch.n_rows, 4)
        if len(sections) != 3:
            _fail("sections must be the numbers of pairs of the three axes")
        try:
            p = _APPEND(heads, _type(k), rot, axes, pairs, n_pos, *sections, eps, q_row, q_head, k_row, k_head, v_row, v_head,
                        out_row, out_head)
        except struct.error as e:
            _fail(f"append's numbers: {e}")
        rc = self.lib.snl_paged_append(self.ref, batch.ref, p, qp, kp, vp, _floats(q_norm, "q_norm", d),
                                       _floats(k_norm, "k_norm", d), tp, rp, op, stream)
        if rc:
            ffi.check(rc)

    def _query(self, batch: PagedBatch, q) -> tuple[int, int, int]:
        at = self._rows(q, "q", batch, q.shape[1])
        if _type(q) != self.type:
            _fail("q must have the cache's type")
        return at

    def _attn(self, batch: PagedBatch, heads, scale, cap, window, slopes, first, last, *types_and_strides: int) -> bytes:
        """snl_paged_attn_p; types_and_strides: gate's and out's type, and q's, gate's and out's strides."""
        try:
            return _ATTN(_floats(slopes, "slopes", heads) or 0, 0 if first is None else _ints(first, "first", batch.n_rows),
                         0 if last is None else _ints(last, "last", batch.n_rows), heads, window,
                         self.head_dim ** -0.5 if scale is None else scale, cap, *types_and_strides)
        except (struct.error, OverflowError) as e:
            _fail(f"the attention's numbers: {e}")

    def attend_workspace(self, batch: PagedBatch, heads: int) -> int:
        """Bytes of scratch that attend needs for such a batch."""
        return self.lib.snl_paged_attend_workspace(self.ref, batch.ref, heads)

    def attend(self, batch: PagedBatch, q, out, work, *, lse=None, gate=None, scale: float | None = None,
               cap: float = 0.0, window: int = 0, slopes=None, first=None, last=None, stream: int = 0) -> None:
        """The rows attend over their sequences (snl_paged_attend): q [rows, heads, d] in the
        cache's type, out and gate like it in any type, lse [rows, heads] f32, work a
        contiguous tensor of scratch bytes. first, last [rows] int32 and slopes [heads] f32
        are the masks and the distance bias; scale is 1 / sqrt(d) unless given."""
        heads = q.shape[1]
        qp, q_row, q_head = self._query(batch, q)
        op, out_row, out_head = self._rows(out, "out", batch, heads)
        gp, gate_type, gate_row, gate_head = None, 0, 0, 0
        if gate is not None:
            gp, gate_row, gate_head = self._rows(gate, "gate", batch, heads)
            gate_type = _type(gate)
        if not work.is_contiguous():  # its elements are counted below, which an expanded view does not hold
            _fail("work must be contiguous")
        p = self._attn(batch, heads, scale, cap, window, slopes, first, last, gate_type, _type(out), q_row, q_head,
                       gate_row, gate_head, out_row, out_head)
        rc = self.lib.snl_paged_attend(self.ref, batch.ref, p, qp, gp, op,
                                       _floats(lse, "lse", batch.n_rows, heads), work.data_ptr(),
                                       work.numel() * work.element_size(), stream)
        if rc:
            ffi.check(rc)

    def weigh(self, batch: PagedBatch, q, lse, *, decay: float = 1.0, scale: float | None = None, cap: float = 0.0,
              window: int = 0, slopes=None, first=None, last=None, stream: int = 0) -> None:
        """weight = decay * weight + what the rows' attention (with attend's lse) gave each
        slot, per KV head (snl_paged_weigh)."""
        heads = q.shape[1]
        qp, q_row, q_head = self._query(batch, q)
        p = self._attn(batch, heads, scale, cap, window, slopes, first, last, 0, 0, q_row, q_head, 0, 0, 0, 0)
        rc = self.lib.snl_paged_weigh(self.ref, batch.ref, p, qp,
                                      _floats(lse, "lse", batch.n_rows, heads), decay, stream)
        if rc:
            ffi.check(rc)

    def evict(self, batch: PagedBatch, budget: int, kept, into=None, new_lens=None, *, sink: int = 0, recent: int = 0,
              stream: int = 0) -> None:
        """Sequences of more than `budget` slots keep `budget` per KV head (snl_paged_evict):
        the first sink, the last recent and the heaviest others, moved in order to the pages
        into [seqs, pages], or in place. kept [seqs, kv heads, budget] and new_lens [seqs]
        receive the kept slots and the lengths; in place new_lens defaults to the batch's."""
        seqs = batch.n_seqs
        ip, width = None, 0
        if into is not None:
            width = into.shape[1]
            ip = _ints(into, "into", seqs, width)
            _need(new_lens is not None, "new_lens is needed with new pages")
        try:
            p = PagedEvictP.from_buffer_copy(_EVICT(budget, sink, recent, width))
        except struct.error as e:
            _fail(f"evict's numbers: {e}")
        lp = batch.c.len if new_lens is None else _ints(new_lens, "new_lens", seqs)
        rc = self.lib.snl_paged_evict(self.ref, batch.ref, p, _ints(kept, "kept", seqs, self.n_kv, budget), ip,
                                      lp, stream)
        if rc:
            ffi.check(rc)


def rope_table(out, theta: float, stream: int = 0) -> None:
    """Fill out [positions, rot / 2, 2] with (cos, sin) of pos * theta^(-2f / rot)
    (snl_rope_table)."""
    n, half, two = out.shape
    _need(two == 2, "rope must be [positions, rot / 2, 2]")
    ffi.check(ffi.load().snl_rope_table(theta, 2 * half, n, _floats(out, "rope", n, half, 2), stream))
