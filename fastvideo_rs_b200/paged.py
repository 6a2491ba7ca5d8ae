"""A paged K/V cache for streaming generation: appending a ragged batch's keys and values (rotated on the way) to pages of
bf16 or of 4 bits, reading rows back, and attention over the pages with a sliding window and sink tokens.

`wan.CausalKvCache` keeps one contiguous buffer per sequence and rolls it by copying; here a sequence is a list of pages, so
a window slides by handing pages back, sequences of any lengths share one pool, query heads may share K/V heads, and
4-bit pages take little more than a quarter of the memory.  One `PagedKv` is one layer's pool; one `PagedBatch` says where
the sequences of a call lie in it and serves every layer that uses the same tables."""
from __future__ import annotations

import ctypes
import struct
from typing import Optional, Tuple

import torch

from . import _lib
from .sdpa import BlockCausal

FORMATS = ("bf16", "q4")
PAIRINGS = {"interleaved": 0, "half": 1}
D = 128
_vp, _int = ctypes.c_void_p, ctypes.c_int
# fv_paged_rows and fv_paged_query, packed: one bytes object is a fifth of what twenty ctypes arguments cost a call.
_rows_struct = struct.Struct("@7P6q4i")
_query_struct = struct.Struct("@3PN2q6if")


class _KvC(ctypes.Structure):
    _fields_ = [("k", _vp), ("v", _vp), ("k_scale", _vp), ("v_scale", _vp), ("format", _int), ("pages", _int),
                ("page_rows", _int), ("kv_heads", _int)]


class _BatchC(ctypes.Structure):
    _fields_ = [("page_table", _vp), ("kv_len", _vp), ("cu_q", _vp), ("seqs", _int), ("table_width", _int),
                ("max_q", _int), ("max_kv", _int)]


# (the handle of the current stream without building a Stream object around it, where torch offers that)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)
_fns = None


def _entries():
    """The C entries with their argument types declared once: a decode step calls them for every layer, and untyped
    ctypes arguments cost more than the launch."""
    global _fns
    if _fns is None:
        L = _lib.lib()
        L.fv_paged_append_bf16.argtypes = [_vp, _vp, _vp, _vp]
        L.fv_paged_read_bf16.argtypes = [_vp, _vp, _vp, _vp, _vp, _int, _vp, _vp]
        L.fv_paged_attn_workspace_bytes.argtypes = [_vp, _vp, _vp]
        L.fv_paged_attn_workspace_bytes.restype = ctypes.c_size_t
        L.fv_paged_attn_bf16.argtypes = [_vp, _vp, _vp, _vp]
        _fns = (L.fv_paged_append_bf16, L.fv_paged_read_bf16, L.fv_paged_attn_workspace_bytes, L.fv_paged_attn_bf16)
    return _fns


def _index(name: str, t: torch.Tensor, shape: Tuple[int, ...], device) -> torch.Tensor:
    if not t.is_cuda or t.device != device or t.dtype != torch.int32 or not t.is_contiguous() or tuple(t.shape) != shape:
        raise ValueError(f"{name} must be a contiguous int32 tensor {list(shape)} on {device}")
    return t


class PagedKv:
    """The pool of one layer.  bf16 pages: k, v [pages, kv_heads, page_rows, 128] bf16.  4-bit pages: k, v [pages, kv_heads,
    page_rows, 64] uint8 (value 2 i in the low half of byte i, as code + 8) and k_scale, v_scale [pages, kv_heads,
    page_rows, 2] bf16 = (step, zero): a row stands for zero + step * code.  page_rows 16, 32, 64, 128 or 256."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: Optional[torch.Tensor] = None,
                 v_scale: Optional[torch.Tensor] = None):
        if k.dim() != 4 or k.dtype not in (torch.bfloat16, torch.uint8):
            raise ValueError("PagedKv: k must be [pages, kv_heads, page_rows, 128] bf16 or [.., 64] uint8")
        q4 = k.dtype == torch.uint8
        if k.shape[3] != (D // 2 if q4 else D) or v.shape != k.shape or v.dtype != k.dtype:
            raise ValueError("PagedKv: k and v must be [pages, kv_heads, page_rows, 128] bf16 or [.., 64] uint8")
        if k.shape[2] not in (16, 32, 64, 128, 256):
            raise ValueError(f"PagedKv: pages of {k.shape[2]} rows (16, 32, 64, 128 or 256)")
        if q4 != (k_scale is not None) or q4 != (v_scale is not None):
            raise ValueError("PagedKv: 4-bit pages have scales, bf16 pages have none")
        for name, t in (("k", k), ("v", v), ("k_scale", k_scale), ("v_scale", v_scale)):
            if t is None:
                continue
            if not t.is_cuda or t.device != k.device or not t.is_contiguous():
                raise ValueError(f"PagedKv: {name} must be a contiguous CUDA tensor on one device: this package has no CPU path")
            if name.endswith("scale") and (t.dtype != torch.bfloat16 or t.shape != (*k.shape[:3], 2)):
                raise ValueError(f"PagedKv: {name} must be bf16 [pages, kv_heads, page_rows, 2]")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.format = "q4" if q4 else "bf16"
        self.pages, self.kv_heads, self.page_rows = k.shape[:3]
        self.device, self.index = k.device, k.get_device()
        ptr = lambda t: t.data_ptr() if t is not None else None
        self._c = _KvC(ptr(k), ptr(v), ptr(k_scale), ptr(v_scale), int(q4), self.pages, self.page_rows, self.kv_heads)
        self._ref = ctypes.addressof(self._c)

    @staticmethod
    def empty(pages: int, page_rows: int, kv_heads: int, format: str = "bf16", device="cuda") -> "PagedKv":
        """A pool of its own; the memory is not cleared (rows are read only after they were appended)."""
        if format not in FORMATS:
            raise ValueError(f"PagedKv: unknown format {format!r} {FORMATS}")
        mk = lambda width, dtype: torch.empty((pages, kv_heads, page_rows, width), dtype=dtype, device=device)
        if format == "bf16":
            return PagedKv(mk(D, torch.bfloat16), mk(D, torch.bfloat16))
        return PagedKv(mk(D // 2, torch.uint8), mk(D // 2, torch.uint8), mk(2, torch.bfloat16), mk(2, torch.bfloat16))


class PagedBatch:
    """The sequences of a call.  page_table [seqs, width] int32: the page of rows i * page_rows .. of each sequence (entries
    that the call does not need may be -1).  kv_len [seqs] int32: tokens of each sequence, those of this call included.
    cu_q [seqs + 1] int32, ascending from 0: rows cu_q[s] .. cu_q[s + 1] of the packed operands are the last tokens of
    sequence s.  max_q and max_kv bound the tokens and lengths; the tensors may change under a captured graph as long as they
    keep to them (but bounds far above what a call holds cost time, since they are what its kernel is chosen and laid out by: one token of each
    of 16 sequences of 4 000 keys, 32 heads on 8, bf16, 39 us with max_q 1, 65 with 256, 143 with 4 096).  Rows of an operand from cu_q[seqs] on
    belong to no sequence: outputs leave them as they were (an output that the call allocates holds anything there)."""

    def __init__(self, page_table: torch.Tensor, kv_len: torch.Tensor, cu_q: torch.Tensor, *, max_q: int, max_kv: int):
        if page_table.dim() != 2:
            raise ValueError("PagedBatch: page_table must be [seqs, width]")
        seqs, width = page_table.shape
        dev = page_table.device
        self.page_table = _index("PagedBatch: page_table", page_table, (seqs, width), dev)
        self.kv_len = _index("PagedBatch: kv_len", kv_len, (seqs,), dev)
        self.cu_q = _index("PagedBatch: cu_q", cu_q, (seqs + 1,), dev)
        if not 0 <= max_q < 1 << 30 or not 0 <= max_kv < 1 << 30:
            raise ValueError("PagedBatch: max_q and max_kv must be 0 .. 2^30 - 1")
        self.seqs, self.max_q, self.max_kv, self.device, self.index = seqs, int(max_q), int(max_kv), dev, page_table.get_device()
        self._need = {}  # scratch bytes by the call's shape: a step asks for every layer
        self._c = _BatchC(page_table.data_ptr(), kv_len.data_ptr(), cu_q.data_ptr(), seqs, width, self.max_q, self.max_kv)
        self._ref = ctypes.addressof(self._c)


_bf16, _f32, _SCALE = torch.bfloat16, torch.float32, D ** -0.5


def _refuse(name: str, t: torch.Tensor, index: int, tokens: int = -1, heads: int = -1) -> None:
    """Says why t is not bf16 [tokens, heads, 128] on device `index` (-1: any number of tokens or heads)."""
    if t.get_device() != index:
        raise ValueError(f"{name} must be a CUDA tensor on cuda:{index}: this package has no CPU path")
    if t.dtype != _bf16 or t.dim() != 3 or t.shape[2] != D or (t.stride(2) != 1 and t.numel() > 0):
        raise ValueError(f"{name} must be bfloat16 [tokens, heads, 128] with adjacent values")
    raise ValueError(f"{name} is {list(t.shape)}: {tokens} tokens of {heads} heads are wanted")


def _heads_in(name: str, t: torch.Tensor, index: int, tokens: int = -1, heads: int = -1) -> Tuple[int, int, int, int]:
    """(tokens, heads, their strides) of a bf16 [tokens, heads, 128] tensor; the stride of an extent of one means nothing and
    counts as a row's.  (Reads each property once: a decode step passes here for every layer, and the time between two
    launches is what it costs.)"""
    shape = t.shape
    if len(shape) != 3 or t.dtype is not _bf16 or t.get_device() != index:
        _refuse(name, t, index)
    n, h, d = shape
    a, b, c = t.stride()
    if d != D or (c != 1 and n * h) or (tokens >= 0 and n != tokens) or (heads >= 0 and h != heads):
        _refuse(name, t, index, tokens, heads)
    return n, h, a if n > 1 else D, b if h > 1 else D


_KEPT = 64  # shapes that a batch remembers


def _scratch_bytes(kv: "PagedKv", batch: "PagedBatch", mask: Optional[BlockCausal], key) -> int:
    """Scratch of an attention call of this shape; the batch remembers it."""
    how, heads, _, tokens, _ = key
    if max(how) > 0x7fffffff or min(how) < 0:
        raise ValueError(f"attend: {mask} is out of range")
    with torch.cuda.device(kv.index):
        need = (_fns or _entries())[2](kv._ref, batch._ref, _query_struct.pack(0, 0, 0, 0, 0, 0, tokens, heads, *how, 0.0))
    if len(batch._need) >= _KEPT:  # (a program whose number of packed rows never comes again)
        batch._need.clear()
    batch._need[key] = need
    return need


def _rows_like(q: torch.Tensor, n: int, h: int) -> torch.Tensor:
    """A contiguous [n, h, 128] result beside q."""
    out = torch.empty_like(q)  # (keeps q's order of extents, which is nearly always this one)
    return out if out.is_contiguous() else q.new_empty((n, h, D))


def _keep_apart(name: str, out: torch.Tensor, other: str, t: torch.Tensor, n: int, h: int, nt: int, nh: int, in_place: bool = False) -> None:
    """Refuses a result (contiguous) that shares memory with rows of an operand t [n, h, 128] (strides nt, nh), which other blocks may
    still have to read; in_place: but for one that is the operand itself."""
    at = (out.data_ptr() - t.data_ptr()) // 2  # in values, of the first byte of out
    size = out.numel()
    if at >= (n - 1) * nt + (h - 1) * nh + D or at + size <= 0 or size == 0 or n * h == 0:
        return
    if in_place and at == 0 and size == n * h * D and (h == 1 or nh == D) and (n == 1 or nt == h * D):
        return
    first = (torch.arange(n)[:, None] * nt + torch.arange(h) * nh).flatten()  # (out may lie in a gap between the rows)
    if bool(((first < at + size) & (first + D > at)).any()):
        raise ValueError(f"{name} overlaps {other}" + (", of which it may only be the whole" if in_place else ""))


def _call(kv: PagedKv, batch: PagedBatch, what: str, fn, *args) -> None:
    """One C entry on the current stream of the cache's device."""
    index = kv.index
    if batch.index != index:
        raise ValueError(f"the cache is on cuda:{index}, the batch on cuda:{batch.index}")
    if torch.cuda.current_device() == index:
        rc = fn(_raw_stream(index), kv._ref, batch._ref, *args)
    else:
        with torch.cuda.device(index):
            rc = fn(_raw_stream(index), kv._ref, batch._ref, *args)
    if rc:
        _lib.check(rc, what)


def append(kv: PagedKv, batch: PagedBatch, k: torch.Tensor, v: torch.Tensor, *, q: Optional[torch.Tensor] = None,
           cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None,
           pairing: str = "interleaved", q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Writes the call's tokens into the cache: k, v [tokens, kv_heads, 128] bf16 (any strides of tokens and heads that are
    multiples of 8: slices of a fused projection are read in place), K rotated on the way when cos / sin f32 [rows, 128] are
    given: token t with row positions[t] (int32), by default its position in its sequence.  pairing "interleaved": values
    2 i and 2 i + 1 (the tables of wan.wan_rope_tables), "half": values i and i + 64.  q [tokens, heads, 128], if given, is
    rotated too and returned as [tokens, heads, 128] (in q_out, which may be q itself, and else shares no memory with q, k and v).  Two tokens of a call must not fall on the same cache row."""
    index = kv.index
    tokens, _, kt, kh = _heads_in("append: k", k, index, -1, kv.kv_heads)
    _, _, vt, vh = _heads_in("append: v", v, index, tokens, kv.kv_heads)
    if pairing not in PAIRINGS:
        raise ValueError(f"append: unknown pairing {pairing!r} {tuple(PAIRINGS)}")
    cp = sp = pp = rows = 0
    if cos is not None and sin is not None:
        shape = cos.shape
        rows = shape[0] if len(shape) == 2 else 0
        for name, t in (("cos", cos), ("sin", sin)):
            if t.shape != (rows, D) or t.dtype is not _f32 or t.get_device() != index or not t.is_contiguous():
                raise ValueError(f"append: {name} must be a contiguous CUDA float32 [rows, 128] tensor on cuda:{index}")
        cp, sp = cos.data_ptr(), sin.data_ptr()
        if positions is not None:
            pp = _index("append: positions", positions, (tokens,), kv.device).data_ptr()
    elif cos is not None or sin is not None or positions is not None:
        raise ValueError("append: cos, sin and positions go together")
    heads = qt = qh = 0
    qp = op = 0
    if q is not None:
        _, heads, qt, qh = _heads_in("append: q", q, index, tokens)
        if q_out is None:
            q_out = _rows_like(q, tokens, heads)
        else:
            _heads_in("append: q_out", q_out, index, tokens, heads)
            if not q_out.is_contiguous():
                raise ValueError("append: q_out must be contiguous")
            _keep_apart("append: q_out", q_out, "q", q, tokens, heads, qt, qh, in_place=True)
            _keep_apart("append: q_out", q_out, "k", k, tokens, kv.kv_heads, kt, kh)
            _keep_apart("append: q_out", q_out, "v", v, tokens, kv.kv_heads, vt, vh)
        if heads:
            qp, op = q.data_ptr(), q_out.data_ptr()
    elif q_out is not None:
        raise ValueError("append: q_out without q")
    if tokens == 0 or batch.seqs == 0 or batch.max_q == 0:
        return q_out
    _call(kv, batch, "paged append", (_fns or _entries())[0],
          _rows_struct.pack(k.data_ptr(), v.data_ptr(), qp, op, cp, sp, pp, kt, kh, vt, vh, qt, qh, tokens, heads, rows, PAIRINGS[pairing]))
    return q_out


def read(kv: PagedKv, batch: PagedBatch, *, rows: int, cu_rows: Optional[torch.Tensor] = None,
         first: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Rows of the sequences as packed (k, v) [rows, kv_heads, 128] bf16, 4-bit rows as the values they stand for: sequence s
    gives rows cu_rows[s] .. cu_rows[s + 1] (int32 [seqs + 1]; default: the batch's own tokens), beginning with its token
    first[s] (int32 [seqs]; default: its last ones).  Rows from cu_rows[seqs] on are zero, as are rows that a sequence does
    not hold; rows below cu_rows[seqs] gives the first ones.  What dense attention, an exchange or a copy of a cache starts from."""
    if rows < 0:
        raise ValueError("read: rows must not be negative")
    cu = batch.cu_q if cu_rows is None else _index("read: cu_rows", cu_rows, (batch.seqs + 1,), kv.device)
    if first is not None:
        _index("read: first", first, (batch.seqs,), kv.device)
    k = (kv.k if kv.k_scale is None else kv.k_scale).new_empty((rows, kv.kv_heads, D))  # (either is bf16)
    v = torch.empty_like(k)  # (cheaper than two views of one tensor)
    if rows == 0:
        return k, v
    if batch.seqs == 0:
        return k.zero_(), v.zero_()
    _call(kv, batch, "paged read", (_fns or _entries())[1], cu.data_ptr(), first.data_ptr() if first is not None else None, rows,
          k.data_ptr(), v.data_ptr())
    return k, v


def attend(kv: PagedKv, batch: PagedBatch, q: torch.Tensor, mask: Optional[BlockCausal] = None, *,
           scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of q [tokens, heads, 128] bf16 (the batch's tokens, rotated; strides as in append, but none 0) over the cache, in place:
    returns [tokens, heads, 128] bf16.  heads is a multiple of kv_heads; head h reads K/V head h // (heads // kv_heads).
    mask None: every key of the sequence.  BlockCausal(block_tokens, window, sink): key j is visible to position p iff
    t_j <= t_p and (window == 0 or t_p - t_j < window or t_j < sink), t = index // block_tokens -- block_tokens 1: causal
    by token, a window of `window` tokens, the first `sink` tokens always visible; block_tokens of a frame: the streaming
    form of the block-causal mask.  A row that sees no key is zero.  Pages of which no row sees a key need not exist; what
    memory holds where no row of the call sees it has no influence, but a key that some row sees must be finite (a NaN may reach
    other rows of the call; one in q reaches only its own row, as an infinity does).  Sums and softmax statistics are f32, probabilities are rounded to the type of the products: bf16, over 4-bit pages f16 (there long
    chunks also take q and the cached values through f16, scaled to its upper end: a value that is 2^-26 and less of the largest that the
    same 256 rows see in its sequence and head loses relative precision).
    With `out` (which may be q itself, and else shares no memory with it), rows that belong to no sequence keep what they hold."""
    tokens, heads, qt, qh = _heads_in("attend: q", q, kv.index)
    if heads < 1 or heads % kv.kv_heads:
        raise ValueError(f"attend: {heads} heads over {kv.kv_heads} K/V heads")
    if out is None:
        out = _rows_like(q, tokens, heads)
    else:
        _heads_in("attend: out", out, kv.index, tokens, heads)
        if not out.is_contiguous():
            raise ValueError("attend: out must be contiguous")
        _keep_apart("attend: out", out, "q", q, tokens, heads, qt, qh, in_place=True)
    if tokens == 0 or batch.seqs == 0 or batch.max_q == 0:
        return out
    how = (1, mask.block_tokens, mask.window, mask.sink) if mask is not None else (0, 0, 0, 0)
    fns = _fns or _entries()
    key = (how, heads, kv.kv_heads, tokens, kv.format)
    need = batch._need.get(key)
    if need is None:
        need = _scratch_bytes(kv, batch, mask, key)
    # (scratch of this call alone, from the stream's own pool: calls on other streams and captured graphs share nothing)
    ws = q.new_empty((need // 2,)) if need else None
    scale = _SCALE if scale is None else float(scale)
    try:
        _call(kv, batch, "paged attention", fns[3],
              _query_struct.pack(q.data_ptr(), out.data_ptr(), ws.data_ptr() if need else 0, need, qt, qh, tokens, heads, *how, scale))
    except _lib.FvError:  # (FV_PAGED_KERNEL may have changed since this shape was first asked for: refused before anything ran)
        fresh = _scratch_bytes(kv, batch, mask, key)
        if fresh <= need:
            raise
        ws = q.new_empty((fresh // 2,))
        _call(kv, batch, "paged attention", fns[3],
              _query_struct.pack(q.data_ptr(), out.data_ptr(), ws.data_ptr(), fresh, qt, qh, tokens, heads, *how, scale))
    return out
