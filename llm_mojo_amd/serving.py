"""What a server calls around the matmuls: the paged key / value cache with
one token's attention over it (llmq_pkv_*), and a sampler's rules on the
logits (llmq_adjust_logits).  No counterpart in the reference, whose caches
hold one sequence (kvcache.mojo:31-87) and whose pick takes the logits as
they are (gpt2t.mojo:792-797).

Tensors are torch tensors on the context's device; their types and shapes
are checked here, since the library sees addresses only.
"""
import ctypes
import math

from ._lib import LogitRules, check, lib

PKV_TYPES = {"int8": 0, "f16": 1}


def _need(ok, what):
    if not ok:
        raise ValueError(what)


# The checks of a decode step's calls are on its critical path: a message is
# formed only where one fails.


torch = None  # imported by whoever makes a tensor; the package itself does not need it


def _torch():
    global torch
    if torch is None:
        import torch as t

        torch = t
    return torch


def _rows(t, heads, hd, dev, name):
    """Row stride of float32 [rows, heads, hd] (or [rows, heads * hd]) on GPU dev with whole rows in one piece."""
    shape, stride = t.shape, t.stride()
    if len(shape) == 3:
        ok = (shape[1] == heads and shape[2] == hd
              and (stride[2] == 1 and (heads == 1 or stride[1] == hd) or shape[0] == 0))
    else:
        ok = len(shape) == 2 and shape[1] == heads * hd and (stride[1] == 1 or shape[0] == 0)
    if not ok or t.dtype is not torch.float32 or t.get_device() != dev:
        raise ValueError(f"{name}: a float32 tensor on GPU {dev} of rows of {heads} heads of {hd} in one piece, "
                         f"got {tuple(shape)} with strides {stride}")
    return stride[0] if shape[0] > 1 else max(stride[0], heads * hd)


def _ints(t, shape, dev, name):
    """Address of a contiguous int32 tensor of that shape."""
    if t.shape != shape or t.dtype is not torch.int32 or not t.is_contiguous() or t.get_device() != dev:
        raise ValueError(f"{name}: a contiguous int32 tensor of shape {shape} on GPU {dev}")
    return t.data_ptr()


class PagedKV:
    """Keys and values of many sequences in pages of `page` positions.

    A table row (int32 [n_seq, width]) names a sequence's pages: position p is
    in page table[seq, p // page].  Positions, lengths and tables are device
    tensors, read when the kernels run.  kind "int8": int8 codes with a scale
    a position and head, as QuantKV8 but for the scale's last bit (max|x| times
    the float 1 / 127, not over 127; codes can differ at ties); "f16": float16
    values.
    """

    def __init__(self, ctx, n_layer, n_pages, page, n_kv, head_dim, kind="int8"):
        _need(kind in PKV_TYPES, f"PagedKV: kind {kind!r}, expected one of {sorted(PKV_TYPES)}")
        _torch()
        self.ctx, self.kind = ctx, kind
        self.n_layer, self.n_pages, self.page, self.n_kv, self.head_dim = n_layer, n_pages, page, n_kv, head_dim
        h = ctypes.c_void_p()
        check(lib().llmq_pkv_create(ctx.h, PKV_TYPES[kind], n_layer, n_pages, page, n_kv, head_dim, ctypes.byref(h)))
        self.h = h
        self._scale = 1.0 / math.sqrt(head_dim)
        self._dev = ctx.device

    def nbytes(self):
        return lib().llmq_pkv_nbytes(self.h)

    def work_bytes(self, rows, n_head):
        """Bytes of device memory that attend and step of `rows` rows take as `work` (fewer rows may take more)."""
        return lib().llmq_pkv_work_bytes(self.h, rows, n_head)

    def _move(self, call, layer, k, v, seq, pos, table):
        ld = _rows(k, self.n_kv, self.head_dim, self._dev, "k")
        n = k.shape[0]
        if v.shape[0] != n or _rows(v, self.n_kv, self.head_dim, self._dev, "v") != ld:
            raise ValueError("k and v: rows of one number and stride")
        n_seq, width = table.shape
        check(call(self.ctx.h, self.h, layer, k.data_ptr(), v.data_ptr(), ld, n, _ints(seq, (n,), self._dev, "seq"),
                   _ints(pos, (n,), self._dev, "pos"), _ints(table, (n_seq, width), self._dev, "table"), n_seq, width))

    def store(self, layer, k, v, seq, pos, table):
        """Rows of keys and values ([T, n_kv, head_dim]) at positions pos[t] of
        sequences seq[t]; seq or pos -1 leaves a row out."""
        self._move(lib().llmq_pkv_store, layer, k, v, seq, pos, table)

    def fetch(self, layer, k, v, seq, pos, table):
        """Those rows as the cache holds them, into k and v."""
        self._move(lib().llmq_pkv_fetch, layer, k, v, seq, pos, table)

    def _queries(self, out, q, slopes, work):
        """(query heads, out's and q's row strides, the slopes' address, work's address and bytes)."""
        hd = self.head_dim
        n_head = q.shape[1] if q.dim() == 3 else q.shape[1] // hd
        ldq, ldo = _rows(q, n_head, hd, self._dev, "q"), _rows(out, n_head, hd, self._dev, "out")
        if out.shape[0] != q.shape[0]:
            raise ValueError("out and q: rows of one number")
        if work.get_device() != self._dev or not work.is_contiguous():
            raise ValueError(f"work: contiguous memory on GPU {self._dev}")
        sl = None
        if slopes is not None:
            if (slopes.dtype is not torch.float32 or slopes.shape != (n_head,) or not slopes.is_contiguous()
                    or slopes.get_device() != self._dev):
                raise ValueError(f"slopes: {n_head} contiguous float32 values on GPU {self._dev}")
            sl = slopes.data_ptr()
        return n_head, ldo, ldq, sl, work.data_ptr(), work.nbytes

    def attend(self, layer, out, q, length, table, work, scale=None, cap=0.0, slopes=None):
        """out[r] = attention of q[r] ([rows, n_head, head_dim]) over positions
        0 .. length[r] - 1 of table row r; scale 1 / sqrt(head_dim) unless
        given, cap: scores through cap * tanh(s / cap), slopes: plus
        slopes[h] * (j - (length - 1))."""
        n, width = q.shape[0], table.shape[1]
        n_head, ldo, ldq, sl, w, nw = self._queries(out, q, slopes, work)
        check(lib().llmq_pkv_attend(self.ctx.h, self.h, layer, out.data_ptr(), ldo, q.data_ptr(), ldq, n, n_head,
                                    _ints(length, (n,), self._dev, "length"),
                                    _ints(table, (n, width), self._dev, "table"), width,
                                    self._scale if scale is None else scale, cap, sl, w, nw))

    def step(self, layer, out, q, k, v, pos, table, work, scale=None, cap=0.0, slopes=None):
        """A decode step: row r's new key and value ([rows, n_kv, head_dim]) go
        to position pos[r] of table row r, then q[r] attends to 0 .. pos[r];
        pos -1: no token, zeros.  q, k and v have one row stride (views of one
        qkv tensor)."""
        n, width = q.shape[0], table.shape[1]
        n_head, ldo, ldq, sl, w, nw = self._queries(out, q, slopes, work)
        ldk = _rows(k, self.n_kv, self.head_dim, self._dev, "k")
        ldv = _rows(v, self.n_kv, self.head_dim, self._dev, "v")
        if k.shape[0] != n or v.shape[0] != n or (n > 1 and not ldk == ldv == ldq):
            raise ValueError("q, k and v: rows of one number and stride")
        check(lib().llmq_pkv_step(self.ctx.h, self.h, layer, out.data_ptr(), ldo, q.data_ptr(), k.data_ptr(),
                                  v.data_ptr(), ldq, n, n_head, _ints(pos, (n,), self._dev, "pos"),
                                  _ints(table, (n, width), self._dev, "table"), width,
                                  self._scale if scale is None else scale, cap, sl, w, nw))

    def free(self):
        if getattr(self, "h", None):
            lib().llmq_pkv_free(self.h)
            self.h = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


def logits_work_bytes(rows, V):
    """Bytes of device memory that adjust_logits of `rows` rows takes as `work` for a pick (fewer rows may take more)."""
    return lib().llmq_adjust_logits_work_bytes(rows, V)


def _vec(t, dtype, n, dev, name):
    """Address of a contiguous 1-d tensor of n elements."""
    if t.shape != (n,) or t.dtype is not dtype or not t.is_contiguous() or t.get_device() != dev:
        raise ValueError(f"{name}: a contiguous {dtype} tensor of {n} on GPU {dev}")
    return t.data_ptr()


def adjust_logits(ctx, out, logits, history=None, repetition=None, presence=None, frequency=None, bias=None, mask=None,
                  pick=None, work=None):
    """out = logits ([rows, V]; out may be logits) under a sampler's rules, in
    this order: history=(ids, offsets) with repetition, presence and frequency
    penalties ([rows] each) of its tokens; bias=(ids, values, offsets); mask
    (int32 [rows, words], a bit a token; 0 forbids it).  pick (int64 [rows]):
    the first token of the largest result, -1 where none is left."""
    t = torch or _torch()
    f32, i32, i64 = t.float32, t.int32, t.int64
    rows, V = logits.shape
    dev = ctx.device
    ld = []
    for t in (out, logits):
        stride = t.stride()
        if t.shape != (rows, V) or t.dtype is not f32 or (stride[1] != 1 and rows) or t.get_device() != dev:
            raise ValueError(f"logits and out: float32 [{rows}, {V}] on GPU {dev} with rows in one piece")
        ld.append(stride[0] if rows > 1 else max(stride[0], V))
    r = LogitRules()
    if history is not None:
        ids, offsets = history
        r.history_len = n = ids.shape[0]
        r.history = _vec(ids, i32, n, dev, "history")
        r.history_offsets = _vec(offsets, i64, rows + 1, dev, "history offsets")
    if repetition is not None:
        r.repetition = _vec(repetition, f32, rows, dev, "repetition")
    if presence is not None:
        r.presence = _vec(presence, f32, rows, dev, "presence")
    if frequency is not None:
        r.frequency = _vec(frequency, f32, rows, dev, "frequency")
    if bias is not None:
        ids, values, offsets = bias
        r.bias_len = n = ids.shape[0]
        r.bias_ids, r.bias = _vec(ids, i32, n, dev, "bias ids"), _vec(values, f32, n, dev, "biases")
        r.bias_offsets = _vec(offsets, i64, rows + 1, dev, "bias offsets")
    if mask is not None:
        words = mask.shape[1]
        stride = mask.stride()
        if (mask.shape[0] != rows or 32 * words < V or (stride[1] != 1 and rows) or mask.dtype is not i32
                or mask.get_device() != dev):
            raise ValueError(f"mask: int32 words on GPU {dev}, {rows} rows of {V} bits")
        r.mask, r.mask_ld = mask.data_ptr(), stride[0] if rows > 1 else max(stride[0], words)
    w, nw, at = None, 0, None
    if pick is not None:
        if work is None or work.get_device() != dev or not work.is_contiguous():
            raise ValueError(f"pick: contiguous work memory on GPU {dev}")
        w, nw, at = work.data_ptr(), work.nbytes, _vec(pick, i64, rows, dev, "pick")
    check(lib().llmq_adjust_logits(ctx.h, out.data_ptr(), ld[0], logits.data_ptr(), ld[1], rows, V, ctypes.byref(r), at,
                                   w, nw))
