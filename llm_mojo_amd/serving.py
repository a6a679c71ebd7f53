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


def _rows(t, heads, hd, name):
    """Row stride of [rows, heads, hd] (or [rows, heads * hd]) float32 with whole rows in one piece."""
    import torch  # whoever has a tensor has it already; the package itself does not need it

    _need(t.dtype == torch.float32 and t.is_cuda, f"{name}: a float32 tensor on the GPU")
    if t.dim() == 3:
        _need(t.shape[1] == heads and t.shape[2] == hd, f"{name}: {tuple(t.shape)}, expected {heads} heads of {hd}")
        _need(t.numel() == 0 or (t.stride(2) == 1 and (heads == 1 or t.stride(1) == hd)),
              f"{name}: a row is not in one piece")
    else:
        _need(t.dim() == 2 and t.shape[1] == heads * hd, f"{name}: {tuple(t.shape)}, expected rows of {heads * hd}")
        _need(t.numel() == 0 or t.stride(1) == 1, f"{name}: a row is not in one piece")
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), heads * hd)


def _ints(t, shape, name):
    import torch

    _need(t.dtype == torch.int32 and t.is_cuda and t.is_contiguous() and tuple(t.shape) == shape,
          f"{name}: a contiguous int32 tensor of shape {shape} on the GPU")
    return t.data_ptr()


class PagedKV:
    """Keys and values of many sequences in pages of `page` positions.

    A table row (int32 [n_seq, width]) names a sequence's pages: position p is
    in page table[seq, p // page].  Positions, lengths and tables are device
    tensors, read when the kernels run.  kind "int8": int8 codes with a scale
    a position and head, as QuantKV8; "f16": float16 values.
    """

    def __init__(self, ctx, n_layer, n_pages, page, n_kv, head_dim, kind="int8"):
        _need(kind in PKV_TYPES, f"PagedKV: kind {kind!r}, expected one of {sorted(PKV_TYPES)}")
        self.ctx, self.kind = ctx, kind
        self.n_layer, self.n_pages, self.page, self.n_kv, self.head_dim = n_layer, n_pages, page, n_kv, head_dim
        h = ctypes.c_void_p()
        check(lib().llmq_pkv_create(ctx.h, PKV_TYPES[kind], n_layer, n_pages, page, n_kv, head_dim, ctypes.byref(h)))
        self.h = h

    def nbytes(self):
        return lib().llmq_pkv_nbytes(self.h)

    def work_bytes(self, rows, n_head):
        """Bytes of device memory that attend and step of `rows` rows take as `work`."""
        return lib().llmq_pkv_work_bytes(self.h, rows, n_head)

    def _move(self, call, layer, k, v, seq, pos, table):
        ld = _rows(k, self.n_kv, self.head_dim, "k")
        _need(v.shape[0] == k.shape[0] and _rows(v, self.n_kv, self.head_dim, "v") == ld,
              "k and v: rows of one number and stride")
        n = k.shape[0]
        check(call(self.ctx.h, self.h, layer, k.data_ptr(), v.data_ptr(), ld, n, _ints(seq, (n,), "seq"),
                   _ints(pos, (n,), "pos"), _ints(table, tuple(table.shape[:2]), "table"), table.shape[0],
                   table.shape[1]))

    def store(self, layer, k, v, seq, pos, table):
        """Rows of keys and values ([T, n_kv, head_dim]) at positions pos[t] of
        sequences seq[t]; seq or pos -1 leaves a row out."""
        self._move(lib().llmq_pkv_store, layer, k, v, seq, pos, table)

    def fetch(self, layer, k, v, seq, pos, table):
        """Those rows as the cache holds them, into k and v."""
        self._move(lib().llmq_pkv_fetch, layer, k, v, seq, pos, table)

    def _work(self, work):
        _need(work.is_cuda and work.is_contiguous(), "work: contiguous memory on the GPU")
        return work.data_ptr(), work.numel() * work.element_size()

    def _queries(self, out, q, slopes):
        """(query heads, out's and q's row strides, the slopes' address)."""
        hd = self.head_dim
        n_head = q.shape[1] if q.dim() == 3 else q.shape[1] // hd
        ldq, ldo = _rows(q, n_head, hd, "q"), _rows(out, n_head, hd, "out")
        _need(out.shape[0] == q.shape[0], "out and q: rows of one number")
        if slopes is not None:
            _need(str(slopes.dtype) == "torch.float32" and slopes.is_cuda and slopes.is_contiguous()
                  and slopes.numel() == n_head, f"slopes: {n_head} contiguous float32 values on the GPU")
        return n_head, ldo, ldq, None if slopes is None else slopes.data_ptr()

    def attend(self, layer, out, q, length, table, work, scale=None, cap=0.0, slopes=None):
        """out[r] = attention of q[r] ([rows, n_head, head_dim]) over positions
        0 .. length[r] - 1 of table row r; scale 1 / sqrt(head_dim) unless
        given, cap: scores through cap * tanh(s / cap), slopes: plus
        slopes[h] * (j - (length - 1))."""
        n = q.shape[0]
        n_head, ldo, ldq, sl = self._queries(out, q, slopes)
        w, nw = self._work(work)
        check(lib().llmq_pkv_attend(self.ctx.h, self.h, layer, out.data_ptr(), ldo, q.data_ptr(), ldq, n, n_head,
                                    _ints(length, (n,), "length"), _ints(table, (n, table.shape[1]), "table"),
                                    table.shape[1], 1.0 / math.sqrt(self.head_dim) if scale is None else scale, cap,
                                    sl, w, nw))

    def step(self, layer, out, q, k, v, pos, table, work, scale=None, cap=0.0, slopes=None):
        """A decode step: row r's new key and value ([rows, n_kv, head_dim]) go
        to position pos[r] of table row r, then q[r] attends to 0 .. pos[r];
        pos -1: no token, zeros.  q, k and v have one row stride (views of one
        qkv tensor)."""
        n = q.shape[0]
        n_head, ldo, ldq, sl = self._queries(out, q, slopes)
        ldk, ldv = (_rows(t, self.n_kv, self.head_dim, s) for t, s in ((k, "k"), (v, "v")))
        _need(k.shape[0] == n and v.shape[0] == n and (n <= 1 or ldk == ldv == ldq),
              "q, k and v: rows of one number and stride")
        w, nw = self._work(work)
        check(lib().llmq_pkv_step(self.ctx.h, self.h, layer, out.data_ptr(), ldo, q.data_ptr(), k.data_ptr(),
                                  v.data_ptr(), ldq, n, n_head, _ints(pos, (n,), "pos"),
                                  _ints(table, (n, table.shape[1]), "table"), table.shape[1],
                                  1.0 / math.sqrt(self.head_dim) if scale is None else scale, cap, sl, w, nw))

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
    """Bytes of device memory that adjust_logits takes as `work` for a pick."""
    return lib().llmq_adjust_logits_work_bytes(rows, V)


def _vec(t, dtype, n, name):
    """Address of a contiguous 1-d tensor of n elements (any number for None)."""
    _need(str(t.dtype) == dtype and t.is_cuda and t.is_contiguous() and t.dim() == 1 and (n is None or t.shape[0] == n),
          f"{name}: a contiguous {dtype[6:]} tensor{'' if n is None else f' of {n}'} on the GPU")
    return t.data_ptr()


def adjust_logits(ctx, out, logits, history=None, repetition=None, presence=None, frequency=None, bias=None, mask=None,
                  pick=None, work=None):
    """out = logits ([rows, V]; out may be logits) under a sampler's rules, in
    this order: history=(ids, offsets) with repetition, presence and frequency
    penalties ([rows] each) of its tokens; bias=(ids, values, offsets); mask
    (int32 [rows, words], a bit a token; 0 forbids it).  pick (int64 [rows]):
    the first token of the largest result, -1 where none is left."""
    rows, V = logits.shape
    for t, name in ((logits, "logits"), (out, "out")):
        _need(str(t.dtype) == "torch.float32" and t.is_cuda and tuple(t.shape) == (rows, V)
              and (t.numel() == 0 or t.stride(1) == 1),
              f"{name}: float32 [{rows}, {V}] on the GPU with rows in one piece")
    r = LogitRules()
    if history is not None:
        r.history, r.history_offsets = (_vec(history[0], "torch.int32", None, "history"),
                                        _vec(history[1], "torch.int64", rows + 1, "history offsets"))
        r.history_len = history[0].shape[0]
    for name, t in (("repetition", repetition), ("presence", presence), ("frequency", frequency)):
        if t is not None:
            setattr(r, name, _vec(t, "torch.float32", rows, name))
    if bias is not None:
        n = r.bias_len = bias[0].shape[0]
        r.bias_ids, r.bias = _vec(bias[0], "torch.int32", n, "bias ids"), _vec(bias[1], "torch.float32", n, "biases")
        r.bias_offsets = _vec(bias[2], "torch.int64", rows + 1, "bias offsets")
    if mask is not None:
        _need(str(mask.dtype) == "torch.int32" and mask.is_cuda and mask.dim() == 2 and mask.shape[0] == rows
              and (mask.numel() == 0 or mask.stride(1) == 1) and 32 * mask.shape[1] >= V,
              f"mask: int32 words on the GPU, {rows} rows of {V} bits")
        r.mask, r.mask_ld = mask.data_ptr(), mask.stride(0) if rows > 1 else max(mask.stride(0), mask.shape[1])
    w, nw = None, 0
    if pick is not None:
        _need(work is not None and work.is_cuda and work.is_contiguous(), "pick: contiguous work memory on the GPU")
        w, nw = work.data_ptr(), work.numel() * work.element_size()
    ld = [t.stride(0) if rows > 1 else max(t.stride(0), V) for t in (out, logits)]
    check(lib().llmq_adjust_logits(ctx.h, out.data_ptr(), ld[0], logits.data_ptr(), ld[1], rows, V, ctypes.byref(r),
                                   None if pick is None else _vec(pick, "torch.int64", rows, "pick"), w, nw))
