"""Drafted decoding over a quantised cache: the op-level entry points of include/pk.h on torch tensors.

  RopeTable, rope      rotary positions (both pair layouts, part of the head, long-context scaling)
  KvCache, KvSeqs      a paged K/V cache in 8 or 4 bits: store, load, keep; and the attention over it, attend
  logit_rules          penalties, biases and token masks on logits

Nothing here waits for the device, and every call can be captured into a CUDA graph once its outputs and scratch are
passed in (or come from the graph's own pool).  Calls run on the tensors' device, on its current stream or on the
`stream` given (a raw cudaStream_t).  With `stream`, what a call makes (outputs, scratch) comes from that stream's
memory, and the tensors that it uses are not given to others before that stream is done with them; the caller orders
what they hold, and its later use of the outputs, against that stream.
"""
from __future__ import annotations

import ctypes as C
import struct

KV_Q8, KV_Q4 = 2, 3  # cache types, as pk_set_kv_type's
ROPE_SCALING = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3}
ROPE_LAYOUT = {"interleaved": 0, "half": 1}
KINDS = {"q8": KV_Q8, "q4": KV_Q4}


class KvCacheC(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("ks", C.c_void_p), ("vs", C.c_void_p)] + \
               [(n, C.c_int) for n in ("type", "n_pages", "page_size", "n_kv", "head_dim")]


class KvSeqsC(C.Structure):
    _fields_ = [("start", C.c_void_p), ("ctx", C.c_void_p), ("pages", C.c_void_p)] + \
               [(n, C.c_int) for n in ("n_seq", "max_pages", "n_tok", "max_new", "max_len")]


class KvQueryC(C.Structure):
    _fields_ = [("q", C.c_void_p), ("out", C.c_void_p), ("mask", C.c_void_p)] + \
               [(n, C.c_int64) for n in ("q_tok_stride", "q_head_stride", "out_tok_stride", "out_head_stride")] + \
               [(n, C.c_int) for n in ("type", "n_head", "mask_words")] + [("scale", C.c_float)]


class RopeSpecC(C.Structure):
    _fields_ = [("n_rot", C.c_int), ("scaling", C.c_int)] + \
               [(n, C.c_double) for n in ("theta", "factor", "n_ctx_train", "low", "high", "gain")] + [("factors", C.c_void_p)]


class RopeArgsC(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("q", "k", "q_out", "k_out", "pos", "turns")] + \
               [(n, C.c_int64) for n in ("q_tok_stride", "q_head_stride", "k_tok_stride", "k_head_stride", "qo_tok_stride",
                                         "qo_head_stride", "ko_tok_stride", "ko_head_stride")] + \
               [(n, C.c_int) for n in ("type", "layout", "n_tok", "n_head", "n_kv", "head_dim", "n_rot")] + [("gain", C.c_float)]


class LogitRulesC(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("repeat", "freq", "presence", "hist", "n_hist", "bias_id", "bias", "allow")] + \
               [(n, C.c_int64) for n in ("hist_stride", "bias_stride", "allow_stride")] + \
               [("n_hist_max", C.c_int), ("n_bias", C.c_int)]


# The structures of a call, packed: immutable bytes, so that two threads' calls share nothing (a quarter of the time of
# filling a ctypes structure, too).  Native alignment; tests compare them with the ctypes layouts above.
PACK_QUERY = struct.Struct("@3P4q3if").pack
PACK_ROPE = struct.Struct("@6P8q7if").pack
PACK_RULES = struct.Struct("@8P3q2i").pack

P, I, I64, SZ = C.c_void_p, C.c_int, C.c_int64, C.c_size_t
SIGNATURES = {
    "pk_kv_store": ([P, P, P, P, I, I64, I64, P], I), "pk_kv_load": ([P, P, P, P, I, I64, I64, P], I),
    "pk_kv_keep": ([P, P, P, I, P, P], I), "pk_kv_attn_scratch_bytes": ([P, P, I, I], SZ),
    "pk_kv_attn": ([P, P, P, P, SZ, P], I), "pk_rope_turns": ([P, P, P], I), "pk_rope": ([P, P], I),
    "pk_apply_logit_rules": ([P, P, I, I, I, I64, I64, P, P], I),
}

torch = None  # set by _init, with the library and the error type
_L = PkError = last_error = raw_stream = current_device = None
_type_of = {}


def _init():
    global torch, _L, PkError, last_error, raw_stream, current_device
    if _L is not None:
        return
    import torch as t

    from . import PkError as err, last_error as last, lib

    torch, PkError, last_error = t, err, last
    _type_of.update({t.float32: 0, t.float16: 1, t.bfloat16: 30})
    # the current stream's handle without building a Stream object for it (2 us a call)
    raw_stream = getattr(t._C, "_cuda_getCurrentRawStream", None) or (lambda i: t.cuda.current_stream(i).cuda_stream)
    current_device = t.cuda.current_device
    _L = lib()


def _bad(msg, code=1):
    raise PkError(code, msg)


def _dtype(t, who):
    code = _type_of.get(t.dtype)
    if code is None:
        _bad(f"{who}: {t.dtype} is not float32, float16 or bfloat16", 2)
    return code


def _call(fn, device, stream, used, *args):
    """fn(*args, stream) on device number `device`; used: with a stream given, the call's tensors and lists of them,
    which may be freed before that stream has come to the call."""
    if stream is None and current_device() == device:
        rc = fn(*args, raw_stream(device))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, raw_stream(device) if stream is None else stream)
        if stream is not None and stream != raw_stream(device):
            other = torch.cuda.ExternalStream(stream, device=device)
            for x in used:
                for t in x if isinstance(x, tuple) else (x,):
                    if t is not None:
                        t.record_stream(other)
    if rc:
        raise PkError(rc, last_error())


def _new(make, device, stream, kept=True):
    """make(), a tensor or some, on device number `device` for a call on `stream`: from that stream's pool, because a
    block freed on the current stream may still be in use there.  kept: the caller gets them and may use them on the
    current stream too, which the allocator then has to know."""
    if stream == raw_stream(device):
        return make()
    here = torch.cuda.current_stream(device)
    with torch.cuda.device(device), torch.cuda.stream(torch.cuda.ExternalStream(stream, device=device)):
        made = make()
    if kept:
        for t in made if isinstance(made, tuple) else (made,):
            t.record_stream(here)
    return made


def _i32(t, device, name, dims):
    if t.dtype != torch.int32 or t.get_device() != device or t.dim() != dims or not t.is_contiguous():
        _bad(f"{name} must be a contiguous int32 tensor of {dims} dimension(s) on device {device}")


def _mask(t, rows, device):
    """(words a row, address).  No words at all have no address, which would mean causal."""
    if t.dtype != torch.int64 or t.dim() != 2 or t.shape[0] != rows or not t.is_contiguous() or t.get_device() != device:
        _bad("attend: mask must be a contiguous int64 tensor [n_tok, words] on the cache's device")
    if t.shape[1] < 1:
        _bad("attend: a mask has one word a token or more")
    return t.shape[1], t.data_ptr()


def _same_strides(k, v):
    """Of tensors of one shape; what steps a dimension of size 1 has means nothing."""
    return all(a == b or n == 1 for a, b, n in zip(k.stride(), v.stride(), k.shape))


def _like(x):
    return torch.empty_like(x) if x.is_contiguous() else torch.empty(x.shape, dtype=x.dtype, device=x.device)


class KvSeqs:
    """The sequences of a call: start [n_seq + 1], ctx [n_seq], pages [n_seq, max_pages] (int32, on the device).  n_tok:
    rows of the token arrays; max_new, max_len: bounds of a sequence's new tokens and of all its positions."""

    def __init__(self, start, ctx, pages, n_tok: int, max_new: int, max_len: int):
        _init()
        for x, name in ((n_tok, "n_tok"), (max_new, "max_new"), (max_len, "max_len")):
            if not 0 <= x <= 0x7FFFFFFF:  # (the structure's field would hold another number, 0 for 2^32)
                _bad(f"{name} {x} is not within 0 .. 2^31 - 1")
        device, n = start.get_device(), ctx.numel()
        for t, name, dims in ((start, "start", 1), (ctx, "ctx", 1), (pages, "pages", 2)):
            _i32(t, device, name, dims)
        if not start.is_cuda or start.numel() != n + 1 or pages.shape[0] != n:
            _bad("start, ctx and pages must agree about the sequences and be on a CUDA device")
        self.start, self.ctx, self.pages = start, ctx, pages
        self.device, self.n_seq, self.n_tok, self.max_new, self.max_len = device, n, n_tok, max_new, max_len
        self.c = KvSeqsC(start.data_ptr(), ctx.data_ptr(), pages.data_ptr(), n, pages.shape[1], n_tok, max_new, max_len)
        self.ref = C.byref(self.c)
        self.tensors = (start, ctx, pages)
        self.scratch = {}  # bytes that attend() needs, by what they depend on besides


class KvCache:
    """A paged cache of one layer in 8 ("q8") or 4 ("q4") bits: codes k, v [n_pages, n_kv, page_size, bytes] (uint8) and
    scales ks, vs [n_pages, n_kv, page_size, 1 or 2] (float32), laid out as include/pk.h says."""

    def __init__(self, k, v, ks, vs, kind: str, head_dim: int):
        _init()
        if kind not in KINDS:
            _bad(f"cache kind {kind!r} is not q8 or q4")
        row, words = (head_dim, 1) if kind == "q8" else (head_dim // 2, 2)
        if not k.is_cuda or k.dim() != 4 or k.shape[3] != row:
            _bad(f"k must be [n_pages, n_kv, page_size, {row}] on a CUDA device")
        for t, dt, shape in ((k, torch.uint8, k.shape), (v, torch.uint8, k.shape), (ks, torch.float32, k.shape[:3] + (words,)),
                             (vs, torch.float32, k.shape[:3] + (words,))):
            if t.dtype != dt or t.shape != shape or t.device != k.device or not t.is_contiguous():
                _bad(f"a cache array is not a contiguous {dt} tensor {tuple(shape)} on {k.device}")
        self.k, self.v, self.ks, self.vs, self.kind, self.head_dim = k, v, ks, vs, kind, head_dim
        self.n_pages, self.n_kv, self.page_size = k.shape[:3]
        self.shape = (kind, self.n_kv, head_dim, self.page_size)  # what the scratch of attend() depends on
        self.device = k.get_device()
        self.c = KvCacheC(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), KINDS[kind], self.n_pages,
                          self.page_size, self.n_kv, head_dim)
        self.ref = C.byref(self.c)
        self.tensors = (k, v, ks, vs)

    @classmethod
    def empty(cls, n_pages: int, page_size: int, n_kv: int, head_dim: int, kind: str = "q8", device="cuda"):
        """A cache of zeros."""
        _init()
        if kind not in KINDS:
            _bad(f"cache kind {kind!r} is not q8 or q4")
        row, words = (head_dim, 1) if kind == "q8" else (head_dim // 2, 2)
        make = lambda w, dt: torch.zeros((n_pages, n_kv, page_size, w), dtype=dt, device=device)  # noqa: E731
        return cls(make(row, torch.uint8), make(row, torch.uint8), make(words, torch.float32), make(words, torch.float32), kind, head_dim)

    def _rows(self, seqs, k, v, who):
        """(type, token stride, head stride) of rows k and v."""
        shape, st = (seqs.n_tok, self.n_kv, self.head_dim), k.stride()
        if seqs.device != self.device:
            _bad(f"{who}: the sequences are on another device")
        if k.shape != shape or v.shape != shape:
            _bad(f"{who}: k and v must be {shape}")
        if k.dtype != v.dtype or k.get_device() != self.device or v.get_device() != self.device or (v.stride() != st and not _same_strides(k, v)) or st[2] != 1:
            _bad(f"{who}: k and v must be on the cache's device and share type and strides, with contiguous heads")
        return _dtype(k, who), st[0], st[1]

    def store(self, seqs: KvSeqs, k, v, stream=None):
        """Quantises rows k, v [n_tok, n_kv, head_dim] of the new tokens into the cache.  k and v have the same strides:
        those of one fused projection do, also after rope() in place (out_q, out_k)."""
        _call(_L.pk_kv_store, self.device, stream, stream is not None and (self.tensors, seqs.tensors, k, v), self.ref, seqs.ref, k.data_ptr(), v.data_ptr(), *self._rows(seqs, k, v, "store"))

    def load(self, seqs: KvSeqs, dtype=None, out=None, stream=None):
        """(k, v) [n_tok, n_kv, head_dim] of positions ctx .. read back; rows that no sequence has keep what they held."""
        if out is None:
            dh, dt, dev = self.head_dim, dtype or torch.float32, self.k.device
            shape, st = (seqs.n_tok, self.n_kv, dh), (self.n_kv * dh, dh, 1)
            make = lambda: torch.empty_strided(shape, st, dtype=dt, device=dev)  # noqa: E731
            out = (make(), make()) if stream is None else _new(lambda: (make(), make()), self.device, stream)
        k, v = out
        _call(_L.pk_kv_load, self.device, stream, stream is not None and (self.tensors, seqs.tensors, k, v), self.ref, seqs.ref, k.data_ptr(), v.data_ptr(), *self._rows(seqs, k, v, "load"))
        return k, v

    def keep(self, seqs: KvSeqs, keep, n_keep, stream=None):
        """Accepts drafts: position ctx + j of sequence s becomes what position ctx + keep[s, j] holds, j < n_keep[s]."""
        _i32(keep, self.device, "keep", 2)
        _i32(n_keep, self.device, "n_keep", 1)
        if keep.shape[0] != seqs.n_seq or n_keep.shape[0] != seqs.n_seq or seqs.device != self.device:
            _bad("keep: one row and one count a sequence, on the cache's device")
        _call(_L.pk_kv_keep, self.device, stream, stream is not None and (self.tensors, seqs.tensors, keep, n_keep), self.ref, seqs.ref, keep.data_ptr(), keep.shape[1], n_keep.data_ptr())

    def attend(self, seqs: KvSeqs, q, mask=None, scale: float | None = None, out=None, scratch=None, stream=None):
        """Attention of the new tokens q [n_tok, n_head, head_dim] over the cache; mask: int64 [n_tok, words], bit j of
        token i set where it sees new token j (None: causal).  scratch: a uint8 tensor of attend_scratch_bytes()."""
        code, shape, s, dev = _dtype(q, "attend"), q.shape, q.stride(), self.device
        if len(shape) != 3 or shape[0] != seqs.n_tok or shape[2] != self.head_dim or s[2] != 1:
            _bad("attend: q must be [n_tok, n_head, head_dim] with contiguous heads")
        if q.get_device() != dev or seqs.device != dev:
            _bad("attend: q and the sequences must be on the cache's device")
        words, bits = (0, 0) if mask is None else _mask(mask, shape[0], dev)
        if out is None:
            out = _like(q) if stream is None else _new(lambda: _like(q), dev, stream)
        elif out.shape != shape or out.dtype != q.dtype or out.get_device() != dev or out.stride(2) != 1:
            _bad("attend: out must be as q")
        ptr, size = None, seqs.scratch.get((shape[1], code, self.shape))
        if size is None:
            size = self.attend_scratch_bytes(seqs, shape[1], q.dtype)
        if scratch is not None:
            if scratch.get_device() != dev or not scratch.is_contiguous():
                _bad("attend: scratch must be contiguous and on the cache's device")
            ptr, size = scratch.data_ptr(), scratch.numel() * scratch.element_size()
        elif size:
            make = lambda: self.ks.new_empty((size + 3) // 4)  # noqa: E731
            scratch = make() if stream is None else _new(make, dev, stream, kept=False)
            ptr = scratch.data_ptr()
        o = out.stride()
        args = PACK_QUERY(q.data_ptr(), out.data_ptr(), bits, s[0], s[1], o[0], o[1], code, shape[1], words,
                          self.head_dim ** -0.5 if scale is None else scale)
        _call(_L.pk_kv_attn, dev, stream, stream is not None and (self.tensors, seqs.tensors, q, mask, out, scratch), self.ref, seqs.ref, args, ptr, size)
        return out

    def attend_scratch_bytes(self, seqs: KvSeqs, n_head: int, dtype) -> int:
        """Bytes of scratch that attend() needs (0: none); kept with the sequences, whose bounds do not change."""
        code = _type_of[dtype]
        n = _L.pk_kv_attn_scratch_bytes(self.ref, seqs.ref, n_head, code)
        seqs.scratch[n_head, code, self.shape] = n
        return n


class RopeTable:
    """The turns a position of n_rot / 2 pairs, on the device, and the gain (pk_rope_turns).  yarn: pairs that turn at
    most `low` times in n_ctx_train positions are slowed by `factor`, those that turn `high` times or more are kept, linear
    in the turns between them.  A ramp that is linear in the pair's index, which some checkpoints were made for, is given
    as factors, 1 / (keep + (1 - keep) / factor) a pair, with the gain."""

    def __init__(self, n_rot: int, theta: float = 10000.0, scaling: str = "none", factor: float = 1.0, n_ctx_train: int = 0,
                 low: float = 1.0, high: float = 32.0, gain: float | None = None, factors=None, device="cuda"):
        _init()
        if scaling not in ROPE_SCALING:
            _bad(f"rope scaling {scaling!r} is not one of {sorted(ROPE_SCALING)}")
        host = (C.c_double * max(n_rot // 2, 1))()
        f = None
        if factors is not None:
            if len(factors) != n_rot // 2:
                _bad("factors: one value a pair")
            f = (C.c_float * len(factors))(*[float(x) for x in factors])
        spec = RopeSpecC(n_rot, ROPE_SCALING[scaling], theta, factor, n_ctx_train, low, high, gain or 0.0,
                         C.cast(f, C.c_void_p) if f else None)
        g = C.c_float()
        rc = _L.pk_rope_turns(C.byref(spec), host, C.byref(g))
        if rc:
            raise PkError(rc, last_error())
        self.n_rot, self.gain = n_rot, g.value
        self.turns = torch.tensor(list(host), dtype=torch.float64).to(device)
        self.device = self.turns.get_device()


_NO_ROWS = (0, 0, 0)


def rope(table: RopeTable, pos, q, k=None, layout: str = "interleaved", out_q=None, out_k=None, stream=None):
    """q [n_tok, n_head, head_dim] and k [n_tok, n_kv, head_dim] (or None) rotated by pos [n_tok] (int32) into new tensors
    or the given ones, which may be q and k themselves; returns (q, k)."""
    pairs = ROPE_LAYOUT.get(layout)
    if pairs is None:
        _bad(f"rope layout {layout!r} is not one of {sorted(ROPE_LAYOUT)}")
    dev = table.device
    if dev < 0:
        _bad("rope: the table is not on a CUDA device")
    _i32(pos, dev, "pos", 1)
    code, shape = _dtype(q, "rope"), q.shape
    n, dh = pos.shape[0], shape[-1]
    qs = q.stride()
    if len(shape) != 3 or shape[0] != n or qs[2] != 1 or q.get_device() != dev:
        _bad("rope: q must be [n_tok, heads, head_dim] on the table's device, with contiguous heads")
    if out_q is None:
        out_q = _like(q) if stream is None else _new(lambda: _like(q), dev, stream)
    elif out_q.shape != shape or out_q.dtype != q.dtype or out_q.get_device() != dev or out_q.stride(2) != 1:
        _bad("rope: an output is not as its input")
    qt, ks, kt, kp, kq, nk = out_q.stride(), _NO_ROWS, _NO_ROWS, 0, 0, 0
    if k is not None:
        kshape, ks = k.shape, k.stride()
        if len(kshape) != 3 or kshape[0] != n or kshape[2] != dh or ks[2] != 1 or k.dtype != q.dtype or k.get_device() != dev:
            _bad("rope: k must be [n_tok, heads, head_dim] of q's type on the table's device, with contiguous heads")
        if out_k is None:
            out_k = _like(k) if stream is None else _new(lambda: _like(k), dev, stream)
        elif out_k.shape != kshape or out_k.dtype != q.dtype or out_k.get_device() != dev or out_k.stride(2) != 1:
            _bad("rope: an output is not as its input")
        kt, kp, kq, nk = out_k.stride(), k.data_ptr(), out_k.data_ptr(), kshape[1]
    args = PACK_ROPE(q.data_ptr(), kp, out_q.data_ptr(), kq, pos.data_ptr(), table.turns.data_ptr(), qs[0], qs[1], ks[0], ks[1], qt[0],
                     qt[1], kt[0], kt[1], code, pairs, n, shape[1], nk, dh, table.n_rot, table.gain)
    _call(_L.pk_rope, dev, stream, stream is not None and (table.turns, pos, q, k, out_q, out_k), args)
    return out_q, out_k


def _row_list(t, name, dt, rows, dev):
    """(address, stride in elements, entries) of a list for every row, or one for all."""
    if t is None:
        return 0, 0, 0
    st = t.stride()
    if t.dtype != dt or len(st) != 2 or t.shape[0] not in (1, rows) or t.get_device() != dev or (st[1] != 1 and t.shape[1] > 1):
        _bad(f"{name} must be a {dt} tensor of {rows} rows or one, on the logits' device")
    return t.data_ptr(), st[0] if t.shape[0] > 1 else 0, t.shape[1]


def _row_value(t, name, dt, rows, dev):
    if t is None:
        return 0
    if t.dtype != dt or t.shape != (rows,) or t.get_device() != dev or not t.is_contiguous():
        _bad(f"{name} must be a contiguous {dt} tensor of {rows} values on the logits' device")
    return t.data_ptr()


def logit_rules(logits, repeat=None, freq=None, presence=None, hist=None, n_hist=None, bias_id=None, bias=None, allow=None,
                out=None, stream=None):
    """Rules on logits [rows, n] (or [n]) before a token is drawn, into a new tensor or `out` (which may be the logits):
    repeat, freq, presence float32 [rows]; hist int32 [rows or 1, ids] with n_hist int32 [rows]; bias_id int32 and bias
    float32 [rows or 1, entries]; allow int32 [rows or 1, at least n / 32 words], bit t & 31 of word t >> 5 for token t."""
    _init()
    code, dev, st, shape = _dtype(logits, "logit_rules"), logits.get_device(), logits.stride(), logits.shape
    if dev < 0 or len(shape) not in (1, 2) or st[-1] != 1:
        _bad("logit_rules: logits must be [rows, n] on a CUDA device, with contiguous rows")
    rows, n = shape if len(shape) == 2 else (1, shape[0])
    if out is None:
        out = _like(logits) if stream is None else _new(lambda: _like(logits), dev, stream)
    elif out.shape != shape or out.dtype != logits.dtype or out.get_device() != dev or out.stride(-1) != 1:
        _bad("logit_rules: out must be as the logits")
    f, i = torch.float32, torch.int32
    hp, hs, hn = _row_list(hist, "hist", i, rows, dev)
    ip, bs, bn = _row_list(bias_id, "bias_id", i, rows, dev)
    bp, bs2, bn2 = _row_list(bias, "bias", f, rows, dev)
    ap, as_, an = _row_list(allow, "allow", i, rows, dev)
    if (bias_id is None) != (bias is None) or bs != bs2 or bn != bn2:
        _bad("bias_id and bias come together, in one shape")
    if allow is not None and an < (n + 31) // 32:
        _bad("allow has fewer than n bits a row")
    args = PACK_RULES(_row_value(repeat, "repeat", f, rows, dev), _row_value(freq, "freq", f, rows, dev),
                      _row_value(presence, "presence", f, rows, dev), hp, _row_value(n_hist, "n_hist", i, rows, dev), ip, bp, ap,
                      hs, bs, as_, hn, bn)
    _call(_L.pk_apply_logit_rules, dev, stream, stream is not None and (logits, out, repeat, freq, presence, hist, n_hist, bias_id, bias, allow), logits.data_ptr(), out.data_ptr(), code, rows, n, st[0] if len(st) == 2 else n,
          out.stride(0) if len(st) == 2 else n, args)
    return out
