"""Drafted decoding over a quantised cache: the op-level entry points of include/pk.h on torch tensors.

  RopeTable, rope      rotary positions (both pair layouts, part of the head, long-context scaling)
  KvCache, KvSeqs      a paged K/V cache in 8 or 4 bits: store, load, keep; and the attention over it, attend
  logit_rules          penalties, biases and token masks on logits

Nothing here waits for the device, and every call can be captured into a CUDA graph once its outputs and scratch are
passed in (or come from the graph's own pool).  Calls run on the tensors' device, on its current stream or on the
`stream` given (a raw cudaStream_t).
"""
from __future__ import annotations

import ctypes as C

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


P, I, I64, SZ = C.c_void_p, C.c_int, C.c_int64, C.c_size_t
SIGNATURES = {
    "pk_kv_store": ([P, P, P, P, I, I64, I64, P], I), "pk_kv_load": ([P, P, P, P, I, I64, I64, P], I),
    "pk_kv_keep": ([P, P, P, I, P, P], I), "pk_kv_attn_scratch_bytes": ([P, P, I, I], SZ),
    "pk_kv_attn": ([P, P, P, P, SZ, P], I), "pk_rope_turns": ([P, P, P], I), "pk_rope": ([P, P], I),
    "pk_apply_logit_rules": ([P, P, I, I, I, I64, I64, P, P], I),
}

_torch = None
_type_of = {}


def _t():
    global _torch
    if _torch is None:
        import torch

        _torch = torch
        _type_of.update({torch.float32: 0, torch.float16: 1, torch.bfloat16: 30})
    return _torch


def _need(ok, msg):
    if not ok:
        from . import PkError

        raise PkError(1, msg)


def _dtype(t, who):
    code = _type_of.get(t.dtype)
    if code is None:
        from . import PkError

        raise PkError(2, f"{who}: {t.dtype} is not float32, float16 or bfloat16")
    return code


def _call(fn, device, stream, *args, used=()):
    """fn(*args, stream) on `device`; `used`: tensors made by this call, which a stream that is not the current one
    must be known to use."""
    torch = _t()
    if stream is None:
        if device.index == torch.cuda.current_device():
            rc = fn(*args, torch.cuda.current_stream(device).cuda_stream)
        else:
            with torch.cuda.device(device):
                rc = fn(*args, torch.cuda.current_stream(device).cuda_stream)
    else:
        with torch.cuda.device(device):
            rc = fn(*args, stream)
        ext = torch.cuda.ExternalStream(stream, device=device)
        for t in used:
            t.record_stream(ext)
    if rc:
        from . import PkError, last_error

        raise PkError(rc, last_error())


def _lib():
    from . import lib

    return lib()


def _i32(t, device, name, dims):
    torch = _t()
    _need(t.dtype == torch.int32 and t.device == device and t.dim() == dims and t.is_contiguous(),
          f"{name} must be a contiguous int32 tensor of {dims} dimension(s) on {device}")


class KvSeqs:
    """The sequences of a call: start [n_seq + 1], ctx [n_seq], pages [n_seq, max_pages] (int32, on the device).  n_tok:
    rows of the token arrays; max_new, max_len: bounds of a sequence's new tokens and of all its positions."""

    def __init__(self, start, ctx, pages, n_tok: int, max_new: int, max_len: int):
        _t()
        for t, name, dims in ((start, "start", 1), (ctx, "ctx", 1), (pages, "pages", 2)):
            _i32(t, start.device, name, dims)
        n = ctx.numel()
        _need(start.is_cuda and start.numel() == n + 1 and pages.shape[0] == n, "start, ctx and pages disagree about the sequences")
        self.start, self.ctx, self.pages = start, ctx, pages
        self.device, self.n_seq, self.n_tok, self.max_new, self.max_len = start.device, n, n_tok, max_new, max_len
        self.c = KvSeqsC(start.data_ptr(), ctx.data_ptr(), pages.data_ptr(), n, pages.shape[1], n_tok, max_new, max_len)
        self.ref = C.byref(self.c)


class KvCache:
    """A paged cache of one layer in 8 ("q8") or 4 ("q4") bits: codes k, v [n_pages, n_kv, page_size, bytes] (uint8) and
    scales ks, vs [n_pages, n_kv, page_size, 1 or 2] (float32), laid out as include/pk.h says."""

    def __init__(self, k, v, ks, vs, kind: str, head_dim: int):
        torch = _t()
        _need(kind in KINDS, f"cache kind {kind!r} is not q8 or q4")
        row, words = (head_dim, 1) if kind == "q8" else (head_dim // 2, 2)
        _need(k.is_cuda and k.dim() == 4 and k.shape[3] == row, f"k must be [n_pages, n_kv, page_size, {row}] on a CUDA device")
        for t, dt, shape in ((k, torch.uint8, k.shape), (v, torch.uint8, k.shape), (ks, torch.float32, k.shape[:3] + (words,)),
                             (vs, torch.float32, k.shape[:3] + (words,))):
            _need(t.dtype == dt and t.shape == shape and t.device == k.device and t.is_contiguous(),
                  f"a cache array is not a contiguous {dt} tensor {tuple(shape)} on {k.device}")
        self.k, self.v, self.ks, self.vs, self.kind, self.head_dim = k, v, ks, vs, kind, head_dim
        self.n_pages, self.n_kv, self.page_size = k.shape[:3]
        self.device = k.device
        self.c = KvCacheC(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), KINDS[kind], *k.shape[:1],
                          self.page_size, self.n_kv, head_dim)
        self.ref = C.byref(self.c)
        self.lib = _lib()

    @classmethod
    def empty(cls, n_pages: int, page_size: int, n_kv: int, head_dim: int, kind: str = "q8", device="cuda"):
        torch = _t()
        _need(kind in KINDS, f"cache kind {kind!r} is not q8 or q4")
        row, words = (head_dim, 1) if kind == "q8" else (head_dim // 2, 2)
        make = lambda w, dt: torch.zeros((n_pages, n_kv, page_size, w), dtype=dt, device=device)  # noqa: E731
        return cls(make(row, torch.uint8), make(row, torch.uint8), make(words, torch.float32), make(words, torch.float32), kind, head_dim)

    def _rows(self, seqs, k, v, who):
        shape = (seqs.n_tok, self.n_kv, self.head_dim)
        _need(seqs.device == self.device, f"{who}: the sequences are on another device")
        _need(k.shape == shape and v.shape == shape, f"{who}: k and v must be {shape}")
        _need(k.dtype == v.dtype and k.device == v.device == self.device and k.stride() == v.stride() and k.stride(2) == 1,
              f"{who}: k and v must share type, device and strides, with contiguous heads")
        return _dtype(k, who)

    def store(self, seqs: KvSeqs, k, v, stream=None):
        """Quantises rows k, v [n_tok, n_kv, head_dim] of the new tokens into the cache."""
        code = self._rows(seqs, k, v, "store")
        s = k.stride()
        _call(self.lib.pk_kv_store, self.device, stream, self.ref, seqs.ref, k.data_ptr(), v.data_ptr(), code, s[0], s[1])

    def load(self, seqs: KvSeqs, dtype=None, out=None, stream=None):
        """(k, v) [n_tok, n_kv, head_dim] of positions ctx .. read back; rows that no sequence has keep what they held."""
        torch = _t()
        made = ()
        if out is None:
            kv = torch.empty((2, seqs.n_tok, self.n_kv, self.head_dim), dtype=dtype or torch.float32, device=self.device)
            made = (kv,)
            out = kv[0], kv[1]
        k, v = out
        code = self._rows(seqs, k, v, "load")
        s = k.stride()
        _call(self.lib.pk_kv_load, self.device, stream, self.ref, seqs.ref, k.data_ptr(), v.data_ptr(), code, s[0], s[1], used=made)
        return k, v

    def keep(self, seqs: KvSeqs, keep, n_keep, stream=None):
        """Accepts drafts: position ctx + j of sequence s becomes what position ctx + keep[s, j] holds, j < n_keep[s]."""
        _i32(keep, self.device, "keep", 2)
        _i32(n_keep, self.device, "n_keep", 1)
        _need(keep.shape[0] == seqs.n_seq and n_keep.numel() == seqs.n_seq and seqs.device == self.device,
              "keep: one row and one count a sequence, on the cache's device")
        _call(self.lib.pk_kv_keep, self.device, stream, self.ref, seqs.ref, keep.data_ptr(), keep.shape[1], n_keep.data_ptr())

    def attend(self, seqs: KvSeqs, q, mask=None, scale: float | None = None, out=None, scratch=None, stream=None):
        """Attention of the new tokens q [n_tok, n_head, head_dim] over the cache; mask: int64 [n_tok, words], bit j of
        token i set where it sees new token j (None: causal).  scratch: a uint8 tensor of attend_scratch_bytes()."""
        torch = _t()
        code = _dtype(q, "attend")
        _need(q.dim() == 3 and q.shape[0] == seqs.n_tok and q.shape[2] == self.head_dim and q.stride(2) == 1,
              "attend: q must be [n_tok, n_head, head_dim] with contiguous heads")
        _need(q.device == seqs.device == self.device, "attend: q and the sequences must be on the cache's device")
        words = 0
        if mask is not None:
            _need(mask.dtype == torch.int64 and mask.dim() == 2 and mask.shape[0] == seqs.n_tok and mask.is_contiguous() and
                  mask.device == self.device, "attend: mask must be a contiguous int64 tensor [n_tok, words]")
            words = mask.shape[1]
        made = ()
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=self.device)
            made = (out,)
        else:
            _need(out.shape == q.shape and out.dtype == q.dtype and out.device == self.device and out.stride(2) == 1,
                  "attend: out must be as q")
        n_head = q.shape[1]
        need = self.lib.pk_kv_attn_scratch_bytes(self.ref, seqs.ref, n_head, code)
        ptr, size = None, 0
        if scratch is not None:
            _need(scratch.device == self.device and scratch.is_contiguous(), "attend: scratch must be contiguous and on the cache's device")
            ptr, size = scratch.data_ptr(), scratch.numel() * scratch.element_size()
        elif need:
            scratch = torch.empty(need, dtype=torch.uint8, device=self.device)
            made += (scratch,)
            ptr, size = scratch.data_ptr(), need
        s, o = q.stride(), out.stride()
        args = KvQueryC(q.data_ptr(), out.data_ptr(), None if mask is None else mask.data_ptr(), s[0], s[1], o[0], o[1], code,
                        n_head, words, self.head_dim ** -0.5 if scale is None else scale)
        _call(self.lib.pk_kv_attn, self.device, stream, self.ref, seqs.ref, C.byref(args), ptr, size, used=made)
        return out

    def attend_scratch_bytes(self, seqs: KvSeqs, n_head: int, dtype) -> int:
        _t()
        return self.lib.pk_kv_attn_scratch_bytes(self.ref, seqs.ref, n_head, _type_of[dtype])


class RopeTable:
    """The turns a position of n_rot / 2 pairs, on the device, and the gain (pk_rope_turns).  yarn: pairs that turn at
    most `low` times in n_ctx_train positions are slowed by `factor`, those that turn `high` times or more are kept."""

    def __init__(self, n_rot: int, theta: float = 10000.0, scaling: str = "none", factor: float = 1.0, n_ctx_train: int = 0,
                 low: float = 1.0, high: float = 32.0, gain: float | None = None, factors=None, device="cuda"):
        torch = _t()
        _need(scaling in ROPE_SCALING, f"rope scaling {scaling!r} is not one of {sorted(ROPE_SCALING)}")
        host = (C.c_double * max(n_rot // 2, 1))()
        f = None
        if factors is not None:
            _need(len(factors) == n_rot // 2, "factors: one value a pair")
            f = (C.c_float * len(factors))(*[float(x) for x in factors])
        spec = RopeSpecC(n_rot, ROPE_SCALING[scaling], theta, factor, n_ctx_train, low, high, gain or 0.0,
                         C.cast(f, C.c_void_p) if f else None)
        g = C.c_float()
        rc = _lib().pk_rope_turns(C.byref(spec), host, C.byref(g))
        if rc:
            from . import PkError, last_error

            raise PkError(rc, last_error())
        self.n_rot, self.gain = n_rot, g.value
        self.turns = torch.tensor(list(host), dtype=torch.float64).to(device)
        self.device = self.turns.device


def rope(table: RopeTable, pos, q, k=None, layout: str = "interleaved", out_q=None, out_k=None, stream=None):
    """q [n_tok, n_head, head_dim] and k [n_tok, n_kv, head_dim] (or None) rotated by pos [n_tok] (int32) into new tensors
    or the given ones, which may be q and k themselves; returns (q, k)."""
    torch = _t()
    _need(layout in ROPE_LAYOUT, f"rope layout {layout!r} is not one of {sorted(ROPE_LAYOUT)}")
    device = table.device
    _i32(pos, device, "pos", 1)
    code, made, c = _dtype(q, "rope"), [], []
    for x, out in ((q, out_q), (k, out_k)):
        if x is None:
            c.append((None, None, (0, 0, 0), (0, 0, 0), 0, None))
            continue
        _need(x.dim() == 3 and x.shape[0] == pos.shape[0] and x.shape[2] == q.shape[2] and x.stride(2) == 1 and x.dtype == q.dtype and
              x.device == device, "rope: q and k must be [n_tok, heads, head_dim] of one type on the table's device, with contiguous heads")
        if out is None:
            out = torch.empty(x.shape, dtype=x.dtype, device=device)
            made.append(out)
        else:
            _need(out.shape == x.shape and out.dtype == x.dtype and out.device == device and out.stride(2) == 1, "rope: an output is not as its input")
        c.append((x.data_ptr(), out.data_ptr(), x.stride(), out.stride(), x.shape[1], out))
    (qp, qo, qs, qt, nh, oq), (kp, ko, ks, kt, nk, ok) = c
    args = RopeArgsC(qp, kp, qo, ko, pos.data_ptr(), table.turns.data_ptr(), qs[0], qs[1], ks[0], ks[1], qt[0], qt[1], kt[0], kt[1],
                     code, ROPE_LAYOUT[layout], pos.shape[0], nh, nk, q.shape[2], table.n_rot, table.gain)
    _call(_lib().pk_rope, device, stream, C.byref(args), used=made)
    return oq, ok


def logit_rules(logits, repeat=None, freq=None, presence=None, hist=None, n_hist=None, bias_id=None, bias=None, allow=None,
                out=None, stream=None):
    """Rules on logits [rows, n] (or [n]) before a token is drawn, into a new tensor or `out` (which may be the logits):
    repeat, freq, presence float32 [rows]; hist int32 [rows or 1, ids] with n_hist int32 [rows]; bias_id int32 and bias
    float32 [rows or 1, entries]; allow int32 [rows or 1, at least n / 32 words], bit t & 31 of word t >> 5 for token t."""
    torch = _t()
    code, device = _dtype(logits, "logit_rules"), logits.device
    _need(logits.is_cuda and logits.dim() in (1, 2) and logits.stride(-1) == 1, "logit_rules: logits must be [rows, n] with contiguous rows")
    rows, n = logits.shape if logits.dim() == 2 else (1, logits.shape[0])
    made = ()
    if out is None:
        out = torch.empty(logits.shape, dtype=logits.dtype, device=device)
        made = (out,)
    else:
        _need(out.shape == logits.shape and out.dtype == logits.dtype and out.device == device and out.stride(-1) == 1,
              "logit_rules: out must be as the logits")
    r = LogitRulesC()
    for name, t in (("repeat", repeat), ("freq", freq), ("presence", presence)):
        if t is not None:
            _need(t.dtype == torch.float32 and t.shape == (rows,) and t.device == device and t.is_contiguous(), f"{name} must be float32 [{rows}]")
            setattr(r, name, t.data_ptr())
    _need((bias_id is None) == (bias is None), "bias_id and bias come together")
    for name, t, dt in (("hist", hist, torch.int32), ("bias_id", bias_id, torch.int32), ("bias", bias, torch.float32), ("allow", allow, torch.int32)):
        if t is not None:
            _need(t.dtype == dt and t.dim() == 2 and t.shape[0] in (1, rows) and t.device == device and (t.shape[1] < 2 or t.stride(1) == 1),
                  f"{name} must be a {dt} tensor of {rows} rows or one")
            setattr(r, name, t.data_ptr())
    if hist is not None:
        r.hist_stride, r.n_hist_max = (0 if hist.shape[0] == 1 else hist.stride(0)), hist.shape[1]
        if n_hist is not None:
            _i32(n_hist, device, "n_hist", 1)
            _need(n_hist.numel() == rows, "n_hist: one count a row")
            r.n_hist = n_hist.data_ptr()
    if bias is not None:
        _need(bias.shape == bias_id.shape and bias.stride() == bias_id.stride(), "bias and bias_id must match")
        r.bias_stride, r.n_bias = (0 if bias.shape[0] == 1 else bias.stride(0)), bias.shape[1]
    if allow is not None:
        _need(allow.shape[1] >= (n + 31) // 32, "allow has fewer than n bits a row")
        r.allow_stride = 0 if allow.shape[0] == 1 else allow.stride(0)
    st = (logits.stride(0), out.stride(0)) if logits.dim() == 2 else (n, n)
    _call(_lib().pk_apply_logit_rules, device, stream, logits.data_ptr(), out.data_ptr(), code, rows, n, st[0], st[1], C.byref(r), used=made)
    return out
