"""A serving step around the quantised cache: the op-level entry points of include/pk.h on torch tensors.

  kv_plan              a step's page tables and slot maps from the requests' lengths, on the device
  KvShared             the prefixes that sequences share, for KvCache.attend(shared=...)
  sample_rows          a token for every row of logits: temperature, top-k, top-p and min-p, from given random numbers

As the drafted-decoding operators (drafts.py): nothing here waits for the device, every call can be captured, and calls
run on the tensors' device, on its current stream or on the `stream` given (a raw cudaStream_t).
"""
from __future__ import annotations

import ctypes as C
import struct
from typing import NamedTuple

from . import drafts as _d
from .drafts import _bad, _call, _dtype, _i32, _init, _new, _row_value


class KvSharedC(C.Structure):
    _fields_ = [("first", C.c_void_p), ("len", C.c_void_p)] + [(n, C.c_int) for n in ("n_group", "max_tok", "max_len", "max_own")]


class KvPlanC(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("ctx", "n_new", "pages", "held", "free", "n_free", "done", "shared", "pages_out", "held_out", "free_out",
                                          "n_free_out", "start", "lacking", "pos", "seq", "slot")] + \
               [(n, C.c_int) for n in ("n_seq", "max_pages", "free_cap", "n_tok", "page_size")]


class SampleC(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("u", "temp", "top_k", "top_p", "min_p", "tok", "prob", "kept")]


# As drafts.py's: packed structures, immutable and the call's own.
PACK_PLAN = struct.Struct("@17P5i").pack
PACK_SAMPLE = struct.Struct("@8P").pack


class KvShared:
    """Groups of sequences that share a prefix: group g is sequences first[g] .. first[g + 1] - 1, whose first len[g]
    positions hold the same K and V and are read from the pages of the first of them (first [n_group + 1], len [n_group]:
    int32, on the device).  max_tok: a bound of a group's new tokens (one with more is not shared); max_len: of len;
    max_own: of a sequence's positions besides the shared ones, new ones included (what is beyond is left out).  A
    sequence whose ctx is less than its group's len is computed by itself."""

    def __init__(self, first, len, max_tok: int, max_len: int, max_own: int):
        _init()
        for x, name in ((max_tok, "max_tok"), (max_len, "max_len"), (max_own, "max_own")):
            if not 0 <= x <= 0x7FFFFFFF:
                _bad(f"{name} {x} is not within 0 .. 2^31 - 1")
        device, n = first.get_device(), len.numel()
        _i32(first, device, "first", 1)
        _i32(len, device, "len", 1)
        if not first.is_cuda or first.numel() != n + 1:
            _bad("first and len must agree about the groups and be on a CUDA device")
        self.first, self.len, self.device, self.n_group = first, len, device, n
        self.max_tok, self.max_len, self.max_own = max_tok, max_len, max_own
        self.c = KvSharedC(first.data_ptr(), len.data_ptr(), n, max_tok, max_len, max_own)
        self.ref = C.byref(self.c)
        self.tensors = (first, len)
        self.key = (n, max_tok, max_len, max_own)  # what the scratch of attend() depends on


class KvPlan(NamedTuple):
    """What kv_plan makes: for KvSeqs start and pages (with the call's ctx), for rope pos; the sequence and the cache slot
    (page * page_size + offset) of each token, -1 where there is none; the tables, pages held and free list after the step;
    lacking [1]: pages that there were not."""

    start: object
    pos: object
    seq: object
    slot: object
    pages: object
    held: object
    free: object
    n_free: object
    lacking: object


def kv_plan(ctx, n_new, pages, held, free, n_free, page_size: int, n_tok: int, done=None, shared=None, in_place: bool = False, stream=None) -> KvPlan:
    """Page tables and slot maps of a step.  ctx, n_new [n_seq]: committed positions and new tokens of each slot; pages
    [n_seq, max_pages], held [n_seq]: its page table and how many pages that holds; free [any], n_free [1]: the list of free
    pages.  Slots with done [n_seq] set first give back their pages (but the first shared [n_seq], which others have too);
    then the others take, from the list's end, what ctx + n_new needs besides held.  All int32, on one device.  n_tok: rows
    of the token arrays (at least the new tokens; rows behind them get position 0, sequence -1, slot -1).  in_place: pages,
    held, free and n_free are updated themselves; otherwise the results are new tensors."""
    _init()
    torch = _d.torch
    i32, dev, n = torch.int32, ctx.get_device(), ctx.shape[0] if ctx.dim() == 1 else -1
    if dev < 0 or n < 0:
        _bad("kv_plan: ctx must be [n_seq] on a CUDA device")
    whole = (n,)
    if done is None or shared is None:
        for t, name in ((done, "done"), (shared, "shared")):
            if t is not None and (t.dtype is not i32 or t.get_device() != dev or t.shape != whole or not t.is_contiguous()):
                _bad(f"kv_plan: {name} must be a contiguous int32 tensor of {n} on device {dev}")
        per_slot, ends = (ctx, n_new, held), (0 if done is None else done.data_ptr(), 0 if shared is None else shared.data_ptr())
    else:
        per_slot, ends = (ctx, n_new, held, done, shared), (done.data_ptr(), shared.data_ptr())
    for t in per_slot:
        if t.dtype is not i32 or t.shape != whole or t.get_device() != dev or not t.is_contiguous():
            _bad(f"kv_plan: ctx, n_new, held, done and shared must be contiguous int32 tensors of {n} on device {dev}")
    for t in (pages, free, n_free):
        if t.dtype is not i32 or t.get_device() != dev or not t.is_contiguous():
            _bad(f"kv_plan: pages, free and n_free must be contiguous int32 tensors on device {dev}")
    ptrs = (ctx.data_ptr(), n_new.data_ptr(), pages.data_ptr(), held.data_ptr(), free.data_ptr(), n_free.data_ptr())
    if pages.dim() != 2 or pages.shape[0] != n or free.dim() != 1 or n_free.shape != (1,):
        _bad("kv_plan: pages must be [n_seq, max_pages], free a list and n_free one number")
    if not 0 <= n_tok <= 1 << 30:
        _bad("kv_plan: n_tok must be 0 to 2^30")
    wide, cap = pages.shape[1], free.shape[0]
    # one block for all results (a tensor of its own each costs more than the launch): first what has to be aligned
    table = 0 if in_place else n * wide + (n * wide & 1)
    sizes = (table, 2 * n_tok, n + 1, n_tok, n_tok, 1) if in_place else (table, 2 * n_tok, n + 1, n_tok, n_tok, 1, n, cap, 1)
    make = lambda: ctx.new_empty(sum(sizes)).split_with_sizes(sizes)  # noqa: E731
    made = make() if stream is None else _new(make, dev, stream)
    slot, start, pos, seq, lacking = made[1].view(torch.int64), made[2], made[3], made[4], made[5]
    if in_place:
        out, to = (pages, held, free, n_free), (ptrs[2], ptrs[3], ptrs[4], ptrs[5])
    else:
        block = made[0] if table == n * wide else made[0][:-1]
        out = (block.view(n, wide), made[6], made[7], made[8])
        to = (block.data_ptr(), made[6].data_ptr(), made[7].data_ptr(), made[8].data_ptr())
    args = PACK_PLAN(*ptrs, *ends, *to, start.data_ptr(), lacking.data_ptr(), pos.data_ptr(), seq.data_ptr(), slot.data_ptr(), n, wide, cap, n_tok, page_size)
    _call(_d._L.pk_kv_plan, dev, stream, stream is not None and (ctx, n_new, pages, held, free, n_free, done, shared, made), args)
    return KvPlan(start, pos, seq, slot, *out, lacking)


def sample_rows(logits, u, temp=None, top_k=None, top_p=None, min_p=None, stream=None):
    """A token for every row of logits [rows, n] (or [n]) from random numbers u float32 [rows] in [0, 1): (tokens int32,
    their probability among the kept ones float32, how many were kept int32), each [rows].  temp, top_p, min_p float32 and
    top_k int32 [rows], or None: 1, all, all, all.  Order: min_p of the likeliest's weight, then top_k, then top_p of what
    these leave; equal logits in the order of their indices; temp <= 0 takes the largest logit.  A row that allows nothing
    (-inf or NaN everywhere) gives token -1."""
    _init()
    code, dev, st, shape = _dtype(logits, "sample_rows"), logits.get_device(), logits.stride(), logits.shape
    if dev < 0 or len(shape) not in (1, 2) or (st[-1] != 1 and shape[-1] > 1):
        _bad("sample_rows: logits must be [rows, n] on a CUDA device, with contiguous rows")
    rows, n = shape if len(shape) == 2 else (1, shape[0])
    f, i = _d.torch.float32, _d.torch.int32
    if u is None:
        _bad("sample_rows: u is missing")

    at_u = _row_value(u, "u", f, rows, dev)
    make = lambda: u.new_empty((3, rows)).unbind()  # noqa: E731
    tok, prob, kept = made = make() if stream is None else _new(make, dev, stream)
    tok, kept = tok.view(i), kept.view(i)
    args = PACK_SAMPLE(at_u, _row_value(temp, "temp", f, rows, dev), _row_value(top_k, "top_k", i, rows, dev),
                       _row_value(top_p, "top_p", f, rows, dev), _row_value(min_p, "min_p", f, rows, dev), tok.data_ptr(), prob.data_ptr(), kept.data_ptr())
    _call(_d._L.pk_sample_rows, dev, stream, stream is not None and (logits, u, temp, top_k, top_p, min_p, made), logits.data_ptr(), code, rows, n,
          st[0] if len(st) == 2 else n, args)
    return tok, prob, kept
