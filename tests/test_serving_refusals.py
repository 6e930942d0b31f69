"""The serving entry points refuse bad arguments before they touch the device, and their structures are laid out as the
compiler lays them out (no GPU needed)."""
import ctypes as C
import os
import subprocess

import pytest

from conftest import ROOT
from pocketinfer import drafts as D
from pocketinfer import serving as S
from test_drafts_refusals import A, BAD_CACHE, BAD_SEQS, INVALID, UNSUPPORTED, cache, query, seqs


def shared(**kw):
    x = S.KvSharedC(A, A, 1, 8, 100, 64)
    for k, v in kw.items():
        setattr(x, k, v)
    return x


def test_shared_attention(pk):
    lib = pk.lib()

    def call(c=None, s=None, sh=None, q=None, scratch=A, size=1 << 40):
        return lib.pk_kv_attn_shared(C.byref(c or cache()), C.byref(s or seqs()), C.byref(sh or shared()), C.byref(q or query()), scratch, size, None)

    for kw, code in BAD_CACHE:
        assert call(c=cache(**kw)) == code, kw
    for kw in BAD_SEQS:
        assert call(s=seqs(**kw)) == INVALID, kw
    for kw in ({"n_group": -1}, {"n_group": 3}, {"max_tok": -1}, {"max_len": -1}, {"max_own": -1}, {"first": None}, {"len": None}, {"first": A + 2}, {"len": A + 1}):
        assert call(sh=shared(**kw)) == INVALID, kw
        assert pk.last_error().startswith("pk_kv_attn_shared")
    for kw, code in (({"type": 12}, UNSUPPORTED), ({"n_head": 3}, INVALID), ({"scale": 0.0}, INVALID), ({"q": None}, INVALID), ({"out": A + 2}, INVALID),
                     ({"mask": A, "mask_words": 0}, INVALID), ({"q_tok_stride": -1}, INVALID), ({"out_tok_stride": 100}, INVALID)):
        assert call(q=query(**kw)) == code, kw
    assert lib.pk_kv_attn_shared(C.byref(cache()), C.byref(seqs()), None, C.byref(query()), A, 1 << 40, None) == INVALID
    for kw in ({"n_seq": 0}, {"n_tok": 0}, {"max_new": 0}, {"max_len": 0}):  # nothing to do
        assert call(s=seqs(**kw, start=None, ctx=None, pages=None), sh=shared(n_group=0, first=None, len=None)) == 0, kw
    # the scratch: what the bytes function says, 16-byte aligned
    c, s, q = cache(), seqs(n_seq=40, n_tok=40, max_len=100000, max_pages=4096), query()
    for sh in (shared(max_len=90000, max_tok=40, max_own=500), shared(max_len=0, max_own=100000), shared(max_len=90000, max_tok=40, max_own=50000)):
        need = lib.pk_kv_attn_shared_scratch_bytes(C.byref(c), C.byref(s), C.byref(sh), 4, 0)
        if need:
            for scratch, size in ((None, need), (A, need - 1), (A + 8, need)):
                assert call(c, s, sh, q, scratch, size) == INVALID
                assert str(need) in pk.last_error()
    assert need > 0
    assert lib.pk_kv_attn_shared_scratch_bytes(C.byref(c), C.byref(s), C.byref(shared()), 3, 0) == 0
    # bounds past what there is mean what there is
    big = (1 << 31) - 1
    for type_ in (0, 1, 30):
        want = lib.pk_kv_attn_shared_scratch_bytes(C.byref(c), C.byref(s), C.byref(shared(max_tok=40, max_len=100000, max_own=100000)), 8, type_)
        assert lib.pk_kv_attn_shared_scratch_bytes(C.byref(c), C.byref(s), C.byref(shared(max_tok=big, max_len=big, max_own=big)), 8, type_) == want


def test_plan(pk):
    lib = pk.lib()

    def call(**kw):
        n = {f: A + 4096 * (i + 1) for i, (f, t) in enumerate(S.KvPlanC._fields_) if t is C.c_void_p}
        n.update(n_seq=4, max_pages=8, free_cap=16, n_tok=10, page_size=16)
        n.update(kw)
        return lib.pk_kv_plan(C.byref(S.KvPlanC(*[n[f] for f, _ in S.KvPlanC._fields_])), None)

    for kw in ({"n_seq": -1}, {"n_seq": 16385}, {"n_tok": -1}, {"n_tok": (1 << 30) + 1}, {"max_pages": -1}, {"free_cap": -1}, {"page_size": 0}, {"page_size": 8},
               {"page_size": 48}, {"page_size": 131072}, {"n_seq": 16384, "max_pages": 1 << 17}, {"ctx": None}, {"n_new": None}, {"pages": None},
               {"held": None}, {"free": None}, {"n_free": None}, {"pages_out": None}, {"held_out": None}, {"free_out": None}, {"n_free_out": None},
               {"start": None}, {"lacking": None}, {"ctx": A + 1}, {"slot": A + 4}, {"done": A + 2}, {"pos": A + 3}):
        assert call(**kw) == INVALID, kw
        assert pk.last_error().startswith("pk_kv_plan")
    # in place: all of them or none
    same = {"pages": A, "pages_out": A, "held": A + 512, "held_out": A + 512, "free": A + 1024, "free_out": A + 1024, "n_free": A + 2048, "n_free_out": A + 2048}
    for name in ("pages_out", "held_out", "free_out", "n_free_out"):
        assert call(**{**same, name: A + 4096}) == INVALID, name
        assert "in place" in pk.last_error()
    assert lib.pk_kv_plan(None, None) == INVALID


def test_sample_rows(pk):
    lib = pk.lib()

    def call(logits=A, ty=0, rows=3, n=100, stride=100, **kw):
        a = S.SampleC(A, A, A, A, A, A, A, A)
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.pk_sample_rows(logits, ty, rows, n, stride, C.byref(a), None)

    for kw, code in (({"ty": 12}, UNSUPPORTED), ({"ty": 8}, UNSUPPORTED), ({"rows": -1}, INVALID), ({"rows": (1 << 24) + 1}, INVALID), ({"n": 0}, INVALID),
                     ({"n": (1 << 30) + 1}, INVALID), ({"stride": -1}, INVALID), ({"stride": 1 << 41}, INVALID), ({"logits": None}, INVALID), ({"logits": A + 2}, INVALID),
                     ({"logits": A + 1, "ty": 1}, INVALID), ({"u": None}, INVALID), ({"tok": None}, INVALID), ({"temp": A + 2}, INVALID), ({"kept": A + 1}, INVALID)):
        assert call(**kw) == code, kw
        assert pk.last_error().startswith("pk_sample_rows")
    assert lib.pk_sample_rows(A, 0, 3, 100, 100, None, None) == INVALID
    assert call(rows=0, logits=None, u=None) == 0


def test_structures_as_the_compiler_lays_them_out(pk, tmp_path):
    """sizeof and every offset of the C structures, and that the packed forms have the same bytes."""
    names = {"pk_kv_shared": S.KvSharedC, "pk_kv_plan_args": S.KvPlanC, "pk_sample_args": S.SampleC}
    lines = ['#include <stddef.h>', '#include <stdio.h>', '#include "pk.h"', "int main(void) {"]
    for c, py in names.items():
        lines.append(f'printf("%zu", sizeof({c}));')
        lines += [f'printf(" %zu", offsetof({c}, {f}));' for f, _ in py._fields_]
        lines.append('printf("\\n");')
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines) + "\nreturn 0; }\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines()
    for (c, py), line in zip(names.items(), out):
        assert [int(x) for x in line.split()] == [C.sizeof(py)] + [getattr(py, f).offset for f, _ in py._fields_], c
    plan = [A + 8 * i for i in range(17)] + [3, 4, 5, 6, 16]
    assert S.PACK_PLAN(*plan).ljust(C.sizeof(S.KvPlanC), b"\0") == bytes(S.KvPlanC(*plan))
    sample = [A + 8 * i for i in range(8)]
    assert S.PACK_SAMPLE(*sample) == bytes(S.SampleC(*sample))


def test_signatures_cover_the_entry_points(pk):
    for n in ("pk_kv_attn_shared_scratch_bytes", "pk_kv_attn_shared", "pk_kv_plan", "pk_sample_rows"):
        assert n in D.SIGNATURES and n in pk.SYMBOLS


@pytest.mark.parametrize("kw", [{"max_tok": -1}, {"max_len": 1 << 31}, {"max_own": -5}])
def test_binding_bounds(pk, kw):
    torch = pytest.importorskip("torch")
    z = torch.zeros(2, dtype=torch.int32)
    args = {"max_tok": 1, "max_len": 1, "max_own": 1, **kw}
    with pytest.raises(pk.PkError):
        pk.KvShared(z, z[:1], **args)
    with pytest.raises(pk.PkError):  # not on a CUDA device
        pk.KvShared(z, z[:1], 1, 1, 1)
    with pytest.raises(pk.PkError):
        pk.kv_plan(z, z, z.view(2, 1), z, z, z[:1], 16, 4)
    with pytest.raises(pk.PkError):
        pk.sample_rows(torch.zeros(2, 5), torch.zeros(2))
