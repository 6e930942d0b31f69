"""The drafted-decoding entry points refuse bad arguments before they touch the device (no GPU needed)."""
import ctypes as C
import math

import pytest

from pocketinfer import drafts as D

INVALID, UNSUPPORTED = 1, 2
A = 1 << 20  # an aligned address that is never followed: every call here returns before a launch


def cache(**kw):
    c = D.KvCacheC(A, A, A, A, D.KV_Q8, 4, 64, 2, 128)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def seqs(**kw):
    s = D.KvSeqsC(A, A, A, 2, 4, 8, 4, 200)
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def query(**kw):
    q = D.KvQueryC(A, A, None, 512, 128, 512, 128, 0, 4, 0, 0.1)
    for k, v in kw.items():
        setattr(q, k, v)
    return q


BAD_CACHE = [({"type": 1}, UNSUPPORTED), ({"type": 9}, UNSUPPORTED), ({"head_dim": 96}, UNSUPPORTED), ({"head_dim": 0}, UNSUPPORTED),
             ({"n_pages": 0}, INVALID), ({"n_kv": 0}, INVALID), ({"page_size": 8}, INVALID), ({"page_size": 48}, INVALID),
             ({"page_size": 131072}, INVALID), ({"k": None}, INVALID), ({"vs": None}, INVALID), ({"v": A + 8}, INVALID), ({"ks": A + 4}, INVALID)]
BAD_SEQS = [{"n_seq": -1}, {"n_tok": -1}, {"max_new": -3}, {"max_len": -1}, {"max_pages": 0}, {"start": None}, {"ctx": None},
            {"pages": None}, {"ctx": A + 2}, {"max_len": (1 << 30) + 1}]


@pytest.mark.parametrize("what", ["store", "load", "keep", "attn"])
def test_bad_cache_and_sequences(pk, what):
    lib = pk.lib()

    def call(c, s):
        c, s = C.byref(c), C.byref(s)
        if what == "keep":
            return lib.pk_kv_keep(c, s, A, 4, A, None)
        if what == "attn":
            return lib.pk_kv_attn(c, s, C.byref(query()), A, 1 << 30, None)
        return getattr(lib, "pk_kv_" + what)(c, s, A, A, 0, 512, 128, None)

    for kw, code in BAD_CACHE:
        assert call(cache(**kw), seqs()) == code, kw
        assert pk.last_error()
    for kw in BAD_SEQS:
        assert call(cache(), seqs(**kw)) == INVALID, kw
    for kw in ({"n_seq": 0}, {"n_tok": 0}, {"max_new": 0}, {"max_len": 0}):  # nothing to do
        assert call(cache(), seqs(**kw, start=None, ctx=None, pages=None)) == 0, kw


def test_rows_and_keep(pk):
    lib, c, s = pk.lib(), cache(), seqs()
    for fn in (lib.pk_kv_store, lib.pk_kv_load):
        for args, code in (((None, A, 0, 512, 128), INVALID), ((A, None, 0, 512, 128), INVALID), ((A + 2, A, 0, 512, 128), INVALID),
                           ((A, A + 1, 1, 512, 128), INVALID), ((A, A, 12, 512, 128), UNSUPPORTED), ((A, A, 0, 512, 127), INVALID),
                           ((A, A, 0, -1, 128), INVALID), ((A, A, 0, 1 << 41, 128), INVALID)):
            assert fn(C.byref(c), C.byref(s), *args, None) == code, args
    assert lib.pk_kv_load(C.byref(c), C.byref(s), A, A, 0, 64, 128, None) == INVALID  # rows would overlap
    for args in ((None, 4, A), (A, 4, None), (A + 1, 4, A), (A, -1, A)):
        assert lib.pk_kv_keep(C.byref(c), C.byref(s), *args, None) == INVALID, args
    assert lib.pk_kv_keep(C.byref(c), C.byref(s), A, 0, A, None) == 0


def test_attention(pk):
    lib, c, s = pk.lib(), cache(), seqs()
    need = lib.pk_kv_attn_scratch_bytes(C.byref(c), C.byref(seqs(max_len=100000, max_pages=4096)), 4, 0)
    assert need > 0 and need % 4 == 0
    assert lib.pk_kv_attn_scratch_bytes(C.byref(c), C.byref(s), 3, 0) == 0
    for kw, code in (({"type": 12}, UNSUPPORTED), ({"n_head": 0}, INVALID), ({"n_head": 3}, INVALID), ({"scale": 0.0}, INVALID),
                     ({"scale": -1.0}, INVALID), ({"scale": math.inf}, INVALID), ({"scale": math.nan}, INVALID), ({"q": None}, INVALID),
                     ({"out": None}, INVALID), ({"q": A + 2}, INVALID), ({"mask": A, "mask_words": 0}, INVALID),
                     ({"mask": A + 4, "mask_words": 1}, INVALID), ({"mask": A, "mask_words": 5000}, INVALID),
                     ({"q_tok_stride": -1}, INVALID), ({"out_head_stride": 64}, INVALID), ({"out_tok_stride": 100}, INVALID)):
        assert lib.pk_kv_attn(C.byref(c), C.byref(s), C.byref(query(**kw)), A, 1 << 30, None) == code, kw
    big = seqs(max_len=100000, max_pages=4096)
    for scratch, size in ((None, need), (A, need - 1), (A + 8, need), (A, 0)):
        assert lib.pk_kv_attn(C.byref(c), C.byref(big), C.byref(query()), scratch, size, None) == INVALID
    assert str(need) in pk.last_error()


def test_attention_bound_of_new_tokens(pk):
    """Any max_new past the tokens that there are means the same: the same scratch, and more rows than a grid has are
    refused."""
    lib = pk.lib()

    def need(n_head, type_=0, **kw):
        return lib.pk_kv_attn_scratch_bytes(C.byref(cache(n_kv=1)), C.byref(seqs(max_len=100000, max_pages=4096, **kw)), n_head, type_)

    for type_ in (0, 1, 30):
        for n_head in (1, 8, 512, 1 << 20):
            want = need(n_head, type_, max_new=8)
            for most in (9, 1 << 20, 1 << 30, (1 << 31) - 1):
                assert need(n_head, type_, max_new=most) == want, (type_, n_head, most)
    assert need(1 << 20, n_tok=1 << 20, max_new=(1 << 31) - 1) == 0
    for kw, n_head in (({"n_tok": 1 << 20}, 1 << 20), ({"n_seq": (1 << 31) - 1}, 4)):
        s, q = seqs(max_new=(1 << 31) - 1, **kw), query(n_head=n_head)
        assert lib.pk_kv_attn(C.byref(cache()), C.byref(s), C.byref(q), A, 1 << 60, None) == INVALID, kw


def test_rope(pk):
    lib = pk.lib()
    out, g = (C.c_double * 64)(), C.c_float()

    def spec(**kw):
        p = D.RopeSpecC(128, 0, 10000.0, 1.0, 4096.0, 1.0, 32.0, 0.0, None)
        for k, v in kw.items():
            setattr(p, k, v)
        return C.byref(p)

    assert lib.pk_rope_turns(spec(), out, C.byref(g)) == 0 and g.value == 1.0 and abs(out[0] * 2 * math.pi - 1) < 1e-15
    for kw in ({"n_rot": 0}, {"n_rot": 7}, {"n_rot": 5000}, {"theta": 0.0}, {"theta": math.nan}, {"scaling": 4}, {"scaling": -1},
               {"scaling": 1, "factor": 0.0}, {"scaling": 3, "factor": 2.0, "n_ctx_train": 0.0}, {"scaling": 3, "factor": 2.0, "low": 40.0},
               {"gain": -1.0}, {"factors": C.cast((C.c_float * 64)(*([1.0] * 63 + [0.0])), C.c_void_p)}):
        assert lib.pk_rope_turns(spec(**kw), out, C.byref(g)) == INVALID, kw
    assert lib.pk_rope_turns(None, out, C.byref(g)) == INVALID

    def args(**kw):
        a = D.RopeArgsC(A, A, A, A, A, A, 512, 128, 256, 128, 512, 128, 256, 128, 0, 0, 3, 4, 2, 128, 128, 1.0)
        for k, v in kw.items():
            setattr(a, k, v)
        return C.byref(a)

    for kw, code in (({"type": 8}, UNSUPPORTED), ({"layout": 2}, INVALID), ({"n_rot": 130}, INVALID), ({"n_rot": 3}, INVALID),
                     ({"n_tok": -1}, INVALID), ({"q": None, "k": None}, INVALID), ({"pos": None}, INVALID), ({"turns": A + 4}, INVALID),
                     ({"q_out": None}, INVALID), ({"k_out": None}, INVALID), ({"q": A + 2}, INVALID), ({"ko_head_stride": 64}, INVALID),
                     ({"q_tok_stride": -4}, INVALID)):
        assert lib.pk_rope(args(**kw), None) == code, kw
    assert lib.pk_rope(args(n_tok=0), None) == 0
    assert lib.pk_rope(args(n_head=0, k=None), None) == 0


def test_logit_rules(pk):
    lib = pk.lib()

    def call(ptr=(A, A), ty=0, rows=2, n=100, st=(100, 100), **kw):
        r = D.LogitRulesC()
        for k, v in kw.items():
            setattr(r, k, v)
        return lib.pk_apply_logit_rules(ptr[0], ptr[1], ty, rows, n, st[0], st[1], C.byref(r), None)

    assert call(ty=12) == UNSUPPORTED
    for kw in ({"ptr": (None, A)}, {"ptr": (A, None)}, {"ptr": (A + 1, A)}, {"rows": -1}, {"n": -1}, {"st": (-1, 100)}, {"st": (100, 99)},
               {"st": (200, 100)}, {"hist": A, "n_hist_max": -1}, {"bias_id": A, "n_bias": 3}, {"bias": A}, {"hist": A, "hist_stride": -1},
               {"allow": A + 2}, {"n_bias": -1}):
        assert call(**kw) == INVALID, kw
    assert lib.pk_apply_logit_rules(A, A, 0, 2, 100, 100, 100, None, None) == INVALID
    assert call(rows=0) == 0 and call(n=0) == 0


def test_binding_refuses_host_tensors(pk):
    torch = pytest.importorskip("torch")
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    for bad in (lambda: pk.KvSeqs(i(3), i(2), i(2, 4), 8, 4, 100), lambda: pk.KvSeqs(i(3).long(), i(2), i(2, 4), 8, 4, 100),
                lambda: pk.KvCache.empty(4, 16, 2, 128, "q6", device="cpu"), lambda: pk.KvCache.empty(4, 16, 2, 128, "q8", device="cpu"),
                lambda: pk.logit_rules(torch.zeros(2, 8)), lambda: pk.RopeTable(127, device="cpu"),
                lambda: pk.rope(pk.RopeTable(64, device="cpu"), i(2), torch.zeros(2, 1, 64), layout="quarter")):
        with pytest.raises(pk.PkError):
            bad()


@pytest.mark.parametrize("bounds", [(2 ** 32, 4, 100), (8, 2 ** 32, 100), (8, 4, 2 ** 32), (8, 4, 2 ** 31), (-1, 4, 100), (8, -4, 100), (8, 4, -2 ** 32)])
def test_bounds_that_the_structure_cannot_hold(pk, bounds):
    torch = pytest.importorskip("torch")
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(pk.PkError, match="not within"):
        pk.KvSeqs(i(3), i(2), i(2, 4), *bounds)


def test_strides_of_single_rows(pk):
    """K and V of one token or one head are alike whatever the strides of those dimensions."""
    torch = pytest.importorskip("torch")
    f = torch.zeros((4, 6, 64))
    for k, v, ok in ((f[:1, :2], torch.zeros(1, 2, 64), True), (f[:, :1], f[:, 5:], True), (f[:1, :1], torch.zeros(1, 1, 64), True),
                     (f[:, :2], f[:, 4:], True), (f[:, :2], torch.zeros(4, 2, 64), False), (f[:, :1], torch.zeros(4, 1, 64), False),
                     (f[:1, :2], torch.zeros(1, 64, 2).transpose(1, 2), False)):
        assert D._same_strides(k, v) == ok, (k.stride(), v.stride())


@pytest.mark.parametrize("n_rot,theta,ctx,factor", [(128, 10000.0, 4096, 8.0), (64, 500000.0, 8192, 32.0), (48, 10000.0, 2048, 4.0)])
def test_ramp_by_index_as_factors(pk, n_rot, theta, ctx, factor):
    """The long-context ramp that is linear in the pair's index, through factors: every turn within the factor's rounding
    to f32.  It is not the one that is linear in the turns."""
    at = lambda turns: n_rot / 2 * math.log(ctx / (turns * 2 * math.pi)) / math.log(theta)  # noqa: E731  (pair that turns so often)
    lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), n_rot - 1)
    want, factors = [], []
    for i in range(n_rot // 2):
        keep = 1.0 - min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0)
        f = theta ** (-2.0 * i / n_rot) / (2 * math.pi)
        want.append(f / factor * (1 - keep) + f * keep)
        factors.append(1.0 / (keep + (1 - keep) / factor))
    gain = 0.1 * math.log(factor) + 1
    table = pk.RopeTable(n_rot, theta, factors=factors, gain=gain, device="cpu")
    assert abs(table.gain - gain) < 1e-7 * gain
    assert all(abs(a - b) <= b * (2.0 ** -24 + 1e-14) for a, b in zip(table.turns.tolist(), want))
    other = pk.RopeTable(n_rot, theta, "yarn", factor, ctx, device="cpu")
    assert max(a / b for a, b in zip(other.turns.tolist(), want)) > 1.3 or min(a / b for a, b in zip(other.turns.tolist(), want)) < 0.8


def test_mask_without_words(pk):
    """A mask of no words is refused: its tensor has no address, and no address means causal."""
    torch = pytest.importorskip("torch")
    with pytest.raises(pk.PkError):  # (sets the binding up)
        pk.logit_rules(torch.zeros(2, 8))
    m = lambda *s: torch.zeros(s, dtype=torch.int64)  # noqa: E731
    assert D._mask(m(3, 1), 3, -1)[0] == 1 and D._mask(m(3, 70), 3, -1)[0] == 70
    for bad in (m(3, 0), m(2, 1), m(3), m(3, 2)[:, :1], m(3, 1).int(), m(0, 0)):
        with pytest.raises(pk.PkError):
            D._mask(bad, 3, -1)


def test_packed_structures_match_the_header():
    """The packed bytes have the fields where the ctypes structures (the C layouts) have them."""
    q = D.PACK_QUERY(1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 0.5)
    r = D.PACK_ROPE(*range(1, 22), 0.5)
    u = D.PACK_RULES(*range(1, 14))
    for cls, data, last in ((D.KvQueryC, q, 0.5), (D.RopeArgsC, r, 0.5), (D.LogitRulesC, u, 13)):
        s = cls.from_buffer_copy(data + bytes(C.sizeof(cls) - len(data)))
        got = [getattr(s, n) for n, _ in cls._fields_]
        assert got == list(range(1, len(got))) + [last], cls


def test_binding_structures_match_the_compiler(tmp_path):
    """sizeof and offsetof of the header's structures, as a C compiler has them."""
    import os
    import subprocess

    from conftest import ROOT

    names = {"pk_kv_cache": D.KvCacheC, "pk_kv_seqs": D.KvSeqsC, "pk_kv_query": D.KvQueryC, "pk_rope_spec": D.RopeSpecC,
             "pk_rope_args": D.RopeArgsC, "pk_logit_rules": D.LogitRulesC}
    lines = [f'printf("{n} %zu", sizeof({n}));' + "".join(f'printf(" %zu", offsetof({n}, {f}));' for f, _ in c._fields_) + 'puts("");'
             for n, c in names.items()]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include "pk.h"\nint main(void) {\n' + "\n".join(lines) + "\nreturn 0;\n}\n")
    exe = str(tmp_path / "layout")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", exe], check=True)
    for line in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.splitlines():
        name, size, *offs = line.split()
        c = names[name]
        assert int(size) == C.sizeof(c) and [int(o) for o in offs] == [getattr(c, f).offset for f, _ in c._fields_], name
