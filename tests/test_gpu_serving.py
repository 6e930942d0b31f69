"""The serving operators against plain 64-bit forms: page tables entry by entry, attention over shared prefixes within the
bounds of the attention that it stands beside, drawn tokens one by one."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_drafts import DT, Setup, attention, check_attention, gen, i32, randn, tree, words_of  # noqa: E402

# ---------------------------------------------------------------- page tables


def plan_ref(ctx, new, pages, held, free, n_free, ps, n_tok, done=None, shared=None):
    """The plan step by step on the host."""
    S, wide = pages.shape
    cap = len(free)
    done = done if done is not None else [0] * S
    shared = shared if shared is not None else [0] * S
    held = [min(max(h, 0), wide) for h in held]
    n_free = min(max(n_free, 0), cap)
    pages, old, pool = pages.copy(), list(free), list(free[:n_free])
    for s in range(S):
        if done[s]:
            pool += pages[s, min(max(shared[s], 0), held[s]):held[s]].tolist()
            pages[s, :held[s]] = -1
    had = [0 if done[s] else held[s] for s in range(S)]
    start, pos, seq, slot, lacking = [0], [], [], [], 0
    for s in range(S):
        n = 0 if done[s] or ctx[s] < 0 else min(max(new[s], 0), n_tok - start[-1])
        start.append(start[-1] + n)
        need = min(-(-(ctx[s] + n) // ps), wide) if n else 0
        for j in range(had[s], need):
            if pool:
                pages[s, j] = pool.pop()
                had[s] += 1
            else:
                pages[s, j] = -1
                lacking += 1
        for p in range(ctx[s], ctx[s] + n):
            pos.append(p)
            seq.append(s)
            j = p // ps
            slot.append(int(pages[s, j]) * ps + p % ps if j < had[s] and pages[s, j] >= 0 else -1)
    rest = n_tok - len(pos)
    left = min(len(pool), cap)
    out = pool[:left]
    out += [-1] * max(0, n_free - left)
    out += old[len(out):]
    return {"start": start, "pages": pages, "held": had, "free": out[:cap], "n_free": [left], "lacking": [lacking], "pos": pos + [0] * rest,
            "seq": seq + [-1] * rest, "slot": slot + [-1] * rest}


def plan_case(S, wide, ps, seed, scarce=False, max_new=40, odd=True):
    """Random slots: running, new, done, left out; some with pages to spare, some sharing a prefix."""
    rng = np.random.default_rng(seed)
    ctx = rng.integers(0, max(1, wide * ps - max_new), S)
    ctx[rng.random(S) < 0.2] = 0
    held = np.minimum(-(-ctx // ps) + (rng.random(S) < 0.3), wide)
    new = np.where(rng.random(S) < 0.5, 1, rng.integers(0, max_new + 1, S))
    done = (rng.random(S) < 0.25).astype(int)
    shared = np.where(rng.random(S) < 0.3, rng.integers(0, 4, S), 0)
    if odd:
        ctx[rng.random(S) < 0.05] = -3
        new[rng.random(S) < 0.05] = -2
        held[rng.random(S) < 0.03] = -1
        held[rng.random(S) < 0.03] = wide + 2
        shared[rng.random(S) < 0.05] = 1000
    cap = int(np.maximum(held, 0).sum()) + int(np.maximum(new, 0).sum()) // ps + S + 3
    ids = rng.permutation(3 * cap + S * wide)
    pages = ids[:S * wide].reshape(S, wide).astype(np.int32)
    n_free = int(rng.integers(0, 3)) if scarce else cap - int(held.clip(0, wide).sum())
    n_free = max(0, n_free)
    free = ids[S * wide:S * wide + cap].astype(np.int32)
    return ctx.tolist(), new.tolist(), pages, held.tolist(), free, n_free, done.tolist(), shared.tolist()


def run_plan(pk, c, ps, n_tok, in_place=False, none=False, **kw):
    ctx, new, pages, held, free, n_free, done, shared = c
    t = [i32(ctx), i32(new), torch.from_numpy(pages.copy()).cuda(), i32(held), torch.from_numpy(free.copy()).cuda(), i32([n_free])]
    more = {} if none else {"done": i32(done), "shared": i32(shared)}
    p = pk.kv_plan(*t, ps, n_tok, in_place=in_place, **more, **kw)
    if in_place:
        assert p.pages is t[2] and p.held is t[3] and p.free is t[4] and p.n_free is t[5]
    else:  # the inputs are as they were
        assert t[3].tolist() == held and torch.equal(t[2].cpu(), torch.from_numpy(pages)) and t[5].tolist() == [n_free]
        assert torch.equal(t[4].cpu(), torch.from_numpy(free))
    return p


def check_plan(p, want):
    for name, w in want.items():
        got = getattr(p, name).cpu().numpy()
        assert np.array_equal(got, np.asarray(w, dtype=got.dtype).reshape(got.shape)), name


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("S, wide, ps", [(1, 1, 16), (1, 8, 64), (3, 5, 16), (31, 40, 32), (513, 36, 16), (600, 1030, 16), (2000, 12, 128), (5, 4100, 16)])
def test_plan(pk, S, wide, ps, in_place):
    for seed, scarce in ((1, False), (2, True), (3, False)):
        c = plan_case(S, wide, ps, seed, scarce, max_new=40 if S > 40 else min(5000, wide * ps))
        total = sum(max(0, n) for n in c[1])
        for n_tok in (total + 7, total // 2):  # rows behind the last token; fewer rows than tokens
            check_plan(run_plan(pk, c, ps, n_tok, in_place), plan_ref(*c[:6], ps, n_tok, *c[6:]))
        check_plan(run_plan(pk, c, ps, total, in_place, none=True), plan_ref(*c[:6], ps, total))


def test_plan_most_slots(pk):
    c = plan_case(16384, 8, 16, 5)
    total = sum(max(0, n) for n in c[1])
    for in_place in (False, True):
        check_plan(run_plan(pk, c, 16, total, in_place), plan_ref(*c[:6], 16, total, *c[6:]))


def test_plan_nothing(pk):
    e = lambda *s: torch.empty(s, dtype=torch.int32, device="cuda")  # noqa: E731
    for in_place in (False, True):
        p = pk.kv_plan(e(0), e(0), e(0, 4), e(0), i32([5, 6, 7]), i32([2]), 16, 3, in_place=in_place)
        assert p.start.tolist() == [0] and p.n_free.tolist() == [2] and p.free.tolist() == [5, 6, 7] and p.lacking.tolist() == [0]
        assert p.seq.tolist() == [-1] * 3 and p.slot.tolist() == [-1] * 3 and p.pos.tolist() == [0] * 3
        # no rows, no columns, no list
        p = pk.kv_plan(i32([3, 0]), i32([1, 2]), e(2, 0), i32([0, 0]), e(0), i32([4]), 16, 0, in_place=in_place)
        assert p.start.tolist() == [0, 0, 0] and p.n_free.tolist() == [0] and p.held.tolist() == [0, 0] and p.lacking.tolist() == [0]
        p = pk.kv_plan(i32([3, 0]), i32([1, 2]), e(2, 0), i32([0, 0]), e(0), i32([0]), 16, 3, in_place=in_place)
        assert p.start.tolist() == [0, 1, 3] and p.pos.tolist() == [3, 0, 1] and p.slot.tolist() == [-1] * 3


def test_plan_far_positions(pk):
    """Positions past what 32 bits and the table hold have no page."""
    top = 2 ** 31 - 1
    p = pk.kv_plan(i32([top - 1, 2 ** 20]), i32([3, 2]), torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4), i32([4, 4]), i32([9]), i32([1]), 65536, 5)
    assert p.pos.tolist() == [top - 1, top, top, 2 ** 20, 2 ** 20 + 1] and p.slot.tolist() == [-1] * 5 and p.n_free.tolist() == [1]
    p = pk.kv_plan(i32([2 ** 17]), i32([1]), i32([[1, 2, 2 ** 31 - 1]]), i32([3]), i32([9]), i32([1]), 65536, 1)
    assert p.slot.tolist() == [(2 ** 31 - 1) * 65536]


# ---------------------------------------------------------------- shared prefixes

class SharedSetup(Setup):
    """Groups of `per` sequences behind prefixes of `shared` positions.  A group's whole shared pages stand in its first
    sequence's table alone: in the others' tables they are no pages (or, `wrong`, other sequences')."""

    def __init__(self, pk, groups, own, new, kind="q8", n_kv=2, dh=64, page=16, seed=0, wrong=False, **kw):
        per = [n for _, n in groups]
        lead = [g for g, (_, n) in enumerate(groups) for _ in range(n)]
        lens = [groups[g][0] + o for g, o in zip(lead, own)]
        super().__init__(pk, lens, new, kind, n_kv, dh, page, seed, **kw)
        self.groups, self.lead = groups, lead
        self.first = np.concatenate([[0], np.cumsum(per)]).astype(np.int32)
        self.fill(pk)
        # the prefix as the group's first sequence has it, in the others' own pages too
        for s, g in enumerate(lead):
            a, n = int(self.first[g]), groups[g][0]
            if s == a or n == 0:
                continue
            p = np.arange(n)
            at = lambda x: (torch.as_tensor(self.table[x, p // page].astype(np.int64)).cuda(), torch.as_tensor(p % page).cuda())  # noqa: E731
            (pa, la), (pb, lb) = at(a), at(s)
            for t in (self.cache.k, self.cache.v, self.cache.ks, self.cache.vs):
                t[pb, :, lb] = t[pa, :, la]
        table = self.table.copy()
        for s, g in enumerate(lead):
            if s != self.first[g]:
                table[s, :groups[g][0] // 16 * 16 // page] = self.table[(s + 1) % len(lead), 0] if wrong else -1
        tok = [int(self.start[self.first[g + 1]] - self.start[self.first[g]]) for g in range(len(groups))]
        self.shared_seqs = pk.KvSeqs(i32(self.start), i32(lens), i32(table), self.n_tok, self.max_new, self.max_len)
        self.shared = pk.KvShared(i32(self.first), i32([n for n, _ in groups]), max(tok), max(n for n, _ in groups),
                                  max(o + n for o, n in zip(own, new)))

    def attend(self, q, **kw):
        return self.cache.attend(self.shared_seqs, q, shared=self.shared, **kw)


GROUPS = [
    # (groups of (positions shared, sequences), own positions, new tokens, query heads, kv heads, page)
    ([(16, 2)], [0, 0], [1, 1], 2, 2, 16),
    ([(100, 3)], [0, 37, 1], [1, 2, 1], 4, 2, 64),
    ([(700, 4)], [60, 60, 5, 0], [1, 1, 1, 1], 8, 1, 64),
    ([(15, 2), (333, 1), (0, 2), (1200, 5)], [3, 0, 40, 7, 0, 0, 300, 5, 1, 64], [2, 1, 3, 1, 1, 2, 1, 1, 4, 1], 4, 2, 16),
    ([(2000, 40)], [(37 * i) % 90 for i in range(40)], [1] * 40, 6, 2, 32),
    ([(1030, 9), (64, 20)], [(91 * i) % 700 for i in range(29)], [1 + i % 4 for i in range(29)], 8, 2, 128),
    ([(300, 3)], [10, 2000, 500], [40, 1, 9], 3, 3, 16),
    ([(9000, 6)], [20, 0, 700, 1, 16, 33], [1, 2, 3, 1, 1, 1], 16, 2, 256),
]


@pytest.mark.parametrize("kind", ["q8", "q4"])
@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("ty", list(DT))
@pytest.mark.parametrize("case", range(len(GROUPS)))
def test_shared_causal(pk, kind, dh, ty, case):
    groups, own, new, n_head, n_kv, page = GROUPS[case]
    su = SharedSetup(pk, groups, own, new, kind, n_kv, dh, page, seed=dh + case, extra_rows=2, wrong=case % 2 == 1)
    q = randn((su.n_tok, n_head, dh), 8, DT[ty], std=1.5)
    out = torch.full_like(q, 7.0)
    su.attend(q, out=out)
    check_attention(su, q, out)
    assert (out[int(su.start[-1]):] == 7).all()  # rows that no sequence has
    # and what the same sequences give without a word about their prefix
    check_attention(su, q, su.cache.attend(su.seqs, q))


@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("ty", list(DT))
def test_shared_tree(pk, dh, ty):
    """Drafted trees of 1 to 70 behind prefixes, rows that see nothing new, and some behind no prefix that see nothing."""
    groups, own, new = [(130, 3), (0, 2), (2100, 4)], [0, 20, 3, 0, 0, 300, 0, 17, 64], [5, 1, 70, 4, 3, 16, 16, 9, 33]
    su = SharedSetup(pk, groups, own, new, "q8" if dh == 64 else "q4", 2, dh, 32, seed=5)
    rows = [tree(n, s, empty=(1, 3) if s % 2 else ()) for s, n in enumerate(new)]
    q = randn((su.n_tok, 8, dh), 8, DT[ty])
    got = su.attend(q, mask=words_of(sum(rows, []), 2))

    def see(s, n):
        return torch.tensor([[(b >> j) & 1 for j in range(n)] for b in rows[s]], dtype=torch.bool, device="cuda").reshape(n, n)

    check_attention(su, q, got, see=see)
    assert (got[int(su.start[3]) + 1] == 0).all() and (got[int(su.start[3]) + 3] == 0).all()


@pytest.mark.parametrize("ty", ["f32", "bf16"])
def test_shared_bounds(pk, ty):
    """What does not fit the bounds: a group of more tokens than max_tok and sequences with fewer committed positions than
    their group shares are computed by themselves, from their own pages; len is cut to max_len; of the rest, positions past
    max_own are left out; a negative ctx leaves rows of 0."""
    groups, own, new = [(200, 3), (400, 2), (100, 2)], [10, 20, 0, 30, 500, 0, 8], [1, 2, 1, 1, 1, 9, 9]
    su = SharedSetup(pk, groups, own, new, "q8", 2, 64, 16, seed=6)
    q = randn((su.n_tok, 4, 64), 3, DT[ty])
    first, ln = su.shared.first, su.shared.len
    full = su.seqs  # every sequence's own pages

    def call(max_tok=100, max_len=400, max_own=1000, ctx=None, ln=ln, first=first):
        sq = full if ctx is None else pk.KvSeqs(full.start, i32(ctx), full.pages, su.n_tok, su.max_new, su.max_len)
        return su.cache.attend(sq, q, shared=pk.KvShared(first, ln, max_tok, max_len, max_own))

    check_attention(su, q, call())
    check_attention(su, q, call(max_tok=17))  # the last group has 18
    check_attention(su, q, call(max_tok=0))
    check_attention(su, q, call(max_len=111))
    check_attention(su, q, call(max_len=0))
    check_attention(su, q, call(max_len=2 ** 31 - 1, max_tok=2 ** 31 - 1, max_own=2 ** 31 - 1))
    e = torch.empty(0, dtype=torch.int32, device="cuda")
    check_attention(su, q, call(first=i32([0]), ln=e))  # no groups
    check_attention(su, q, call(first=i32([1, 3]), ln=i32([200])))  # some sequences in no group
    check_attention(su, q, call(first=i32([0, 3, 3, 3, 5, 7]), ln=i32([200, 7, 900, 400, 100])))  # empty groups
    check_attention(su, q, call(ln=i32([200, 10 ** 9, -5])))  # (longer than their ctx: by themselves)
    # fewer committed positions than shared: by itself
    lens = list(su.lens)
    lens[1], lens[3] = 150, 399
    keep, su.lens = su.lens, lens
    check_attention(su, q, call(ctx=lens))
    su.lens = keep
    lens = list(keep)
    lens[2] = lens[5] = -1
    got = call(ctx=lens)
    want = call()
    for s in range(len(lens)):
        a, b = int(su.start[s]), int(su.start[s + 1])
        assert (got[a:b] == 0).all() if s in (2, 5) else torch.equal(got[a:b], want[a:b])
    # max_own 64 leaves of sequence 4 the positions 400 .. 463, and of those alone the first 64
    got = call(max_own=64)
    sq = pk.KvSeqs(full.start, i32([64 - n if s == 99 else c for s, (c, n) in enumerate(zip(su.lens, new))]), full.pages, su.n_tok, su.max_new, 464)
    cut = su.cache.attend(sq, q)
    a = int(su.start[4])
    lim = 3e-2 if ty == "bf16" else 1e-5
    assert (got[a].double() - cut[a].double()).abs().max() <= lim * cut[a].double().abs().max()


@pytest.mark.parametrize("kind", ["q8", "q4"])
@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("ty", list(DT))
def test_shared_many_rows(pk, kind, dh, ty):
    """Hundreds of rows a group: several tiles, a prefix of several chunks that ends inside a tile, pages of it missing,
    garbage where nothing is read, V rows far apart in size, and rows of NaN and infinities that stay their own."""
    groups, new = [(9300, 45), (260, 30), (2000, 3)], [2] * 45 + [1] * 30 + [7, 1, 60]
    own = [(7 * i) % 40 for i in range(78)]
    su = SharedSetup(pk, groups, own, new, kind, 2, dh, 32, seed=3)
    c = su.cache
    table = su.shared_seqs.pages
    holes = {}
    for g, gone in ((0, (0, 5, 100, 200)), (1, (3,)), (2, (0, 1, 2))):  # pages of the prefix that are none
        table[int(su.first[g]), list(gone)] = -1
        for s in range(int(su.first[g]), int(su.first[g + 1])):
            holes[s] = gone
    free = sorted(set(range(c.n_pages)) - set(su.table.ravel().tolist()))
    for t in (c.ks, c.vs):
        t[free, ..., 0] = math.nan
    for s in range(45):  # a few large rows, in every copy of the prefix
        c.vs[torch.as_tensor(su.table[s, :9].astype(np.int64)).cuda(), :, ::3, 0] *= 300.0
    q = randn((su.n_tok, 8, dh), 8, DT[ty], std=1.5)

    def gone(s):
        p = torch.arange(su.lens[s] + su.new[s], device="cuda")
        return ((p[:, None] // 32) == torch.tensor(holes[s], device="cuda")[None]).any(1) & (p < groups[su.lead[s]][0] // 16 * 16)

    got = su.attend(q)
    check_attention(su, q, got, holes=gone)
    bad = q.clone()
    bad[5, 3] = math.nan
    bad[91, 0, 7] = math.inf
    other = su.attend(bad)
    assert torch.isnan(other[5, 3]).all() and torch.isnan(other[91, 0]).all()
    same = torch.ones(q.shape[:2], dtype=torch.bool, device="cuda")
    same[5, 3] = same[91, 0] = False
    assert (other[same].double() - got[same].double()).abs().max() <= 4 * torch.finfo(DT[ty]).eps * got.double().abs().max()


@pytest.mark.parametrize("kind,dh,ty", [("q8", 128, "bf16"), ("q8", 64, "f16"), ("q4", 128, "f16"), ("q4", 64, "bf16")])
def test_shared_whole_tiles_missing(pk, kind, dh, ty):
    """Pages that are none over whole runs of 128 positions, a chunk's first among them: what follows still counts."""
    gone = tuple(range(4)) + tuple(range(16, 20)) + tuple(range(36, 48))
    su = SharedSetup(pk, [(2000, 40), (300, 25)], [(5 * i) % 30 for i in range(65)], [2] * 40 + [4] * 25, kind, 2, dh, 32, seed=12)
    table = su.shared_seqs.pages
    holes = {s: gone if s < 40 else (0, 1, 2, 3) for s in range(65)}
    for g in range(2):
        table[int(su.first[g]), list(holes[int(su.first[g])])] = -1
    q = randn((su.n_tok, 8, dh), 4, DT[ty], std=1.5)

    def missing(s):
        p = torch.arange(su.lens[s] + su.new[s], device="cuda")
        return ((p[:, None] // 32) == torch.tensor(holes[s], device="cuda")[None]).any(1) & (p < (2000 if s < 40 else 288))

    check_attention(su, q, su.attend(q), holes=missing)


@pytest.mark.parametrize("ty", list(DT))
def test_shared_nothing_of_ones_own(pk, ty):
    """max_own 0: every row sees its group's prefix alone, and of a sequence in no group nothing."""
    groups = [(208, 20), (96, 2)]
    su = SharedSetup(pk, groups, [0] * 22, [1] * 22, "q8", 2, 64, 16, seed=6)
    q = randn((su.n_tok, 16, 64), 3, DT[ty])
    sh = pk.KvShared(i32([0, 20]), i32([208]), 20, 208, 0)
    got = su.cache.attend(su.shared_seqs, q, shared=sh)
    cut = Setup.__new__(Setup)
    cut.__dict__.update(su.__dict__)
    cut.lens, cut.new = [207] * 20, [1] * 20  # (its last position as if it were the token's own)
    cut.start = su.start[:21]
    want, absv, dots = attention(cut, q[:20])
    from test_gpu_drafts import attn_bound

    assert ((got[:20].double() - want).abs() <= attn_bound(q[:20], want, absv, dots, 64)).all()
    assert (got[20:] == 0).all()


def test_shared_side_by_side(pk):
    """Calls of different shapes at once on two streams and in captured graphs, each with its own scratch."""
    runs = []
    for i, (ty, dh, case) in enumerate((("f16", 128, 5), ("f32", 64, 4), ("bf16", 64, 7), ("f16", 64, 2), ("bf16", 128, 6))):
        groups, own, new, n_head, n_kv, page = GROUPS[case]
        su = SharedSetup(pk, groups, own, new, "q4" if i % 2 else "q8", n_kv, dh, page, seed=i)
        q = randn((su.n_tok, n_head, dh), i, DT[ty])
        runs.append((su, q, su.attend(q)))
    streams = [torch.cuda.Stream() for _ in range(3)]
    graphs = []
    for j, (su, q, want) in enumerate(runs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = su.attend(q)
        graphs.append((g, out))
    torch.cuda.synchronize()
    for turn in range(10):
        got = []
        for w, st in enumerate(streams):
            with torch.cuda.stream(st):
                for j in range(len(runs)):
                    k = (j + w + turn) % len(runs)
                    if w == 2:
                        graphs[k][0].replay()
                    else:
                        got.append((k, runs[k][0].attend(runs[k][1])))
        torch.cuda.synchronize()
        for k, o in got + [(k, o) for k, (_, o) in enumerate(graphs)]:
            assert torch.equal(o, runs[k][2]), k


def test_shared_strides_scratch_and_order(pk):
    """Strided and unaligned rows, a given scratch, a second call that gives the same bits, and rows in any place."""
    su = SharedSetup(pk, *GROUPS[5][:3], "q8", 2, 128, 64, seed=9)
    for ty in DT.values():
        n = su.n_tok
        wide = randn((n, 11, 131), 3, ty)
        q = wide[:, 2:10, 1:129]
        want = su.attend(q.contiguous())
        out = torch.full((n, 9, 130), 5.0, dtype=ty, device="cuda")
        size = su.cache.attend_scratch_bytes(su.shared_seqs, 8, ty, su.shared)
        scratch = torch.full((size,), 255, dtype=torch.uint8, device="cuda")  # NaN, were it read
        su.attend(q, out=out[:, :8, 1:129], scratch=scratch)
        assert torch.equal(out[:, :8, 1:129], want) and (out[:, 8] == 5).all() and (out[..., 0] == 5).all() and (out[..., 129] == 5).all()
        assert torch.equal(su.attend(q), want)


# ---------------------------------------------------------------- drawing tokens

def draw_ref(x, u, temp=None, top_k=None, top_p=None, min_p=None):
    """One row in 64 bits: (token, prob, kept), and how near u is to a border, relative to the sum."""
    x = np.asarray(x, dtype=np.float64) + 0.0
    x = np.where(np.isnan(x), -np.inf, x)
    ok = x > -np.inf
    if not ok.any():
        return -1, 0.0, 0, 1.0
    order = np.lexsort((np.arange(len(x)), -x))
    order = order[ok[order]]
    t = 1.0 if temp is None else float(temp)
    p = 1.0 if top_p is None or np.isnan(top_p) else float(top_p)
    m = 0.0 if min_p is None or np.isnan(min_p) else float(min_p)
    if not t > 0:
        return int(order[0]), 1.0, 1, 1.0
    top = x[order[0]]
    with np.errstate(invalid="ignore", over="ignore"):
        y = np.where(x == top, 0.0, (x - top) / t)
        w = np.where(np.isnan(y), 0.0, np.exp(y))
    n = len(order)
    ids = order
    if m > 0:
        ids = ids[:max(1, int((w[ids] >= m).sum()))]
    if top_k is not None and top_k > 0:
        ids = ids[:top_k]
    if p < 1:
        ids = ids[:max(1, int(np.searchsorted(np.cumsum(w[ids]), p * w[ids].sum(), side="left")) + 1)]
    n = len(ids)
    ids = np.sort(ids)
    s = np.cumsum(w[ids])
    u = 0.0 if np.isnan(u) else max(float(u), 0.0)  # (u below 0 and NaN count as 0)
    at = int(np.searchsorted(s, u * s[-1], side="right"))
    if at >= n:
        at = int(np.searchsorted(s, s[-1], side="left"))
    near = np.abs(s / s[-1] - u)
    return int(ids[at]), w[ids[at]] / s[-1], n, float(near.min())


def check_draw(pk, x, u, **kw):
    tok, prob, kept = pk.sample_rows(x, u, **kw)
    rows = x.reshape(-1, x.shape[-1])
    host, uh = rows.double().cpu().numpy(), u.double().cpu().numpy()
    kh = {n: None if t is None else t.cpu().numpy() for n, t in kw.items()}
    for r in range(len(host)):
        t, p, n, near = draw_ref(host[r], uh[r], **{k: None if v is None else v[r] for k, v in kh.items()})
        # the kernel's sums of n weights, each within 2^-46 and 1.4e-13 of itself, over the largest's 1
        slack = 2e-13 + len(host[r]) * 2.0 ** -46
        assert int(kept[r]) == n, (r, int(kept[r]), n)
        assert int(tok[r]) == t or near < slack, (r, int(tok[r]), t, near)
        assert abs(float(prob[r]) - p) <= p * 2.0 ** -24 + slack or near < slack, (r, float(prob[r]), p)
    return tok, prob, kept


def likely(rows, n, seed, ty, std=3.0):
    """Rows of logits with a few likely tokens."""
    x = randn((rows, n), seed, std=std)
    at = (torch.randint(0, n, (rows, 1), generator=gen(seed + 1), device="cuda") + torch.arange(20, device="cuda") * max(1, n // 20)) % n
    x.scatter_(1, at, 8 + randn((rows, 20), seed + 2, std=3.0))
    return x.to(DT[ty])


SIZES = [1, 2, 7, 31, 1000, 1025, 4097, 16383, 16385, 32000, 73448]


@pytest.mark.parametrize("ty", list(DT))
@pytest.mark.parametrize("n", SIZES)
def test_draw(pk, ty, n):
    rows = 13
    x, u = likely(rows, n, n, ty) if n > 20 else randn((rows, n), n, DT[ty]), torch.rand(rows, generator=gen(n + 5), device="cuda")
    f = lambda *v: torch.tensor([v[i % len(v)] for i in range(rows)], dtype=torch.float32, device="cuda")  # noqa: E731
    k = i32([(0, 1, 2, 40, 300, n, n + 5, n - 1, -4)[i % 9] for i in range(rows)])
    temp, top_p, min_p = f(1.0, 0.7, 1.5, 3.0), f(0.9, 0.5, 1.0, 0.99, 0.1, 2.0), f(0.0, 0.05, 0.3, 1e-6, 1.0)
    for kw in ({}, {"temp": temp}, {"top_k": k}, {"top_p": top_p}, {"min_p": min_p}, {"temp": temp, "top_k": k, "top_p": top_p},
               {"temp": temp, "top_k": k, "top_p": top_p, "min_p": min_p}, {"top_p": top_p, "min_p": min_p}):
        check_draw(pk, x, u, **kw)


@pytest.mark.parametrize("ty, n", [("f32", 128256), ("bf16", 128256), ("f32", 262144), ("f16", 250001), ("f32", 500003), ("bf16", 1000000)])
def test_draw_long_rows(pk, ty, n):
    """More than one CTA holds three times an SM, than a cluster holds, and than fits it at all; hot rows, whose nucleus is
    far more than what is sorted."""
    rows = 4
    x, u = likely(rows, n, 3, ty), torch.rand(rows, generator=gen(6), device="cuda")
    for t, p, k in ((1.0, 0.9, 50), (2.0, 0.95, 0), (4.0, 0.9, 3000), (8.0, 0.99, n - 3), (30.0, 0.5, 0)):
        check_draw(pk, x, u, temp=torch.full((rows,), t, device="cuda"), top_p=torch.full((rows,), p, device="cuda"), top_k=i32([k] * rows))
    check_draw(pk, x, u)


@pytest.mark.parametrize("ty", list(DT))
def test_draw_equal_logits(pk, ty):
    """Ties by thousands: the lower index first, at every cut."""
    for n in (600, 5000, 40000):
        x = torch.zeros((6, n), dtype=DT[ty], device="cuda")
        x[1] = -7.5
        x[2, ::2] = 1.0
        x[3] = (torch.arange(n, device="cuda") % 3).to(DT[ty])
        x[4, n // 2:] = -math.inf
        x[5, ::3] = -0.0
        u = torch.tensor([0.0, 0.3, 0.9999999, 0.5, 0.77, 0.1], device="cuda")
        full = lambda v: torch.full((6,), v, device="cuda")  # noqa: E731
        for k, p in ((0, 1.0), (3, 1.0), (550, 1.0), (n - 1, 1.0), (0, 0.3141), (0, 0.9998), (n // 3, 0.777), (17, 0.55)):
            check_draw(pk, x, u, top_k=i32([k] * 6), top_p=full(p))


@pytest.mark.parametrize("ty", list(DT))
def test_draw_edges(pk, ty):
    """Rows of nothing, infinities, NaN, and settings at their ends."""
    n = 3001
    x = likely(12, n, 4, ty)
    x[0] = -math.inf
    x[1] = math.nan
    x[2, 7:] = -math.inf
    x[3, ::2] = math.nan
    x[4, 100] = math.inf
    x[5, [5, 900]] = math.inf
    x[6] = -math.inf
    x[6, 2222] = -5.0
    u = torch.rand(12, generator=gen(1), device="cuda")
    full = lambda v: torch.full((12,), v, device="cuda")  # noqa: E731
    one = {"temp": (0.0, -1.0, 1e-3, 1e-30, 1e30, math.inf, math.nan, 1e-45), "top_p": (0.0, -1.0, 1e-9, 0.9999999, math.nan, 5.0),
           "min_p": (1.0, 2.0, math.nan, -1.0, 1e-40)}
    for name, vals in one.items():
        for v in vals:
            for more in ({}, {"top_k": i32([30] * 12)}):
                check_draw(pk, x, u, **{name: full(v)}, **more)
    for v in (0.0, -1.0, 1.0, 7.0, math.nan, 1.0 - 2.0 ** -24, 2.0 ** -149):
        check_draw(pk, x, full(v))
        check_draw(pk, x, full(v), top_k=i32([5] * 12))
    top = float(torch.finfo(DT[ty]).max)
    y = torch.tensor([[top, -top, 0.0, top], [-top, -top, -math.inf, -top], [0.0, -0.0, 0.0, -0.0]], device="cuda").to(DT[ty])
    for v in (0.1, 0.6, 0.99):
        check_draw(pk, y, torch.full((3,), v, device="cuda"))
        check_draw(pk, y, torch.full((3,), v, device="cuda"), min_p=torch.full((3,), 1e-30, device="cuda"), top_k=i32([3, 2, 3]))


def test_draw_frequencies(pk):
    """Over evenly spaced numbers every kept token comes up in proportion (each border moves one count at the most)."""
    n, rows = 50, 20000
    x = randn((1, n), 3).expand(rows, n)
    u = (torch.arange(rows, device="cuda", dtype=torch.float64) + 0.5).div(rows).float()
    tok, prob, kept = pk.sample_rows(x, u, top_k=i32([20]).expand(rows).contiguous())
    w = torch.softmax(x[0].double().masked_fill(x[0] < x[0].topk(20).values[-1], -math.inf), -1)
    count = torch.bincount(tok.long(), minlength=n).double()
    assert (count - w * rows).abs().max() <= 2 and (kept == 20).all()
    assert (prob.double() - w[tok.long()]).abs().max() <= 1e-7


@pytest.mark.parametrize("ty", list(DT))
def test_draw_strides(pk, ty):
    """Rows at odd addresses, rows of a wider tensor, one row for all, a single row without a dimension for it."""
    wide = likely(5, 20011, 2, ty)
    u = torch.rand(5, generator=gen(2), device="cuda")
    k = i32([50, 3, 0, 700, 9])
    for a, b in ((0, 20011), (1, 20010), (3, 5000), (7, 8), (5, 16390)):
        x = wide[:, a:b]
        got = check_draw(pk, x, u, top_k=k)
        for s, t in zip(got, pk.sample_rows(x.contiguous(), u, top_k=k)):
            assert torch.equal(s, t)
    check_draw(pk, wide[:1].expand(5, 20011), u, top_k=k)
    tok, prob, kept = pk.sample_rows(wide[3], u[:1])
    assert torch.equal(tok, pk.sample_rows(wide[3:4], u[:1])[0])


def test_draw_repeats_bit_for_bit(pk):
    x, u = likely(40, 128256, 7, "f32"), torch.rand(40, generator=gen(8), device="cuda")
    kw = {"temp": torch.full((40,), 1.7, device="cuda"), "top_p": torch.full((40,), 0.97, device="cuda"), "top_k": i32([0, 500, 5000, 20] * 10)}
    first = pk.sample_rows(x, u, **kw)
    for _ in range(5):
        for a, b in zip(first, pk.sample_rows(x, u, **kw)):
            assert torch.equal(a, b)


# ---------------------------------------------------------------- together

class Server:
    """A few slots on one cache: each step the plan, rotary positions, K and V stored, attention (over the shared prefix),
    rules and a draw, all on the device."""

    def __init__(self, pk, slots, shared, wide=12, page=16, vocab=3000, seed=0):
        self.pk, self.slots, self.page, self.vocab, self.shared_len = pk, slots, page, vocab, shared
        n_pages = slots * wide + 8
        self.cache = pk.KvCache.empty(n_pages, page, 2, 64, "q8")
        self.table = pk.RopeTable(64)
        self.pages = torch.full((slots, wide), -1, dtype=torch.int32, device="cuda")
        self.held = torch.zeros(slots, dtype=torch.int32, device="cuda")
        self.free = torch.randperm(n_pages, generator=gen(seed), device="cuda").to(torch.int32)
        self.n_free = i32([n_pages])
        self.ctx = torch.zeros(slots, dtype=torch.int32, device="cuda")
        self.emb = {n: randn((vocab, h, 64), seed + i, torch.float16) for i, (n, h) in enumerate((("q", 4), ("k", 2), ("v", 2)))}
        self.head = randn((256, vocab), seed + 9, torch.float16, std=0.1)

    def step(self, ids, n_new, u, n_tok, max_new, groups=None, done=None, shared=None):
        pk = self.pk
        p = pk.kv_plan(self.ctx, n_new, self.pages, self.held, self.free, self.n_free, self.page, n_tok, done=done, shared=shared, in_place=True)
        q, k, v = (self.emb[n][ids] for n in "qkv")
        q, k = pk.rope(self.table, p.pos, q, k, layout="half")
        seqs = pk.KvSeqs(p.start, self.ctx, p.pages, n_tok, max_new, self.pages.shape[1] * self.page)
        self.cache.store(seqs, k, v.contiguous())
        o = self.cache.attend(seqs, q, shared=groups)
        last = p.start[1:].long() - 1
        logits = o[last].reshape(self.slots, 256) @ self.head
        tok, prob, kept = pk.sample_rows(logits, u, temp=torch.full((self.slots,), 0.8, device="cuda"), top_k=i32([40]).expand(self.slots).contiguous())
        return tok, o, p


def test_a_served_batch(pk):
    """Slots admitted behind one prompt's pages, decoded for some steps, one of them finished: the same tokens with the
    prefix shared and with every slot attending by itself, pages neither lost nor held twice."""
    slots, shared = 5, 32
    outs = []
    for share in (True, False):
        sv = Server(pk, slots, shared, seed=3)
        n_pages = sv.cache.n_pages
        prompt = torch.randint(0, sv.vocab, (shared + 5,), generator=gen(4), device="cuda")
        one = i32([shared + 5] + [0] * (slots - 1))
        sv.step(prompt, one, torch.rand(slots, generator=gen(5), device="cuda"), shared + 5, shared + 5)
        # the others get the prompt's whole pages, and its last 5 tokens as their own
        whole = shared // sv.page
        sv.pages[1:, :whole] = sv.pages[:1, :whole]
        sv.held[1:] = whole
        sv.ctx.copy_(i32([shared + 5] + [shared] * (slots - 1)))
        groups = pk.KvShared(i32([0, slots]), i32([shared]), slots * 5, shared, 300) if share else None
        tail = prompt[shared:].repeat(slots - 1)
        sv.step(tail, i32([0] + [5] * (slots - 1)), torch.rand(slots, generator=gen(6), device="cuda"), 5 * (slots - 1), 5, groups)
        sv.ctx.copy_(i32([shared + 5] * slots))
        ids = prompt[-1:].repeat(slots)
        seen = []
        for turn in range(20):
            tok, o, p = sv.step(ids, i32([1] * slots), torch.rand(slots, generator=gen(10 + turn), device="cuda"), slots, 1, groups)
            assert p.lacking.tolist() == [0]
            sv.ctx.add_(1)
            ids = tok.long()
            seen.append((tok, o))
        # slot 3 is done: its own pages go back
        n0, h3 = int(sv.n_free), int(sv.held[3])
        done, sh = i32([0, 0, 0, 1, 0]), i32([0] + [whole] * (slots - 1))
        p = pk.kv_plan(sv.ctx, i32([0] * slots), sv.pages, sv.held, sv.free, sv.n_free, sv.page, 0, done=done, shared=sh, in_place=True)
        assert int(sv.n_free) == n0 + h3 - whole and int(sv.held[3]) == 0
        used = [sv.pages[s, (0 if s == 0 else whole):int(sv.held[s])].tolist() for s in range(slots) if s != 3]
        listed = sum(used, []) + sv.free[:int(sv.n_free)].tolist()
        assert sorted(listed) == list(range(n_pages))
        outs.append(seen)
    for (ta, oa), (tb, ob) in zip(*outs):
        assert torch.equal(ta, tb)
        # both are within the attention's bound of 2^-11 on weights and scores that differ by their order of sums
        assert (oa.double() - ob.double()).abs().max() <= 2.0 ** -9 * ob.double().abs().max()


def test_captured_and_on_another_stream(pk):
    """A step in one graph, replayed, and on a side stream, gives what the calls give one by one."""
    def inputs(seed):
        c = plan_case(40, 20, 16, seed, odd=False, max_new=3)
        return [i32(c[0]), i32(c[1]), torch.from_numpy(c[2]).cuda(), i32(c[3]), torch.from_numpy(c[4]).cuda(), i32([c[5]])], {"done": i32(c[6]), "shared": i32(c[7])}

    su = SharedSetup(pk, *GROUPS[5][:3], "q8", 2, 64, 16, seed=2)
    q, x, u = randn((su.n_tok, 8, 64), 1, torch.float16), likely(9, 30000, 2, "f32"), torch.rand(9, generator=gen(3), device="cuda")
    kw = {"top_k": i32([0, 5, 900] * 3), "top_p": torch.full((9,), 0.95, device="cuda")}
    t, more = inputs(1)

    def calls():
        p = pk.kv_plan(*t, 16, 120, **more)
        return (*p, su.attend(q), *pk.sample_rows(x, u, **kw))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        calls()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = calls()
    for seed in range(2, 6):
        t2, more2 = inputs(seed)
        for a, b in zip(t + list(more.values()), t2 + list(more2.values())):
            if a.shape == b.shape:
                a.copy_(b)
        q.copy_(randn(q.shape, seed, torch.float16))
        u.copy_(torch.rand(9, generator=gen(seed), device="cuda"))
        graph.replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = calls()
        torch.cuda.current_stream().wait_stream(side)
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_raw_stream_argument(pk):
    """A call on `stream` while the current stream is busy, with memory of its own and tensors that the caller drops."""
    su = SharedSetup(pk, *GROUPS[3][:3], "q8", 2, 64, 16, seed=2)
    q, x, u = randn((su.n_tok, 4, 64), 1), likely(3, 9000, 2, "f32"), torch.rand(3, generator=gen(3), device="cuda")
    c = plan_case(40, 20, 16, 4)
    want = su.attend(q), pk.sample_rows(x, u, top_k=i32([9] * 3)), run_plan(pk, c, 16, 200)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        torch.cuda._sleep(20_000_000)
        got = (su.attend(q, stream=side.cuda_stream), pk.sample_rows(x.clone(), u.clone(), top_k=i32([9] * 3), stream=torch.cuda.current_stream().cuda_stream))
        side.synchronize()
        assert torch.equal(got[0], want[0])
        assert all(torch.equal(a, b) for a, b in zip(got[1], want[1]))
    k = i32([9] * 3)
    torch.cuda.synchronize()
    got = pk.sample_rows(x, u, top_k=k, stream=side.cuda_stream)
    t = [i32(c[0]), i32(c[1]), torch.from_numpy(c[2]).cuda(), i32(c[3]), torch.from_numpy(c[4]).cuda(), i32([c[5]]), 16, 200]
    d = {"done": i32(c[6]), "shared": i32(c[7])}
    torch.cuda.synchronize()
    p = pk.kv_plan(*t, **d, stream=side.cuda_stream)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[1])) and all(torch.equal(a, b) for a, b in zip(p, want[2]))


def test_refusals_on_the_device(pk):
    x, u = randn((3, 50), 1), torch.rand(3, device="cuda")
    for bad in (lambda: pk.sample_rows(x.double(), u), lambda: pk.sample_rows(x, u[:2]), lambda: pk.sample_rows(x, u, top_k=u), lambda: pk.sample_rows(x, None),
                lambda: pk.sample_rows(x.t(), torch.rand(50, device="cuda")), lambda: pk.sample_rows(x.cpu(), u), lambda: pk.sample_rows(x, u.cpu()),
                lambda: pk.sample_rows(x[:, :0], u), lambda: pk.KvShared(i32([0, 1]), i32([1, 2]), 1, 1, 1), lambda: pk.KvShared(i32([0, 1]), i32([1]), -1, 1, 1),
                lambda: pk.KvShared(u, i32([1]), 1, 1, 1)):
        with pytest.raises(pk.PkError):
            bad()
    good = dict(ctx=i32([1]), n_new=i32([1]), pages=i32([[0, 1]]), held=i32([1]), free=i32([5]), n_free=i32([1]), page_size=16, n_tok=1)
    pk.kv_plan(**good)
    for kw in ({"n_new": i32([1, 2])}, {"pages": i32([0])}, {"held": torch.ones(1, device="cuda")}, {"n_free": i32([1, 2])}, {"page_size": 24}, {"n_tok": -1},
               {"done": i32([1, 0])}, {"shared": i32([[0]])}, {"free": i32([5]).cpu()}):
        with pytest.raises(pk.PkError):
            pk.kv_plan(**{**good, **kw})
    su = SharedSetup(pk, [(64, 2)], [1, 2], [1, 1], seed=1)
    with pytest.raises(pk.PkError):
        su.attend(randn((2, 4, 64), 1), scratch=torch.empty(16, dtype=torch.uint8, device="cuda"))
    with pytest.raises(pk.PkError):  # more groups than sequences
        su.cache.attend(su.seqs, randn((2, 4, 64), 1), shared=pk.KvShared(i32([0, 1, 1, 2]), i32([4, 4, 4]), 2, 4, 100))
