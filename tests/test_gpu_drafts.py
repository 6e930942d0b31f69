"""The drafted-decoding operators against plain 64-bit forms: the quantised cache bit for bit, attention, rotary positions
and logit rules within bounds counted from their roundings."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BIG = 2.0 ** 127


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(shape, seed, dtype=torch.float32, std=1.0):
    return (torch.randn(shape, generator=gen(seed), device="cuda") * std).to(dtype)


def half_step(want, t):
    """A rounding to t is off by at most half a step: eps / 2 of the value, and below the smallest normal value, where
    steps stay smallest_normal * eps wide (f16: 2^-24), half of that."""
    f = torch.finfo(t)
    return (want.abs() * (f.eps / 2)).clamp(min=f.smallest_normal * f.eps / 2)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ---------------------------------------------------------------- plain forms

def f32(x):
    return x.float().double()  # one rounding to f32 of a 64-bit value


def stored(x, kind):
    """(values a row reads back as, in f32; rows x [..., dh])."""
    x = x.double().nan_to_num(nan=0.0, posinf=BIG, neginf=-BIG).clamp(-BIG, BIG)
    amax = x.abs().amax(-1, keepdim=True)
    if kind == "q8":
        d = f32(amax / 127)
        c = torch.where(d > 0, torch.round(x / d.clamp(min=1e-300)), torch.zeros_like(x)).clamp(-127, 127)
        return (c * d).float()
    d = f32(amax / 105)
    y = x.unflatten(-1, (-1, 32))
    seven = f32(7 * d).unsqueeze(-1)
    s = torch.ceil(f32(y.abs().amax(-1, keepdim=True) / seven.clamp(min=1e-300))).clamp(1, 15)
    s = torch.where(seven > 0, s, torch.ones_like(s))
    step = f32(d.unsqueeze(-1) * s)
    c = torch.where(step > 0, torch.round(y / step.clamp(min=1e-300)), torch.zeros_like(y)).clamp(-8, 7)
    return ((c * s).flatten(-2) * d).float()


def decoded(cache):
    """(k, v) [n_pages, n_kv, page_size, dh] in 64 bits."""
    out = []
    for codes, sc in ((cache.k, cache.ks), (cache.v, cache.vs)):
        if cache.kind == "q8":
            out.append((codes.double() - 128) * sc.double())
            continue
        nib = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).double() - 8
        word = sc[..., 1:].contiguous().view(torch.int32)
        s = (word >> (4 * torch.arange(cache.head_dim // 32, device="cuda", dtype=torch.int32))) & 15
        out.append((nib.unflatten(-1, (-1, 32)) * s.unsqueeze(-1).double()).flatten(-2) * sc[..., :1].double())
    return out


class Setup:
    """A cache with random pages, its sequences, and everything on the host too."""

    def __init__(self, pk, lens, new, kind="q8", n_kv=2, dh=64, page=16, seed=0, extra_rows=0, slack=0, pool=None):
        rng = np.random.default_rng(seed)
        self.lens, self.new, self.page, self.kind = lens, new, page, kind
        need = [max(1, -(-(c + n) // page)) for c, n in zip(lens, new)]
        n_pages = pool or sum(need) + 2
        order = rng.permutation(n_pages)[:sum(need)]
        table = np.full((len(lens), max(need) + slack), -1, np.int32)
        at = 0
        for s, n in enumerate(need):
            table[s, :n] = order[at:at + n]
            at += n
        self.table = table
        self.start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.n_tok = int(self.start[-1]) + extra_rows
        self.cache = pk.KvCache.empty(n_pages, page, n_kv, dh, kind)
        self.max_new, self.max_len = max(max(new), 1), max(max(c + n for c, n in zip(lens, new)), 1)
        self.seqs = pk.KvSeqs(i32(self.start), i32(lens), i32(table), self.n_tok, self.max_new, self.max_len)

    def fill(self, pk, seed=1, std_v=1.0):
        """Every position of every sequence written through store()."""
        total = [c + n for c, n in zip(self.lens, self.new)]
        start = np.concatenate([[0], np.cumsum(total)])
        t = int(start[-1])
        if t == 0:
            return
        k = randn((t, self.cache.n_kv, self.cache.head_dim), seed)
        k[..., ::9] *= 3
        v = randn((t, self.cache.n_kv, self.cache.head_dim), seed + 1, std=std_v) * (0.2 + torch.rand((t, 1, 1), generator=gen(seed + 2), device="cuda"))
        self.cache.store(pk.KvSeqs(i32(start), i32([0] * len(total)), self.seqs.pages, t, max(total), max(total)), k, v)

    def rows(self, s):
        """(page, slot) of sequence s's positions."""
        p = np.arange(self.lens[s] + self.new[s])
        return torch.as_tensor(self.table[s, p // self.page].astype(np.int64)).cuda(), torch.as_tensor(p % self.page).cuda()


def attention(su, q, see=None, scale=None, holes=None):
    """(out, bound's parts) in 64 bits; see(s, n) -> bool [n, n] of the new tokens; holes(s) -> bool [total] of
    positions without a page."""
    k64, v64 = decoded(su.cache)
    n_kv, dh = su.cache.n_kv, su.cache.head_dim
    group = q.shape[1] // n_kv
    scale = dh ** -0.5 if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    absv, dots = torch.zeros_like(out), torch.zeros(q.shape[:2], dtype=torch.float64, device="cuda")
    for s, n in enumerate(su.new):
        if n == 0:
            continue
        c, a = su.lens[s], int(su.start[s])
        pg, sl = su.rows(s)
        vis = torch.ones((n, c + n), dtype=torch.bool, device="cuda")
        vis[:, c:] = torch.ones((n, n), dtype=torch.bool, device="cuda").tril() if see is None else see(s, n)
        if holes is not None:
            vis &= ~holes(s)[None]
        for h in range(q.shape[1]):
            k, v = k64[pg, h // group, sl], v64[pg, h // group, sl]
            x = q[a:a + n, h].double()
            w = (x @ k.T * scale).masked_fill(~vis, -math.inf)
            p = torch.softmax(w, -1).nan_to_num(nan=0.0)
            out[a:a + n, h] = p @ v
            absv[a:a + n, h] = p @ v.abs()
            dots[a:a + n, h] = (x.abs() @ k.abs().T * scale).amax(-1)
    return out, absv, dots


def attn_bound(q, want, absv, dots, dh):
    """Per element: the weights' rounding to f16 (2^-11 relative; 2^-22 as two terms), the error of the scores (each of
    the dh products and sums, the scales and the exponent's argument off by at most 2^-23 of sum |q k|, on both sides of
    the quotient), the sums over positions (2^-20 covers 8 accumulations in a chunk's order), and the output's rounding."""
    t = q.dtype
    weights = 2.0 ** -21 if t == torch.float32 else 2.0 ** -11
    # queries: exact in f16 for half types (2^-25 of the row's largest below its normal range), 2^-22 as two terms
    score = (dh + 8) * 2.0 ** -23 + 2.0 ** -22
    return absv * (weights + 2.0 ** -20 + 2 * score * dots.unsqueeze(-1)) + half_step(want, t) + 1e-30


def check_attention(su, q, got, **kw):
    want, absv, dots = attention(su, q, **kw)
    rows = int(su.start[-1])
    err = (got.double() - want).abs()[:rows]
    lim = attn_bound(q, want, absv, dots, su.cache.head_dim)[:rows]
    worst = (err / lim).max().item() if rows else 0.0
    assert torch.isfinite(got[:rows].double()).all()
    assert worst <= 1.0, worst


# ---------------------------------------------------------------- the cache

@pytest.mark.parametrize("kind", ["q8", "q4"])
@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("ty", list(DT))
def test_store_then_load(pk, kind, dh, ty):
    """Codes and scales are the definition's, bit for bit, at ragged lengths, from one token to several pages."""
    for lens, new, n_kv, page in (([0], [1], 1, 16), ([5, 0, 31, 16], [3, 0, 18, 40], 3, 16), ([100, 7], [1, 130], 5, 64)):
        su = Setup(pk, lens, new, kind, n_kv, dh, page, seed=dh, extra_rows=2)
        k = randn((su.n_tok, n_kv, dh), 3, DT[ty])
        v = randn((su.n_tok, n_kv, dh), 4, DT[ty], std=30.0)
        k[..., ::13] *= 9
        su.cache.store(su.seqs, k, v)
        rows = int(su.start[-1])
        gk, gv = su.cache.load(su.seqs, torch.float32)
        assert torch.equal(gk[:rows], stored(k, kind)[:rows]) and torch.equal(gv[:rows], stored(v, kind)[:rows])
        for t in ("f16", "bf16"):
            hk, hv = su.cache.load(su.seqs, DT[t])
            assert torch.equal(hk[:rows], gk[:rows].to(DT[t])) and torch.equal(hv[:rows], gv[:rows].to(DT[t]))


@pytest.mark.parametrize("kind", ["q8", "q4"])
def test_store_edge_values(pk, kind):
    """Zero rows, zero blocks, ties between codes, the largest and smallest magnitudes, NaN and infinities."""
    dh = 128
    x = torch.zeros((12, 1, dh), device="cuda")
    x[1] = 1.0
    x[2, 0, 5] = -3.0                                                     # one value, three zero blocks
    x[3] = torch.arange(dh, device="cuda") - 64.0
    x[4] = (torch.arange(dh, device="cuda") % 32 - 15.5) * 2 + 0.0        # halves of a step
    x[4, 0, 0] = 127.0
    x[5] = torch.randn(dh, generator=gen(1), device="cuda") * 1e-44       # subnormal
    x[6] = torch.randn(dh, generator=gen(2), device="cuda") * 1e38
    x[7, 0, 3], x[7, 0, 4] = math.inf, 1.0
    x[8, 0, 3], x[8, 0, 4] = math.nan, 2.0
    x[9] = -math.inf
    x[10] = torch.where(torch.arange(dh, device="cuda") < 32, 105.0, 3.5)
    x[11] = torch.arange(dh, device="cuda").float().remainder(7).sub(3) * 0.5
    su = Setup(pk, [3], [12], kind, 1, dh, 16)
    su.cache.store(su.seqs, x, -x)
    k, v = su.cache.load(su.seqs)
    assert torch.isfinite(k).all() and torch.isfinite(v).all()
    assert torch.equal(k, stored(x, kind)) and torch.equal(v, stored(-x, kind))
    assert k[0].abs().max() == 0 and k[9].max() == k[9].min() < -1.6e38


@pytest.mark.parametrize("kind", ["q8", "q4"])
def test_store_leaves_the_rest(pk, kind):
    """Only the new tokens' slots change; tokens with no page, no sequence or no room are dropped; strided and unaligned
    inputs are read where they lie, and load() leaves rows without a sequence as they were."""
    dh, n_kv = 64, 2
    su = Setup(pk, [10, 30], [4, 9], kind, n_kv, dh, 16, extra_rows=3)
    su.fill(pk)
    before = [t.clone() for t in (su.cache.k, su.cache.v, su.cache.ks, su.cache.vs)]
    big = randn((su.n_tok, n_kv + 3, dh + 6), 9, torch.float16)
    k, v = big[:, 1:1 + n_kv, 3:3 + dh], big[:, 2:2 + n_kv, 5:5 + dh]
    table = su.table.copy()
    table[1, 2] = -1                                                       # positions 32 .. of sequence 1
    bad = pk.KvSeqs(su.seqs.start, su.seqs.ctx, i32(table), su.n_tok, su.max_new, 37)  # and none from 37 on
    su.cache.store(bad, k, v)
    wk, wv = stored(k, kind), stored(v, kind)
    touched = torch.zeros(su.cache.k.shape[:3], dtype=torch.bool, device="cuda")
    k64, v64 = decoded(su.cache)
    for s in range(2):
        for i in range(su.new[s]):
            p = su.lens[s] + i
            page = table[s, p // 16]
            if page < 0 or p >= 37:
                continue
            touched[page, :, p % 16] = True
            row = int(su.start[s]) + i
            assert torch.equal(k64[page, :, p % 16].float(), wk[row]) and torch.equal(v64[page, :, p % 16].float(), wv[row])
    assert touched.sum() == (4 + 2) * n_kv
    for a, b in zip((su.cache.k, su.cache.v, su.cache.ks, su.cache.vs), before):
        assert torch.equal(a[~touched].view(torch.uint8), b[~touched].view(torch.uint8))
    out = torch.full((2, su.n_tok, n_kv + 1, dh + 1), 7.0, device="cuda")
    ko, vo = out[0, :, :n_kv, 1:], out[1, :, :n_kv, 1:]
    su.cache.load(bad, out=(ko, vo))
    assert (out[:, -3:] == 7).all() and (out[:, :, n_kv] == 7).all() and (out[..., 0] == 7).all()
    assert (ko[4 + 2:4 + 9] == 0).all()                                    # without a page: zero
    assert torch.equal(ko[:4], k64[table[0, 0], :, 10:14].float().transpose(0, 1))


def test_store_and_load_single_rows(pk):
    """One token or one head: K and V of different strides in that dimension."""
    for n_tok, n_kv in ((1, 3), (5, 1), (1, 1)):
        su = Setup(pk, [7], [n_tok], "q8", n_kv, 64, 16)
        k = randn((n_tok, n_kv, 64), 1)
        v = randn((n_tok, n_kv + 2, 64), 2)[:, 1:1 + n_kv] if n_tok == 1 else randn((n_tok, n_kv, 64), 2)[:, ::2]
        su.cache.store(su.seqs, k, v)
        out = torch.zeros_like(k), torch.zeros((n_tok, n_kv + 3, 64), device="cuda")[:, :n_kv] if n_tok == 1 else torch.zeros_like(v)
        su.cache.load(su.seqs, out=out)
        assert torch.equal(out[0], stored(k, "q8")) and torch.equal(out[1], stored(v, "q8"))


@pytest.mark.parametrize("kind", ["q8", "q4"])
@pytest.mark.parametrize("dh", [64, 128])
def test_keep_moves_the_accepted_path(pk, kind, dh):
    lens, new = [13, 0, 47, 5], [33, 5, 1, 70]
    su = Setup(pk, lens, new, kind, 3, dh, 16, seed=5)
    su.fill(pk)
    k64, v64 = decoded(su.cache)
    before = [(k64[pg, :, sl].clone(), v64[pg, :, sl].clone()) for pg, sl in (su.rows(s) for s in range(4))]
    paths = [[0, 2, 3, 9, 17, 32], [], [0], [1] + list(range(5, 70, 3))]
    keep = np.zeros((4, max(map(len, paths)) + 2), np.int32)
    for s, p in enumerate(paths):
        keep[s, :len(p)] = p
    su.cache.keep(su.seqs, i32(keep), i32([len(p) for p in paths]))
    k64, v64 = decoded(su.cache)
    for s, p in enumerate(paths):
        pg, sl = su.rows(s)
        for x, old in ((k64[pg, :, sl], before[s][0]), (v64[pg, :, sl], before[s][1])):
            want = old.clone()
            for j, i in enumerate(p):
                want[lens[s] + j] = old[lens[s] + i]
            assert torch.equal(x, want), s
    # entries below their place, out of range, or counts past the row's end move nothing
    before = [t.clone() for t in (su.cache.k, su.cache.vs)]
    keep[:] = -1
    keep[3] = 70
    keep[0, 3] = 2
    su.cache.keep(su.seqs, i32(keep), i32([1000, 1000, -5, 1000]))
    assert torch.equal(su.cache.k, before[0]) and torch.equal(su.cache.vs, before[1])


def test_cache_beyond_4_gib(pk):
    """Rows at byte offsets past 2^32 of a large pool."""
    n_pages = 80000  # x 8 heads x 64 slots x 128 B = 5.2 GB a side
    su = Setup(pk, [200], [3], "q8", 8, 128, 64, pool=n_pages)
    table = np.array([[n_pages - 1, n_pages - 2, 1, n_pages - 3]], np.int32)
    su.table = table
    su.seqs = pk.KvSeqs(i32([0, 3]), i32([200]), i32(table), 3, 3, 203)
    su.fill(pk)
    k = randn((3, 8, 128), 5)
    su.cache.store(su.seqs, k, -k)
    gk, gv = su.cache.load(su.seqs)
    assert torch.equal(gk, stored(k, "q8")) and torch.equal(gv, stored(-k, "q8"))
    q = randn((3, 8, 128), 6, torch.float16)
    got = su.cache.attend(su.seqs, q)
    small = pk.KvCache(*(t[torch.as_tensor(table[0].astype(np.int64)).cuda()].contiguous() for t in (su.cache.k, su.cache.v, su.cache.ks, su.cache.vs)), "q8", 128)
    want = small.attend(pk.KvSeqs(i32([0, 3]), i32([200]), i32([[0, 1, 2, 3]]), 3, 3, 203), q)
    assert torch.equal(got, want)


@pytest.mark.parametrize("kind,n_pages", [("q8", 80000), ("q4", 160000)])
def test_attention_of_many_rows_beyond_4_gib(pk, kind, n_pages):
    """The same for many query rows a kv head, whose codes and scales are read by another kernel."""
    at = [n_pages - 1, n_pages - 2, 1, n_pages - 3]
    cache, small = (pk.KvCache.empty(n, 64, 8, 128, kind) for n in (n_pages, 4))
    k, v = randn((243, 8, 128), 1), randn((243, 8, 128), 2)
    for c, pages in ((cache, at), (small, [0, 1, 2, 3])):
        c.store(pk.KvSeqs(i32([0, 243]), i32([0]), i32([pages]), 243, 243, 243), k, v)
    for ty in ("f16", "f32"):
        q = randn((43, 8, 128), 6, DT[ty])
        got, want = (c.attend(pk.KvSeqs(i32([0, 43]), i32([200]), i32([p]), 43, 43, 243), q) for c, p in ((cache, at), (small, [0, 1, 2, 3])))
        assert torch.equal(got, want)
        got = cache.load(pk.KvSeqs(i32([0, 43]), i32([200]), i32([at]), 43, 43, 243))
        assert torch.equal(got[0], stored(k, kind)[200:]) and torch.equal(got[1], stored(v, kind)[200:])


# ---------------------------------------------------------------- attention

SHAPES = [
    # lens, new, n_head, n_kv, page
    ([0], [1], 1, 1, 16),
    ([1, 15, 16, 17, 0, 300], [1, 1, 1, 1, 1, 1], 4, 2, 16),
    ([700, 3, 0, 64, 129], [5, 0, 7, 1, 16], 8, 2, 32),
    ([40, 2000, 511], [1, 1, 1], 21, 3, 64),
    ([1000, 77], [64, 33], 8, 1, 128),
    ([0, 250], [130, 70], 6, 6, 16),
    ([5000], [2], 64, 8, 256),
]


@pytest.mark.parametrize("kind", ["q8", "q4"])
@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("ty", list(DT))
@pytest.mark.parametrize("shape", SHAPES)
def test_attention_causal(pk, kind, dh, ty, shape):
    lens, new, n_head, n_kv, page = shape
    su = Setup(pk, lens, new, kind, n_kv, dh, page, seed=dh + n_head, extra_rows=1, slack=1)
    su.fill(pk)
    q = randn((su.n_tok, n_head, dh), 8, DT[ty], std=1.5)
    check_attention(su, q, su.cache.attend(su.seqs, q))


WIDE = [
    # row counts around a block of 128 and two, of one tile of positions and of many (two f32 prompts are split over a
    # cluster, the last one's over the scratch), with sequences that have nothing
    ([0], [33], 1, 1, 16),
    ([0, 90, 0], [129, 0, 1], 1, 1, 16),
    ([63, 64, 1], [64, 1, 40], 8, 2, 16),
    ([0, 700], [257, 31], 3, 3, 32),
    ([2500, 40], [200, 130], 2, 2, 64),
    ([1700], [64], 40, 20, 64),
]


@pytest.mark.parametrize("kind", ["q8", "q4"])
@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("ty", list(DT))
@pytest.mark.parametrize("shape", WIDE)
def test_attention_wide(pk, kind, dh, ty, shape):
    lens, new, n_head, n_kv, page = shape
    su = Setup(pk, lens, new, kind, n_kv, dh, page, seed=dh + n_head, extra_rows=1)
    su.fill(pk)
    q = randn((su.n_tok, n_head, dh), 8, DT[ty], std=1.5)
    check_attention(su, q, su.cache.attend(su.seqs, q))
    see = {s: torch.rand((n, n), generator=gen(50 + s), device="cuda") < 0.3 for s, n in enumerate(new)}
    words = max(1, -(-max(new) // 64))
    mask = torch.zeros((su.n_tok, words), dtype=torch.int64)
    for s, n in enumerate(new):
        for i in range(n):
            bits = sum(1 << int(j) for j in see[s][i].nonzero()[:, 0].tolist())
            for w in range(words):
                x = (bits >> (64 * w)) & (2 ** 64 - 1)
                mask[int(su.start[s]) + i, w] = x - 2 ** 64 if x >= 2 ** 63 else x
    check_attention(su, q, su.cache.attend(su.seqs, q, mask=mask.cuda()), see=lambda s, n: see[s])


def test_attention_wide_side_by_side(pk):
    """Kernels that take a half or all of an SM's tensor memory, on two streams at once and replayed from graphs: the
    results of each alone."""
    runs = []
    for i, (ty, dh, lens, new, heads) in enumerate((("f32", 64, [900, 3], [300, 140], 12), ("f16", 128, [2000], [90], 24), ("bf16", 64, [50, 800], [33, 64], 16))):
        su = Setup(pk, lens, new, "q8", heads // 2, dh, 64, seed=i)
        su.fill(pk)
        q = randn((su.n_tok, heads, dh), 8 + i, DT[ty])
        want = su.cache.attend(su.seqs, q)
        out = [torch.empty_like(q) for _ in range(2)]
        scratch = [torch.empty(max(16, su.cache.attend_scratch_bytes(su.seqs, heads, q.dtype)), dtype=torch.uint8, device="cuda") for _ in range(2)]
        runs.append((su, q, want, out, scratch))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()

    def go(w, order):
        for j in order:
            su, q, _, out, scratch = runs[j]
            su.cache.attend(su.seqs, q, out=out[w], scratch=scratch[w])

    graphs = []
    for w, order in enumerate(([0, 1, 2], [2, 0, 1])):
        with torch.cuda.stream(streams[w]):
            go(w, order)
        streams[w].synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=streams[w]):
            go(w, order)
        graphs.append(g)
    for _, _, _, out, _ in runs:
        for o in out:
            o.zero_()
    torch.cuda.synchronize()
    for _ in range(20):
        for w in range(2):
            with torch.cuda.stream(streams[w]):
                go(w, [w, 2, 1 - w])
                graphs[w].replay()
    torch.cuda.synchronize()
    for _, _, want, out, _ in runs:
        assert torch.equal(out[0], want) and torch.equal(out[1], want)


def test_attention_clusters_side_by_side(pk):
    """Kernels whose CTAs wait for their cluster's and share an SM's tensor memory, on four streams at once."""
    runs = []
    for i, (ty, dh) in enumerate((("f16", 64), ("bf16", 64), ("f16", 128), ("f32", 64))):
        su = Setup(pk, [6000], [40 if ty == "f32" else 20], "q8", 32, dh, 64, seed=i)
        su.fill(pk)
        q = randn((su.n_tok, 32, dh), 8 + i, DT[ty])
        assert su.cache.attend_scratch_bytes(su.seqs, 32, q.dtype) == 0  # (a cluster's sums, or one chunk)
        runs.append((su, q, su.cache.attend(su.seqs, q), torch.empty_like(q), torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(60):
        for su, q, _, out, st in runs:
            with torch.cuda.stream(st):
                su.cache.attend(su.seqs, q, out=out)
    torch.cuda.synchronize()
    for _, _, want, out, _ in runs:
        assert torch.equal(out, want)


@pytest.mark.parametrize("ty", list(DT))
@pytest.mark.parametrize("dh", [64, 128])
def test_attention_query_range(pk, dh, ty):
    """Rows of very different sizes side by side, rows of zeros, and rows of infinities and NaN, which spoil no other."""
    su = Setup(pk, [333], [140], "q8", 1, dh, 16, seed=4)
    su.fill(pk)
    q = randn((140, 2, dh), 8, torch.float32)
    q[0::7] *= 100.0
    q[1::7] *= 6e-8 if ty == "f16" else 1e-30
    q[2::7] = 0
    q = q.to(DT[ty])
    bad = torch.zeros(140, dtype=torch.bool, device="cuda")
    bad[[5, 12, 61, 139]] = True
    q[5], q[12, :, 3], q[61, 1] = math.inf, math.nan, -math.inf
    q[139, 0, 0] = math.nan
    clean = torch.where(bad[:, None, None], torch.zeros_like(q), q)
    # Rows of large scores may have one weight that counts, and a V code of 0 there: then what is left are products
    # w D^V below f16's normal values, off by 2^-25 each, where the row's largest is 2^6 or more.  With D <= max |v| / 97
    # (Q4's codes go to 97 at least, Q8's to 127) and |c| <= 127, n positions are off by n 2^-31 127 / 97 of the largest
    # p max |v|; n 2^-30 of it is allowed.
    k64, v64 = decoded(su.cache)
    pg, sl = su.rows(0)
    for scale, x in ((dh ** -0.5, q), (dh ** -0.5, clean), (0.3, clean), (1e-3, clean)):
        got = su.cache.attend(su.seqs, x, scale=scale)
        want, absv, dots = attention(su, clean, scale=scale)
        p = (clean.double() @ k64[pg, 0, sl].T * scale).masked_fill(torch.ones((140, 473), device="cuda").triu(334).bool()[:, None], -math.inf)
        most = (torch.softmax(p, -1) * v64[pg, 0, sl].abs().amax(-1)).amax(-1, keepdim=True)
        ok = ~bad if x is q else torch.ones_like(bad)
        assert torch.isfinite(got[ok].double()).all()
        lim = attn_bound(clean, want, absv, dots, dh) + 473 * 2.0 ** -30 * most
        assert ((got.double() - want).abs() <= lim)[ok].all(), scale


@pytest.mark.parametrize("ty", list(DT))
@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("heads", [4, 64])
def test_attention_bad_query_rows(pk, dh, ty, heads):
    """Query rows with an infinity or NaN give NaN wherever they see something, also where all their scores are -inf
    (codes of one sign, one position); they give 0 where they see nothing, and leave the other rows as they were."""
    for lens, new in (([0], [2]), ([70], [3])):
        su = Setup(pk, lens, new, "q8", 1, dh, 16)
        t = lens[0] + new[0]
        k = randn((t, 1, dh), 1).abs() + 0.1
        su.cache.store(pk.KvSeqs(i32([0, t]), i32([0]), su.seqs.pages, t, t, t), k, k)
        q = randn((new[0], heads, dh), 2).to(DT[ty])
        clean = su.cache.attend(su.seqs, q)
        last = new[0] - 1
        for h, (d, x) in enumerate(((0, -math.inf), (5, math.inf), (dh - 1, math.nan))):
            q[last, h, d] = x
        got = su.cache.attend(su.seqs, q)
        assert torch.isnan(got[last, :3]).all()
        got[last, :3] = clean[last, :3]
        assert torch.equal(got, clean)
        none = su.cache.attend(pk.KvSeqs(su.seqs.start, i32([0]), su.seqs.pages, new[0], new[0], t), q,
                               mask=torch.zeros((new[0], 1), dtype=torch.int64, device="cuda"))
        assert (none == 0).all()


@pytest.mark.parametrize("ty,heads", [("f32", 2), ("f32", 64), ("bf16", 2), ("bf16", 64), ("f16", 2)])
def test_attention_scores_below_f32(pk, ty, heads):
    """Scale and query so small that their product has no f32 value: all that is seen counts alike, the rest not at all."""
    su = Setup(pk, [20], [3], "q8", 1, 64, 16)
    su.fill(pk)
    q = (randn((3, heads, 64), 1) * (1e-7 if ty == "f16" else 1e-32)).to(DT[ty])
    for scale in (1e-20, 1e-38):
        check_attention(su, q, su.cache.attend(su.seqs, q, scale=scale), scale=scale)


def tree(n, seed, empty=()):
    """Ancestor bits of a random tree, parents first; rows of `empty` see nothing new."""
    rng = np.random.default_rng(seed)
    bits = []
    for i in range(n):
        par = int(rng.integers(-1, i)) if i else -1
        bits.append((bits[par] if par >= 0 else 0) | (1 << i))
    return [0 if i in empty else b for i, b in enumerate(bits)]


def words_of(rows, words):
    out = [[(b >> (64 * w)) & (2 ** 64 - 1) for w in range(words)] for b in rows]
    return torch.tensor([[x - 2 ** 64 if x >> 63 else x for x in r] for r in out], dtype=torch.int64).reshape(-1, words).cuda()


@pytest.mark.parametrize("kind", ["q8", "q4"])
@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("ty", list(DT))
def test_attention_tree(pk, kind, dh, ty):
    """Trees of 1 to 150 drafts, several mask words, rows that see nothing at all (no context either)."""
    for lens, new, n_head, n_kv in (([300, 0, 31, 900], [9, 5, 64, 33], 8, 2), ([0, 100], [150, 70], 4, 4), ([17], [63], 32, 4)):
        su = Setup(pk, lens, new, kind, n_kv, dh, 16, seed=3)
        su.fill(pk)
        rows = [tree(n, s, empty=(1, 3) if s % 2 else ()) for s, n in enumerate(new)]
        words = (max(new) + 63) // 64
        mask = words_of(sum(rows, []), words)
        q = randn((su.n_tok, n_head, dh), 8, DT[ty])
        got = su.cache.attend(su.seqs, q, mask=mask)

        def see(s, n):
            return torch.tensor([[(b >> j) & 1 for j in range(n)] for b in rows[s]], dtype=torch.bool, device="cuda").reshape(n, n)

        check_attention(su, q, got, see=see)
        for s, n in enumerate(new):
            if s % 2 and lens[s] == 0:
                assert (got[int(su.start[s]) + 1] == 0).all()


def test_attention_masked_garbage(pk):
    """Slots beyond the sequences' ends, masked drafts and pages that are none hold NaN scales and never reach a result."""
    for kind in ("q8", "q4"):
        su = Setup(pk, [37, 90], [6, 3], kind, 2, 128, 16, slack=1)
        su.fill(pk)
        used = torch.zeros(su.cache.ks.shape[:3], dtype=torch.bool, device="cuda")
        for s in range(2):
            pg, sl = su.rows(s)
            used[pg, :, sl] = True
        pg, sl = su.rows(0)
        used[pg[38], :, sl[38]] = False  # draft 1 of sequence 0: masked for every row
        table = su.table.copy()
        table[1, 2] = su.cache.n_pages   # positions 32 .. 47 of sequence 1
        for t in (su.cache.ks, su.cache.vs):
            t[~used] = math.nan
        mask = words_of([0b1, 0, 0b101, 0b1101, 0b11101, 0b111101, 1, 3, 7], 1)
        q = randn((9, 4, 128), 8, torch.float16)
        seqs = pk.KvSeqs(su.seqs.start, su.seqs.ctx, i32(table), 9, 6, 93)
        got = su.cache.attend(seqs, q, mask=mask)
        for t in (su.cache.ks, su.cache.vs):
            t[~used] = 0.0
        rows = [[0b1, 0, 0b101, 0b1101, 0b11101, 0b111101], [1, 3, 7]]
        see = lambda s, n: torch.tensor([[(b >> j) & 1 for j in range(n)] for b in rows[s]], dtype=torch.bool, device="cuda")  # noqa: E731
        holes = lambda s: (torch.arange(su.lens[s] + su.new[s], device="cuda") // 16 == 2) & (s == 1)  # noqa: E731
        check_attention(su, q, got, see=see, holes=holes)


def test_attention_extremes(pk):
    """Scores far apart, V rows of very different sizes, large and tiny queries, another scale, and NaN only where a NaN
    query asks."""
    su = Setup(pk, [600], [4], "q8", 2, 128, 16)
    su.fill(pk)
    pg, sl = su.rows(0)
    su.cache.vs[pg[::7], :, sl[::7]] *= 1e4
    su.cache.vs[pg[::5], :, sl[::5]] *= 1e-6
    for ty, std in (("f32", 1e-20), ("f32", 12.0), ("bf16", 1e-30), ("f16", 8.0), ("f16", 0.0)):
        q = randn((4, 4, 128), 8, DT[ty], std=std)
        check_attention(su, q, su.cache.attend(su.seqs, q))
        check_attention(su, q, su.cache.attend(su.seqs, q, scale=0.02), scale=0.02)
    q = randn((4, 4, 128), 8)
    good = su.cache.attend(su.seqs, q)
    q[2, 1, 5] = math.nan
    got = su.cache.attend(su.seqs, q)
    assert torch.isnan(got[2, 1]).all()
    got[2, 1] = good[2, 1]
    assert torch.equal(got, good)


@pytest.mark.parametrize("kind", ["q8", "q4"])
@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("ty", list(DT))
@pytest.mark.parametrize("new,heads", [(4, 8), (40, 8)])
def test_attention_scales_apart(pk, kind, dh, ty, new, heads):
    """V rows 10^10 apart in size under weights of every size, for few rows and for many (another kernel), in a chunk of
    its own and split.  The products w D^V lie on a grid of 2^-24 where the row's largest is 2^6 or more, so each is off by
    2^-25 2^-6 of that largest, p max |v| 127 / 97 at the most: n positions by n 2^-30 of the largest p max |v|."""
    for lens in ([600], [5000]):
        su = Setup(pk, lens, [new], kind, 2, dh, 16, seed=6)
        su.fill(pk)
        pg, sl = su.rows(0)
        su.cache.vs[pg[::7], :, sl[::7], 0] *= 1e4
        su.cache.vs[pg[::5], :, sl[::5], 0] *= 1e-6
        k64, v64 = decoded(su.cache)
        total = lens[0] + new
        vis = (torch.arange(total, device="cuda")[None] <= lens[0] + torch.arange(new, device="cuda")[:, None])[:, None]
        for std in (1e-4, 1.0, 12.0):
            q = randn((new, heads, dh), 8, DT[ty], std=std)
            got = su.cache.attend(su.seqs, q)
            want, absv, dots = attention(su, q)
            most = torch.empty((new, heads, 1), dtype=torch.float64, device="cuda")
            for h in range(2):
                k, v = k64[pg, h, sl], v64[pg, h, sl]
                mine = slice(h * heads // 2, (h + 1) * heads // 2)
                p = torch.softmax((q[:, mine].double() @ k.T * dh ** -0.5).masked_fill(~vis, -math.inf), -1)
                most[:, mine] = (p * v.abs().amax(-1)).amax(-1, keepdim=True)
            lim = attn_bound(q, want, absv, dots, dh) + total * 2.0 ** -30 * most
            assert torch.isfinite(got).all()
            assert ((got.double() - want).abs() <= lim).all(), (std, ((got.double() - want).abs() / lim).max().item())


@pytest.mark.parametrize("kind", ["q8", "q4"])
@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("ty", list(DT))
def test_attention_wide_masked_garbage(pk, kind, dh, ty):
    """Many rows: NaN and infinite scales behind the sequences' ends, under masked drafts and in pages that are none, also
    whole tiles of those, never reach a result."""
    lens, new = [37, 290, 0], [40, 70, 33]
    su = Setup(pk, lens, new, kind, 2, dh, 16, slack=1)
    su.fill(pk)
    hidden = {0: (1, 17), 1: (0, 33, 69), 2: (32,)}  # drafts that no row sees
    gone = {0: (), 1: (2, 8, 9, 10, 11, 12), 2: (1,)}  # pages that are none
    used = torch.zeros(su.cache.ks.shape[:3], dtype=torch.bool, device="cuda")
    table = su.table.copy()
    for s in range(3):
        pg, sl = su.rows(s)
        used[pg, :, sl] = True
        for j in hidden[s]:
            used[pg[lens[s] + j], :, sl[lens[s] + j]] = False
        for i, j in enumerate(gone[s]):
            used[pg[j * 16]] = False
            table[s, j] = (-1, su.cache.n_pages, -2 ** 31, 2 ** 31 - 1)[i % 4]
    see = {}
    for s, n in enumerate(new):
        see[s] = torch.rand((n, n), generator=gen(70 + s), device="cuda") < 0.4
        see[s][:, list(hidden[s])] = False
        see[s][3] = False
    rows = [[sum(1 << int(j) for j in r.nonzero()[:, 0].tolist()) for r in see[s]] for s in range(3)]
    mask = words_of(sum(rows, []), 2)
    q = randn((sum(new), 8, dh), 8, DT[ty])
    seqs = pk.KvSeqs(su.seqs.start, su.seqs.ctx, i32(table), su.n_tok, su.max_new, su.max_len)
    holes = lambda s: torch.isin(torch.arange(lens[s] + new[s], device="cuda") // 16, torch.tensor(gone[s], device="cuda"))  # noqa: E731
    for bad in (math.nan, math.inf):
        for t in (su.cache.ks, su.cache.vs):
            t[..., 0][~used] = bad
        got = su.cache.attend(seqs, q, mask=mask)
        for t in (su.cache.ks, su.cache.vs):
            t[..., 0][~used] = 0.0
        check_attention(su, q, got, see=lambda s, n: see[s], holes=holes)
        assert (got[su.start[2] + 3] == 0).all()


@pytest.mark.parametrize("ty", list(DT))
def test_attention_strides(pk, ty):
    """Queries and outputs inside larger tensors, unaligned; rows behind the last sequence and everything between keep
    what they held; a null mask's words and a long max_len bound change nothing."""
    su = Setup(pk, [400, 30], [3, 2], "q8", 2, 64, 32, extra_rows=2, slack=5)
    su.fill(pk)
    big = randn((su.n_tok, 9, 71), 4, DT[ty])
    out = torch.full((su.n_tok, 10, 67), 5.0, dtype=DT[ty], device="cuda")
    q, o = big[:, 2:8, 3:67], out[:, 1:7, 1:65]
    su.cache.attend(su.seqs, q, out=o)
    check_attention(su, q, o)
    rest = out.clone()
    rest[:5, 1:7, 1:65] = 5.0
    assert (rest == 5).all()
    plain = su.cache.attend(su.seqs, q.contiguous())
    assert torch.equal(plain[:5], o[:5])
    long = pk.KvSeqs(su.seqs.start, su.seqs.ctx, su.seqs.pages, su.n_tok, 64, 1 << 20)
    check_attention(su, q, su.cache.attend(long, q))


def test_attention_bounds_are_kept(pk):
    """Device arrays that disagree with the host's bounds are cut to them, and rows outside are not touched."""
    su = Setup(pk, [100], [6], "q8", 1, 64, 16)
    su.fill(pk)
    q = randn((6, 2, 64), 3)
    out = torch.full_like(q, 9.0)
    few = pk.KvSeqs(su.seqs.start, su.seqs.ctx, su.seqs.pages, 6, 4, 106)  # four of six new tokens
    su.cache.attend(few, q, out=out)
    assert (out[4:] == 9).all() and torch.equal(out[:4], su.cache.attend(su.seqs, q)[:4])
    for start, ctx in (([-3, 6], [100]), ([0, 900], [100]), ([5, 2], [100]), ([0, 6], [-7]), ([0, 6], [2 ** 31 - 1])):
        seqs = pk.KvSeqs(i32(start), i32(ctx), su.seqs.pages, 6, 6, 106)
        su.cache.attend(seqs, q, out=out)
        su.cache.store(seqs, q[:, :1].contiguous(), q[:, 1:].contiguous())
        su.cache.load(seqs)
    torch.cuda.synchronize()


@pytest.mark.parametrize("ty,heads", [("f32", 2), ("f32", 64), ("f16", 2), ("bf16", 64)])
@pytest.mark.parametrize("start,ctx", [([-3, 6], 100), ([0, 900], 100), ([5, 2], 100), ([2, 4], 100), ([7, 9], 100), ([0, 6], -7), ([0, 6], 103),
                                       ([0, 6], 106), ([0, 6], 110), ([0, 6], 2 ** 31 - 1), ([0, 6], -2 ** 31)])
def test_arrays_that_contradict_the_bounds(pk, start, ctx, ty, heads):
    """start and ctx outside the host's bounds mean what is left of them within: every row, slot and page of the calls'
    outputs against that, and everything around them (more pages, rows and elements) as it was."""
    dh, n_tok, max_len, page = 64, 6, 106, 16
    a, b = (min(max(x, 0), n_tok) for x in start)
    n, total = max(b - a, 0), 0 if ctx < 0 else min(ctx + max(b - a, 0), max_len)
    pool = [torch.full((11, 2, page, w), 77, dtype=t, device="cuda") for w, t in ((dh, torch.uint8), (dh, torch.uint8), (1, torch.float32), (1, torch.float32))]
    cache = pk.KvCache(*(t[2:9] for t in pool), "q8", dh)
    table = i32([[4, 0, 6, 1, 3, 2, 5]])
    cache.store(pk.KvSeqs(i32([0, max_len]), i32([0]), table, max_len, max_len, max_len), randn((max_len, 2, dh), 1), randn((max_len, 2, dh), 2))
    seqs = pk.KvSeqs(i32(start), i32([ctx]), table, n_tok, n_tok, max_len)
    k, v = randn((n_tok, 2, dh), 3, DT[ty]), randn((n_tok, 2, dh), 4, DT[ty])
    want = [t.clone() for t in pool]
    codes = pk.KvCache.empty(1, page, 2, dh)
    codes.store(pk.KvSeqs(i32([0, n_tok]), i32([0]), i32([[0]]), n_tok, n_tok, n_tok), k, v)
    for i in range(n):
        p = ctx + i
        if 0 <= ctx and p < total:
            for w, c in zip(want, (codes.k, codes.v, codes.ks, codes.vs)):
                w[2 + int(table[0, p // page]), :, p % page] = c[0, :, a + i]
    cache.store(seqs, k, v)
    same = lambda x, y: torch.equal(x.view(torch.uint8), y.view(torch.uint8))  # noqa: E731
    assert all(same(x, w) for x, w in zip(pool, want))

    k64, v64 = decoded(cache)
    at = torch.arange(total, device="cuda")
    k64, v64 = (x[table[0, at // page].long(), :, at % page] for x in (k64, v64))  # [total, 2, dh]
    big = torch.full((2, n_tok + 4, 2, dh), 5.0, dtype=DT[ty], device="cuda")
    cache.load(seqs, out=(big[0, 2:-2], big[1, 2:-2]))
    for x, y in ((big[0], k64), (big[1], v64)):
        for i in range(n):
            got = x[2 + a + i].double()
            assert torch.equal(got, y[ctx + i].float().to(DT[ty]).double()) if 0 <= ctx and ctx + i < total else (got == 0).all()
        assert (x[:2 + a] == 5).all() and (x[2 + a + n:] == 5).all()

    q = randn((n_tok, heads, dh), 5, DT[ty])
    out = torch.full((n_tok + 4, heads, dh), 5.0, dtype=DT[ty], device="cuda")
    cache.attend(seqs, q, out=out[2:-2])
    assert (out[:2 + a] == 5).all() and (out[2 + a + n:] == 5).all()
    for i in range(n):
        see = (at < ctx) | (at - ctx <= i)
        for h in range(heads):
            x, kk, vv = q[a + i, h].double(), k64[:, h * 2 // heads], v64[:, h * 2 // heads]
            p = torch.softmax((kk @ x * dh ** -0.5).masked_fill(~see, -math.inf), 0)
            y, absv = (p @ vv, p @ vv.abs()) if total else (torch.zeros(dh, dtype=torch.float64, device="cuda"),) * 2
            dots = (kk.abs() @ x.abs() * dh ** -0.5).amax() if total else torch.tensor(0.0, device="cuda")
            assert ((out[2 + a + i, h].double() - y).abs() <= attn_bound(q, y, absv, dots.double()[None], dh)).all()
    keep = i32([[3, 2, 5]])
    moved = [t.clone() for t in pool]
    for j, x in enumerate((3, 2, 5)):
        if 0 <= ctx and x < n and ctx + x < total:
            for w, t in zip(moved, pool):
                w[2 + int(table[0, (ctx + j) // page]), :, (ctx + j) % page] = t[2 + int(table[0, (ctx + x) // page]), :, (ctx + x) % page]
    cache.keep(seqs, keep, i32([3]))
    assert all(same(x, w) for x, w in zip(pool, moved))


@pytest.mark.parametrize("ty", list(DT))
def test_attention_wide_bound_of_new_tokens(pk, ty):
    """A max_new far past the tokens that there are changes nothing."""
    su = Setup(pk, [900, 3], [2, 1], "q8", 2, 64, 16)
    su.fill(pk)
    q = randn((3, 128, 64), 8, DT[ty])
    for most in (3, 1000, 2 ** 31 - 1):
        seqs = pk.KvSeqs(su.seqs.start, su.seqs.ctx, su.seqs.pages, 3, most, su.max_len)
        got = su.cache.attend(seqs, q)
        check_attention(su, q, got)
        if most > 3:
            assert torch.equal(got, last)
        last = got


@pytest.mark.parametrize("ty,total", [("f16", 131072), ("bf16", 262144), ("f32", 131072)])
@pytest.mark.parametrize("heads", [1, 40])
def test_attention_sums_of_long_histories(pk, ty, total, heads):
    """V of one sign over long histories, so many sequences that each would be one sum: what the sums drop must not show.
    Single errors are as large as the weights' and outputs' roundings, their mean over 16 rows of 64 is not: a rounding
    within half a step u has a standard deviation of u / sqrt(3), the mean of 1024 a 32nd of it, and 5 of those pass by
    chance once in a million runs; an eighth of u is what the sums may drop.  f32: total / 16 additions, each within half a
    step of the sum, 5 standard deviations likewise."""
    dh, page, n = 64, 4096, 640
    cache = pk.KvCache.empty(total // page, page, 1, dh)
    pages = torch.arange(total // page, dtype=torch.int32, device="cuda")[None]
    v = randn((total, 1, dh), 2).abs() + 0.25
    cache.store(pk.KvSeqs(i32([0, total]), i32([0]), pages, total, total, total), randn((total, 1, dh), 1), v)
    q = randn((16, heads, dh), 3, DT[ty]).repeat(n // 16, 1, 1)
    seqs = pk.KvSeqs(i32(range(n + 1)), i32([total - 1] * n), pages.expand(n, -1).contiguous(), n, 1, total)
    got = cache.attend(seqs, q)[:16, heads - 1].double()
    k64, v64 = (x[:, 0].reshape(total, dh) for x in decoded(cache))
    want = torch.softmax(q[:16, heads - 1].double() @ k64.T * dh ** -0.5, -1) @ v64
    off = ((got - want) / want).mean().abs().item()
    u = torch.finfo(DT[ty]).eps / 2
    assert off <= (5 * u * math.sqrt(total / 16) if ty == "f32" else u / 8 + 5 * u / math.sqrt(3) / 32), off


@pytest.mark.parametrize("kind,dh,ty,total", [("q8", 64, "f16", 100003), ("q4", 128, "f16", 70001), ("q8", 128, "bf16", 140009), ("q4", 64, "bf16", 140009)])
@pytest.mark.parametrize("n", [37, 100, 592])
def test_attention_long_sums_in_parts(pk, kind, dh, ty, total, n):
    """Sums longer than one that the tensor core keeps, for as many sequences as make a cluster's chunks, chunks in the
    scratch, and one chunk each: scores that grow along the history, so that rows' references move late, and two new
    tokens with a mask."""
    page, heads = 1024, 20
    np_ = -(-total // page)
    cache = pk.KvCache.empty(np_, page, 1, dh, kind)
    pages = torch.arange(np_, dtype=torch.int32, device="cuda").flip(0)[None].contiguous()
    up = torch.linspace(-0.5, 2.5, total, device="cuda")[:, None, None]
    k, v = randn((total, 1, dh), 1, std=0.3) + up, randn((total, 1, dh), 2)
    cache.store(pk.KvSeqs(i32([0, total]), i32([0]), pages, total, total, total), k, v)
    q = (randn((2 * n, heads, dh), 3, std=0.5) + 0.8).to(DT[ty])
    seqs = pk.KvSeqs(i32(range(0, 2 * n + 1, 2)), i32([total - 2] * n), pages.expand(n, -1).contiguous(), 2 * n, 2, total)
    mask = torch.tensor([[1], [2]], device="cuda").repeat(n, 1)
    got = cache.attend(seqs, q, mask=mask)
    k64, v64 = (x.flip(0)[:, 0].reshape(-1, dh)[:total] for x in decoded(cache))
    for t in (0, 1, 5, 2 * n - 2, 2 * n - 1):
        x = q[t].double()
        w = x @ k64.T * dh ** -0.5
        w[:, total - 1 if t % 2 == 0 else total - 2] = -math.inf
        p = torch.softmax(w, -1)
        want, absv, dots = p @ v64, p @ v64.abs(), (x.abs() @ k64.abs().T * dh ** -0.5).amax(-1)
        most = (p * v64.abs().amax(-1)).amax(-1, keepdim=True)
        # (the sums may drop an eighth of the output's rounding, eps / 16, of what they add up)
        lim = attn_bound(q, want, absv, dots, dh) + absv * torch.finfo(DT[ty]).eps / 16 + total * 2.0 ** -30 * most
        assert ((got[t].double() - want).abs() <= lim).all(), (t, ((got[t].double() - want).abs() / lim).max().item())


@pytest.mark.parametrize("ty,heads", [("f32", 2), ("f32", 32), ("f16", 2), ("bf16", 32)])
def test_attention_mask_of_few_words(pk, ty, heads):
    """New tokens past the mask's words are seen by none; sequences share the pages of a prefix; the output may be the
    query itself."""
    lens, n = [64, 64, 64], 100
    su = Setup(pk, lens, [n] * 3, "q4", 2, 64, 16, seed=9)
    su.fill(pk)
    su.table[:, :4] = su.table[0, :4]
    su.seqs = pk.KvSeqs(su.seqs.start, su.seqs.ctx, i32(su.table), su.n_tok, n, su.max_len)
    q = randn((3 * n, heads, 64), 8, DT[ty])
    see = torch.rand((3, n, n), generator=gen(3), device="cuda") < 0.5
    mask = words_of([sum(1 << int(j) for j in r.nonzero()[:, 0].tolist() if j < 64) for s in range(3) for r in see[s]], 1)
    see[:, :, 64:] = False
    want = su.cache.attend(su.seqs, q, mask=mask)
    check_attention(su, q, want, see=lambda s, n: see[s])
    again = q.clone()
    assert su.cache.attend(su.seqs, again, mask=mask, out=again) is again and torch.equal(again, want)


def test_attention_repeats_bit_for_bit(pk):
    su = Setup(pk, [3000, 1200, 5], [7, 1, 3], "q4", 2, 128, 16)
    su.fill(pk)
    q = randn((11, 8, 128), 8, torch.float16)
    first = su.cache.attend(su.seqs, q).clone()
    for _ in range(5):
        assert torch.equal(su.cache.attend(su.seqs, q), first)


# ---------------------------------------------------------------- rotary positions

@pytest.mark.parametrize("ty", list(DT))
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dh,n_rot", [(128, 128), (64, 64), (64, 48), (128, 2), (80, 74), (96, 96), (33, 10)])
def test_rope(pk, ty, layout, dh, n_rot):
    pos = i32([0, 1, 2, 4095, 131071, 1000003, 2 ** 31 - 1, 77])
    q, k = randn((8, 5, dh), 1, DT[ty]), randn((8, 2, dh), 2, DT[ty])
    for kw in ({}, {"scaling": "linear", "factor": 4.0}, {"scaling": "ntk", "factor": 8.0, "theta": 5e5},
               {"scaling": "yarn", "factor": 16.0, "n_ctx_train": 4096},
               {"scaling": "yarn", "factor": 8.0, "n_ctx_train": 8192, "high": 4.0, "gain": 1.0, "factors": [1.0 + 0.1 * i for i in range(n_rot // 2)]}):
        table = pk.RopeTable(n_rot, **kw)
        gq, gk = pk.rope(table, pos, q, k, layout=layout)
        i = np.arange(0, n_rot, 2)
        theta, gain, fac = kw.get("theta", 1e4), 1.0, kw.get("factor", 1.0)
        if kw.get("scaling") == "ntk" and n_rot > 2:
            theta *= fac ** (n_rot / (n_rot - 2))
        f = theta ** (-i / n_rot) / (2 * math.pi)
        if "factors" in kw:
            f = f / np.array(kw["factors"], np.float32).astype(np.float64)
        if kw.get("scaling") == "linear":
            f = f / fac
        if kw.get("scaling") == "yarn":
            keep = np.clip((f * kw["n_ctx_train"] - 1) / (kw.get("high", 32.0) - 1), 0, 1)
            f = f / fac * (1 - keep) + f * keep
            gain = kw.get("gain") or 0.1 * math.log(fac) + 1
        assert abs(table.gain - gain) < 1e-6
        turns = torch.as_tensor(f).cuda() if len(f) else None
        # far positions: the product's own rounding in 64 bits is up to 2^31 * 2^-53 turns on either side
        ang = (pos.double()[:, None] * turns) % 1.0 * 2 * math.pi
        for x, g in ((q, gq), (k, gk)):
            a, b = (x[..., 0:n_rot:2], x[..., 1:n_rot:2]) if layout == "interleaved" else (x[..., :n_rot // 2], x[..., n_rot // 2:n_rot])
            z = torch.polar(torch.full_like(ang, table.gain), ang)[:, None] * torch.complex(a.double(), b.double())
            u, v = (g[..., 0:n_rot:2], g[..., 1:n_rot:2]) if layout == "interleaved" else (g[..., :n_rot // 2], g[..., n_rot // 2:n_rot])
            # angle to f32 2^-24 turns, cosine and sine 2^-23, four roundings of 2^-24 of the pair's length, the output's
            lim = z.abs() * (2 * math.pi * 2.0 ** -24 + 2.0 ** -23 + 4 * 2.0 ** -24 + 2 * math.pi * 2.0 ** -21)
            for got, want in ((u, z.real), (v, z.imag)):
                assert ((got.double() - want).abs() <= lim + half_step(want, DT[ty]) + 1e-30).all()
            assert torch.equal(g[..., n_rot:], x[..., n_rot:])


@pytest.mark.parametrize("ty", ["f32", "f16"])
def test_rope_in_place_and_strided(pk, ty):
    table = pk.RopeTable(48, scaling="linear", factor=2.0)
    pos = i32(np.arange(700) * 13)
    for layout in ("half", "interleaved"):
        big = randn((700, 7, 70), 4, DT[ty])
        q, k = big[:, 0:4, 3:67], big[:, 4:6, 3:67]
        wq, wk = pk.rope(table, pos, q, k, layout=layout)
        cq, ck = pk.rope(table, pos, q.contiguous(), k.contiguous(), layout=layout)
        assert torch.equal(wq, cq) and torch.equal(wk, ck)
        only, none = pk.rope(table, pos, k, layout=layout)
        assert none is None and torch.equal(only, wk)
        copy = big.clone()
        pk.rope(table, pos, q, k, layout=layout, out_q=q, out_k=k)
        assert torch.equal(q, wq) and torch.equal(k, wk)
        copy[:, 0:4, 3:67], copy[:, 4:6, 3:67] = wq, wk
        assert torch.equal(copy, big)
    e = pk.rope(table, i32([]).reshape(0), torch.empty((0, 4, 64), device="cuda"))
    assert e[0].shape == (0, 4, 64)


# ---------------------------------------------------------------- logit rules

def rules64(x, row, repeat=None, freq=None, presence=None, hist=None, n_hist=None, bias_id=None, bias=None, allow=None):
    y, size = x.double().clone(), x.double().abs()
    n = x.numel()
    if hist is not None:
        ids = hist[row % hist.shape[0]].long()
        ids = ids[:int(n_hist[row])] if n_hist is not None else ids
        ids = ids[(ids >= 0) & (ids < n)]
        u, c = torch.unique(ids, return_counts=True)
        r = 1.0 if repeat is None else float(repeat[row])
        f, p = (0.0 if a is None else float(a[row]) for a in (freq, presence))
        y[u] = torch.where(y[u] > 0, y[u] / r, y[u] * r) - c.double() * f - p
        size[u] = size[u] * max(r, 1 / r) + c.double() * abs(f) + abs(p)
    if bias is not None:
        ids, b = bias_id[row % bias_id.shape[0]].long(), bias[row % bias.shape[0]].double()
        ok = (ids >= 0) & (ids < n)
        y.index_add_(0, ids[ok], b[ok])
        size.index_add_(0, ids[ok], b[ok].abs())
    if allow is not None:
        t = torch.arange(n, device=x.device)
        y[((allow[row % allow.shape[0]].long()[t // 32] >> (t % 32)) & 1) == 0] = -math.inf
    return y, size


@pytest.mark.parametrize("ty", list(DT))
@pytest.mark.parametrize("rows,n,nh,nb", [(1, 1, 1, 1), (3, 31, 5, 2), (2, 2047, 700, 40), (5, 2049, 33, 100), (4, 73448, 3000, 300), (1, 128256, 1, 0),
                                          (3, 30000, 6000, 900), (2, 9001, 3413, 0), (2, 9001, 3400, 13), (700, 300, 40, 5)])
def test_logit_rules(pk, ty, rows, n, nh, nb):
    g = gen(rows * n)
    x = randn((rows, n), n, DT[ty], std=4.0)
    kw = {"repeat": 0.8 + torch.rand(rows, generator=g, device="cuda"), "freq": torch.rand(rows, generator=g, device="cuda") - 0.3,
          "presence": torch.rand(rows, generator=g, device="cuda"),
          "hist": (torch.rand((rows, nh), generator=g, device="cuda") ** 4 * (n + 3)).to(torch.int32) - 1,  # some ids out of range
          "n_hist": torch.randint(0, nh + 1, (rows,), generator=g, device="cuda").to(torch.int32),
          "allow": torch.randint(-2 ** 31, 2 ** 31, (rows, (n + 31) // 32), generator=g, device="cuda").to(torch.int32)}
    if nb:
        kw["bias_id"] = (torch.rand((rows, nb), generator=g, device="cuda") ** 3 * (n + 2)).to(torch.int32) - 1
        kw["bias"] = randn((rows, nb), 5)
    some = [kw, {k: v for k, v in kw.items() if k not in ("allow", "bias", "bias_id")}, {"allow": kw["allow"][:1]}, {},
            {"hist": kw["hist"][:1].expand(1, -1), "presence": kw["presence"]}]
    if nb:
        some.append({"bias_id": kw["bias_id"][:1], "bias": kw["bias"][:1]})
    for s in some:
        got = pk.logit_rules(x, **s)
        for r in range(rows):
            want, size = rules64(x[r], r, **s)
            inf = torch.isinf(want)
            assert torch.equal(torch.isneginf(got[r]), inf)
            # the quotient or product, the penalty's two and its difference, nb biases: 2^-24 of the sizes each; the output's
            lim = size * (4 + min(nb, n)) * 2.0 ** -24 + half_step(want, DT[ty]) + 1e-30
            assert ((got[r].double() - want).abs()[~inf] <= lim[~inf]).all()
    same = x.clone()
    assert pk.logit_rules(same, **kw, out=same) is same and torch.equal(same, pk.logit_rules(x, **kw))


@pytest.mark.parametrize("n", [61440, 61441, 65536, 128256])
def test_logit_rules_many_rows(pk, n):
    """Enough rows that a row is few, long parts: the tokens at the parts' ends and the row's, in place too."""
    rows = 600
    x = randn((rows, n), 3)
    ends = [0, 2047, 2048, 4095, 43007, 43008, 45055, 45056, 61439, 61440, 63487, 63488, 65534, 65535, 65536, n - 2, n - 1]
    hist = i32([[t for t in ends if t < n] + [n, 2 ** 31 - 1]])
    pr = torch.rand(rows, generator=gen(1), device="cuda")
    bias = randn((1, hist.shape[1]), 4)
    want, total = x.clone(), {}
    for t, b in zip(hist[0, :-2].tolist(), bias[0]):  # (an id may be twice among the ends)
        total[t] = total[t] + b if t in total else b
    for t, b in total.items():
        want[:, t] = (x[:, t] - pr) + b
    assert torch.equal(pk.logit_rules(x, presence=pr, hist=hist, bias_id=hist, bias=bias), want)
    assert torch.equal(pk.logit_rules(x, presence=pr, hist=hist, bias_id=hist, bias=bias, out=x), want)


def test_logit_rules_edges(pk):
    """The same bias id many times adds up in the list's order, bit for bit; NaN and -inf logits; a row with nothing
    allowed; strided rows; a one-dimensional vector."""
    n = 5000
    x = randn((3, n), 2)
    ids = torch.full((1, 500), 4097, dtype=torch.int32, device="cuda")
    ids[0, ::3] = 7
    b = randn((1, 500), 3, std=100.0)
    want = {7: np.float32(0), 4097: np.float32(0)}
    for i, v in zip(ids[0].tolist(), b[0].cpu().numpy()):
        want[i] = np.float32(want[i] + v)
    got = pk.logit_rules(x, bias_id=ids, bias=b)
    for t, w in want.items():
        assert torch.equal(got[:, t].cpu(), x[:, t].cpu() + torch.tensor(w))
    x[0, 5], x[1, 6], x[2, 9] = math.nan, -math.inf, math.inf
    hist = i32([[5, 6, 9, 5]])
    two = torch.full((3,), 2.0, device="cuda")
    got = pk.logit_rules(x, hist=hist, repeat=two, freq=two)
    assert torch.isnan(got[0, 5]) and got[1, 6] == -math.inf and got[2, 9] == math.inf
    assert torch.equal(got[:, 10:], x[:, 10:])
    none = torch.zeros((3, 157), dtype=torch.int32, device="cuda")
    assert (pk.logit_rules(x, allow=none) == -math.inf).all()
    wide = randn((3, n + 9), 4)
    assert torch.equal(pk.logit_rules(wide[:, 3:3 + n], hist=hist, freq=two), pk.logit_rules(wide[:, 3:3 + n].contiguous(), hist=hist, freq=two))
    assert torch.equal(pk.logit_rules(x[1], hist=hist, n_hist=i32([2]), presence=two[:1]), pk.logit_rules(x, hist=hist, n_hist=i32([2, 2, 2]), presence=two)[1])


# ---------------------------------------------------------------- together

def step(pk, su, table, pos, q, k, v, mask, layout="half"):
    rq, rk = pk.rope(table, pos, q, k, layout=layout)
    su.cache.store(su.seqs, rk, v)
    return su.cache.attend(su.seqs, rq, mask=mask)


def test_a_drafted_step(pk):
    """Rotate, store, attend over a tree, accept a path, and go on: the accepted tokens' cache and the next step's output
    equal those of a run that had only the accepted tokens."""
    kind, n_kv, dh, n_head = "q8", 2, 64, 8
    lens, new = [50, 121], [7, 7]
    parent = [-1, 0, 0, 1, 3, 2, 4]
    path = [0, 1, 3, 4]
    depth, bits = [], []
    for i, p in enumerate(parent):
        depth.append(0 if p < 0 else depth[p] + 1)
        bits.append((0 if p < 0 else bits[p]) | 1 << i)
    table = pk.RopeTable(dh)
    a, b = (Setup(pk, lens, n, kind, n_kv, dh, 16, seed=2, slack=2) for n in (new, [4, 4]))
    for su in (a, b):
        hist = pk.KvSeqs(i32([0, 50, 171]), i32([0, 0]), su.seqs.pages, 171, 121, 121)
        su.cache.store(hist, randn((171, n_kv, dh), 1), randn((171, n_kv, dh), 2))
    q, k, v = randn((14, n_head, dh), 3), randn((14, n_kv, dh), 4), randn((14, n_kv, dh), 5)
    rows = path + [7 + p for p in path]
    pos = i32([c + d for c in lens for d in depth])
    out_a = step(pk, a, table, pos, q, k, v, words_of(bits * 2, 1))
    out_b = step(pk, b, table, pos[rows], q[rows], k[rows], v[rows], None)
    assert (out_a[rows] - out_b).abs().max() < 1e-5 * out_b.abs().max()
    a.cache.keep(a.seqs, i32([path] * 2), i32([4, 4]))
    got = [t for su in (a, b) for t in su.cache.load(pk.KvSeqs(i32([0, 54, 179]), i32([0, 0]), su.seqs.pages, 179, 125, 125))]
    assert torch.equal(got[0], got[2]) and torch.equal(got[1], got[3])
    q1, k1, v1 = randn((2, n_head, dh), 6), randn((2, n_kv, dh), 7), randn((2, n_kv, dh), 8)
    nxt = [54, 125]
    outs = []
    for su in (a, b):
        su.seqs = pk.KvSeqs(i32([0, 1, 2]), i32(nxt), su.seqs.pages, 2, 1, 126)
        outs.append(step(pk, su, table, i32(nxt), q1, k1, v1, None))
    assert torch.equal(outs[0], outs[1])


def test_captured_and_on_another_stream(pk):
    """One graph of rotate, store, attend, keep and rules, replayed as the context grows (only device arrays change), and
    the same calls on a side stream, give what the calls give one by one."""
    n_kv, dh, n_head, vocab = 2, 128, 8, 5000
    table = pk.RopeTable(dh)

    def fresh():
        su = Setup(pk, [0, 0], [3, 3], "q8", n_kv, dh, 16, seed=4, pool=64)
        su.table = np.arange(60, dtype=np.int32).reshape(2, 30)
        su.seqs = pk.KvSeqs(i32([0, 3, 6]), i32([5, 300]), i32(su.table), 6, 3, 480)
        return su

    a, b = fresh(), fresh()
    q, k, v = randn((6, n_head, dh), 3, torch.float16), randn((6, n_kv, dh), 4, torch.float16), randn((6, n_kv, dh), 5, torch.float16)
    logits, keep, n_keep = randn((6, vocab), 6), i32([[0, 2], [1, 2]]), i32([2, 1])
    hist, two = i32([[1, 2, 3, 3]]), torch.full((6,), 2.0, device="cuda")
    pos = i32([5, 6, 7, 300, 301, 302])

    def calls(su, p):
        o = step(pk, su, table, p, q, k, v, None)
        su.cache.keep(su.seqs, keep, n_keep)
        return o, pk.logit_rules(logits, hist=hist, freq=two)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        calls(a, pos)
    torch.cuda.current_stream().wait_stream(side)
    a = fresh()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = calls(a, pos)
    for t in (a.cache.k, a.cache.v, a.cache.ks, a.cache.vs):
        t.zero_()
    a.seqs.ctx.copy_(i32([5, 300]))
    for turn in range(6):
        p = i32([5 + 2 * turn + i for i in range(3)] + [300 + turn + i for i in range(3)])
        pos.copy_(p)
        graph.replay()
        if turn % 2:
            want = calls(b, p)
        else:
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                want = calls(b, p)
            torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert torch.equal(a.cache.k, b.cache.k) and torch.equal(a.cache.vs, b.cache.vs)
        for su in (a, b):
            su.seqs.ctx.add_(i32([2, 1]))


def test_raw_stream_argument(pk):
    su = Setup(pk, [900], [2], "q8", 2, 64, 16)
    su.fill(pk)
    q = randn((2, 4, 64), 3)
    want = su.cache.attend(su.seqs, q)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = [su.cache.attend(su.seqs, q, stream=side.cuda_stream) for _ in range(4)]
    side.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_memory_of_a_call_on_another_stream(pk):
    """What a call on `stream` makes is never a block that was freed on the current stream, where work that still reads
    it may be queued; and once the caller lets go of it, it is not reused before the current stream is done with it."""
    su = Setup(pk, [6000], [2], "q8", 2, 64, 16, seed=1)
    su.fill(pk)
    q, x, pos = randn((2, 4, 64), 3), randn((2, 1000), 4), i32([3, 4])
    table = pk.RopeTable(64)
    size = su.cache.attend_scratch_bytes(su.seqs, 4, q.dtype)
    assert size > 0
    calls = {"attend": lambda st: su.cache.attend(su.seqs, q, stream=st), "load": lambda st: su.cache.load(su.seqs, stream=st),
             "rope": lambda st: pk.rope(table, pos, q, q[:, :2], stream=st), "rules": lambda st: pk.logit_rules(x, stream=st)}
    want = {n: f(None) for n, f in calls.items()}
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    flat = lambda r: r if isinstance(r, tuple) else (r,)  # noqa: E731
    for n, f in calls.items():
        f(side.cuda_stream)  # (the side stream's own pool has what the call needs)
        torch.cuda.synchronize()
        # blocks of the sizes that the call makes, whose copies wait behind a long kernel when they are freed
        sizes = [t.numel() * t.element_size() for t in flat(want[n])] + ([size] if n == "attend" else [])
        blocks = [torch.full((s,), 7, dtype=torch.uint8, device="cuda") for s in sizes]
        at = {b.data_ptr() for b in blocks}
        torch.cuda._sleep(200_000_000)
        copies = [b.clone() for b in blocks]
        del blocks
        got = f(side.cuda_stream)
        assert not at & {t.data_ptr() for t in flat(got)}, n
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(flat(got), flat(want[n]))), n
        assert all((c == 7).all() for c in copies), n
    for n, f in calls.items():
        got = f(side.cuda_stream)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda._sleep(200_000_000)
        copies = [t.clone() for t in flat(got)]
        del got
        with torch.cuda.stream(side):
            for t in flat(want[n]):
                torch.full_like(t, 9.0)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(copies, flat(want[n]))), n
    with torch.cuda.stream(side):  # the current stream by its number
        assert torch.equal(su.cache.attend(su.seqs, q, stream=side.cuda_stream), want["attend"])
    torch.cuda.synchronize()


def test_tensors_of_a_call_on_another_stream(pk):
    """Tensors that the caller lets go of right after a call on `stream` are not reused before that stream has come to it."""
    su = Setup(pk, [6000], [2], "q8", 2, 64, 16, seed=1)
    su.fill(pk)
    q, kv, x = randn((2, 4, 64), 3), randn((2, 2, 64), 5), randn((2, 1000), 4)
    table = lambda: pk.RopeTable(64)  # noqa: E731
    one = torch.ones(2, device="cuda")

    def seqs():
        return pk.KvSeqs(su.seqs.start.clone(), su.seqs.ctx.clone(), su.seqs.pages.clone(), 2, 2, 6002)

    def store(st):
        cache = pk.KvCache(*(t.clone() for t in (su.cache.k, su.cache.v, su.cache.ks, su.cache.vs)), "q8", 64)
        if st is not None:
            side.wait_stream(torch.cuda.current_stream())
        cache.store(seqs(), kv.clone(), (kv * 2).clone(), stream=st)
        return cache.load(su.seqs, stream=st)

    calls = {"attend": lambda st: su.cache.attend(seqs(), q.clone(), stream=st), "rope": lambda st: pk.rope(table(), i32([3, 4]), q.clone(), kv.clone(), stream=st),
             "rules": lambda st: pk.logit_rules(x.clone(), hist=i32([[1, 2, 3]]), presence=one.clone(), bias_id=i32([[5]]), bias=one[:1].clone()[None], stream=st),
             "store": store}
    flat = lambda r: r if isinstance(r, tuple) else (r,)  # noqa: E731
    side = torch.cuda.Stream()
    for n, f in calls.items():
        want = f(None)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(400_000_000)
        got = f(side.cuda_stream)  # (its inputs are ready long before the sleep is over)
        junk = [torch.full((m,), 255, dtype=torch.uint8, device="cuda") for m in (8, 512, 1024, 2048, 4096, 8192, 32768) for _ in range(40)]
        junk += [torch.full_like(su.cache.k, 255) for _ in range(2)] + [torch.full_like(su.cache.ks, 9.0) for _ in range(2)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(flat(got), flat(want))), n
        del junk


def test_scratch_of_two_page_sizes(pk):
    """The same sequences over caches of other page sizes: a page table reaches further there, and the scratch is sized
    for each."""
    pages = i32(range(40)).reshape(1, 40)
    seqs = pk.KvSeqs(i32([0, 1]), i32([600]), pages, 1, 1, 1 << 20)
    q = randn((1, 2, 64), 1)
    sizes, outs = [], []
    for page in (16, 256, 16):
        cache = pk.KvCache.empty(40, page, 2, 64)
        cache.store(pk.KvSeqs(i32([0, 601]), i32([0]), pages, 601, 601, 601), randn((601, 2, 64), 2), randn((601, 2, 64), 3))
        outs.append(cache.attend(seqs, q))
        sizes.append(cache.attend_scratch_bytes(seqs, 2, q.dtype))
        assert torch.equal(cache.attend(seqs, q), outs[-1])
    assert sizes[0] == sizes[2] < sizes[1] and torch.equal(outs[0], outs[2])
    assert (outs[0] - outs[1]).abs().max() <= 2.0 ** -18 * outs[0].abs().max()


def test_refusals_on_the_device(pk):
    su = Setup(pk, [5], [2], "q8", 2, 64, 16)
    k = randn((2, 2, 64), 1)
    q = randn((2, 4, 64), 1)
    for bad in (lambda: su.cache.store(su.seqs, k, k.half()), lambda: su.cache.store(su.seqs, k[:1], k[:1]),
                lambda: su.cache.store(su.seqs, k.double(), k.double()), lambda: su.cache.store(su.seqs, k.cpu(), k.cpu()),
                lambda: su.cache.attend(su.seqs, q[..., :32]), lambda: su.cache.attend(su.seqs, randn((2, 3, 64), 1)),
                lambda: su.cache.attend(su.seqs, q, mask=torch.zeros((2, 1), dtype=torch.int32, device="cuda")),
                lambda: su.cache.attend(su.seqs, q, scale=0.0), lambda: su.cache.attend(su.seqs, q.transpose(1, 2).contiguous().transpose(1, 2)),
                lambda: su.cache.keep(su.seqs, i32([0, 1]), i32([1])), lambda: pk.KvSeqs(i32([0, 2]), i32([5]), i32([[0], [1]]), 2, 2, 7),
                lambda: pk.logit_rules(q), lambda: pk.logit_rules(k[0], allow=i32([[1]] * 2).expand(2, 1)),
                lambda: pk.rope(pk.RopeTable(66), i32([1, 2]), q), lambda: pk.rope(pk.RopeTable(64), i32([1]), q)):
        with pytest.raises(pk.PkError):
            bad()
