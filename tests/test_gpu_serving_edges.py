"""The serving operators where settings and sizes are at their ends: equal logits at temperatures that are no power of two,
temperatures of every size, shared prefixes shorter than a tile, calls right behind what they read; and the forms of the
attention that f32 rows take by their number."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_drafts import DT, Setup, check_attention, gen, i32, randn, words_of  # noqa: E402
from test_gpu_serving import SharedSetup, check_draw, likely  # noqa: E402


def halves():
    """(largest logit, temperature) whose product of 32 largest / temperature lies next to a half in f32, rounded up to it
    or, below 0, down: to the nearest number it is then more than a half away.  The logits have 8 bits."""
    tops = np.unique(np.outer(np.arange(1, 256), 2.0 ** -np.arange(10)))
    tops = np.concatenate([tops, -tops])
    out = []
    for temp in (0.3, 0.35, 0.6, 0.7, 0.9, 1.2):
        per = np.float64(np.float32(32) / np.float32(temp))
        product = (tops * per).astype(np.float32).astype(np.float64)
        at = np.nonzero(np.rint(product) - tops * per > 0.5)[0]
        out += [(float(tops[i]), temp) for i in at[:: max(1, len(at) // 5)]]
    return out


@pytest.mark.parametrize("ty", list(DT))
def test_draw_equal_logits_at_temperatures(pk, ty):
    """The largest logit is in the first bin of the order also where its product with the bins a unit is a rounded half."""
    pairs = halves()
    assert len(pairs) >= 20
    rows = len(pairs)
    temp = torch.tensor([t for _, t in pairs], dtype=torch.float32, device="cuda")
    u = torch.rand(rows, generator=gen(3), device="cuda")
    for n in (900, 20000):
        x = torch.tensor([v for v, _ in pairs], device="cuda")[:, None].expand(rows, n).to(DT[ty]).contiguous()
        for spread in (False, True):
            if spread:
                x[:, ::3] -= 5.0
                x[:, 7] = -math.inf
            for k in (17, 250, n // 2, n - 3):
                for p in (1.0, 0.6):
                    check_draw(pk, x, u, temp=temp, top_k=i32([k] * rows), top_p=torch.full((rows,), p, device="cuda"))


@pytest.mark.parametrize("ty", list(DT))
@pytest.mark.parametrize("n", [3, 50, 3001, 40000])
def test_draw_top_p_at_all_temperatures(pk, ty, n):
    """Temperatures that are subnormal, infinite, or so large that differences of logits overflow, beside top_p."""
    top = float(torch.finfo(DT[ty]).max)
    x = torch.empty((7, n), device="cuda")
    x[:4] = likely(4, n, 5, "f32") if n > 20 else torch.tensor([1.0, 0.5, 2.0], device="cuda")
    x[1, ::2] = -math.inf
    x[2, n // 2] = math.inf
    x[4] = torch.where(torch.arange(n, device="cuda") % 3 == 1, top, -top)
    x[5] = top * torch.linspace(-1, 1, n, device="cuda")
    x[6] = -1e-40 * (torch.arange(n, device="cuda") % 50)  # (0 in half precision)
    x = x.to(DT[ty])
    u = torch.rand(7, generator=gen(n), device="cuda")
    full = lambda v: torch.full((7,), v, device="cuda")  # noqa: E731
    for t in (1e-45, 1e-40, 4e-39, 4.3e-39, 1e-30, 1e-20, 1e20, 1e38, 3e38, math.inf):
        for p in (0.0, 1e-6, 0.37, 0.9, 0.9999999):
            check_draw(pk, x, u, temp=full(t), top_p=full(p))
        check_draw(pk, x, u, temp=full(t), top_p=full(0.6), top_k=i32([0, 5, 600, n - 1, 2, 0, 7]), min_p=full(1e-3))


def test_draw_top_p_at_all_temperatures_of_long_rows(pk):
    """The same where a row does not fit its CTAs' shared memory."""
    x = likely(3, 700001, 5, "f32")
    x[1] = 3e38 * torch.linspace(-1, 1, 700001, device="cuda")
    u = torch.rand(3, generator=gen(2), device="cuda")
    for t in (1e-45, 4e-39, 1.0, 3e38, math.inf):
        check_draw(pk, x, u, temp=torch.full((3,), t, device="cuda"), top_p=torch.full((3,), 0.37, device="cuda"))


@pytest.mark.parametrize("ty", list(DT))
@pytest.mark.parametrize("n", [20, 3001, 40000])
def test_draw_small_temperatures(pk, ty, n):
    """Temperatures at which the next float below the largest logit has a weight of 2^-100 to 2^-(10^9): the largest alone
    counts, or all that are equal to it, and the others have none."""
    x = torch.empty((5, n), device="cuda")
    x[:4] = likely(4, n, 5, "f32")
    x[1] = 12.0 + x[1].abs().clamp(max=3.0)
    x[2, n // 3] = 60.0
    x[3, ::4] = 21.5
    x[4] = 9.75
    x = x.to(DT[ty])
    x[4, ::2] = torch.nextafter(x[4, :1].float(), torch.zeros((), device="cuda")).to(DT[ty]) if ty == "f32" else x[4, 0] - x[4, 0] * torch.finfo(DT[ty]).eps
    u = torch.rand(5, generator=gen(n), device="cuda")
    full = lambda v: torch.full((5,), v, device="cuda")  # noqa: E731
    for t in (1e-6, 1e-7, 3e-8, 1e-8, 3e-9, 2.5e-9, 2e-9, 1.5e-9, 1e-9, 7e-10, 5e-10, 3e-10, 1e-10, 1e-11, 1e-12, 1e-14, 2.4e-17, 1e-18):
        for kw in ({}, {"top_p": full(0.9)}, {"top_k": i32([15] * 5)}, {"min_p": full(1e-3), "top_p": full(0.4)}):
            check_draw(pk, x, u, temp=full(t), **kw)


SHORT = [
    # (groups of (positions shared, sequences), own positions, new tokens): the longest prefix is under a tile
    ([(1, 3)], [0, 40, 7], [1, 1, 1]),
    ([(8, 2), (0, 1)], [60, 0, 20], [1, 3, 1]),
    ([(15, 4), (3, 2)], [3, 0, 90, 700, 5, 0], [2, 1, 1, 1, 4, 2]),
    ([(15, 30)], [(11 * i) % 70 for i in range(30)], [3] * 30),
]


@pytest.mark.parametrize("kind, dh", [("q8", 64), ("q8", 128), ("q4", 64), ("q4", 128)])
@pytest.mark.parametrize("ty", list(DT))
@pytest.mark.parametrize("case", range(len(SHORT)))
def test_shared_short_prefixes(pk, kind, dh, ty, case):
    """max_own is of the positions besides the shared ones also where those are too few to be computed for all."""
    su = SharedSetup(pk, *SHORT[case], kind, 2, dh, 16, seed=case)
    assert su.shared.max_len == max(n for n, _ in SHORT[case][0]) < 16
    for heads in (2, 16):
        q = randn((su.n_tok, heads, dh), 8, DT[ty], std=1.5)
        check_attention(su, q, su.attend(q))


@pytest.mark.parametrize("ty", list(DT))
def test_shared_bounds_under_a_tile(pk, ty):
    """The same where the sequences' own bound, or max_len alone, is under a tile; and no tokens of a group at all."""
    su = SharedSetup(pk, [(8, 3)], [2, 0, 4], [1, 3, 2], "q8", 2, 64, 16, seed=1)
    assert su.max_len < 16
    q = randn((su.n_tok, 4, 64), 8, DT[ty])
    check_attention(su, q, su.attend(q))
    su = SharedSetup(pk, [(15, 3), (12, 2)], [20, 0, 37, 50, 1], [1, 3, 2, 1, 1], "q8", 2, 64, 16, seed=2)
    q = randn((su.n_tok, 4, 64), 8, DT[ty])
    for max_len in (15, 17):
        check_attention(su, q, su.cache.attend(su.seqs, q, shared=pk.KvShared(su.shared.first, su.shared.len, su.shared.max_tok, max_len, 51)))
    # (cut to 9, six positions more of a sequence are besides them; max_tok 0: all of a sequence are)
    check_attention(su, q, su.cache.attend(su.seqs, q, shared=pk.KvShared(su.shared.first, su.shared.len, su.shared.max_tok, 9, 51 + 6)))
    check_attention(su, q, su.cache.attend(su.seqs, q, shared=pk.KvShared(su.shared.first, su.shared.len, 0, 9, 15 + 51 + 6)))


@pytest.mark.parametrize("ty, dh, heads", [("f16", 128, 16), ("bf16", 64, 40), ("f32", 64, 4), ("f32", 64, 40), ("f32", 128, 16)])
def test_shared_reads_what_was_just_written(pk, ty, dh, heads):
    """Queries, lengths, tables and the cache are written by the calls right before, which nobody waits for: the results are
    those of calls that were waited for, bit by bit, also from a captured graph."""
    su = SharedSetup(pk, [(700, 6), (90, 3)], [(37 * i) % 120 for i in range(9)], [2] * 9, "q8", 2, dh, 32, seed=4)
    sq, c, n = su.shared_seqs, su.cache, su.n_tok
    k, v = (randn((n, 2, dh), 40 + i, DT[ty]) for i in range(2))
    qs = [randn((n, heads, dh), i, DT[ty]) for i in range(6)]
    ctx = [sq.ctx - i for i in range(6)]  # (the first of a group keeps its prefix: own positions 0 .. only shrink)
    for x in ctx:
        x[[0, 6]] = sq.ctx[[0, 6]]
    q = torch.empty_like(qs[0])
    cells = [t.clone() for t in (c.k, c.v, c.ks, c.vs)]

    def step(i):
        for t, was in zip((c.k, c.v, c.ks, c.vs), cells):
            t.copy_(was)
        sq.ctx.copy_(ctx[i])
        sq.pages.copy_(table)
        c.store(sq, k * (1 + i), v * (1 + i))
        q.copy_(qs[i])

    table = sq.pages.clone()
    want = []
    for i in range(6):
        step(i)
        torch.cuda.synchronize()
        want.append(su.attend(q))
        torch.cuda.synchronize()
    got = []
    for i in range(30):
        sq.pages.fill_(-1)
        step(i % 6)
        got.append(su.attend(q))
        q.fill_(math.nan)
    torch.cuda.synchronize()
    assert all(torch.equal(got[i], want[i % 6]) for i in range(30))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = []
        for i in range(6):
            sq.pages.fill_(-1)
            step(i)
            out.append(su.attend(q))
            q.fill_(math.nan)
    for _ in range(5):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.parametrize("kind", ["q8", "q4"])
@pytest.mark.parametrize("lens, new, n_kv, heads", [
    ([700, 0, 33], [64, 40, 1], 3, 3),            # few CTAs: of two blocks, one without rows, several chunks
    ([900, 30, 0, 871, 512, 64], [33, 1, 40, 7, 33, 2], 36, 36),  # many: of one block, two an SM
    ([6400, 5000, 10, 6000], [3, 1, 40, 16], 36, 36),             # of one block, chunks in clusters
    ([3000] * 30, [5] * 30, 8, 64),               # eight query heads a kv head
    ([20000], [100], 36, 36),                     # chunks through the scratch
    ([8000], [64], 36, 36),                       # of two blocks, chunks through the scratch
    ([150] * 20, [128] * 20, 8, 8),               # of one block without a row to spare, many of few tiles
])
def test_attention_of_33_to_128_f32_rows(pk, kind, lens, new, n_kv, heads):
    """Every form that f32 rows of head_dim 64 take on the tensor cores, causal and with a mask of one's own token alone."""
    su = Setup(pk, lens, new, kind, n_kv, 64, 64, seed=3)
    su.fill(pk)
    q = randn((su.n_tok, heads, 64), 8)
    check_attention(su, q, su.cache.attend(su.seqs, q))
    alone = words_of([1 << j for n in new for j in range(n)], 2)  # (token 64 of a sequence is in the second word)
    check_attention(su, q, su.cache.attend(su.seqs, q, mask=alone), see=lambda s, n: torch.eye(n, dtype=torch.bool, device="cuda"))
