"""The quantised K/V cache options of the engine (pk_set_kv_type(PK_KV_Q8 / PK_KV_Q4)): layer 0's rotation and attention
against a 64-bit computation over the stored values, prompts in lanes against the same chunks one by one, streams against
the engine alone, and the whole model against its f32 cache."""
import math

import numpy as np
import pytest

from pocketinfer import synth

pytestmark = pytest.mark.gpu
DH128 = synth.ModelSpec("tiny-dh128", n_layer=2, n_embd=256, n_head=2, n_head_kv=1, head_dim=128, n_ff=512, n_vocab=1000)
DH32 = synth.ModelSpec("tiny-dh32", n_layer=1, n_embd=256, n_head=8, n_head_kv=2, head_dim=32, n_ff=512, n_vocab=1000)
MODELS = {"tiny": synth.TINY, "q8down": synth.SMALL_Q8DOWN, "q40": synth.SMALL_Q40, "dh128": DH128}


@pytest.fixture(scope="module")
def paths(tmp_path_factory):
    d = tmp_path_factory.mktemp("kvq")
    out = {}
    for name, spec in list(MODELS.items()) + [("dh32", DH32)]:
        out[name] = str(d / f"{name}.gguf")
        synth.write_gguf(out[name], spec, seed=33)
    return out


def rotated(x, spec):
    """x [n, heads, dh] at positions 0 .., in 64 bits, neighbouring pairs."""
    n_rot = spec.n_rot or spec.head_dim
    ang = np.arange(x.shape[0])[:, None] * spec.rope_theta ** (-2.0 * np.arange(n_rot // 2) / n_rot)[None]
    c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
    y = x.astype(np.float64).copy()
    a, b = x[..., 0:n_rot:2].astype(np.float64), x[..., 1:n_rot:2].astype(np.float64)
    y[..., 0:n_rot:2], y[..., 1:n_rot:2] = a * c - b * s, a * s + b * c
    return y


@pytest.mark.parametrize("kind", ["q8", "q4"])
@pytest.mark.parametrize("name", list(MODELS))
def test_layer_zero(pk, paths, name, kind):
    """Batches of 32, 1, 31, 1 and 7 tokens (over the page edge at 64).  The attention is held to the error of rows that
    are known: those that pk_kv_store keeps of the rotated K and V."""
    import torch

    spec = MODELS[name]
    H, KV, dh = spec.n_head, spec.n_head_kv, spec.head_dim
    e = pk.Engine(paths[name], n_ctx=128, kv=kind)
    ids = synth.prompt_ids(7, 72, spec.n_vocab)
    ks, vs, qs, ropes, outs, at = [], [], [], [], [], 0
    for n in (32, 1, 31, 1, 7):
        e.set_debug(True)
        e.forward(ids[at:at + n], list(range(at, at + n)))
        for to, key, heads in ((qs, "Qcur-0", H), (ks, "Kcur-0", KV), (vs, "Vcur-0", KV), (ropes, "Qrope-0", H), (outs, "kqv_out-0", H)):
            to.append(e.dump(key).reshape(n, heads, dh))
        at += n
    q, k, v, rope, out = (np.concatenate(x) for x in (qs, ks, vs, ropes, outs))
    # a result of two products and a sum in f32 of a sine and cosine rounded to f32: within 4 half steps of |a| + |b|
    pair = np.abs(q).astype(np.float64)
    pair = np.repeat(pair[..., 0::2] + pair[..., 1::2], 2, axis=-1)
    want_q = rotated(q, spec)
    assert (np.abs(rope - want_q) <= 4 * 2.0 ** -24 * pair).all()
    # K rotated and both stored by the public calls, read back
    table = pk.RopeTable(spec.n_rot or dh, spec.rope_theta)
    pos = torch.arange(72, dtype=torch.int32, device="cuda")
    kr = torch.from_numpy(k).cuda()
    _, kr = pk.rope(table, pos, torch.from_numpy(q).cuda(), kr)
    cache = pk.KvCache.empty(2, 64, KV, dh, kind)
    one = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    seqs = pk.KvSeqs(one([0, 72]), one([0]), one([[0, 1]]), 72, 72, 72)
    cache.store(seqs, kr, torch.from_numpy(v).cuda())
    k64, v64 = (x.double().cpu().numpy() for x in cache.load(seqs, torch.float32))
    for h in range(H):
        w = rope[:, h].astype(np.float64) @ k64[:, h // (H // KV)].T / math.sqrt(dh)
        w[np.triu_indices(72, 1)] = -np.inf
        p = np.exp(w - w.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        want, absv = p @ v64[:, h // (H // KV)], p @ np.abs(v64[:, h // (H // KV)])
        dots = (np.abs(rope[:, h]).astype(np.float64) @ np.abs(k64[:, h // (H // KV)]).T / math.sqrt(dh)).max(1, keepdims=True)
        # weights 2^-21 as two f16 terms, sums 2^-20, scores (dh + 8) 2^-23 + 2^-22 of sum |q k| on both sides of the
        # quotient, the scale's and the output's rounding
        lim = absv * (2.0 ** -21 + 2.0 ** -20 + 2 * ((dh + 9) * 2.0 ** -23 + 2.0 ** -22) * dots) + np.abs(want) * 2.0 ** -24
        assert (np.abs(out[:, h] - want) <= lim + 1e-30).all(), (h, (np.abs(out[:, h] - want) / (lim + 1e-30)).max())


@pytest.mark.parametrize("kind", ["q8", "q4"])
@pytest.mark.parametrize("name", list(MODELS))
def test_prompts_in_lanes(pk, paths, name, kind):
    """A prompt of several chunks runs them in lanes; one by one they give the same logits bit for bit (below 257
    positions no row's history is split), and so do the tokens that follow; a prompt that goes on reuses the prefix."""
    spec = MODELS[name]
    ids = synth.prompt_ids(19, 225, spec.n_vocab)
    a, b = pk.Engine(paths[name], n_ctx=256, kv=kind), pk.Engine(paths[name], n_ctx=256, kv=kind)
    r = a.generate(ids, 20, stop_at_eog=False)
    for o in range(0, 225, 32):
        m = min(32, 225 - o)
        b.forward(ids[o:o + m], list(range(o, o + m)), want_logits=o + m == 225)
    toks, tok = [], int(np.argmax(b.logits()))
    for i in range(20):
        toks.append(tok)
        if i < 19:
            b.forward([tok], [225 + i])
            tok = int(np.argmax(b.logits()))
    assert r["gen_ids"] == toks
    assert np.array_equal(a.logits().view(np.uint32), b.logits().view(np.uint32))
    assert a.generate(np.concatenate([ids, ids[:9]]), 2, stop_at_eog=False)["prefill_cached_tokens"] > 0


def test_lanes_with_the_tensor_memory_matvecs(pk, paths):
    """Six lanes of chunks whose matvecs and attention both use tensor memory: the default matvecs' tokens (the two
    paths give the same bits)."""
    ids = synth.prompt_ids(31, 250, synth.SMALL_Q40.n_vocab)
    want = pk.Engine(paths["q40"], n_ctx=320, kv="q8").generate(ids, 12, stop_at_eog=False)["gen_ids"]
    pk.set_matmul_path("tcgen05")
    try:
        e = pk.Engine(paths["q40"], n_ctx=320, kv="q8")
        for _ in range(3):
            assert e.generate(ids, 12, stop_at_eog=False)["gen_ids"] == want
            e.forward(ids[:1], [0])  # (drops the prefix)
    finally:
        pk.set_matmul_path("mma.sync")


@pytest.mark.parametrize("kind", ["q8", "q4"])
@pytest.mark.parametrize("name", ["tiny", "q8down", "dh128"])
def test_streams(pk, paths, name, kind):
    """Streams of different lengths in one batched step a token: each stream's tokens are the engine's for it alone."""
    spec = MODELS[name]
    prompts = [synth.prompt_ids(51 + i, n, spec.n_vocab) for i, n in enumerate((1, 20, 70, 131))]
    want = [pk.Engine(paths[name], n_ctx=256, kv=kind).generate(p, 24, stop_at_eog=False)["gen_ids"] for p in prompts]
    e = pk.Engine(paths[name], n_ctx=256, kv=kind)
    e.streams_begin(len(prompts))
    for s in (2, 0, 3, 1):
        e.stream_prefill(s, prompts[s])
    a, b = e.streams_decode(9), e.streams_decode(15)
    assert [x + y for x, y in zip(a, b)] == want
    # the engine's own sequence lies in pages of its own
    assert e.generate(prompts[1], 24, stop_at_eog=False)["gen_ids"] == want[1]
    e.stream_prefill(3, prompts[0])
    assert e.streams_decode(24)[3] == want[0]


@pytest.mark.parametrize("name,n_ctx,n", [("tiny", 256, 200), ("q8down", 256, 200), ("q40", 256, 200), ("dh128", 256, 200), ("dh128", 2000, 1900)])
def test_near_the_f32_cache(pk, paths, name, n_ctx, n):
    """Logits of a prompt beside those of the f32 cache.  A Q8 row is off by at most half a step of its largest / 127, in
    the mean 0.6% of the row for rows of normal values, a Q4 row by half a step of a block's largest / 7, 9%.  Each layer
    adds that to its attention's output at the most, the attention is at most one of the two equal parts of a layer's
    sum, and the layers' errors add as independent ones: under sqrt(3) of it in at most three layers, doubled for K.
    Twice that is allowed: 5% and 60% of the logits' size.  A wrong page, layer or position gives 100% and more."""
    spec = MODELS[name]
    ids = synth.prompt_ids(23, n, spec.n_vocab)
    logits = {}
    for kind in ("f32", "q8", "q4"):
        e = pk.Engine(paths[name], n_ctx=n_ctx, kv=kind)
        e.generate(ids, 1, stop_at_eog=False)
        logits[kind] = e.logits().astype(np.float64)
        if kind != "f32":
            per = 2 * spec.n_layer * spec.n_head_kv * (spec.head_dim + 4 if kind == "q8" else spec.head_dim // 2 + 8)
            assert e.model_info()["kv_bytes"] == -(-n_ctx // 64) * 64 * per
    size = np.linalg.norm(logits["f32"])
    assert np.linalg.norm(logits["q8"] - logits["f32"]) <= 0.05 * size
    assert np.linalg.norm(logits["q4"] - logits["f32"]) <= 0.6 * size


def test_long_history(pk, paths):
    """Histories that are split over CTAs, in lanes, alone and in streams: every path reads the same cache, so logits
    agree to the sums' order, which the 8-bit activations of the next product can turn into a step of 1/127 of a block's
    largest here and there: 2% of the logits' size."""
    spec = DH128
    ids = synth.prompt_ids(29, 1500, spec.n_vocab)
    a, b = pk.Engine(paths["dh128"], n_ctx=1536, kv="q8"), pk.Engine(paths["dh128"], n_ctx=1536, kv="q8")
    a.generate(ids, 1, stop_at_eog=False)
    for o in range(0, 1500, 20):
        b.forward(ids[o:o + 20], list(range(o, o + 20)), want_logits=o == 1480)
    x, y = a.logits().astype(np.float64), b.logits().astype(np.float64)
    assert np.linalg.norm(x - y) <= 0.02 * np.linalg.norm(x)


@pytest.mark.parametrize("kind", ["q8", "q4"])
def test_device_steps(pk, paths, kind):
    """Steps kept on the device (one graph a step), a rewound position, the fast order, and the per-kernel profile."""
    ids = synth.prompt_ids(37, 70, synth.TINY.n_vocab)
    want = pk.Engine(paths["tiny"], n_ctx=256, kv=kind).generate(ids, 20, stop_at_eog=False)["gen_ids"]
    e = pk.Engine(paths["tiny"], n_ctx=256, kv=kind, order="fast")
    e.generate(ids, 1, stop_at_eog=False)
    assert list(e.decode_steps_device(20)) == want
    e.set_position(70)
    e.generate(ids, 1, stop_at_eog=False)
    assert list(e.decode_steps_device(5)) == want[:5]
    names = {r["name"] for r in e.decode_profile()}
    assert {"k_rope", "k_kv_store", "k_kv_attn"} <= names
    e.generate(ids, 1, stop_at_eog=False)
    assert list(e.decode_steps_device(5)) == want[:5]


def test_refusals(pk, paths):
    e = pk.Engine(paths["tiny"], n_ctx=128, kv="q8")
    ids = synth.prompt_ids(3, 4, synth.TINY.n_vocab)
    for pos in ([0, 2, 3, 4], [3, 2, 1, 0], [5, 5, 5, 5]):
        with pytest.raises(Exception, match="consecutive"):
            e.forward(ids, pos)
    e.forward(ids, [0, 1, 2, 3])
    with pytest.raises(Exception, match="head_dim"):
        pk.Engine(paths["dh32"], n_ctx=128, kv="q4")
    assert pk.lib().pk_set_kv_type(e.h, pk.KV_Q8) != 0
    with pytest.raises(KeyError):
        pk.Engine(paths["tiny"], n_ctx=128, kv="q5")


def test_a_wait_that_runs_out_is_an_error(pk, paths):
    """An attention launch whose codes never arrive ends after its bounded waits, the engine reports it, and goes on as
    one that has not seen it."""
    spec = synth.SMALL_Q40
    ids = synth.prompt_ids(31, 40, spec.n_vocab)
    ref, e = (pk.Engine(paths["q40"], n_ctx=128, kv="q8") for _ in range(2))
    want = ref.generate(ids, 8, stop_at_eog=False)["gen_ids"]
    assert e.generate(ids, 8, stop_at_eog=False)["gen_ids"] == want
    assert e.selftest_bounded_wait() == 8  # PK_ERR_TIMEOUT
    e.forward(ids[:32], list(range(32)))
    ref.forward(ids[:32], list(range(32)))
    assert np.array_equal(e.logits().view(np.uint32), ref.logits().view(np.uint32))
    assert e.generate(ids, 8, stop_at_eog=False)["gen_ids"] == want
    with pytest.raises(pk.PkError):  # (no attention with waits at head_dim 128 in f32)
        pk.Engine(paths["dh128"], n_ctx=128, kv="q8").selftest_bounded_wait()
