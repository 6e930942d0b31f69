"""Measured cases of the drafted-decoding operators: rotary positions, the quantised paged K/V cache, attention of
drafted tokens over it, and the rules applied to logits before a token is drawn.

`run` computes a case either through pocketinfer (`own`) or with elementary torch operations in 32 bits.

The cache's entries, as include/pk.h documents them.  A row is one (position, kv head) of K or V:
  q8  code byte = c + 128 with c = rint(x / D), |c| <= 127, D = amax / 127; the row stands for D * c
  q4  nibble j = c + 8 with c = rint(x / (D * s_b)), -8 <= c <= 7, D = amax / 105, s_b = ceil(amax_b / (7 * D)) in
      1..15 for each 32 dimensions b (nibble b of the word beside D); the row stands for D * (c * s_b)
Codes are [page][kv head][slot][bytes], scales [page][kv head][slot][1 or 2 words].
"""
import math
import os
import sys

import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
BIG = 2.0 ** 127  # larger magnitudes are stored as this


def _pk():
    path = os.path.join(os.getcwd(), "pocket-workbench-android_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import pocketinfer

    return pocketinfer


# ------------------------------------------------------------------ the cases

M70 = {"heads": 64, "kv": 8, "dh": 128}  # the 70B-shaped stack's attention
M26 = {"heads": 36, "kv": 36, "dh": 64}  # the 2.6B-shaped stack's: one query head a kv head


def listed():
    return [
        # the drafts of one sequence far beyond the trained context: a handful of rows, where launch latency counts
        {"name": "rope_drafts", "op": "rope", **M70, "tok": 9, "type": "f32", "layout": "half", "n_rot": 128,
         "scaling": "yarn", "far": 120000},
        # a long prompt in half precision, part of each head rotated
        {"name": "rope_prompt", "op": "rope", **M26, "tok": 8191, "type": "f16", "layout": "interleaved", "n_rot": 48,
         "scaling": "linear", "far": 16384},
        # one token of each of 64 streams, written and read back
        {"name": "kv_step", "op": "kv", **M70, "seqs": 64, "ctx": 4000, "new": 1, "page": 64, "kv_type": "q8",
         "type": "bf16", "ragged": 1},
        # the prompts of five requests written at once in 4 bits, and read back, as for a cache that moves elsewhere
        {"name": "kv_prompts", "op": "kv", **M26, "seqs": 5, "ctx": 700, "new": 3500, "page": 16, "kv_type": "q4",
         "type": "f16", "ragged": 1},
        # around a verification: the drafts are written, the accepted path is moved up behind the context and read back
        {"name": "kv_accept", "op": "keep", **M70, "seqs": 24, "ctx": 9000, "new": 33, "page": 32, "kv_type": "q8",
         "type": "f32", "ragged": 1},
        # one user, one token: the smallest call of a decode step
        {"name": "attn_token", "op": "attn", **M70, "seqs": 1, "ctx": 1500, "new": 1, "page": 64, "kv_type": "q8",
         "type": "f16", "ragged": 0, "tree": 0},
        # eight streams at 16K positions, as the streams benchmark has them
        {"name": "attn_streams", "op": "attn", **M26, "seqs": 8, "ctx": 16256, "new": 1, "page": 256, "kv_type": "q8",
         "type": "f32", "ragged": 0, "tree": 0},
        # a ragged serving batch, a few drafts a request, 4-bit cache
        {"name": "attn_drafts", "op": "attn", **M70, "seqs": 40, "ctx": 15000, "new": 5, "page": 16, "kv_type": "q4",
         "type": "bf16", "ragged": 1, "tree": 1},
        # wide trees over long histories: the most arithmetic
        {"name": "attn_tree", "op": "attn", **M70, "seqs": 8, "ctx": 32000, "new": 64, "page": 128, "kv_type": "q8",
         "type": "f16", "ragged": 0, "tree": 1},
        # a chunk of two prompts behind earlier parts of them, in the engine's own type
        {"name": "attn_chunk", "op": "attn", **M26, "seqs": 2, "ctx": 2900, "new": 509, "page": 64, "kv_type": "q8",
         "type": "f32", "ragged": 1, "tree": 0},
        # one row of logits before sampling
        {"name": "rules_row", "op": "rules", "rows": 1, "vocab": 73448, "type": "f32", "hist": 600, "bias": 20},
        # a serving batch's logits, each row with its own history, biases and grammar
        {"name": "rules_batch", "op": "rules", "rows": 250, "vocab": 128256, "type": "f32", "hist": 3000, "bias": 300},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "kv", "kv", "keep", "attn", "attn", "attn", "rules"])
    heads = rng.choice([M70, M26, {"heads": 4, "kv": 2, "dh": 64}, {"heads": 8, "kv": 8, "dh": 64}, {"heads": 21, "kv": 3, "dh": 128}])
    c = {"op": op, "type": rng.choice(["f32", "f16", "bf16"])}
    if op == "rope":
        return {**c, **heads, "tok": _log(rng, 1, 8191), "layout": rng.choice(["half", "interleaved"]),
                "n_rot": rng.choice([heads["dh"], heads["dh"] // 2, 2 * rng.randint(1, heads["dh"] // 2)]),
                "scaling": rng.choice(["none", "linear", "ntk", "yarn"]), "far": _log(rng, 100, 1000000)}
    if op == "rules":
        rows = _log(rng, 1, 250)
        return {**c, "rows": rows, "vocab": _log(rng, 1000, 128256), "hist": _log(rng, 1, 3000), "bias": rng.choice([0, _log(rng, 1, 300)])}
    c |= {**heads, "page": rng.choice([16, 32, 64, 128, 256]), "kv_type": rng.choice(["q8", "q4"]), "ragged": rng.randint(0, 1)}
    if op == "kv":
        seqs = _log(rng, 1, 64)
        return {**c, "seqs": seqs, "ctx": _log(rng, 1, 4000), "new": _log(rng, 1, max(1, min(3500, 12000 // seqs)))}
    if op == "keep":
        return {**c, "seqs": _log(rng, 1, 24), "ctx": _log(rng, 1, 9000), "new": _log(rng, 1, 33)}
    seqs = _log(rng, 1, 40)
    return {**c, "seqs": seqs, "ctx": _log(rng, 1, min(32000, 250000000 // (seqs * c["kv"] * c["dh"]))), "new": rng.choice([1, _log(rng, 1, 64)]),
            "tree": rng.randint(0, 1)}


def _lens(case):
    """Committed positions and new tokens of each sequence: even, or ragged with a first one of full size."""
    ctx, new = [], []
    for s in range(case["seqs"]):
        f = 1.0 if s == 0 or not case["ragged"] else (0.05 + 0.95 * ((s * 0.6180339887) % 1.0))
        g = 1.0 if s == 0 or not case["ragged"] or case["new"] == 1 else (s * 0.7548776662) % 1.0
        ctx.append(int(case["ctx"] * f))
        new.append(max(0 if case["new"] > 2 else 1, int(case["new"] * g)))
    return ctx, new


def _kept(case):
    """How many drafts of each sequence were accepted."""
    return [min(n, 1 + (3 * s) % 7) for s, n in enumerate(_lens(case)[1])]


def _row_bytes(case):
    return case["dh"] + 4 if case["kv_type"] == "q8" else case["dh"] // 2 + 8


def work(case):
    op = case["op"]
    if op == "rules":
        n, v = case["rows"], case["vocab"]
        return {"bytes": n * (2 * v * SIZE[case["type"]] + 4 * ((v + 31) // 32) + 4 * case["hist"] + 8 * case["bias"]), "flops": 4 * n * v}
    if op == "rope":
        x = case["tok"] * (case["heads"] + case["kv"])
        return {"bytes": 2 * x * case["dh"] * SIZE[case["type"]] + 4 * case["tok"], "flops": 3 * x * case["n_rot"]}
    ctx, new = _lens(case)
    kv, dh, e, row = case["kv"], case["dh"], SIZE[case["type"]], _row_bytes(case)
    if op == "kv":
        x = 2 * sum(new) * kv
        return {"bytes": 2 * x * (dh * e + row), "flops": 6 * x * dh}
    if op == "keep":
        x, y = 2 * sum(new) * kv, 2 * sum(_kept(case)) * kv
        return {"bytes": x * (dh * e + row) + y * (3 * row + dh * e), "flops": 4 * x * dh}
    seen = sum((c + n) for c, n in zip(ctx, new) if n)
    each = sum(n * (c + n) for c, n in zip(ctx, new))
    q = 2 * sum(new) * case["heads"] * dh * e
    return {"bytes": 2 * seen * kv * row + q + 8 * sum(new) * case["tree"], "flops": 4 * each * case["heads"] * dh}


# ------------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)


def _normal(g, shape, dtype=torch.float32, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def _keys(g, shape, dtype):
    """K rows as projections give them: some dimensions far larger than the rest, a size of its own for each row."""
    x = torch.randn(shape, generator=g, device="cuda")
    x[..., :: 11] *= 4.0
    return (x * (0.5 + torch.rand(shape[:-1], generator=g, device="cuda")).unsqueeze(-1)).to(dtype)


def _pages(case, g, room):
    """A page table over a shuffled pool, with no page behind a sequence's last one."""
    ps = case["page"]
    need = [(n + ps - 1) // ps for n in room]
    order = (torch.randperm(sum(need) + 3, generator=g, device="cuda") if sum(need) else torch.zeros(0, device="cuda")).to(torch.int32)
    table = torch.full((case["seqs"], max(max(need), 1)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    return table, sum(need) + 3


def _tree_masks(case, seed, new):
    """For every drafted token the bits of its ancestors and itself, for random trees in which a parent comes first."""
    rng = torch.Generator().manual_seed(int(seed) + 5)
    rows = []
    for n in new:
        bits = []
        for i in range(n):
            parent = int(torch.randint(max(0, i - 8), i, (1,), generator=rng)) if i else -1
            bits.append((bits[parent] if parent >= 0 else 0) | (1 << i))
        rows += [b - (1 << 64) if b >> 63 else b for b in bits]
    return torch.tensor(rows, dtype=torch.int64).reshape(-1, 1).cuda()


def prepare(case, seed):
    g, op, dt = _gen(seed), case["op"], DT[case["type"]]
    st = {"case": case}
    if op == "rope":
        st["pos"] = (case["far"] + torch.randint(0, 64, (case["tok"],), generator=g, device="cuda")
                     if case["tok"] < 100 else torch.arange(case["tok"], device="cuda") + case["far"]).to(torch.int32)
        st["q"] = _normal(g, (case["tok"], case["heads"], case["dh"]), dt)
        st["k"] = _normal(g, (case["tok"], case["kv"], case["dh"]), dt)
        st["turns"], st["gain"] = _turns(case)
        if own:
            st["rope"] = _pk().RopeTable(case["n_rot"], **_rope_args(case))
        return st
    if op == "rules":
        n, v = case["rows"], case["vocab"]
        x = torch.rand((n, case["hist"]), generator=g, device="cuda")
        st["hist"] = (v * x ** 6).to(torch.int32).clamp(max=v - 1)  # few tokens often, many once
        st["n_hist"] = torch.tensor([max(1, int(case["hist"] * (1.0 if r == 0 else (r * 0.6180339887) % 1.0))) for r in range(n)],
                                    dtype=torch.int32, device="cuda")
        st["logits"] = _normal(g, (n, v), torch.float32, 4.0).to(dt)
        st["repeat"] = 1.0 + 0.3 * torch.rand(n, generator=g, device="cuda")
        st["freq"] = 0.5 * torch.rand(n, generator=g, device="cuda")
        st["presence"] = 0.5 * torch.rand(n, generator=g, device="cuda")
        words = torch.randint(-2 ** 31, 2 ** 31, (n, (v + 31) // 32), generator=g, device="cuda")
        keep = torch.rand(words.shape, generator=g, device="cuda") < 0.4  # runs of forbidden tokens
        st["allow"] = torch.where(keep, words, torch.zeros_like(words)).to(torch.int32)
        st["bias_id"] = st["bias"] = None
        if case["bias"]:
            st["bias_id"] = torch.randint(0, v, (n, case["bias"]), generator=g, device="cuda").to(torch.int32)
            st["bias"] = _normal(g, (n, case["bias"]), std=2.0)
        return st
    ctx, new = _lens(case)
    st["table"], n_pages = _pages(case, g, [c + n for c, n in zip(ctx, new)])
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    st["start"] = torch.tensor(start, dtype=torch.int32, device="cuda")
    st["ctx"] = torch.tensor(ctx, dtype=torch.int32, device="cuda")
    tok, kv, dh, ps = start[-1], case["kv"], case["dh"], case["page"]
    row, words = (dh, 1) if case["kv_type"] == "q8" else (dh // 2, 2)
    for name in ("k", "v"):
        st["c" + name] = torch.empty((n_pages, kv, ps, row), dtype=torch.uint8, device="cuda")
        st["s" + name] = torch.zeros((n_pages, kv, ps, words), dtype=torch.float32, device="cuda")
    if op == "attn":
        step = max(1, (1 << 25) // (kv * ps * dh))
        for p in range(0, n_pages, step):
            m = min(step, n_pages - p)
            for name, make in (("k", _keys), ("v", _normal)):
                _quantise(make(g, (m, kv, ps, dh), torch.float32), case["kv_type"], st["c" + name][p:p + m], st["s" + name][p:p + m])
        st["q"] = _normal(g, (tok, case["heads"], dh), dt)
        st["mask"] = _tree_masks(case, seed, new) if case["tree"] else None
    else:
        st["new_k"], st["new_v"] = _keys(g, (tok, kv, dh), dt), _normal(g, (tok, kv, dh), dt)
    st["most"] = (max(new), max(c + n for c, n in zip(ctx, new)))
    if op == "keep":
        kept = _kept(case)
        st["n_keep"] = torch.tensor(kept, dtype=torch.int32, device="cuda")
        path = torch.zeros((case["seqs"], max(kept)), dtype=torch.int32)
        rng = torch.Generator().manual_seed(int(seed))
        for s, (a, n) in enumerate(zip(kept, new)):
            path[s, :a] = torch.sort(torch.randperm(n, generator=rng)[:a]).values
        st["path"] = path.cuda()
        at = [0]
        for a in kept:
            at.append(at[-1] + a)
        st["kept_start"] = torch.tensor(at, dtype=torch.int32, device="cuda")
        st["kept_most"] = (max(kept), max(c + a for c, a in zip(ctx, kept)), at[-1])
    if own:
        pk = _pk()
        st["cache"] = pk.KvCache(st["ck"], st["cv"], st["sk"], st["sv"], case["kv_type"], dh)
        st["seqs"] = pk.KvSeqs(st["start"], st["ctx"], st["table"], tok, *st["most"])
        if op == "keep":
            st["kept_seqs"] = pk.KvSeqs(st["kept_start"], st["ctx"], st["table"], st["kept_most"][2], *st["kept_most"][:2])
    return st


# ------------------------------------------------------------------ rotary positions

def _rope_args(case):
    return {"theta": 10000.0, "scaling": case["scaling"], "factor": 1.0 if case["scaling"] == "none" else 8.0,
            "n_ctx_train": 4096}


def _turns(case):
    """Turns a position of each pair, and the gain: the pair's frequency theta^(-2i/n_rot) over 2 pi.  linear divides it
    by the factor, ntk stretches theta so that the slowest pair is divided by it, yarn divides the pairs that turn less
    than once in the trained context, keeps those that turn over 32 times and goes over in between."""
    a, n = _rope_args(case), case["n_rot"]
    i = torch.arange(0, n, 2, dtype=torch.float64)
    theta, gain = a["theta"], 1.0
    if a["scaling"] == "ntk" and n > 2:
        theta *= a["factor"] ** (n / (n - 2))
    f = theta ** (-i / n) / (2.0 * math.pi)
    if a["scaling"] == "linear":
        f = f / a["factor"]
    if a["scaling"] == "yarn":
        keep = ((f * a["n_ctx_train"] - 1.0) / 31.0).clamp(0.0, 1.0)
        f = f / a["factor"] * (1.0 - keep) + f * keep
        gain = 0.1 * math.log(a["factor"]) + 1.0
    return f.cuda(), gain


def _rotate(x, cos, sin, n, layout):
    x32, out = x.float(), x.float().clone()
    a, b = (x32[..., 0:n:2], x32[..., 1:n:2]) if layout == "interleaved" else (x32[..., :n // 2], x32[..., n // 2:n])
    u, v = a * cos - b * sin, a * sin + b * cos
    if layout == "interleaved":
        out[..., 0:n:2], out[..., 1:n:2] = u, v
    else:
        out[..., :n // 2], out[..., n // 2:n] = u, v
    return out.to(x.dtype)


def _run_rope(st):
    c = st["case"]
    if own:
        q, k = _pk().rope(st["rope"], st["pos"], st["q"], st["k"], layout=c["layout"])
        return {"q": q, "k": k}
    angle = 2.0 * math.pi * ((st["pos"].double()[:, None] * st["turns"]) % 1.0)  # far positions: 64 bits
    cos, sin = (angle.cos() * st["gain"]).float()[:, None], (angle.sin() * st["gain"]).float()[:, None]
    return {"q": _rotate(st["q"], cos, sin, c["n_rot"], c["layout"]), "k": _rotate(st["k"], cos, sin, c["n_rot"], c["layout"])}


# ------------------------------------------------------------------ the quantised cache

def _quantise(x, kind, codes, scales):
    """Rows x [..., dh] into codes [..., bytes] and scales [..., 1 or 2]."""
    x = x.float().nan_to_num(nan=0.0, posinf=BIG, neginf=-BIG).clamp(-BIG, BIG)
    amax = x.abs().amax(-1, keepdim=True)
    if kind == "q8":
        d = amax / torch.full_like(amax, 127.0)  # a division by a plain number is a product with its rounded inverse
        q = torch.round(x.double() / d.double()).nan_to_num(nan=0.0).clamp(-127, 127)
        codes.copy_((q + 128).to(torch.uint8))
        scales.copy_(d)
        return
    d = amax / torch.full_like(amax, 105.0)
    blocks = x.unflatten(-1, (-1, 32))
    s = torch.ceil(blocks.abs().amax(-1) / (7.0 * d)).nan_to_num(nan=1.0, posinf=15.0).clamp(1, 15)
    step = (d * s).unsqueeze(-1)
    q = torch.round(blocks.double() / step.double()).nan_to_num(nan=0.0).clamp(-8, 7).flatten(-2) + 8
    q = q.to(torch.uint8)
    codes.copy_(q[..., 0::2] | (q[..., 1::2] << 4))
    word = (s.to(torch.int64) << (4 * torch.arange(s.shape[-1], device=s.device))).sum(-1, keepdim=True)
    scales.copy_(torch.cat([d, torch.where(word >= 2 ** 31, word - 2 ** 32, word).to(torch.int32).view(torch.float32)], -1))


def _values(codes, scales, kind):
    """The values that codes [..., bytes] with scales [..., 1 or 2] stand for, in 32 bits."""
    if kind == "q8":
        return (codes.float() - 128.0) * scales
    nib = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float() - 8.0
    word = scales[..., 1:].contiguous().view(torch.int32)
    s = (word >> (4 * torch.arange(nib.shape[-1] // 32, device=nib.device, dtype=torch.int32))) & 15
    return (nib.unflatten(-1, (-1, 32)) * s.unsqueeze(-1).float()).flatten(-2) * scales[..., :1]


def _where(start, first, table, page, n_tok):
    """Page and slot of each token: token t of sequence s is position first[s] + t - start[s]."""
    t = torch.arange(n_tok, device="cuda")
    s = torch.searchsorted(start[1:].contiguous(), t, right=True, out_int32=False)
    p = first[s].long() + t - start[s].long()
    return table[s, p // page].long(), p % page


def _run_kv(st):
    c = st["case"]
    keep = c["op"] == "keep"
    if own:
        cache, seqs = st["cache"], st["seqs"]
        cache.store(seqs, st["new_k"], st["new_v"])
        if keep:
            cache.keep(seqs, st["path"], st["n_keep"])
            seqs = st["kept_seqs"]
        k, v = cache.load(seqs, DT[c["type"]])
        return {"k": k, "v": v}
    tok, kind, page = st["new_k"].shape[0], c["kv_type"], c["page"]
    pg, sl = _where(st["start"], st["ctx"], st["table"], page, tok)
    out = {}
    for name in ("k", "v"):
        codes, scales, x = st["c" + name], st["s" + name], st["new_" + name]
        to = torch.empty((tok,) + codes.shape[1:2] + codes.shape[3:], dtype=torch.uint8, device="cuda")
        sc = torch.empty((tok,) + scales.shape[1:2] + scales.shape[3:], device="cuda")
        _quantise(x, kind, to, sc)
        codes[pg, :, sl] = to
        scales[pg, :, sl] = sc
    if keep:
        n = st["kept_most"][2]
        t = torch.arange(n, device="cuda")
        s = torch.searchsorted(st["kept_start"][1:].contiguous(), t, right=True)
        at = st["path"][s, t - st["kept_start"][s].long()].long() + st["ctx"][s].long()
        from_pg, from_sl = st["table"][s, at // page].long(), at % page
        pg, sl = _where(st["kept_start"], st["ctx"], st["table"], page, n)
        for a in ("ck", "cv", "sk", "sv"):
            st[a][pg, :, sl] = st[a][from_pg, :, from_sl]
    for name in ("k", "v"):
        out[name] = _values(st["c" + name][pg, :, sl], st["s" + name][pg, :, sl], kind).to(DT[c["type"]])
    return out


# ------------------------------------------------------------------ attention of drafted tokens

def _run_attn(st):
    c = st["case"]
    if own:
        return st["cache"].attend(st["seqs"], st["q"], mask=st["mask"])
    q, start, ctx, table = st["q"], st["start"].long(), st["ctx"].long(), st["table"]
    (most, length), kv, page = st["most"], c["kv"], c["page"]
    group = c["heads"] // kv
    t = torch.arange(length, device="cuda")
    pg, sl = table[:, t // page].long().clamp(min=0), (t % page).expand(table.shape[0], -1)
    n = (start[1:] - start[:-1])[:, None]
    i = torch.arange(most, device="cuda")
    rows = (start[:-1, None] + i).clamp(max=q.shape[0] - 1)             # [S, most]
    k = _values(st["ck"][pg, :, sl], st["sk"][pg, :, sl], c["kv_type"])  # [S, L, kv, dh]
    x = q[rows].float().unflatten(2, (kv, group))                       # [S, most, kv, group, dh]
    w = torch.matmul(x.permute(0, 2, 3, 1, 4).flatten(2, 3), k.permute(0, 2, 3, 1)) * c["dh"] ** -0.5
    del k
    j = t[None] - ctx[:, None]                                          # the draft that a position holds, [S, L]
    if st["mask"] is None:
        see = j[:, None, :] <= i[None, :, None]
    else:
        bits = st["mask"][rows][..., 0]                                 # [S, most]
        see = (j[:, None, :] < 0) | (((bits[..., None] >> j.clamp(0, 63)[:, None, :]) & 1) != 0)
    see = see & (j < n)[:, None, :]
    see = see[:, None].expand(-1, group, -1, -1).flatten(1, 2)[:, None]  # [S, 1, group * most, L]
    w = w.masked_fill_(~see, -math.inf)
    top = w.amax(-1, keepdim=True)
    w = torch.exp_(w.sub_(top.masked_fill(top == -math.inf, 0.0)))
    total = w.sum(-1, keepdim=True)
    v = _values(st["cv"][pg, :, sl], st["sv"][pg, :, sl], c["kv_type"])
    o = torch.matmul(w, v.permute(0, 2, 1, 3)) / total.masked_fill(total == 0, 1.0)
    o = o.unflatten(2, (group, most)).permute(0, 3, 1, 2, 4).flatten(2, 3)  # [S, most, heads, dh]
    return o[i[None] < n].to(q.dtype)


# ------------------------------------------------------------------ rules on logits

def _run_rules(st):
    if own:
        return _pk().logit_rules(st["logits"], repeat=st["repeat"], freq=st["freq"], presence=st["presence"],
                                 hist=st["hist"], n_hist=st["n_hist"], bias_id=st["bias_id"], bias=st["bias"],
                                 allow=st["allow"])
    x = st["logits"].float()
    n, v = x.shape
    seen = (torch.arange(st["hist"].shape[1], device="cuda") < st["n_hist"][:, None]).float()
    count = torch.zeros((n, v), device="cuda").scatter_add_(1, st["hist"].long(), seen)
    r = st["repeat"][:, None]
    x = torch.where(count > 0, torch.where(x > 0, x / r, x * r) - (count * st["freq"][:, None] + st["presence"][:, None]), x)
    if st["bias"] is not None:
        x = x + torch.zeros((n, v), device="cuda").scatter_add_(1, st["bias_id"].long(), st["bias"])
    bit = (st["allow"][:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
    x = x.masked_fill(bit.flatten(1)[:, :v] == 0, -math.inf)
    return x.to(st["logits"].dtype)


def run(state):
    return {"rope": _run_rope, "kv": _run_kv, "keep": _run_kv, "attn": _run_attn, "rules": _run_rules}[state["case"]["op"]](state)


# ------------------------------------------------------------------ the definitions in 64 bits

def _stored64(x, kind):
    """What rows x [..., dh] read back as: D rounded to 32 bits, everything else in 64."""
    x = x.double()
    x = torch.where(torch.isnan(x), torch.zeros_like(x), x.clamp(-BIG, BIG))
    amax = x.abs().max(-1, keepdim=True).values
    if kind == "q8":
        d = (amax / 127).float().double()
        c = torch.where(d > 0, torch.round(x / d), torch.zeros_like(x)).clamp(-127, 127)
        return c * d
    d = (amax / 105).float().double()
    out = torch.zeros_like(x)
    for b in range(0, x.shape[-1], 32):
        y = x[..., b:b + 32]
        seven = (7 * d).float()
        s = torch.ceil((y.abs().max(-1, keepdim=True).values.float().double() / seven.double()).float().double()).clamp(1, 15)
        s = torch.where(d > 0, s, torch.ones_like(s))
        step = (d * s).float().double()
        c = torch.where(step > 0, torch.round(y / step), torch.zeros_like(y)).clamp(-8, 7)
        out[..., b:b + 32] = c * s * d
    return out


def _decoded64(codes, scales, kind):
    if kind == "q8":
        return (codes.double() - 128) * scales.double()
    dh = codes.shape[-1] * 2
    out = torch.empty(codes.shape[:-1] + (dh,), dtype=torch.float64, device=codes.device)
    out[..., 0::2], out[..., 1::2] = (codes % 16).double() - 8, (codes // 16).double() - 8
    word = scales[..., 1].contiguous().view(torch.int32)
    for b in range(dh // 32):
        out[..., 32 * b:32 * b + 32] *= (((word >> (4 * b)) & 15).double() * scales[..., 0].double())[..., None]
    return out


def _exact_attn(st):
    c = st["case"]
    start, ctx, table = st["start"].tolist(), st["ctx"].tolist(), st["table"].cpu()
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    group, page = c["heads"] // c["kv"], c["page"]
    for s in range(c["seqs"]):
        n, total = start[s + 1] - start[s], ctx[s] + start[s + 1] - start[s]
        if n == 0:
            continue
        pages = table[s, :(total + page - 1) // page].long().cuda()
        see = torch.ones((n, total), dtype=torch.bool, device="cuda")
        if st["mask"] is None:
            see[:, ctx[s]:] = torch.ones((n, n), dtype=torch.bool, device="cuda").tril()
        else:
            bits = [int(b) % (1 << 64) for b in st["mask"][start[s]:start[s + 1], 0].tolist()]
            see[:, ctx[s]:] = torch.tensor([[(b >> j) & 1 for j in range(n)] for b in bits], dtype=torch.bool, device="cuda")
        for h in range(c["kv"]):
            k = _decoded64(st["ck"][pages, h].flatten(0, 1)[:total], st["sk"][pages, h].flatten(0, 1)[:total], c["kv_type"])
            v = _decoded64(st["cv"][pages, h].flatten(0, 1)[:total], st["sv"][pages, h].flatten(0, 1)[:total], c["kv_type"])
            q = st["q"][start[s]:start[s + 1], h * group:(h + 1) * group].double()
            w = torch.einsum("ngd,td->ngt", q, k) / math.sqrt(c["dh"])
            w = torch.where(see[:, None], w, torch.full_like(w, -math.inf))
            w = torch.where(see.any(-1)[:, None, None], torch.softmax(w, -1), torch.zeros_like(w))
            out[start[s]:start[s + 1], h * group:(h + 1) * group] = torch.einsum("ngt,td->ngd", w, v)
    return out


def _exact_rules(st):
    x, out = st["logits"].double(), []
    for r in range(x.shape[0]):
        y = x[r].clone()
        ids, count = torch.unique(st["hist"][r, :int(st["n_hist"][r])].long(), return_counts=True)
        f, p, rep = (float(st[a][r]) for a in ("freq", "presence", "repeat"))
        y[ids] = torch.where(y[ids] > 0, y[ids] / rep, y[ids] * rep) - f * count.double() - p
        if st["bias"] is not None:
            y.index_add_(0, st["bias_id"][r].long(), st["bias"][r].double())
        t = torch.arange(y.numel(), device="cuda")
        y[((st["allow"][r].long()[t // 32] >> (t % 32)) & 1) == 0] = -math.inf
        out.append(y)
    return torch.stack(out)


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "attn":
        return _exact_attn(st)
    if case["op"] == "rules":
        return _exact_rules(st)
    if case["op"] == "rope":
        out = {}
        for name in ("q", "k"):
            x, n = st[name].double(), case["n_rot"]
            y = x.clone()
            first = list(range(0, n, 2)) if case["layout"] == "interleaved" else list(range(n // 2))
            other = [i + 1 for i in first] if case["layout"] == "interleaved" else [i + n // 2 for i in first]
            angle = st["pos"].double()[:, None, None] * (st["turns"] * (2 * math.pi))
            z = torch.polar(torch.full_like(angle, st["gain"]), angle) * torch.complex(x[..., first], x[..., other])
            y[..., first], y[..., other] = z.real, z.imag
            out[name] = y
        return out
    if case["op"] == "kv":
        return {name: _stored64(st["new_" + name], case["kv_type"]) for name in ("k", "v")}
    start, out = st["start"].tolist(), {"k": [], "v": []}
    for s, n in enumerate(st["n_keep"].tolist()):
        rows = st["path"][s, :n].long() + start[s]
        for name in ("k", "v"):
            out[name].append(_stored64(st["new_" + name][rows], case["kv_type"]))
    return {name: torch.cat(rows) for name, rows in out.items()}
