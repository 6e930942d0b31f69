"""Measured cases of a serving step's operators over the quantised paged cache: page tables and slot maps from the
requests' lengths, attention of a batch whose sequences share a prefix, and tokens drawn from rows of logits.

`run` computes a case either through pocketinfer (`own`) or with elementary torch operations.

Page tables.  Of S slots, slot s holds held[s] pages, pages[s, :held[s]], for its ctx[s] positions and gets new[s] tokens.
First the slots that are done give back pages[s, shared[s]:held[s]], behind the list of free pages; then every other slot
takes, from the list's end, the pages that its ctx + new positions need besides those that it holds.

A shared prefix.  Group g is the sequences first[g] .. first[g + 1] - 1, whose first len[g] positions hold the same K and
V; the first of them says where.

Drawing.  w_t = exp((x_t - max x) / temp).  Tokens in the order of their logits (equal ones: the lower index first); kept
are those with w_t >= min_p, of these the first top_k, of these the shortest run from the first on that has top_p of their
weight.  The token is the first kept one, by index, up to which the kept weights come to more than u times their sum.

The cache's entries (include/pk.h):  q8  value D * (byte - 128), one scale D a row;  q4  value D * s_b * (nibble - 8), D
and the sub-scales s_b of 32 dimensions each in a row's two scale words.
"""
import math
import os
import sys

import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


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
        # a decode step of a few streams: every one grows by a token, some by a page
        {"name": "plan_step", "op": "plan", "seqs": 24, "ctx": 4000, "new": 1, "page": 64, "room": 16384, "turn": 0.0, "scarce": 0},
        # a step of a full server: an eighth of the slots are done, an eighth get prompts, the others a token
        {"name": "plan_turn", "op": "plan", "seqs": 1000, "ctx": 6000, "new": 900, "page": 16, "room": 16384, "turn": 0.25, "scarce": 0},
        # four answers to one prompt, a token each: the smallest batch with a prefix
        {"name": "shared_samples", "op": "attn", **M70, "groups": 1, "per": 4, "shared": 700, "own": 60, "new": 1, "page": 64,
         "kv_type": "q8", "type": "f16", "ragged": 0, "tree": 0},
        # 64 users behind one system prompt
        {"name": "shared_streams", "op": "attn", **M70, "groups": 1, "per": 64, "shared": 4001, "own": 500, "new": 1, "page": 64,
         "kv_type": "q8", "type": "bf16", "ragged": 1, "tree": 0},
        # 33 streams behind a long document, in the engine's own type
        {"name": "shared_document", "op": "attn", **M26, "groups": 1, "per": 33, "shared": 16000, "own": 1200, "new": 1, "page": 256,
         "kv_type": "q8", "type": "f32", "ragged": 1, "tree": 0},
        # eight answers to each of a dozen prompts, three drafts each, 4-bit cache
        {"name": "shared_groups", "op": "attn", **M70, "groups": 12, "per": 8, "shared": 2500, "own": 300, "new": 3, "page": 16,
         "kv_type": "q4", "type": "f16", "ragged": 1, "tree": 1},
        # drafted trees of 100 users behind two system prompts: the most arithmetic
        {"name": "shared_trees", "op": "attn", **M70, "groups": 2, "per": 50, "shared": 24000, "own": 1500, "new": 16, "page": 128,
         "kv_type": "q8", "type": "bf16", "ragged": 0, "tree": 1},
        # one user's row
        {"name": "draw_row", "op": "draw", "rows": 1, "vocab": 73448, "type": "f32", "temp": 0.8, "top_k": 40, "top_p": 0.95, "min_p": 0.05},
        # a decode step of 64 streams, the nucleus only
        {"name": "draw_step", "op": "draw", "rows": 64, "vocab": 73448, "type": "bf16", "temp": 1.0, "top_k": 0, "top_p": 0.9, "min_p": 0.0},
        # drafts of a batch drawn from the whole distribution
        {"name": "draw_all", "op": "draw", "rows": 250, "vocab": 32000, "type": "f16", "temp": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0},
        # a serving batch's rows, each with its own settings, hot ones among them
        {"name": "draw_batch", "op": "draw", "rows": 250, "vocab": 128256, "type": "f32", "temp": 1.5, "top_k": -1, "top_p": -1.0, "min_p": -1.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "attn", "attn", "attn", "draw", "draw"])
    if op == "plan":
        seqs, page = _log(rng, 1, 1000), rng.choice([16, 32, 64, 128, 256])
        return {"op": op, "seqs": seqs, "ctx": _log(rng, 1, 6000), "new": rng.choice([1, _log(rng, 1, 900)]), "page": page, "room": 16384,
                "turn": rng.choice([0.0, 0.25, 0.5]), "scarce": rng.randint(0, 1)}
    if op == "draw":
        pick = lambda *v: rng.choice(v)  # noqa: E731
        return {"op": op, "rows": _log(rng, 1, 250), "vocab": _log(rng, 1000, 128256), "type": rng.choice(list(DT)), "temp": pick(0.5, 0.8, 1.0, 1.5),
                "top_k": pick(0, -1, _log(rng, 1, 500)), "top_p": pick(1.0, -1.0, 0.9, 0.99), "min_p": pick(0.0, -1.0, 0.02)}
    heads = rng.choice([M70, M26, {"heads": 4, "kv": 2, "dh": 64}, {"heads": 8, "kv": 8, "dh": 64}, {"heads": 21, "kv": 3, "dh": 128}])
    groups = rng.choice([1, 1, _log(rng, 2, 12)])
    per = _log(rng, 1, 100 // groups)
    seqs, most = groups * per, 200000000 // (heads["kv"] * heads["dh"])  # positions that a cache has at most
    new = rng.choice([1, _log(rng, 1, 16)])
    shared = _log(rng, 16, max(17, min(24000, most // (2 * groups))))
    return {"op": op, **heads, "groups": groups, "per": per, "shared": shared, "own": _log(rng, 1, max(2, min(1500, most // (2 * seqs)))),
            "new": new, "page": rng.choice([16, 32, 64, 128, 256]), "kv_type": rng.choice(["q8", "q4"]), "type": rng.choice(list(DT)),
            "ragged": rng.randint(0, 1), "tree": rng.randint(0, 1)}


def _part(i):
    return (i * 0.6180339887) % 1.0


def _plan_lens(case):
    """(ctx, new, done) of each slot.  Of the share `turn` half are done and half just admitted."""
    ctx, new, done = [], [], []
    for s in range(case["seqs"]):
        f, r = 0.05 + 0.95 * _part(s), (s * 0.7548776662 + 0.5) % 1.0
        c, n, d = int(case["ctx"] * f), 1, 0
        if case["turn"] and r < case["turn"] / 2:
            n, d = 0, 1
        elif r < case["turn"] or (case["new"] > 1 and not case["turn"]):
            c, n = (0 if case["turn"] else c), max(1, int(case["new"] * (1 - f)))
        ctx.append(c)
        new.append(n)
        done.append(d)
    return ctx, new, done


def _attn_lens(case):
    """Positions that each group shares, and ctx and new tokens of each sequence."""
    shared, ctx, new = [], [], []
    for g in range(case["groups"]):
        shared.append(case["shared"] if g == 0 or not case["ragged"] else 1 + int((case["shared"] - 1) * (0.3 + 0.7 * _part(g))))
        for i in range(case["per"]):
            s = g * case["per"] + i
            f = 1.0 if s == 0 or not case["ragged"] else _part(s)
            ctx.append(shared[g] + int(case["own"] * f))
            new.append(case["new"] if s == 0 or not case["ragged"] or case["new"] == 1 else max(1, int(case["new"] * (s * 0.7548776662 % 1.0))))
    return shared, ctx, new


def _starts(n):
    at = [0]
    for x in n:
        at.append(at[-1] + x)
    return at


def work(case):
    if case["op"] == "plan":
        ctx, new, done = _plan_lens(case)
        wide = case["room"] // case["page"]
        cap = _plan_pages(case)[2]
        return {"bytes": 4 * (2 * case["seqs"] * wide + 2 * cap + 8 * case["seqs"]) + 16 * sum(new), "flops": 4 * sum(new)}
    if case["op"] == "draw":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * SIZE[case["type"]] + 32 * case["rows"], "flops": 2 * n}
    shared, ctx, new = _attn_lens(case)
    kv, dh, e = case["kv"], case["dh"], SIZE[case["type"]]
    row = dh + 4 if case["kv_type"] == "q8" else dh // 2 + 8
    seen = sum(shared) + sum(c + n - shared[s // case["per"]] for s, (c, n) in enumerate(zip(ctx, new)))
    each = sum(n * (c + n) for c, n in zip(ctx, new))
    q = 2 * sum(new) * case["heads"] * dh * e
    return {"bytes": 2 * seen * kv * row + q + 8 * sum(new) * case["tree"], "flops": 4 * each * case["heads"] * dh}


# ------------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)


def _normal(g, shape, dtype=torch.float32, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _plan_pages(case):
    """(pages held, of them shared, capacity of the list) of each slot; a quarter of the slots share a page of a prefix."""
    ctx, new, done = _plan_lens(case)
    held = [-(-c // case["page"]) + (s % 5 == 3 and c > 0) for s, c in enumerate(ctx)]  # some kept the page of rejected drafts
    shared = [int(s % 4 == 1 and h > 1) for s, h in enumerate(held)]
    return held, shared, sum(held) + sum(-(-(c + n) // case["page"]) for c, n in zip(ctx, new)) + 7


def _prepare_plan(case, st, g):
    ctx, new, done = _plan_lens(case)
    held, shared, cap = _plan_pages(case)
    wide = case["room"] // case["page"]
    order = torch.randperm(cap, generator=g, device="cuda").to(torch.int32)
    h = _i32(held)
    table = torch.full((case["seqs"], wide), -1, dtype=torch.int32, device="cuda")
    table[torch.arange(wide, device="cuda")[None] < h[:, None]] = order[:sum(held)]
    free = torch.full((cap,), -1, dtype=torch.int32, device="cuda")
    rest = cap - sum(held)
    if case["scarce"]:  # fewer pages than the step asks for
        rest //= 3
    free[:rest] = order[sum(held):sum(held) + rest]
    st.update(ctx=_i32(ctx), new=_i32(new), done=_i32(done), held=h, shared=_i32(shared), pages=table, free=free, n_free=_i32([rest]),
              n_tok=sum(new) + 5)  # some rows of a graph's fixed size stay empty
    return st


def _prepare_draw(case, st, g):
    n, v = case["rows"], case["vocab"]
    st["logits"] = _normal(g, (n, v), std=3.0).to(DT[case["type"]])
    ids = torch.randint(0, v, (n, 1), generator=g, device="cuda") + torch.arange(40, device="cuda") * (v // 40)
    st["logits"].scatter_(1, ids % v, (8.0 + _normal(g, (n, 40), std=3.0)).to(DT[case["type"]]))  # a few likely tokens, as a model's rows have
    st["u"] = torch.rand(n, generator=g, device="cuda")
    one = lambda x: torch.full((n,), x, device="cuda")  # noqa: E731
    rand = torch.rand((4, n), generator=g, device="cuda")
    st["temp"] = one(case["temp"])
    st["top_k"] = st["top_p"] = st["min_p"] = None
    if case["top_k"]:
        st["top_k"] = (torch.where(rand[0] < 0.5, 0.0, 2.0 + 200.0 * rand[0]) if case["top_k"] < 0 else one(case["top_k"])).to(torch.int32)
    if case["top_p"] < 1:
        st["top_p"] = torch.where(rand[1] < 0.4, 1.0, 0.5 + 0.5 * rand[1]) if case["top_p"] < 0 else one(case["top_p"])
    if case["min_p"]:
        st["min_p"] = torch.where(rand[2] < 0.5, 0.0, 0.1 * rand[2]) if case["min_p"] < 0 else one(case["min_p"])
    return st


def _tree_masks(case, seed, new):
    """For every drafted token the bits of its ancestors and itself, for random trees in which a parent comes first."""
    rng = torch.Generator().manual_seed(int(seed) + 5)
    rows = []
    for n in new:
        bits = []
        for i in range(n):
            parent = int(torch.randint(max(0, i - 8), i, (1,), generator=rng)) if i else -1
            bits.append((bits[parent] if parent >= 0 else 0) | (1 << i))
        rows += bits
    return torch.tensor(rows, dtype=torch.int64).reshape(-1, 1).cuda()


def _prepare_attn(case, st, g, seed):
    shared, ctx, new = _attn_lens(case)
    kv, dh, ps, per = case["kv"], case["dh"], case["page"], case["per"]
    # whole pages of a group's prefix are one for all, the rest of it is copied into each sequence's own pages
    need = [-(-(c + n) // ps) for c, n in zip(ctx, new)]
    lead = [shared[s // per] // ps for s in range(len(ctx))]
    n_pages = sum(x // ps for x in shared) + sum(a - b for a, b in zip(need, lead)) + 3
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32).cpu()
    table = torch.full((len(ctx), max(need)), -1, dtype=torch.int32)
    at, copies = 0, []
    for s in range(len(ctx)):
        first = s - s % per
        if s == first:
            table[s, :lead[s]] = order[at:at + lead[s]]
            at += lead[s]
        table[s, :lead[s]] = table[first, :lead[s]]
        table[s, lead[s]:need[s]] = order[at:at + need[s] - lead[s]]
        at += need[s] - lead[s]
        if s != first and shared[s // per] % ps:
            copies.append((int(table[first, lead[s]]), int(table[s, lead[s]]), shared[s // per] % ps))
    row, words = (dh, 1) if case["kv_type"] == "q8" else (dh // 2, 2)
    for name in ("k", "v"):
        # codes as rows of a normal distribution have them, scales a size of their own for each row
        codes, scales = torch.empty((n_pages, kv, ps, row), dtype=torch.uint8, device="cuda"), torch.zeros((n_pages, kv, ps, words), device="cuda")
        step = max(1, (1 << 25) // (kv * ps * dh))
        for p in range(0, n_pages, step):
            m = min(step, n_pages - p)
            x = torch.randn((m, kv, ps, dh), generator=g, device="cuda")
            if name == "k":
                x[..., ::11] *= 2.5
            size = (0.5 + torch.rand((m, kv, ps), generator=g, device="cuda")) if name == "k" else 1.0
            if case["kv_type"] == "q8":
                codes[p:p + m] = (x * 30).round().clamp(-127, 127).add(128).to(torch.uint8)
                scales[p:p + m, ..., 0] = size / 30
            else:
                sub = torch.randint(5, 9, (m, kv, ps, dh // 32), generator=g, device="cuda")
                q = (x.unflatten(-1, (-1, 32)) * (20.0 / sub.unsqueeze(-1))).round().clamp(-8, 7).flatten(-2).add(8).to(torch.uint8)
                codes[p:p + m] = q[..., 0::2] | (q[..., 1::2] << 4)
                scales[p:p + m, ..., 0] = size / 20
                scales[p:p + m, ..., 1] = (sub << (4 * torch.arange(dh // 32, device="cuda"))).sum(-1).to(torch.int32).view(torch.float32)
        for a, b, n in copies:
            codes[b, :, :n], scales[b, :, :n] = codes[a, :, :n], scales[a, :, :n]
        st["c" + name], st["s" + name] = codes, scales
    start = _starts(new)
    st.update(table=table.cuda(), start=_i32(start), ctx=_i32(ctx), first=_i32([per * i for i in range(case["groups"] + 1)]), len=_i32(shared))
    st["q"] = _normal(g, (start[-1], case["heads"], dh), DT[case["type"]])
    st["mask"] = _tree_masks(case, seed, new) if case["tree"] else None
    if own:
        pk = _pk()
        st["cache"] = pk.KvCache(st["ck"], st["cv"], st["sk"], st["sv"], case["kv_type"], dh)
        st["seqs"] = pk.KvSeqs(st["start"], st["ctx"], st["table"], start[-1], max(new), max(c + n for c, n in zip(ctx, new)))
        rows = max(sum(new[i * per:(i + 1) * per]) for i in range(case["groups"]))
        alone = max(c + n - shared[s // per] for s, (c, n) in enumerate(zip(ctx, new)))
        st["shared"] = pk.KvShared(st["first"], st["len"], rows, max(shared), alone)
    return st


def prepare(case, seed):
    g, st = _gen(seed), {"case": case}
    if case["op"] == "plan":
        return _prepare_plan(case, st, g)
    if case["op"] == "draw":
        return _prepare_draw(case, st, g)
    return _prepare_attn(case, st, g, seed)


# ------------------------------------------------------------------ page tables and slot maps

def _run_plan(st):
    ps, n_tok = st["case"]["page"], st["n_tok"]
    if own:
        p = _pk().kv_plan(st["ctx"], st["new"], st["pages"], st["held"], st["free"], st["n_free"], ps, n_tok, done=st["done"],
                          shared=st["shared"])
        return {"start": p.start, "pages": p.pages, "held": p.held, "free": p.free, "n_free": p.n_free, "lacking": p.lacking, "pos": p.pos,
                "seq": p.seq, "slot": p.slot}
    ctx, held, pages, free = st["ctx"].long(), st["held"].long(), st["pages"], st["free"]
    wide, dev, zero = pages.shape[1], pages.device, torch.zeros(1, dtype=torch.int64, device="cuda")
    done = st["done"] != 0
    new = torch.where(done, 0, st["new"].long().clamp(min=0))
    start = torch.cat([zero, new.cumsum(0)]).clamp(max=n_tok)
    new = start[1:] - start[:-1]
    back = torch.where(done, held - st["shared"].long(), 0)
    back_at = torch.cat([zero, back.cumsum(0)])
    take = torch.where(new > 0, ((ctx + new + ps - 1) // ps).clamp(max=wide) - held, 0).clamp(min=0)
    take_at = torch.cat([zero, take.cumsum(0)])
    total = st["n_free"].long() + back_at[-1:]

    def listed_page(i):  # entry i of the list, the pages given back behind the others
        s = torch.searchsorted(back_at[1:], i - st["n_free"], right=True).clamp(max=len(held) - 1)
        j = (st["shared"].long()[s] + i - st["n_free"] - back_at[s]).clamp(0, wide - 1)
        return torch.where(i < st["n_free"], free[i.clamp(0, len(free) - 1)], pages[s, j])

    j = torch.arange(wide, device=dev)[None]
    k = take_at[:-1, None] + j - held[:, None]                        # which page taken entry j of a slot would be
    fresh = (j >= held[:, None]) & (j < (held + take)[:, None])
    got = fresh & (k < total)
    out = torch.where(got, listed_page((total - 1 - k).clamp(min=0)), pages)
    out = torch.where((fresh & ~got) | (done[:, None] & (j < held[:, None])), -1, out)
    had = torch.where(done, 0, held + got.sum(1))
    left = (total - take_at[-1:]).clamp(min=0)
    i = torch.arange(len(free), device=dev)
    list_out = torch.where(i < left, listed_page(i), torch.where(i < st["n_free"], -1, free))
    t = torch.arange(n_tok, device=dev)
    s = torch.searchsorted(start[1:].contiguous(), t, right=True)
    on = s < len(held)
    s = s.clamp(max=len(held) - 1)
    pos = ctx[s] + t - start[s]
    page = out[s, (pos // ps).clamp(0, wide - 1)].long()
    slot = torch.where(on & (pos // ps < had[s]), page * ps + pos % ps, -1)
    i32 = torch.int32
    return {"start": start.to(i32), "pages": out.to(i32), "held": had.to(i32), "free": list_out.to(i32), "n_free": left.to(i32),
            "lacking": (take_at[-1:] - total).clamp(min=0).to(i32), "pos": torch.where(on, pos, 0).to(i32), "seq": torch.where(on, s, -1).to(i32),
            "slot": slot}


def _exact_plan(st):
    ps, n_tok, wide = st["case"]["page"], st["n_tok"], st["pages"].shape[1]
    ctx, new, done, held, shared = (st[n].tolist() for n in ("ctx", "new", "done", "held", "shared"))
    pages, old = st["pages"].cpu().numpy().copy(), st["free"].tolist()
    pool, n_free = old[:st["n_free"].item()], st["n_free"].item()
    for s, d in enumerate(done):
        if d:
            pool += pages[s, shared[s]:held[s]].tolist()
            pages[s, :held[s]] = -1
            held[s] = 0
    start, pos, seq, slot, lacking = [0], [], [], [], 0
    for s in range(len(ctx)):
        n = 0 if done[s] else min(new[s], n_tok - start[-1])
        start.append(start[-1] + n)
        need = min(-(-(ctx[s] + n) // ps), wide) if n > 0 else 0
        for j in range(held[s], need):
            pages[s, j] = pool.pop() if pool else -1
            lacking += pages[s, j] < 0
            held[s] += pages[s, j] >= 0
        for p in range(ctx[s], ctx[s] + n):
            pos.append(p)
            seq.append(s)
            slot.append(int(pages[s, p // ps]) * ps + p % ps if p // ps < held[s] else -1)
    rest = n_tok - len(pos)
    left = len(pool)
    pool += [-1] * max(0, n_free - left)
    pool += old[len(pool):]
    i = lambda x, t=torch.int32: torch.tensor(x, dtype=t, device="cuda")  # noqa: E731
    return {"start": i(start), "pages": torch.from_numpy(pages).cuda(), "held": i([int(h) for h in held]), "free": i(pool[:len(old)]),
            "n_free": i([left]), "lacking": i([int(lacking)]), "pos": i(pos + [0] * rest), "seq": i(seq + [-1] * rest),
            "slot": i(slot + [-1] * rest, torch.int64)}


# ------------------------------------------------------------------ attention over shared prefixes

def _values(codes, scales, kind):
    """The values that codes [..., bytes] with scales [..., 1 or 2] stand for, in 32 bits."""
    if kind == "q8":
        return (codes.float() - 128.0) * scales
    nib = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float() - 8.0
    word = scales[..., 1:].contiguous().view(torch.int32)
    s = (word >> (4 * torch.arange(nib.shape[-1] // 32, device=nib.device, dtype=torch.int32))) & 15
    return (nib.unflatten(-1, (-1, 32)) * s.unsqueeze(-1).float()).flatten(-2) * scales[..., :1]


def _run_attn(st):
    c = st["case"]
    if own:
        return st["cache"].attend(st["seqs"], st["q"], mask=st["mask"], shared=st["shared"])
    shared, ctx, new = _attn_lens(c)
    per, kv, page, kind, dh = c["per"], c["kv"], c["page"], c["kv_type"], c["dh"]
    group, start, q = c["heads"] // kv, _starts(new), st["q"]
    out = torch.empty_like(q)
    for g in range(c["groups"]):
        a, b, n = g * per, (g + 1) * per, new[g * per:(g + 1) * per]
        rows, most = slice(start[a], start[b]), max(n)
        x = q[rows].float().unflatten(1, (kv, group)).permute(1, 0, 2, 3).flatten(1, 2)         # [kv, rows * group, dh]
        t = torch.arange(shared[g], device="cuda")
        pg, sl = st["table"][a, t // page].long(), t % page
        k = _values(st["ck"][pg, :, sl], st["sk"][pg, :, sl], kind)                               # [L, kv, dh]
        w = torch.matmul(x, k.permute(1, 2, 0)) * dh ** -0.5
        m = w.amax(-1, keepdim=True)
        w = torch.exp_(w.sub_(m))
        v = _values(st["cv"][pg, :, sl], st["sv"][pg, :, sl], kind)
        back = lambda y: y.unflatten(1, (-1, group)).permute(1, 0, 2, 3)                          # noqa: E731
        m, total, o = back(m), back(w.sum(-1, keepdim=True)), back(torch.matmul(w, v.transpose(0, 1)))  # [rows, kv, group, ..]
        del w, k, v
        # each sequence's own positions, padded to the longest's
        length = max(y + z - shared[g] for y, z in zip(ctx[a:b], n))
        t = shared[g] + torch.arange(length, device="cuda")
        pg, sl = st["table"][a:b][:, (t // page).clamp(max=st["table"].shape[1] - 1)].long().clamp(min=0), (t % page).expand(per, -1)
        k = _values(st["ck"][pg, :, sl], st["sk"][pg, :, sl], kind)                               # [S, length, kv, dh]
        i, n_t = torch.arange(most, device="cuda"), (st["start"][a + 1:b + 1] - st["start"][a:b])[:, None]
        at = (st["start"][a:b, None] + i).clamp(max=q.shape[0] - 1).long()                       # [S, most]
        w = torch.matmul(q[at].float().unflatten(2, (kv, group)).permute(0, 2, 3, 1, 4).flatten(2, 3), k.permute(0, 2, 3, 1)) * dh ** -0.5
        j = t[None] - st["ctx"][a:b, None]                                                         # the draft that a position holds
        if st["mask"] is None:
            see = j[:, None, :] <= i[None, :, None]
        else:
            see = (j[:, None, :] < 0) | (((st["mask"][at][..., :1] >> j.clamp(0, 63)[:, None, :]) & 1) != 0)
        see = (see & (j < n_t)[:, None, :])[:, None].expand(-1, group, -1, -1).flatten(1, 2)[:, None]
        w = w.masked_fill_(~see, -math.inf)
        top = w.amax(-1, keepdim=True)
        w = torch.exp_(w.sub_(top.masked_fill(top == -math.inf, 0.0)))
        v = _values(st["cv"][pg, :, sl], st["sv"][pg, :, sl], kind)
        on = i[None] < n_t
        back = lambda y: y.unflatten(2, (group, most)).permute(0, 3, 1, 2, 4)[on]                 # noqa: E731
        m2, total2, o2 = back(top), back(w.sum(-1, keepdim=True)), back(torch.matmul(w, v.permute(0, 2, 1, 3)))
        both = torch.maximum(m, m2)
        f, f2 = torch.exp(m - both), torch.exp(m2 - both)
        out[rows] = ((o * f + o2 * f2) / (total * f + total2 * f2)).flatten(1, 2).to(q.dtype)
    return out


def _decoded64(codes, scales, kind):
    if kind == "q8":
        return (codes.double() - 128) * scales.double()
    out = torch.empty(codes.shape[:-1] + (codes.shape[-1] * 2,), dtype=torch.float64, device=codes.device)
    out[..., 0::2], out[..., 1::2] = (codes % 16).double() - 8, (codes // 16).double() - 8
    word = scales[..., 1].contiguous().view(torch.int32)
    for b in range(out.shape[-1] // 32):
        out[..., 32 * b:32 * b + 32] *= (((word >> (4 * b)) & 15).double() * scales[..., 0].double())[..., None]
    return out


def _exact_attn(st):
    """Every sequence by itself, over all its positions."""
    c = st["case"]
    start, ctx, table = st["start"].tolist(), st["ctx"].tolist(), st["table"].cpu()
    group, page = c["heads"] // c["kv"], c["page"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    for s in range(len(ctx)):
        n, total = start[s + 1] - start[s], ctx[s] + start[s + 1] - start[s]
        if n == 0:
            continue
        pages = table[s, :(total + page - 1) // page].long().cuda()
        see = torch.ones((n, total), dtype=torch.bool, device="cuda")
        see[:, ctx[s]:] = torch.ones((n, n), dtype=torch.bool, device="cuda").tril()
        if st["mask"] is not None:
            bits = [int(b) % (1 << 64) for b in st["mask"][start[s]:start[s + 1], 0].tolist()]
            see[:, ctx[s]:] = torch.tensor([[(b >> j) & 1 for j in range(n)] for b in bits], dtype=torch.bool, device="cuda")
        for h in range(c["kv"]):
            k = _decoded64(st["ck"][pages, h].flatten(0, 1)[:total], st["sk"][pages, h].flatten(0, 1)[:total], c["kv_type"])
            v = _decoded64(st["cv"][pages, h].flatten(0, 1)[:total], st["sv"][pages, h].flatten(0, 1)[:total], c["kv_type"])
            q = st["q"][start[s]:start[s + 1], h * group:(h + 1) * group].double()
            w = torch.einsum("ngd,td->ngt", q, k) / math.sqrt(c["dh"])
            w = torch.softmax(torch.where(see[:, None], w, torch.full_like(w, -math.inf)), -1)
            out[start[s]:start[s + 1], h * group:(h + 1) * group] = torch.einsum("ngt,td->ngd", w, v)
    return out


# ------------------------------------------------------------------ tokens drawn from logits

def _run_draw(st):
    if own:
        tok, prob, kept = _pk().sample_rows(st["logits"], st["u"], temp=st["temp"], top_k=st["top_k"], top_p=st["top_p"], min_p=st["min_p"])
        return {"token": tok, "prob": prob, "kept": kept}
    x = st["logits"].double()  # sums over a vocabulary, next to whose borders u may lie: 64 bits
    rows, v = x.shape
    w = torch.exp((x - x.amax(-1, keepdim=True)) / st["temp"].double()[:, None])
    if st["top_k"] is None and st["top_p"] is None and st["min_p"] is None:
        keep = torch.ones_like(w, dtype=torch.bool)
    else:
        order = torch.sort(x, dim=-1, descending=True, stable=True).indices
        y = w.gather(1, order)
        on = torch.ones_like(y, dtype=torch.bool)
        if st["min_p"] is not None:
            on &= y >= st["min_p"].double()[:, None]
        if st["top_k"] is not None:
            k = st["top_k"].long()
            on &= torch.arange(v, device="cuda")[None] < torch.where(k > 0, k, v)[:, None]
        if st["top_p"] is not None:
            y = torch.where(on, y, 0.0)
            before = y.cumsum(-1) - y
            p = st["top_p"].double()[:, None]
            on &= (before < p * y.sum(-1, keepdim=True)) | (p >= 1)
            on[:, 0] = True
        keep = torch.zeros_like(on).scatter_(1, order, on)
    w = torch.where(keep, w, 0.0)
    s = w.cumsum(-1)
    total = s[:, -1:]
    tok = torch.searchsorted(s, st["u"].double()[:, None] * total, right=True).clamp(max=v - 1)
    return {"token": tok[:, 0].to(torch.int32), "prob": (w.gather(1, tok) / total)[:, 0].float(), "kept": keep.sum(-1).to(torch.int32)}


def _exact_draw(st):
    """A row at a time, in numpy's 64 bits on the host."""
    import numpy as np

    out = {"token": [], "prob": [], "kept": []}
    logits, u, temp = st["logits"].double().cpu().numpy(), st["u"].double().tolist(), st["temp"].double().tolist()
    get = lambda n: None if st[n] is None else st[n].double().tolist()  # noqa: E731
    top_k, top_p, min_p = get("top_k"), get("top_p"), get("min_p")
    for r in range(len(logits)):
        w = np.exp((logits[r] - logits[r].max()) / temp[r])
        ids = np.arange(len(w))
        if top_k is not None or top_p is not None or min_p is not None:
            ids = np.argsort(-logits[r], kind="stable")
            if min_p is not None:
                ids = ids[w[ids] >= min_p[r]]
            if top_k is not None and top_k[r] > 0:
                ids = ids[:int(top_k[r])]
            if top_p is not None and top_p[r] < 1:
                cut = int(np.searchsorted(np.cumsum(w[ids]), top_p[r] * math.fsum(w[ids]), side="left")) + 1
                ids = ids[:cut]
            ids = np.sort(ids)
        s = np.cumsum(w[ids])
        at = min(int(np.searchsorted(s, u[r] * s[-1], side="right")), len(ids) - 1)
        out["token"].append(int(ids[at]))
        out["prob"].append(w[ids[at]] / s[-1])
        out["kept"].append(len(ids))
    return {"token": torch.tensor(out["token"], dtype=torch.int32), "prob": torch.tensor(out["prob"], dtype=torch.float64),
            "kept": torch.tensor(out["kept"], dtype=torch.int32)}


def run(state):
    return {"plan": _run_plan, "attn": _run_attn, "draw": _run_draw}[state["case"]["op"]](state)


def exact(case, seed):
    st = prepare(case, seed)
    return {"plan": _exact_plan, "attn": _exact_attn, "draw": _exact_draw}[case["op"]](st)
