"""Decoding with trees of drafted tokens over the paged KV cache: what its operators are measured on.

A row's chunk is a tree (or a forest): node i continues its parent, an earlier
node of the row, and sits in the cache at start + i whatever its depth. A step
of a server that drafts trees, behind page_tables:

  tables      tree_tables: from the parents, the set of each node's ancestors
              as bits and its position, start + depth
  rope        rope_append: the rotation of q and k at those positions, the QK
              norm, and K and V into their slots (a layer)
  attention   tree_attention: each node against what its row holds, the shared
              prefix and its own ancestors (a layer)
  accept      tree_accept: the longest path on which the target's choices
              follow the drafted tokens
  commit      tree_commit: that path's K and V moved to the front of the row's
              chunk, in all layers

A case's lengths and trees follow from its `mix` alone, so that its work is
known without its inputs. Model shapes are the repository's own (6, 12 or 12/4
heads of 128) and generic ones (heads of 64, one KV head).
"""

import math

import numpy as np
import torch

own = False  # False: the plain forms; True: the framework's operators

_DT = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ---------------------------------------------------------------- the cases
def _case(kind, name, **kw):
    return dict(name=name, kind=kind, **kw)


def listed():
    return [
        # a step's bookkeeping for the trees of 64 rows (the smallest call: latency alone)
        _case("tables", "tables_64_rows", batch=64, nodes=64, spread=8, ragged=False, mix=1),
        # a large batch, trees of more nodes than a word of the mask has bits, chains among the rows
        _case("tables", "tables_500_rows", batch=500, nodes=300, spread=20, ragged=True, mix=2),
        # small trees of a few rows, cut out of the fused fp32 projection, with the QK norm (latency again)
        _case("rope", "rope_small_trees", tokens=128, run=8, spread=3, heads=12, kv=12, hd=128, rot=128, page=64,
              interleaved=False, norm=1.2, span=2000, stretch=1.0, src="fp32", dtype="bf16", mix=3),
        # prompts far into a long context, half of each head rotated, adjacent pairs, stretched positions
        _case("rope", "rope_prompts", tokens=16000, run=500, spread=1, heads=12, kv=4, hd=128, rot=64, page=128,
              interleaved=True, norm=0.0, span=130000, stretch=4.0, src="bf16", dtype="bf16", mix=4),
        # one conversation's tree (latency)
        _case("attention", "attention_one_row", batch=1, nodes=16, spread=4, ragged=False, heads=6, kv=6, hd=128,
              prefix=0, ctx_lo=640, ctx_hi=641, page=64, window=0, dtype="bf16", mix=5),
        # full trees of 64 nodes for a batch in the middle of its answers
        _case("attention", "attention_trees_64", batch=32, nodes=64, spread=8, ragged=False, heads=12, kv=12, hd=128,
              prefix=0, ctx_lo=1024, ctx_hi=1536, page=64, window=0, dtype="bf16", mix=6),
        # trees of unequal size for a large batch behind a long system prompt, 12 query heads on 4 KV heads
        _case("attention", "attention_prefix_gqa", batch=128, nodes=25, spread=6, ragged=True, heads=12, kv=4, hd=128,
              prefix=6144, ctx_lo=50, ctx_hi=2000, page=128, window=0, dtype="bf16", mix=7),
        # the fp32 mode that a port is checked with, a sliding-window layer with heads of 64
        _case("attention", "attention_window_fp32", batch=8, nodes=12, spread=3, ragged=True, heads=12, kv=4, hd=64,
              prefix=700, ctx_lo=1, ctx_hi=1500, page=32, window=1024, dtype="fp32", mix=8),
        # the decision of a step: the target's choices against the drafted tokens
        _case("accept", "accept_64_rows", batch=64, nodes=64, spread=8, ragged=False, mix=9),
        _case("accept", "accept_500_rows", batch=500, nodes=300, spread=20, ragged=True, mix=10),
        # accepted paths of 32 rows in one layer, and of 64 rows in all 24 layers of a GQA model's pool
        _case("commit", "commit_layer", layers=1, batch=32, nodes=16, spread=4, ragged=True, kv=12, hd=128, page=64,
              dtype="bf16", mix=11),
        _case("commit", "commit_all_layers", layers=24, batch=64, nodes=64, spread=8, ragged=False, kv=4, hd=128,
              page=64, dtype="bf16", mix=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tables", "rope", "rope", "attention", "attention", "attention", "attention", "accept", "commit"])
    mix = rng.randrange(1 << 20)
    page = rng.choice([32, 64, 64, 96, 128, 256])
    nodes = rng.choice([rng.randrange(1, 17), rng.randrange(17, 65), _log(rng, 65, 300)])
    spread = rng.choice([1, rng.randrange(2, 9), _log(rng, 9, 100)])  # 1: chains
    if kind in ("tables", "accept"):
        batch = _log(rng, 1, 2000)
        nodes = max(1, min(nodes, 150000 // batch))
        return dict(kind=kind, batch=batch, nodes=nodes, spread=spread, ragged=rng.random() < 0.6, mix=mix)
    if kind == "rope":
        heads, kv, hd = rng.choice([(6, 6, 128), (12, 12, 128), (12, 4, 128), (24, 8, 64), (16, 1, 128), (10, 2, 96)])
        src, dtype = rng.choice([("fp32", "bf16"), ("bf16", "bf16"), ("fp32", "fp32")])
        run = rng.choice([1, rng.randrange(2, 65), _log(rng, 65, 1000)])
        return dict(kind=kind, tokens=_log(rng, 1, 16000 * 4 // max(4, kv)), run=run, spread=spread, heads=heads,
                    kv=kv, hd=hd, rot=rng.choice([hd, hd, hd // 2, hd // 4, 2 * rng.randrange(1, hd // 2)]),
                    page=page, interleaved=rng.random() < 0.4, norm=rng.choice([0.0, 1.2, 1.0]),
                    span=_log(rng, 1, 130000), stretch=rng.choice([1.0, 1.0, 4.0, 2.5]), src=src, dtype=dtype, mix=mix)
    if kind == "commit":
        kv, hd = rng.choice([(6, 128), (12, 128), (4, 128), (8, 64), (1, 128), (2, 96)])
        layers, batch = _log(rng, 1, 24), _log(rng, 1, 64)
        return dict(kind=kind, layers=layers, batch=batch, nodes=min(nodes, 64 * 64 // batch), spread=spread,
                    ragged=rng.random() < 0.6, kv=kv, hd=hd, page=rng.choice([32, 64, 64]),
                    dtype=rng.choice(["bf16", "bf16", "fp32"]) if layers * kv * hd <= 6144 else "bf16", mix=mix)
    while True:
        heads, kv, hd = rng.choice([(6, 6, 128), (12, 12, 128), (12, 4, 128), (12, 4, 128), (24, 8, 64), (8, 1, 128)])
        dtype = rng.choice(["bf16", "bf16", "bf16", "bf16", "bf16", "fp32"])
        ctx_hi = _log(rng, 1, 12000)
        c = dict(kind=kind, batch=_log(rng, 1, 128), nodes=nodes, spread=spread, ragged=rng.random() < 0.6,
                 heads=heads, kv=kv, hd=hd, prefix=rng.choice([0, 0, _log(rng, 1, 16000), _log(rng, 500, 16000)]),
                 ctx_lo=rng.randrange(0, ctx_hi), ctx_hi=ctx_hi, page=page,
                 window=rng.choice([0, 0, 0, 1024, _log(rng, 10, 4000)]), dtype=dtype, mix=mix)
        # fp32 is the mode of small checks; nothing costs more than the largest listed case
        pairs = c["batch"] * nodes * heads * hd * (c["prefix"] + ctx_hi + nodes)
        held = c["batch"] * kv * hd * (ctx_hi + nodes) + kv * hd * c["prefix"]
        if pairs <= (3e10 if dtype == "bf16" else 1e9) and held <= (4e8 if dtype == "bf16" else 1e8):
            return c
        nodes = rng.choice([rng.randrange(1, 17), rng.randrange(17, 65), _log(rng, 65, 300)])


# ---------------------------------------------------------------- lengths and trees
def _shape(case):
    """A case's rows: nodes, context and parents [batch][most nodes] (-1: a root, or no node), from its `mix` alone."""
    rs = np.random.RandomState(case["mix"])
    if case["kind"] == "rope":
        n, at = [], 0
        while at < case["tokens"]:
            n.append(min(int(rs.randint(1, case["run"] + 1)), case["tokens"] - at))
            at += n[-1]
        n = np.array(n, np.int64)
    else:
        B, m = case["batch"], case["nodes"]
        n = rs.randint(0, m + 1, B) if case["ragged"] else np.full(B, m)
        n[rs.randint(0, B)] = m
        n = n.astype(np.int64)
    B, most = len(n), int(n.max())
    i = np.arange(most)
    back = rs.randint(0, case["spread"], (B, most))
    back[rs.random_sample(B) < 0.1] = 0  # rows that drafted a chain
    parent = np.maximum(i - 1 - back, 0)
    if case["spread"] > 1:
        parent[rs.random_sample((B, most)) < 0.01] = -1  # a second root
    parent[:, :1] = -1
    parent[i[None] >= n[:, None]] = -1
    if case["kind"] == "rope":
        ctx = rs.randint(0, 3 * case["page"], B)
    elif case["kind"] == "attention":
        ctx = rs.randint(case["ctx_lo"], max(case["ctx_hi"], case["ctx_lo"] + 1), B)
    else:
        ctx = rs.randint(0, 2 * case.get("page", 1000), B)
    return dict(n=n, ctx=ctx.astype(np.int64), parent=parent, most=most)


def _ancestors(parent):
    """[batch][n][n] truth values: node j is i itself or above it."""
    B, n = parent.shape
    anc = np.zeros((B, n, n), bool)
    rows = np.arange(B)
    for i in range(n):
        p = parent[:, i]
        anc[:, i] = np.where((p >= 0)[:, None], anc[rows, np.maximum(p, 0)], False)
        anc[:, i, i] = True
    return anc


def _depth(parent):
    d = np.zeros(parent.shape, np.int64)
    rows = np.arange(len(parent))
    for i in range(1, parent.shape[1]):
        p = parent[:, i]
        d[:, i] = np.where(p >= 0, d[rows, np.maximum(p, 0)] + 1, 0)
    return d


def _words(anc):
    """The mask of [..][n] truth values: [..][n / 64, rounded up] words, bit j % 64 of word j / 64."""
    n = anc.shape[-1]
    w = max(1, -(-n // 64))
    bits = np.zeros(anc.shape[:-1] + (64 * w,), np.uint8)
    bits[..., :n] = anc
    return np.packbits(bits, axis=-1, bitorder="little").view(np.int64)


def _pages(x, page):
    return -(-x // page)


def _packed(n):
    """Row and place in it of every token."""
    row = np.repeat(np.arange(len(n)), n)
    off = np.concatenate([[0], np.cumsum(n)])
    return row, np.arange(off[-1]) - off[row], off


# ---------------------------------------------------------------- layouts
# A page of the pool holds [kv head][page / 32 blocks of 32 positions]. V blocks are [hd][32]; K blocks are
# row-major [32][hd], except with bf16 and heads of 128: there position 8 a + 4 c + e and dim 32 s + 8 g + x of a
# block sit at [s][c][g][a][e][x].
def _fragment(dtype, hd):
    return dtype == torch.bfloat16 and hd == 128


def _k_rows(p):
    """K pages [..][kv][page][hd] in positions' order."""
    *lead, page, hd = p.shape
    if not _fragment(p.dtype, hd):
        return p
    x = p.reshape(*lead, page // 32, 4, 2, 4, 4, 4, 8)  # [blk][s][c][g][a][e][x]
    d = len(lead)
    return x.permute(*range(d + 1), d + 4, d + 2, d + 5, d + 1, d + 3, d + 6).reshape(*lead, page, hd)


def _v_rows(p):
    """V pages [..][kv][page / 32][hd][32] in positions' order: [..][kv][page][hd]."""
    *lead, nb, hd, _ = p.shape
    return p.transpose(-1, -2).reshape(*lead, nb * 32, hd)


def _places(kp, slot):
    """Flat elements [..][kv][hd] of K and of V of slots [..] in a pool [n_pages][kv][page][hd]."""
    N, G, page, hd = kp.shape
    base, at = (slot // page)[..., None, None] * (G * page * hd), (slot % page)[..., None, None]
    g, d = torch.arange(G, device=kp.device)[:, None], torch.arange(hd, device=kp.device)
    blk, p = at // 32, at % 32
    k_in = ((((d // 32 * 2 + p // 4 % 2) * 4 + d // 8 % 4) * 4 + p // 8) * 4 + p % 4) * 8 + d % 8 \
        if _fragment(kp.dtype, hd) else p * hd + d
    base = base + (g * (page // 32) + blk) * (32 * hd)
    return base + k_in, base + d * 32 + p


# ---------------------------------------------------------------- prepare
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    rs = np.random.RandomState(seed % (1 << 32))
    up = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(dev)  # noqa: E731
    L, kind = _shape(case), case["kind"]
    n, ctx, B, most = L["n"], L["ctx"], len(L["n"]), L["most"]
    row, place, off = _packed(n)
    tail = 3 if case.get("ragged") else 0  # a chunk's capacity may pass its tokens
    pad = lambda a, v=-1: np.concatenate([a, np.full(tail, v, np.int64)])  # noqa: E731
    s = dict(case=case, row_off=up(off), most=most)
    if kind in ("tables", "accept"):
        s["parent"] = up(pad(L["parent"][row, place]))
        if kind == "tables":
            s["start"] = up(rs.randint(0, 8000, B))
            return s
        vocab = 65536
        target = rs.randint(0, vocab, len(row))
        tokens = rs.randint(0, vocab, len(row))
        p = L["parent"][row, place]
        same = (rs.random_sample(len(row)) < 0.6) & (p >= 0)  # drafted tokens that the target chose as well
        tokens[same] = target[(off[row] + np.maximum(p, 0))[same]]
        s["tokens"], s["target"] = up(pad(tokens, 0)), up(pad(target, 0))
        return s
    kv, hd, dt, page = case["kv"], case["hd"], _DT[case["dtype"]], case["page"]
    rnd = lambda *z, dtype=dt: torch.randn(*z, generator=g, device=dev, dtype=dtype)  # noqa: E731
    P = case.get("prefix", 0)
    npre, nrow = int(_pages(P, page)), _pages(ctx + n, page)
    N = npre + int(nrow.sum()) + 3
    ids = rs.permutation(N)
    W = int(max(nrow.max(), 1))
    tables = np.full((B, W), -1, np.int64)
    tables[np.arange(W)[None] < nrow[:, None]] = ids[npre:npre + int(nrow.sum())]
    pos = ctx[row] + place
    slots = tables[row, pos // page] * page + pos % page
    # whatever earlier requests left in the slots that no row holds is as finite as the rest
    lead = (case["layers"], N) if kind == "commit" else (N,)
    s["k_pages"], s["v_pages"] = rnd(*lead, kv, page, hd).mul_(1.2), rnd(*lead, kv, page // 32, hd, 32)
    if kind == "commit":
        # the path of a node drawn among each row's: what tree_accept gave
        anc = _ancestors(L["parent"])
        best = np.minimum((rs.random_sample(B) * np.maximum(n, 1)).astype(np.int64), np.maximum(n - 1, 0))
        path = np.full(len(row), -1, np.int64)
        for b in range(B):
            if n[b]:
                on = np.flatnonzero(anc[b, best[b]])
                path[off[b]:off[b] + len(on)] = on
        s["path"], s["slots"] = up(pad(path)), up(pad(slots))
        return s
    H = case["heads"]
    if kind == "rope":
        slots[rs.random_sample(len(slots)) < 0.02] = -1  # tokens that keep nothing
        pos = rs.randint(0, case["span"], B)[row] + _depth(L["parent"])[row, place]
        if len(row) > 8:
            pos[-2:], slots[-2:] = -1, -1  # the padding of a captured chunk
        half, length = case["rot"] // 2, case["span"] + most
        freq = 100000.0 ** (-torch.arange(half, device=dev, dtype=torch.float64) / half)
        angle = (torch.arange(length, device=dev, dtype=torch.float64) / case["stretch"])[:, None] * freq
        qkv = rnd(len(slots), H + 2 * kv, hd, dtype=_DT[case["src"]])
        return dict(s, q=qkv[:, :H], k=qkv[:, H:H + kv], v=qkv[:, H + kv:], tok_pos=up(pos), slots=up(slots),
                    cos=angle.cos().float(), sin=angle.sin().float())
    # keys as the QK norm leaves them (1.2 times unit rows)
    anc = _ancestors(L["parent"])
    mask = np.concatenate([_words(anc)[row, place], np.zeros((tail, max(1, -(-most // 64))), np.int64)])
    depth = anc.sum(-1) - 1
    return dict(s, q=rnd(len(row) + tail, H, hd).mul_(1.2), tables=up(tables), start=up(P + ctx),
                mask=torch.from_numpy(mask).to(dev), tok_pos=up(pad(P + ctx[row] + depth[row, place])),
                prefix_pages=up(ids[:npre]))


# ---------------------------------------------------------------- run
def run(state):
    s, case = state, state["case"]
    kind = case["kind"]
    if own:
        import flaxchat_amd.torch_ops  # noqa: F401  (registers torch.ops.flaxchat_mi355x)
        ops = torch.ops.flaxchat_mi355x
        if kind == "tables":
            return ops.tree_tables(s["parent"], s["row_off"], s["start"], s["most"])
        if kind == "accept":
            return ops.tree_accept(s["parent"], s["tokens"], s["target"], s["row_off"], s["most"])
        if kind == "commit":
            ops.tree_commit(s["path"], s["slots"], s["row_off"], s["most"], s["k_pages"], s["v_pages"])
            return [s["k_pages"], s["v_pages"]]
        if kind == "rope":
            q = ops.rope_append(s["q"], s["k"], s["v"], s["tok_pos"], s["slots"], s["cos"], s["sin"], s["k_pages"],
                                s["v_pages"], case["interleaved"], case["norm"])
            return [q, s["k_pages"], s["v_pages"]]
        return ops.tree_attention(s["q"], s["k_pages"], s["v_pages"], s["tables"], s["row_off"], s["start"], s["mask"],
                                  s["tok_pos"], s["most"], case["window"], s["prefix_pages"], case["prefix"])
    return {"tables": _plain_tables, "accept": _plain_accept, "commit": _plain_commit, "rope": _plain_rope,
            "attention": _plain_attention}[kind](s)


def _rows(s, T):
    """[batch][most] token of each row's places, T where it has none."""
    off = s["row_off"].long()
    i = torch.arange(s["most"], device=off.device)
    return torch.where(i < (off[1:] - off[:-1])[:, None], off[:-1, None] + i, T)


def _rounds(n):
    return max(1, (n - 1).bit_length())


def _plain_tables(s):
    T, n = s["parent"].numel(), s["most"]
    dev = s["parent"].device
    tok = _rows(s, T)
    up = torch.cat([s["parent"].long(), tok.new_full((1,), -1)])[tok]
    anc = torch.eye(n, device=dev, dtype=torch.bool).repeat(len(up), 1, 1)
    for _ in range(_rounds(n)):  # what is up to 2^k above
        there, at = up >= 0, up.clamp(min=0)
        anc = anc | (anc.gather(1, at[:, :, None].expand(-1, -1, n)) & there[:, :, None])
        up = torch.where(there, up.gather(1, at), -1)
    w = -(-n // 64)
    bits = torch.cat([anc, anc.new_zeros(len(up), n, 64 * w - n)], -1).view(len(up), n, w, 64).long()
    words = (bits << torch.arange(64, device=dev)).sum(-1)
    pos = s["start"].long()[:, None] + anc.sum(-1) - 1
    mask = words.new_zeros(T + 1, w)
    mask[tok] = words
    out = pos.new_full((T + 1,), -1)
    out[tok] = pos
    return mask[:T].contiguous(), out[:T].to(torch.int32)


def _plain_accept(s):
    T, n = s["parent"].numel(), s["most"]
    dev = s["parent"].device
    tok = _rows(s, T)
    pick = lambda x, v: torch.cat([x.long(), tok.new_full((1,), v)])[tok]  # noqa: E731
    up, real = pick(s["parent"], -1), tok < T
    target = pick(s["target"], -1)
    good = real & ((up < 0) | (pick(s["tokens"], -2) == target.gather(1, up.clamp(min=0))))
    anc = torch.eye(n, device=dev, dtype=torch.bool).repeat(len(up), 1, 1)
    for _ in range(_rounds(n)):
        there, at = up >= 0, up.clamp(min=0)
        good = good & (good.gather(1, at) | ~there)
        anc = anc | (anc.gather(1, at[:, :, None].expand(-1, -1, n)) & there[:, :, None])
        up = torch.where(there, up.gather(1, at), -1)
    count = torch.where(good, anc.sum(-1), 0)
    most = count.amax(1)
    i = torch.arange(n, device=dev)
    best = torch.where((count == most[:, None]) & good, i, n).amin(1)  # the lowest index among equals
    some = best < n
    line = anc[torch.arange(len(up), device=dev), best.clamp(max=n - 1)] & some[:, None]
    at = line.cumsum(1) - 1  # its place on the path
    path = tok.new_full((len(up), n + 1), -1)
    path.scatter_(1, torch.where(line, at, n), i.expand_as(at))
    out = tok.new_full((T + 1,), -1)
    out[tok] = torch.where(real, path[:, :n], -1)
    nxt = torch.where(some, target.gather(1, best.clamp(max=n - 1)[:, None])[:, 0], -1)
    return most.to(torch.int32), nxt.to(torch.int32), out[:T].to(torch.int32)


def _plain_commit(s):
    kp, vp = s["k_pages"], s["v_pages"]
    T = s["path"].numel()
    tok = _rows(s, T)
    path = torch.cat([s["path"].long(), tok.new_full((1,), -1)])[tok]
    slot = torch.cat([s["slots"].long(), tok.new_full((1,), -1)])[tok]
    src = slot.gather(1, path.clamp(min=0))
    moved = (path > torch.arange(s["most"], device=tok.device)) & (src >= 0) & (slot >= 0)
    (ks, vs), (kd, vd) = _places(kp[0], src[moved]), _places(kp[0], slot[moved])
    for pages, a, b in ((kp, ks, kd), (vp, vs, vd)):
        flat = pages.view(len(pages), -1)
        flat[:, b] = flat[:, a]
    return [kp, vp]


def _plain_rope(s):
    case, kp, vp = s["case"], s["k_pages"], s["v_pages"]
    N, G, page, hd = kp.shape
    rot, slot = case["rot"], s["slots"].long()
    pos = s["tok_pos"].long()
    there = ((pos >= 0) & (pos < len(s["cos"])))[:, None, None]
    c, sn = (s[x][pos.clamp(0, len(s["cos"]) - 1)][:, None] for x in ("cos", "sin"))

    def turned(x):
        x = x.float()
        a, b = (x[..., :rot:2], x[..., 1:rot:2]) if case["interleaved"] else (x[..., :rot // 2], x[..., rot // 2:rot])
        y = [a * c + b * sn, b * c - a * sn]
        y = torch.stack(y, -1).flatten(-2) if case["interleaved"] else torch.cat(y, -1)
        y = torch.cat([y, x[..., rot:]], -1)
        if case["norm"] > 0:
            y = y * (case["norm"] / (y.square().mean(-1, keepdim=True) + 1e-6).sqrt())
        return torch.where(there, y, 0)

    # tokens that keep nothing write their slot's own value back: of slot 0 of a page of spare elements
    keep = (slot >= 0) & (slot < N * page) & there[:, 0, 0]
    k_at, v_at = _places(kp, torch.where(keep, slot, N * page))
    for pages, x, at in ((kp, turned(s["k"]), k_at), (vp, s["v"].float(), v_at)):
        flat = torch.cat([pages.view(-1), pages.new_zeros(G * page * hd)])
        flat[at] = x.to(pages.dtype)
        pages.copy_(flat[:pages.numel()].view_as(pages))
    return [turned(s["q"]).to(kp.dtype), kp, vp]


def _plain_attention(s):
    case = s["case"]
    q, start, n = s["q"].float(), s["start"].long(), s["most"]
    kp, vp, tables = s["k_pages"], s["v_pages"], s["tables"].long()
    T, H, hd = q.shape
    N, G, page, _ = kp.shape
    (B, W), P, window, rep = tables.shape, case["prefix"], case["window"], H // G
    # each row's queries side by side, [B][G][n rep][hd]
    tok = _rows(s, T)
    qr = torch.cat([q, q.new_zeros(1, H, hd)])[tok].view(B, n, G, rep, hd).transpose(1, 2).reshape(B, G, n * rep, hd)
    spread = lambda x: x.view(B, 1, n, 1, -1).expand(B, 1, n, rep, x.shape[-1]).reshape(B, 1, n * rep, -1)  # noqa: E731
    pos = spread(torch.cat([s["tok_pos"].long(), tok.new_zeros(1)])[tok][..., None])
    scale = 1 / math.sqrt(hd)

    def rows(pages, ids):  # [.., W] page ids -> [.., G][W page][hd]
        x = pages[ids.clamp(0, N - 1)].float()
        return x.transpose(-4, -3).reshape(*ids.shape[:-1], G, ids.shape[-1] * page, hd)

    kr, vr = _k_rows(kp), _v_rows(vp)
    # what the rows hold: keys before `start`, then the chunk's own nodes by their bits
    key = P + torch.arange(W * page, device=q.device)
    node = key - start[:, None]
    words = torch.cat([s["mask"], s["mask"].new_zeros(1, s["mask"].shape[1])])[tok]
    bits = (words[..., None] >> torch.arange(64, device=q.device) & 1).flatten(-2)
    chunk = (node >= 0) & (node < (tok < T).sum(1)[:, None])
    seen = bits.gather(2, torch.where(chunk, node, 0)[:, None].expand(-1, n, -1)).bool() & chunk[:, None]
    ok = spread(seen)
    held = (node < 0)[:, None, None] & ((pos - key <= window) if window > 0 else True)
    ok = (ok | held) & (tables >= 0).repeat_interleave(page, 1)[:, None, None]
    x = (torch.matmul(qr, rows(kr, tables).transpose(-1, -2)) * scale).masked_fill(~ok, -math.inf)
    mx = x.amax(-1, keepdim=True)
    if P > 0:
        pre = s["prefix_pages"].long()
        key = torch.arange(P, device=q.device)
        qa = qr.transpose(0, 1).reshape(G, B * n * rep, hd)
        xp = torch.matmul(qa, rows(kr, pre)[:, :P].transpose(-1, -2)) * scale
        xp = xp.view(G, B, n * rep, P).transpose(0, 1)
        if window > 0:
            xp = xp.masked_fill(pos - key > window, -math.inf)
        mx = torch.maximum(mx, xp.amax(-1, keepdim=True))
    mx = mx.masked_fill(mx == -math.inf, 0)
    x = (x - mx).exp()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x, rows(vr, tables))
    if P > 0:
        xp = (xp - mx).exp()
        total = total + xp.sum(-1, keepdim=True)
        op = torch.matmul(xp.transpose(0, 1).reshape(G, B * n * rep, P), rows(vr, pre)[:, :P])
        o = o + op.view(G, B, n * rep, hd).transpose(0, 1)
    o = torch.where(total > 0, o / total, 0)
    o = o.view(B, G, n, rep, hd).transpose(1, 2).reshape(B, n, H, hd)
    y = q.new_zeros(T + 1, H, hd)
    y[tok] = o
    y[T] = 0
    return y[:T].reshape(T, H * hd).to(s["q"].dtype)


# ---------------------------------------------------------------- work
def work(case):
    L, kind = _shape(case), case["kind"]
    n, ctx, B = L["n"], L["ctx"], len(L["n"])
    tokens, words = int(n.sum()), max(1, -(-L["most"] // 64))
    if kind == "tables":  # parents; offsets and starts; mask and positions
        return dict(bytes=4 * tokens + 8 * B + tokens * (8 * words + 4), flops=0)
    if kind == "accept":  # parents, tokens, choices; offsets; the path, the count and the next token
        return dict(bytes=12 * tokens + 4 * B + 4 * tokens + 8 * B, flops=0)
    kv, hd, es = case["kv"], case["hd"], 2 if case["dtype"] == "bf16" else 4
    if kind == "commit":
        # a path of the mean node's length, all of whose nodes but the first change places
        moves = int(np.maximum(_depth(L["parent"]) * (np.arange(L["most"]) < n[:, None]), 0).sum(1)[n > 0].dot(
            1 / n[n > 0]))
        return dict(bytes=4 * case["layers"] * moves * kv * hd * es + 8 * tokens, flops=0)
    H = case["heads"]
    if kind == "rope":
        ss = 2 if case["src"] == "bf16" else 4
        return dict(bytes=tokens * ((H + 2 * kv) * hd * (ss + es) + 8 * (case["rot"] // 2) + 8),
                    flops=tokens * (H + kv) * (3 * case["rot"] + (3 * hd if case["norm"] > 0 else 0)))
    P, window = case["prefix"], case["window"]
    anc = _ancestors(L["parent"]).sum(-1)
    pairs, keys, pre_lo = 0, 0, P
    for b, (c, m) in enumerate(zip(ctx.tolist(), n.tolist())):
        if m == 0:
            continue
        pos = P + c + anc[b, :m] - 1
        lo = np.clip(pos - window, 0, P + c) if window > 0 else np.zeros(m, np.int64)
        pairs += int((P + c - lo + anc[b, :m]).sum())
        keys += int(P + c + m - max(P, lo.min()))  # the row's own keys that some node sees
        pre_lo = min(pre_lo, int(lo.min()))
    keys += P - pre_lo  # the prefix, once
    return dict(bytes=2 * keys * kv * hd * es + 2 * tokens * H * hd * es + tokens * (8 * words + 4),
                flops=4 * pairs * H * hd)


# ---------------------------------------------------------------- exact
def exact(case, seed):
    s, L = prepare(case, seed), _shape(case)
    return {"tables": _exact_tables, "accept": _exact_accept, "commit": _exact_commit, "rope": _exact_rope,
            "attention": _exact_attention}[case["kind"]](case, s, L)


def _exact_tables(case, s, L):
    """Node by node on the host: each one's chain walked to its root."""
    T, W = s["parent"].numel(), max(1, -(-L["most"] // 64))
    start, at = s["start"].tolist(), 0
    mask, pos = [[0] * W for _ in range(T)], [-1] * T
    for b, m in enumerate(L["n"].tolist()):
        for i in range(m):
            j, deep = i, 0
            while j >= 0:
                mask[at + i][j // 64] |= 1 << (j % 64)
                j, deep = int(L["parent"][b, j]), deep + 1
            pos[at + i] = start[b] + deep - 1
        at += m
    return (torch.from_numpy(np.array(mask, np.uint64).view(np.int64)), torch.tensor(pos, dtype=torch.int32))


def _exact_accept(case, s, L):
    T, at = s["parent"].numel(), 0
    tokens, target = s["tokens"].tolist(), s["target"].tolist()
    count, nxt, path = [], [], [-1] * T
    for b, m in enumerate(L["n"].tolist()):
        par, lines, best = L["parent"][b], {}, []
        for i in range(m):
            p = int(par[i])
            if p < 0:
                lines[i] = [i]
            elif p in lines and tokens[at + i] == target[at + p]:
                lines[i] = lines[p] + [i]
            if i in lines and len(lines[i]) > len(best):
                best = lines[i]
        count.append(len(best))
        nxt.append(target[at + best[-1]] if best else -1)
        path[at:at + len(best)] = best
        at += m
    return tuple(torch.tensor(x, dtype=torch.int32) for x in (count, nxt, path))


def _element(case, page, g, p, d, transposed):
    """Flat element of (page id, KV head, position in the page, dim) in a pool."""
    size, hd, kv = case["page"], case["hd"], case["kv"]
    at = (page * kv + g) * size * hd + p // 32 * 32 * hd
    w = p % 32
    if transposed:
        return at + d * 32 + w
    if case["dtype"] == "bf16" and hd == 128:
        return at + ((2 * (d // 32) + (w // 4) % 2) * 64 + 4 * (w // 8) + w % 4 + 16 * ((d // 8) % 4)) * 8 + d % 8
    return at + w * hd + d


def _exact_commit(case, s, L):
    """Row by row, all sources of a row read first."""
    page, dev, at = case["page"], s["slots"].device, 0
    path, slots = s["path"].tolist(), s["slots"].tolist()
    src, dst = [], []
    for m in L["n"].tolist():
        for j in range(m):
            if path[at + j] > j:
                src.append(slots[at + path[at + j]])
                dst.append(slots[at + j])
        at += m
    src, dst = (torch.tensor(x, device=dev, dtype=torch.int64)[:, None, None] for x in (src, dst))
    g, d = torch.arange(case["kv"], device=dev)[:, None], torch.arange(case["hd"], device=dev)
    out = []
    for pages, transposed in ((s["k_pages"], False), (s["v_pages"], True)):
        a, b = (_element(case, x // page, g, x % page, d, transposed).flatten() for x in (src, dst))
        o = pages.double()
        for layer in range(len(o)):
            one = o[layer].view(-1)
            one[b] = one[a]
        out.append(o)
    return out


def _exact_rope(case, s, L):
    """By the angle of each pair as a complex number."""
    slot, page, dev, rot = s["slots"].long(), case["page"], s["slots"].device, case["rot"]
    pos = s["tok_pos"].long()
    there = (pos >= 0) & (pos < len(s["cos"]))
    at = torch.where(there, pos, 0)
    turn = torch.complex(s["cos"][at].double(), -s["sin"][at].double())[:, None]
    out = []
    for x in (s["q"], s["k"]):
        y = x.double().clone()
        z = y[..., :rot].unflatten(-1, (-1, 2)) if case["interleaved"] else y[..., :rot].unflatten(-1, (2, -1)).mT
        z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * turn)
        y[..., :rot] = (z if case["interleaved"] else z.mT).flatten(-2)
        if case["norm"] > 0:
            y = y * case["norm"] / torch.sqrt((y * y).sum(-1, keepdim=True) / y.shape[-1] + 1e-6)
        y[~there] = 0
        out.append(y)
    live = (slot >= 0) & there
    g, d = torch.arange(case["kv"], device=dev)[None, :, None], torch.arange(case["hd"], device=dev)
    pid, p = (slot // page)[live][:, None, None], (slot % page)[live][:, None, None]
    res = [out[0]]
    for pages, x, transposed in ((s["k_pages"], out[1], False), (s["v_pages"], s["v"], True)):
        o = pages.double().flatten()
        o[_element(case, pid, g, p, d, transposed).flatten()] = x[live].double().flatten()
        res.append(o.view_as(pages))
    return res


def _exact_attention(case, s, L):
    """Row by row in 64 bits, every key by its flat element; the nodes' visibility from the parents themselves."""
    page, P, window = case["page"], case["prefix"], case["window"]
    H, kv, hd, dev = case["heads"], case["kv"], case["hd"], s["q"].device
    kf, vf = s["k_pages"].view(-1), s["v_pages"].view(-1)
    y = torch.zeros(s["q"].shape[0], H, hd, dtype=torch.float64, device=dev)
    g, d = torch.arange(kv, device=dev)[:, None, None], torch.arange(hd, device=dev)
    at = 0
    for b, (c, m) in enumerate(zip(L["ctx"].tolist(), L["n"].tolist())):
        if m == 0:
            continue
        above = np.zeros((m, m), bool)
        for i in range(m):
            j = i
            while j >= 0:
                above[i, j] = True
                j = int(L["parent"][b, j])
        pos = torch.from_numpy(P + c + above.sum(1) - 1).to(dev)
        first = max(0, P + c - window) if window > 0 else 0
        key = torch.arange(first, P + c + m, device=dev)
        local = torch.where(key < P, key, key - P)
        book = torch.cat([s["prefix_pages"], s["tables"][b]]).long()
        pid = book[torch.where(key < P, 0, len(s["prefix_pages"])) + local // page][:, None]
        p = (local % page)[:, None]
        k = kf[_element(case, pid, g, p, d, False)].double()  # [kv][keys][hd]
        v = vf[_element(case, pid, g, p, d, True)].double()
        q = s["q"][at:at + m].double().view(m, kv, H // kv, hd).permute(1, 0, 2, 3).reshape(kv, -1, hd)
        x = q @ k.mT / math.sqrt(hd)
        gone = torch.zeros(m, len(key), dtype=torch.bool, device=dev)
        if window > 0:
            gone |= pos[:, None] - key[None] > window
        gone[:, len(key) - m:] = torch.from_numpy(~above).to(dev)
        x = x.masked_fill(gone.repeat_interleave(H // kv, 0), -math.inf)
        o = torch.softmax(x, -1) @ v
        y[at:at + m] = o.view(kv, m, H // kv, hd).transpose(0, 1).reshape(m, H, hd)
        at += m
    return y.view(-1, H * hd)
