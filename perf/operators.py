"""The paged KV cache whose rows share a prefix: what its operators are measured on.

A server that decodes many rows at once keeps each row's K and V in pages of
a pool (one layer of the cache layout cut into pages of 32 positions and
multiples) and holds the prompt that all rows have in common once. Per step:

  tables      page_tables: from the rows' lengths, on the GPU, the pages each
              row takes from the free stack, the packed chunk's row offsets
              and every new token's row, position and slot
  append      page_append: the new tokens' K and V into their slots
  attention   paged_attention: the chunk's queries against the shared prefix,
              computed once for all rows, and each row's own pages

A case's lengths follow from its `mix` alone, so that its work is known
without its inputs. The model shapes are the repository's own (6, 12 or 12/4
heads of 128, windows of 1024) and generic ones (heads of 64, one KV head).
"""

import math

import numpy as np
import torch

own = False  # False: the plain forms; True: the framework's operators

_DT = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ---------------------------------------------------------------- the cases
def _tables(name, **kw):
    return dict(name=name, kind="tables", **kw)


def _append(name, **kw):
    return dict(name=name, kind="append", **kw)


def _attention(name, **kw):
    return dict(name=name, kind="attention", **kw)


def listed():
    return [
        # a decode step's bookkeeping: one token for each of 64 rows, a few
        # rows ending (the smallest call: latency alone)
        _tables("tables_decode_64", batch=64, q=1, page=64, ctx_lo=0, ctx_hi=2000, prefix=1000, ends=3, pool=1.0,
                mix=1),
        # verify chunks (6 drafts and 1 pending token) of many rows, with a pool that runs short
        _tables("tables_verify_1000", batch=1000, q=7, page=32, ctx_lo=0, ctx_hi=4000, prefix=0, ends=40, pool=0.5,
                mix=2),
        # admission of a batch of prompts of unequal length
        _tables("tables_prompts_200", batch=200, q=700, page=128, ctx_lo=0, ctx_hi=1, prefix=6144, ends=0, pool=1.0,
                mix=3),
        # K and V of a verify chunk of 64 rows, cut out of the fused projection
        _append("append_verify_64", tokens=448, run=7, heads=12, kv=12, hd=128, page=64, src="fp32", dtype="bf16",
                mix=4),
        # K and V of prompt chunks: runs of up to a few hundred positions
        _append("append_prompts", tokens=16000, run=500, heads=12, kv=4, hd=128, page=128, src="bf16", dtype="bf16",
                mix=5),
        # one conversation's decode step, no prefix (latency again)
        _attention("attention_one_row", batch=1, q=1, heads=6, kv=6, hd=128, prefix=0, ctx_lo=640, ctx_hi=641,
                   page=64, window=0, ragged=False, dtype="bf16", mix=6),
        # sampling 64 continuations of one prompt (a length that ends inside a page)
        _attention("attention_samples_64", batch=64, q=1, heads=12, kv=12, hd=128, prefix=5000, ctx_lo=1, ctx_hi=600,
                   page=64, window=0, ragged=False, dtype="bf16", mix=7),
        # the verify chunk of a large batch behind a long system prompt, 12 query heads on 4 KV heads
        _attention("attention_verify_gqa", batch=128, q=9, heads=12, kv=4, hd=128, prefix=6144, ctx_lo=50,
                   ctx_hi=2000, page=128, window=0, ragged=True, dtype="bf16", mix=8),
        # prompt chunks behind the shared prompt, rows of unequal length, some without a token
        _attention("attention_prompts", batch=16, q=512, heads=12, kv=12, hd=128, prefix=4001, ctx_lo=0, ctx_hi=700,
                   page=64, window=0, ragged=True, dtype="bf16", mix=9),
        # a sliding-window layer: the window reaches back into the prefix for some rows and not for others
        _attention("attention_window_hd64", batch=48, q=5, heads=24, kv=8, hd=64, prefix=1500, ctx_lo=1,
                   ctx_hi=1800, page=32, window=1024, ragged=True, dtype="bf16", mix=10),
        # long contexts without a prefix: a pool of more than 2^31 elements
        _attention("attention_long", batch=17, q=1, heads=32, kv=8, hd=128, prefix=0, ctx_lo=98000, ctx_hi=131000,
                   page=256, window=0, ragged=False, dtype="bf16", mix=11),
        # the fp32 mode that a port is checked with
        _attention("attention_fp32", batch=8, q=5, heads=6, kv=6, hd=128, prefix=1000, ctx_lo=1, ctx_hi=900, page=32,
                   window=0, ragged=True, dtype="fp32", mix=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tables", "append", "attention", "attention", "attention", "attention"])
    mix = rng.randrange(1 << 20)
    page = rng.choice([32, 64, 64, 96, 128, 256])
    if kind == "tables":
        batch, q = _log(rng, 1, 2000), rng.choice([1, 1, rng.randrange(2, 18), _log(rng, 18, 1000)])
        q = min(q, max(1, 100000 // batch))
        return dict(kind=kind, batch=batch, q=q, page=page, ctx_lo=0, ctx_hi=_log(rng, 1, 8000),
                    prefix=rng.choice([0, _log(rng, 1, 20000)]), ends=rng.randrange(0, batch // 4 + 1),
                    pool=rng.choice([1.0, 1.0, 0.4]), mix=mix)
    if kind == "append":
        heads, kv, hd = rng.choice([(6, 6, 128), (12, 12, 128), (12, 4, 128), (24, 8, 64), (16, 1, 128)])
        src, dtype = rng.choice([("fp32", "bf16"), ("bf16", "bf16"), ("fp32", "fp32")])
        return dict(kind=kind, tokens=_log(rng, 1, 16000 * 4 // max(4, kv)), run=rng.choice([1, 7, _log(rng, 2, 1000)]),
                    heads=heads, kv=kv, hd=hd, page=page, src=src, dtype=dtype, mix=mix)
    while True:
        heads, kv, hd = rng.choice([(6, 6, 128), (12, 12, 128), (12, 4, 128), (12, 4, 128), (24, 8, 64), (8, 1, 128)])
        dtype = rng.choice(["bf16", "bf16", "bf16", "bf16", "bf16", "fp32"])
        q = rng.choice([1, 1, 1, 5, 7, 9, rng.randrange(2, 18), _log(rng, 18, 600)])
        ctx_hi = _log(rng, 1, 12000)
        c = dict(kind=kind, batch=_log(rng, 1, 128), q=q, heads=heads, kv=kv, hd=hd,
                 prefix=rng.choice([0, _log(rng, 1, 16000), _log(rng, 500, 16000)]), ctx_lo=rng.randrange(0, ctx_hi),
                 ctx_hi=ctx_hi, page=page, window=rng.choice([0, 0, 0, 1024, _log(rng, 10, 4000)]),
                 ragged=rng.random() < 0.6, dtype=dtype, mix=mix)
        # fp32 is the mode of small checks; nothing costs more than the largest listed case
        pairs = c["batch"] * q * heads * hd * (c["prefix"] + ctx_hi + q)
        held = c["batch"] * kv * hd * (ctx_hi + q) + kv * hd * c["prefix"]
        if pairs <= (4e10 if dtype == "bf16" else 1e9) and held <= (1e9 if dtype == "bf16" else 1e8):
            return c


# ---------------------------------------------------------------- lengths
def _shape(case):
    """The lengths of a case, from its `mix` alone."""
    rs = np.random.RandomState(case["mix"])
    if case["kind"] == "append":
        n, at = [], 0
        while at < case["tokens"]:
            n.append(min(int(rs.randint(1, case["run"] + 1)), case["tokens"] - at))
            at += n[-1]
        n = np.array(n, np.int64)
        return dict(n=n, ctx=rs.randint(0, 3 * case["page"], len(n)).astype(np.int64))
    B, q = case["batch"], case["q"]
    ctx = rs.randint(case["ctx_lo"], max(case["ctx_hi"], case["ctx_lo"] + 1), B).astype(np.int64)
    if case["kind"] == "tables":
        n = np.full(B, q) if q < 18 else rs.randint(0, q + 1, B)
        n = n.astype(np.int64)
        n[rs.permutation(B)[:case["ends"]]] = -1
        # rows hold the pages of their positions; some kept one more, from a chunk that was rolled back
        return dict(n=n, ctx=ctx, held=_pages(ctx, case["page"]) + (rs.random_sample(B) < 0.1))
    n = rs.randint(0, q + 1, B) if case["ragged"] else np.full(B, q)
    if case["ragged"]:
        n[rs.randint(0, B)] = q
    return dict(n=n.astype(np.int64), ctx=ctx)


def _pages(x, page):
    return -(-x // page)


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


# ---------------------------------------------------------------- prepare
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    rs = np.random.RandomState(seed % (1 << 32))
    up = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(dev)  # noqa: E731
    L, page = _shape(case), case["page"]
    n, ctx, B = L["n"], L["ctx"], len(L["n"])
    if case["kind"] == "tables":
        held = L["held"]
        want = np.maximum(0, _pages(ctx + np.maximum(n, 0), page) - held)
        W = int(max((held + want).max(), 1)) + 2
        spare = int(np.ceil(want.sum() * case["pool"])) + (8 if case["pool"] >= 1 else 0)
        ids = rs.permutation(int(held.sum()) + spare)
        tables = np.full((B, W), -1, np.int64)
        tables[np.arange(W)[None] < held[:, None]] = ids[:int(held.sum())]
        free = np.full(len(ids), -1, np.int64)
        free[:spare] = ids[int(held.sum()):]
        T = int(np.maximum(n, 0).sum()) + 5
        z = lambda k: torch.zeros(k, dtype=torch.int32, device=dev)  # noqa: E731
        return dict(case=case, tables=up(tables), held=up(held), free=up(free), n_free=up([spare]), length=up(ctx),
                    n_new=up(n), row_off=z(B + 1), start=z(B), tok_row=z(T), tok_pos=z(T), slots=z(T))
    kv, hd, dt = case["kv"], case["hd"], _DT[case["dtype"]]
    rnd = lambda *s, dtype=dt: torch.randn(*s, generator=g, device=dev, dtype=dtype)  # noqa: E731
    P = case.get("prefix", 0)
    npre, nrow = int(_pages(P, page)), _pages(ctx + n, page)
    N = npre + int(nrow.sum()) + 3
    ids = rs.permutation(N)
    W = int(max(nrow.max(), 1))
    tables = np.full((B, W), -1, np.int64)
    tables[np.arange(W)[None] < nrow[:, None]] = ids[npre:npre + int(nrow.sum())]
    # whatever earlier requests left in the slots that no row holds is as finite as the rest; keys as the
    # QK norm leaves them (1.2 times unit rows)
    k_pages, v_pages = rnd(N, kv, page, hd).mul_(1.2), rnd(N, kv, page // 32, hd, 32)
    off = np.concatenate([[0], np.cumsum(n)])
    if case["kind"] == "append":
        pos = np.concatenate([np.arange(c, c + m) for c, m in zip(ctx, n)])
        row = np.repeat(np.arange(B), n)
        slots = tables[row, pos // page] * page + pos % page
        slots[rs.random_sample(len(slots)) < 0.02] = -1  # tokens that keep nothing: the padding of a captured chunk
        H = case["heads"]
        qkv = rnd(len(slots), H + 2 * kv, hd, dtype=_DT[case["src"]])
        return dict(case=case, k=qkv[:, H:H + kv], v=qkv[:, H + kv:], slots=up(slots), k_pages=k_pages,
                    v_pages=v_pages)
    T = int(off[-1]) + (3 if case["ragged"] else 0)  # a chunk's capacity may pass its tokens
    q = rnd(T, case["heads"], hd).mul_(1.2)
    return dict(case=case, q=q, k_pages=k_pages, v_pages=v_pages, tables=up(tables), row_off=up(off),
                start=up(P + ctx), prefix_pages=up(ids[:npre]), max_per_row=int(max(n.max(), 1)))


# ---------------------------------------------------------------- run
def run(state):
    case = state["case"]
    if own:
        import flaxchat_amd.torch_ops  # noqa: F401  (registers torch.ops.flaxchat_mi355x)
        ops = torch.ops.flaxchat_mi355x
        s = state
        if case["kind"] == "tables":
            ops.page_tables(s["tables"], s["held"], s["free"], s["n_free"], s["length"], s["n_new"], s["row_off"],
                            s["start"], s["tok_row"], s["tok_pos"], s["slots"], case["page"], case["prefix"])
            return [s[k] for k in _TABLE_OUT]
        if case["kind"] == "append":
            ops.page_append(s["k"], s["v"], s["slots"], s["k_pages"], s["v_pages"])
            return [s["k_pages"], s["v_pages"]]
        return ops.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["tables"], s["row_off"], s["start"],
                                   s["max_per_row"], case["window"], s["prefix_pages"], case["prefix"])
    return {"tables": _plain_tables, "append": _plain_append, "attention": _plain_attention}[case["kind"]](state)


_TABLE_OUT = ("tables", "held", "free", "n_free", "row_off", "start", "tok_row", "tok_pos", "slots")


def _plain_tables(s):
    case = s["case"]
    page, prefix = case["page"], case["prefix"]
    tables, free = s["tables"], s["free"]
    B, W = tables.shape
    T, F = s["slots"].numel(), free.numel()
    held, n, length, n_free = (s[k].long() for k in ("held", "n_new", "length", "n_free"))
    # rows that end (n < 0) give their pages back, in row order on top of the stack
    gives = torch.where(n < 0, held, 0)
    give_at = n_free + gives.cumsum(0) - gives
    col = torch.arange(W, device=tables.device)
    into = torch.where(col < gives[:, None], give_at[:, None] + col, F)
    stack = torch.cat([free, free.new_zeros(1)])
    stack[into] = torch.where(into < F, tables, 0)
    avail = n_free + gives.sum()
    # rows that ask: their pages have to fit the stack, their tokens the chunk
    asks = (n > 0) & (length >= 0) & (length + n <= W * page) & ((length + page - 1) // page <= held) & (held <= W)
    need = torch.where(asks, ((length + n + page - 1) // page - held).clamp(min=0), 0)
    fits = asks & ((need == 0) | (need.cumsum(0) <= avail))
    n_fit = torch.where(fits, n, 0)
    takes = fits & (n_fit.cumsum(0) <= T)
    n_in, need_in = torch.where(takes, n, 0), torch.where(takes, need, 0)
    row_off = torch.cat([n.new_zeros(1), n_in.cumsum(0)])
    # new pages, from the top of the stack down
    j = col - held[:, None]
    new = (j >= 0) & (j < need_in[:, None])
    at = avail - 1 - (need_in.cumsum(0) - need_in)[:, None] - j
    tables_new = torch.where(new, stack[torch.where(new, at, 0)], tables)
    length = torch.where(n < 0, 0, length)
    # every token's row, position and slot
    t = torch.arange(T, device=tables.device)
    row = torch.searchsorted(row_off[1:], t, right=True).clamp(max=B - 1)
    real = t < row_off[-1]
    at = length[row] + t - row_off[row]
    slot = tables_new[row, (at // page).clamp(0, W - 1)].long() * page + at % page
    s["tables"].copy_(tables_new)
    s["held"].copy_(torch.where(n < 0, 0, held + need_in))
    s["free"].copy_(stack[:F])
    s["n_free"].copy_(avail - need_in.sum())
    s["row_off"].copy_(row_off)
    s["start"].copy_(prefix + length)
    s["tok_row"].copy_(torch.where(real, row, -1))
    s["tok_pos"].copy_(torch.where(real, prefix + at, -1))
    s["slots"].copy_(torch.where(real, slot, -1))
    return [s[k] for k in _TABLE_OUT]


def _plain_append(s):
    k, v, kp, vp = s["k"], s["v"], s["k_pages"], s["v_pages"]
    N, G, page, hd = kp.shape
    slot = s["slots"].long()
    keep = (slot >= 0) & (slot < N * page)
    # tokens that keep nothing write their slot's own value back: of slot 0 of a row of spare elements
    base = torch.where(keep, slot // page, N)[:, None, None] * (G * page * hd)
    at = torch.where(keep, slot % page, 0)[:, None, None]
    g, d = torch.arange(G, device=k.device)[:, None], torch.arange(hd, device=k.device)
    blk, p = at // 32, at % 32
    if _fragment(kp.dtype, hd):
        inner = ((((d // 32 * 2 + p // 4 % 2) * 4 + d // 8 % 4) * 4 + p // 8) * 4 + p % 4) * 8 + d % 8
    else:
        inner = p * hd + d
    k_at = base + (g * (page // 32) + blk) * (32 * hd) + inner
    v_at = base + (g * (page // 32) + blk) * (32 * hd) + d * 32 + p
    for pages, x, at in ((kp, k, k_at), (vp, v, v_at)):
        flat = torch.cat([pages.view(-1), pages.new_zeros(G * page * hd)])
        flat[at] = x.float().to(pages.dtype)
        pages.copy_(flat[:pages.numel()].view_as(pages))
    return [kp, vp]


def _plain_attention(s):
    case = s["case"]
    q, row_off, start, n = s["q"].float(), s["row_off"].long(), s["start"].long(), s["max_per_row"]
    kp, vp, tables = s["k_pages"], s["v_pages"], s["tables"].long()
    T, H, hd = q.shape
    N, G, page, _ = kp.shape
    (B, W), P, window, rep = tables.shape, case["prefix"], case["window"], H // G
    # each row's queries side by side, [B][G][n rep][hd]
    i = torch.arange(n, device=q.device)
    tok = torch.where(i < (row_off[1:] - row_off[:-1])[:, None], row_off[:-1, None] + i, T)
    qr = torch.cat([q, q.new_zeros(1, H, hd)])[tok].view(B, n, G, rep, hd).transpose(1, 2).reshape(B, G, n * rep, hd)
    pos = (start[:, None] + i).view(B, 1, n, 1).expand(B, G, n, rep).reshape(B, G, n * rep, 1)
    scale = 1 / math.sqrt(hd)

    def scores(qs, k, key, there):
        x = torch.matmul(qs, k.transpose(-1, -2)) * scale
        ok = there & (key <= pos) & ((pos - key <= window) if window > 0 else True)
        return x.view(B, G, n * rep, -1) if qs.dim() == 4 else \
            x.view(G, B, n * rep, -1).transpose(0, 1), ok

    def rows(pages, ids):  # [.., W] page ids -> [.., G][W page][hd]
        x = pages[ids.clamp(0, N - 1)].float()
        return x.transpose(-4, -3).reshape(*ids.shape[:-1], G, ids.shape[-1] * page, hd)

    kr, vr = _k_rows(kp), _v_rows(vp)
    key = P + torch.arange(W * page, device=q.device)
    there = (tables >= 0).repeat_interleave(page, 1)[:, None, None]
    x, ok = scores(qr, rows(kr, tables), key, there)
    x = x.masked_fill(~ok, -math.inf)
    mx = x.amax(-1, keepdim=True)
    if P > 0:
        pre = s["prefix_pages"].long()
        key = torch.arange(P, device=q.device)
        qa = qr.transpose(0, 1).reshape(G, B * n * rep, hd)
        xp, okp = scores(qa, rows(kr, pre)[:, :P], key, torch.ones(1, device=q.device, dtype=torch.bool))
        xp = xp.masked_fill(~okp, -math.inf)
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
    return y[:T].reshape(T, H * hd).to(s["q"].dtype)


# ---------------------------------------------------------------- work
def work(case):
    L, page = _shape(case), case["page"]
    n, ctx, B = L["n"], L["ctx"], len(L["n"])
    if case["kind"] == "tables":
        tokens = int(np.maximum(n, 0).sum())
        pages = int((_pages(ctx + n, page) - ctx // page)[n > 0].sum())
        # lengths, additions and pages held of each row; its offset, position and pages held after; its tokens'
        # row, position and slot; the table entries that the tokens lie in
        return dict(bytes=4 * (6 * B + 3 * tokens + pages), flops=0)
    kv, hd, es = case["kv"], case["hd"], 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "append":
        each = case["tokens"] * kv * hd
        return dict(bytes=2 * each * ((2 if case["src"] == "bf16" else 4) + es) + 4 * case["tokens"], flops=0)
    H, P, window = case["heads"], case["prefix"], case["window"]
    pairs, keys, pre_lo = 0, 0, P
    for c, m in zip(ctx.tolist(), n.tolist()):
        if m == 0:
            continue
        pos = P + c + np.arange(m)
        lo = np.maximum(0, pos - window) if window > 0 else np.zeros(m, np.int64)
        pairs += int((pos - lo + 1).sum())
        keys += int(pos[-1] + 1 - max(P, lo[0]))  # the row's own keys that some query sees
        pre_lo = min(pre_lo, int(lo[0]))
    keys += P - pre_lo  # the prefix, once
    return dict(bytes=2 * keys * kv * hd * es + 2 * int(n.sum()) * H * hd * es, flops=4 * pairs * H * hd)


# ---------------------------------------------------------------- exact
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "tables":
        return _exact_tables(case, s)
    if case["kind"] == "append":
        return _exact_append(case, s)
    return _exact_attention(case, s)


def _exact_tables(case, s):
    """Row by row on the host: the free stack as a list."""
    page, prefix = case["page"], case["prefix"]
    h = {k: v.cpu().numpy().astype(np.int64) for k, v in s.items() if torch.is_tensor(v)}
    T, (B, W) = len(h["slots"]), h["tables"].shape
    n_free, free = int(h["n_free"][0]), h["free"].tolist()
    stack = free[:n_free]
    for b in range(B):
        if h["n_new"][b] < 0:
            stack += h["tables"][b, :h["held"][b]].tolist()
    free[:len(stack)] = stack
    avail, asked, used, off = len(stack), 0, 0, [0]
    tok = dict(tok_row=[], tok_pos=[], slots=[])
    start, full = [], False
    for b in range(B):
        n, c, held = int(h["n_new"][b]), int(h["length"][b]), int(h["held"][b])
        start.append(prefix + (0 if n < 0 else c))
        took = 0
        if n < 0:
            h["held"][b] = 0
        elif n > 0 and c + n <= W * page and -(-c // page) <= held <= W:
            need = max(0, -(-(c + n) // page) - held)
            asked += need
            if need == 0 or asked <= avail:
                full = full or used + n > T
                if not full:
                    for j in range(need):
                        h["tables"][b, held + j] = stack.pop()
                    h["held"][b] += need
                    took = n
                    used += n
                    for p in range(c, c + n):
                        tok["tok_row"].append(b)
                        tok["tok_pos"].append(prefix + p)
                        tok["slots"].append(int(h["tables"][b, p // page]) * page + p % page)
        off.append(off[-1] + took)
    pad = lambda v: np.array(v + [-1] * (T - len(v)), np.int64)  # noqa: E731
    out = dict(tables=h["tables"], held=h["held"], free=np.array(free), n_free=np.array([len(stack)]),
               row_off=np.array(off), start=np.array(start), **{k: pad(v) for k, v in tok.items()})
    return [torch.from_numpy(np.ascontiguousarray(out[k])).to(torch.int32) for k in _TABLE_OUT]


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


def _exact_append(case, s):
    slot, page, dev = s["slots"].long(), case["page"], s["slots"].device
    live = slot >= 0
    g, d = torch.arange(case["kv"], device=dev)[None, :, None], torch.arange(case["hd"], device=dev)
    pid, p = (slot // page)[live][:, None, None], (slot % page)[live][:, None, None]
    out = []
    for pages, x, transposed in ((s["k_pages"], s["k"], False), (s["v_pages"], s["v"], True)):
        o = pages.double().flatten()
        o[_element(case, pid, g, p, d, transposed).flatten()] = x[live].double().flatten()
        out.append(o.view_as(pages))
    return out


def _exact_attention(case, s):
    """Row by row in 64 bits, every key by its flat element."""
    L, page, P, window = _shape(case), case["page"], case["prefix"], case["window"]
    H, kv, hd, dev = case["heads"], case["kv"], case["hd"], s["q"].device
    kf, vf = s["k_pages"].view(-1), s["v_pages"].view(-1)
    y = torch.zeros(s["q"].shape[0], H, hd, dtype=torch.float64, device=dev)
    g, d = torch.arange(kv, device=dev)[:, None, None], torch.arange(hd, device=dev)
    at = 0
    for b, (c, m) in enumerate(zip(L["ctx"].tolist(), L["n"].tolist())):
        if m == 0:
            continue
        pos = P + c + torch.arange(m, device=dev)
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
        gone = key[None] > pos[:, None]
        if window > 0:
            gone = gone | (pos[:, None] - key[None] > window)
        x = x.masked_fill(gone.repeat_interleave(H // kv, 0), -math.inf)
        o = torch.softmax(x, -1) @ v
        y[at:at + m] = o.view(kv, m, H // kv, hd).transpose(0, 1).reshape(m, H, hd)
        at += m
    return y.view(-1, H * hd)
