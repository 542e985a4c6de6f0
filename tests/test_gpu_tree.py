"""tree_tables, rope_append, tree_attention, tree_accept and tree_commit on the
GPU against 64-bit references (tests/tree_cases.py), at the sizes, trees and
masks where they can go wrong, and a run of them together as a decode loop
uses them."""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import flaxchat_amd.torch_ops  # noqa: E402,F401
from tests.paged_cases import in_pages, rounded  # noqa: E402
from tests.test_gpu_kernels import _say  # noqa: E402
from tests.tree_cases import Tree, accept_plain, moves_plain, packed, rope_plain, tables_plain  # noqa: E402

pytestmark = pytest.mark.gpu
OPS = torch.ops.flaxchat_mi355x
DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
NAN, INF = float("nan"), float("inf")


def dev():
    return torch.device("cuda", 0)


def up(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(dev())


def same(got, want, what=""):
    np.testing.assert_array_equal(got.cpu().numpy(), want, err_msg=what)


# ---------------------------------------------------------------- tree_tables, tree_accept
ROWS = [
    # nodes, kinds, max_per_row (None: the most), tokens behind the last row
    ([1], ["chain"], None, 0),
    ([0, 1, 0], ["chain"], None, 3),
    ([0, 0], ["chain"], 1, 4),
    ([64] * 3, ["chain", "4", "star"], None, 0),
    ([63, 1, 64, 0, 17], ["8", "chain", "roots", "star", "odd"], None, 2),
    ([65, 3, 128, 40], ["chain", "4", "20", "odd"], None, 5),
    ([512, 0, 511, 300], ["chain", "3", "odd", "64"], None, 1),
    ([512], ["star"], None, 0),
    ([7, 20, 9], ["3"], 9, 0),                     # a row of more nodes than max_per_row
    ([70, 200, 130], ["3", "odd"], 130, 2),
    ([3] * 700, ["chain", "2", "odd"], None, 9),
    ([5, 66, 0, 1] * 1024, ["2", "chain", "9"], None, 0),  # 4096 rows
]


@pytest.mark.parametrize("case", range(len(ROWS)))
def test_tables(case):
    ns, kinds, most, tail = ROWS[case]
    _say(f"tree_tables case {case}")
    rng = np.random.default_rng(case)
    off, parent, _ = packed(rng, ns, kinds)
    T, most = int(off[-1]) + tail, most or max(1, max(ns))
    parent = np.concatenate([parent, rng.integers(-1, 9, tail)])
    start = rng.integers(0, 2 ** 31 - 600, len(ns))
    mask, pos = OPS.tree_tables(up(parent), up(off), up(start), most)
    want_mask, want_pos = tables_plain(off, parent, start, T, most)
    same(mask, want_mask.view(np.int64), "mask")
    same(pos, want_pos, "tok_pos")


@pytest.mark.parametrize("agree", [0.0, 0.6, 1.0])
@pytest.mark.parametrize("case", range(len(ROWS)))
def test_accept(case, agree):
    """Equal tokens among siblings (a small vocabulary) and paths of one length: the lowest index is taken."""
    ns, kinds, most, tail = ROWS[case]
    _say(f"tree_accept case {case}, {agree} agree")
    rng = np.random.default_rng(100 + case)
    off, parent, _ = packed(rng, ns, kinds)
    T, most = int(off[-1]) + tail, most or max(1, max(ns))
    parent = np.concatenate([parent, rng.integers(-1, 9, tail)])
    target = rng.integers(0, 5, T)
    tokens = rng.integers(0, 5, T) if agree < 1 else np.zeros(T, np.int64)
    if agree == 0:
        tokens, target = tokens + 7, target - 2 ** 31
    row = np.repeat(np.arange(len(ns)), ns)
    place = np.arange(len(row)) - off[row]
    p = parent[:len(row)]
    ok = (p >= 0) & (p < place) & (rng.random(len(row)) < agree)
    at = np.flatnonzero(ok)
    tokens[at] = target[off[row[at]] + p[at]]
    got = OPS.tree_accept(up(parent), up(tokens), up(target), up(off), most)
    for g, w, what in zip(got, accept_plain(off, parent, tokens, target, T, most), ("n_accepted", "next", "path")):
        same(g, w, what)


def test_rows_past_the_chunk():
    """Row offsets past the chunk's tokens: that row is empty, its tokens are of no row."""
    _say("tree_tables, tree_accept, tree_commit: a row past the chunk")
    off, parent = up([0, 3, 9]), up([-1, 0, 1, -1, 0, 0])
    mask, pos = OPS.tree_tables(parent, off, up([10, 20]), 8)
    assert mask[:, 0].tolist() == [1, 3, 7, 0, 0, 0] and pos.tolist() == [10, 11, 12, -1, -1, -1]
    n, nxt, path = OPS.tree_accept(parent, up([4] * 6), up([4, 4, 5, 4, 4, 4]), off, 8)
    assert n.tolist() == [3, 0] and nxt.tolist() == [5, -1] and path.tolist() == [0, 1, 2, -1, -1, -1]
    k, v = torch.ones(1, 1, 32, 64, device=dev()), torch.ones(1, 1, 1, 64, 32, device=dev())
    k *= torch.arange(32, device=dev())[:, None]
    OPS.tree_commit(up([2, -1, -1, 2, -1, -1]), up([0, 1, 2, 3, 4, 5]), off, 8, k, v)
    assert k[0, 0, :6, 7].tolist() == [2, 1, 2, 3, 4, 5]
    e = up([])
    n, nxt, path = OPS.tree_accept(e, e, e, up([0, 0, 0]), 4)
    assert n.tolist() == [0, 0] and nxt.tolist() == [-1, -1] and path.shape == (0,)
    assert OPS.tree_tables(e, up([0, 0]), up([0]), 65)[0].shape == (0, 2)


# ---------------------------------------------------------------- tree_commit
COMMITS = [
    # KV heads, head_dim, page, layers (0: one layer's tensors), nodes, kinds
    (1, 128, 32, 0, [1, 0, 2], ["star"]),
    (12, 128, 64, 0, [64, 7, 30], ["2", "chain", "8"]),
    (4, 128, 64, 3, [40, 64, 1], ["3", "2"]),
    (2, 64, 96, 2, [9, 50], ["2"]),
    (3, 96, 32, 2, [33, 12], ["2"]),
    (2, 40, 32, 0, [70, 5], ["2"]),
    (1, 256, 64, 0, [100, 31], ["2"]),
    (2, 7, 32, 2, [20], ["2"]),
    (2, 128, 32, 0, [512, 200], ["2", "3"]),  # paths of hundreds of nodes
]


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("order", ["layers", "pages"])
@pytest.mark.parametrize("case", range(len(COMMITS)))
def test_commit(case, dtype, order):
    G, hd, page, layers, ns, kinds = COMMITS[case]
    _say(f"tree_commit {dtype} {COMMITS[case]} {order}")
    rng = np.random.default_rng(case)
    off, parent, par = packed(rng, ns, kinds)
    T, most = int(off[-1]) + 2, max(ns)
    path = np.full(T, -1, np.int64)
    slots = np.full(T, -1, np.int64)
    ctx = rng.integers(0, 2 * page, len(ns))
    per = [-(-int(c + n) // page) for c, n in zip(ctx, ns)]
    N = sum(per) + 2
    ids, at = rng.permutation(N), 0
    for b, n in enumerate(ns):
        pos = np.arange(ctx[b], ctx[b] + n)
        slots[off[b]:off[b] + n] = ids[at:at + per[b]][pos // page] * page + pos % page
        at += per[b]
        if n:
            on, i = [], n - 1 - int(rng.integers(0, min(3, n)))
            while i >= 0:
                on.append(i)
                i = int(par[b][i]) if 0 <= par[b][i] < i else -1
            path[off[b]:off[b] + len(on)] = on[::-1]
    if most > 30:  # slots outside the pool, and entries that are no later node of the row
        slots[off[1] - 2], slots[off[1] - 3] = -1, N * page
        path[off[1] - 5:off[1] - 2] = (2 ** 31 - 1, -2 ** 31, most)
    shape = (max(1, layers), N) if order == "layers" else (N, max(1, layers))
    K, V = (rounded(rng.standard_normal((*shape, G, page, hd)), DT[dtype]) for _ in range(2))
    kp, vp = (t.to(dev()) for t in in_pages(K, V, DT[dtype]))
    if order == "pages":
        kp, vp, K, V = kp.transpose(0, 1), vp.transpose(0, 1), K.swapaxes(0, 1), V.swapaxes(0, 1)
    a = [up(path), up(slots), up(off)]
    if layers:
        OPS.tree_commit(*a, most, kp, vp)
    else:
        OPS.tree_commit(*a, most, kp[0], vp[0])
    torch.cuda.synchronize()
    moves = moves_plain(off, path, slots, N * page, most, T)
    assert moves or max(ns) < 3
    for X in (K, V):
        old = X.copy()
        for s, d in moves:
            X[:, d // page, :, d % page] = old[:, s // page, :, s % page]
    wk, wv = in_pages(np.ascontiguousarray(K), np.ascontiguousarray(V), DT[dtype])
    assert torch.equal(kp.cpu(), wk) and torch.equal(vp.cpu(), wv)


# ---------------------------------------------------------------- rope_append
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("B,layers,G,hd", [(40, 24, 12, 64), (300, 7, 9, 128), (2, 700, 12, 64)])
def test_commit_of_many_heads(B, layers, G, hd, dtype):
    """All layers at once, more KV heads than the launch has workgroups for, and layer by layer: the same."""
    _say(f"tree_commit {dtype}: {B} rows, {layers} layers of {G} heads of {hd}")
    rng = np.random.default_rng(B)
    ns = rng.integers(0, 24, B)
    off, par, _ = packed(rng, ns, ["3", "chain", "star"])
    T, page = int(off[-1]), 32
    N = -(-T // page) + 2
    slots = up(rng.permutation(N * page)[:T])
    _, _, path = OPS.tree_accept(up(par), up(np.zeros(T)), up(np.zeros(T)), up(off), 24)
    k = torch.randn(layers, N, G, page, hd, device=dev()).to(DT[dtype])
    v = torch.randn(layers, N, G, 1, hd, 32, device=dev()).to(DT[dtype])
    k0, v0, k1, v1 = k.clone(), v.clone(), k.clone(), v.clone()
    OPS.tree_commit(path, slots, up(off), 24, k, v)
    for i in range(layers):
        OPS.tree_commit(path, slots, up(off), 24, k1[i], v1[i])
    assert torch.equal(k, k1) and torch.equal(v, v1)
    assert all((k[i] != k0[i]).any() and (v[i] != v0[i]).any() for i in range(layers))


ROPES = [
    # heads, KV heads, head_dim, rot, page, runs, strided
    (1, 1, 128, 128, 32, [1], False),
    (12, 12, 128, 128, 64, [7, 1, 40, 130, 3], True),
    (12, 4, 128, 64, 96, [200, 31, 33, 64], True),
    (6, 2, 128, 32, 64, [8, 24, 9], False),
    (6, 3, 64, 64, 32, [5, 77, 1, 1, 1], True),
    (2, 1, 64, 16, 32, [100], True),
    (3, 1, 128, 128, 32, [300], True),
    (4, 2, 96, 96, 64, [50, 2], False),
    (4, 2, 40, 10, 32, [35, 9], True),
    (2, 1, 256, 256, 128, [129], False),
    (2, 1, 256, 130, 128, [40], True),
    (5, 5, 7, 6, 32, [40, 1], True),
    (3, 1, 128, 2, 32, [33], False),
    (3, 1, 128, 126, 32, [33], True),
    (9, 3, 2, 2, 32, [12], True),
]


@pytest.mark.parametrize("dtype,src", [("bf16", "bf16"), ("bf16", "fp32"), ("fp32", "fp32")])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [0.0, 1.2])
@pytest.mark.parametrize("case", range(len(ROPES)))
def test_rope_append(case, dtype, src, interleaved, norm):
    H, G, hd, rot, page, runs, strided = ROPES[case]
    _say(f"rope_append {src} -> {dtype} {ROPES[case]} interleaved={interleaved} norm={norm}")
    rng = np.random.default_rng(G * hd + rot)
    ctx = rng.integers(0, 2 * page, len(runs))
    M = sum(runs)
    per = [-(-(c + r) // page) for c, r in zip(ctx, runs)]
    N = sum(per) + 2
    ids = rng.permutation(N)
    slots, at = [], 0
    for c, r, p in zip(ctx, runs, per):
        pos = np.arange(c, c + r)
        slots.append(ids[at:at + p][pos // page] * page + pos % page)
        at += p
    slots = np.concatenate(slots)
    slots[rng.random(M) < 0.1] = -1
    length = 5000
    pos = np.sort(rng.integers(0, length, M))
    pos[0] = 0
    if M > 6:
        slots[1], slots[2] = N * page, 2 ** 31 - 1           # outside the pool
        pos[3], pos[4], pos[5], pos[6] = -1, length, 2 ** 31 - 1, length - 1  # outside the tables, but the last
    half = rot // 2
    angle = np.outer(np.arange(length) * 25.0, 100000.0 ** (-np.arange(half) / half))
    cos, sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
    x = rounded(rng.standard_normal((M, H + 2 * G, hd)) * 2, DT[src])
    qkv = torch.from_numpy(x).to(dev(), DT[src])
    q, k, v = qkv[:, :H], qkv[:, H:H + G], qkv[:, H + G:]
    if not strided:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    old = rng.standard_normal((2, N, 2, G, page, hd)).astype(np.float32)
    pools = [in_pages(old[0][:, i], old[1][:, i], DT[dtype]) for i in range(2)]
    kp, vp = (torch.stack([p[j] for p in pools], 1).to(dev()) for j in range(2))
    kl, vl = (kp[:, 1], vp[:, 1]) if strided else (kp[:, 1].contiguous(), vp[:, 1].contiguous())
    got = OPS.rope_append(q, k, v, up(pos), up(slots), torch.from_numpy(cos).to(dev()), torch.from_numpy(sin).to(dev()),
                          kl, vl, interleaved, norm)
    torch.cuda.synchronize()

    def check(g, y, tol, what):
        if dtype == "bf16":  # half a step of the result's rounding: 2^-8 of it
            tol = tol + 2.0 ** -8 * (abs(y) + tol)
        bad = ~(abs(g.astype(np.float64) - y) <= tol)
        assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, first at {np.argwhere(bad)[0]}"

    y, tol = rope_plain(x[:, :H], pos, cos, sin, interleaved, norm)
    check(got.float().cpu().numpy(), y, tol, "q")
    y, tol = rope_plain(x[:, H:H + G], pos, cos, sin, interleaved, norm)
    K, V = (rounded(old[j][:, 1], DT[dtype]).copy() for j in range(2))
    live = [m for m, s in enumerate(slots) if 0 <= s < N * page and 0 <= pos[m] < length]
    # what the kernel wrote, in positions' order: through the layout of a pool of slot numbers
    number = np.arange(N * page, dtype=np.float32).reshape(N, 1, page, 1) + np.zeros((N, G, page, hd), np.float32)
    place = [t.reshape(-1).numpy().astype(np.int64) for t in in_pages(number, number, torch.float32)]
    if dtype == "bf16" and hd == 128:
        from tests.paged_cases import k_blocks
        place[0] = k_blocks(number).reshape(-1).astype(np.int64)
    kept = np.isin(place[0], [slots[m] for m in live])
    flat, was = kl.float().cpu().numpy().reshape(-1), in_pages(K, V, DT[dtype])[0].float().numpy().reshape(-1)
    np.testing.assert_array_equal(flat[~kept], was[~kept], err_msg="K that no token holds")
    wk, wt = np.zeros((2, N, G, page, hd))
    for m in live:
        wk[slots[m] // page, :, slots[m] % page], wt[slots[m] // page, :, slots[m] % page] = y[m], tol[m]
        V[slots[m] // page, :, slots[m] % page] = rounded(x[m, H + G:], DT[dtype])
    if dtype == "bf16" and hd == 128:
        from tests.paged_cases import k_blocks
        wk, wt = k_blocks(wk), k_blocks(wt)
    check(flat[kept], wk.reshape(-1)[kept], wt.reshape(-1)[kept], "K")
    assert torch.equal(vl.cpu(), in_pages(K, V, DT[dtype])[1])
    if strided:  # the other layer is as it was
        assert torch.equal(kp[:, 0].cpu(), pools[0][0]) and torch.equal(vp[:, 0].cpu(), pools[0][1])


@pytest.mark.parametrize("dtype,src", [("bf16", "bf16"), ("bf16", "fp32"), ("fp32", "fp32")])
@pytest.mark.parametrize("M,H,G,hd", [(7000, 10, 5, 128), (10001, 10, 5, 128), (14000, 10, 5, 128), (13999, 20, 10, 64),
                                      (4000, 1, 1, 128)])
def test_rope_append_of_many_tokens(M, H, G, hd, dtype, src):
    """A chunk whose workgroups take several heads each, 2 to 4 of 15 or 30, gives what the same tokens give in calls of
    300, where they take one: a token's arithmetic is the same whoever does it, so the results are equal."""
    _say(f"rope_append {src} -> {dtype}: {M} tokens of {H} and {G} heads of {hd}")
    rng = np.random.default_rng(M)
    page, length = 64, 9000
    N = -(-M // page) + 3
    slots = up(np.where(rng.random(M) < 0.01, -1, rng.permutation(N * page)[:M] if M % 2 else np.arange(M) + 70))
    pos = up(rng.integers(-1, length + 1, M))
    cos, sin = (torch.randn(length, hd // 4, device=dev()) for _ in range(2))
    qkv = torch.randn(M, H + 2 * G, hd, device=dev()).to(DT[src])
    pools = [[torch.zeros(N, G, *z, dtype=DT[dtype], device=dev()) for z in ((page, hd), (page // 32, hd, 32))]
             for _ in range(2)]
    call = lambda a, b, p: OPS.rope_append(qkv[a:b, :H], qkv[a:b, H:H + G], qkv[a:b, H + G:], pos[a:b], slots[a:b],  # noqa: E731
                                           cos, sin, *p, False, 1.2)
    whole = call(0, M, pools[0])
    parts = torch.cat([call(a, min(a + 300, M), pools[1]) for a in range(0, M, 300)])
    assert torch.equal(whole, parts)
    assert torch.equal(pools[0][0], pools[1][0]) and torch.equal(pools[0][1], pools[1][1])
    assert pools[0][0].abs().amax((1, 2, 3)).gt(0).any() and torch.isfinite(whole).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_rope_is_the_prologue(dtype):
    """On this model's own tables rope_append does what attn_prologue does to q and k, value by value in bf16 steps."""
    _say(f"rope_append {dtype}: against attn_prologue")
    import ctypes
    from flaxchat_amd.config import GPTConfig
    from flaxchat_amd.gpt import GPT
    from flaxchat_amd.runtime import DeviceModel
    cfg = GPTConfig(sequence_len=64, vocab_size=512, n_layer=2, n_head=2, n_kv_head=1, n_embd=256,
                    window_pattern="L")
    dm = DeviceModel.from_host(GPT.init_normal(cfg, seed=0, std=0.02), dtype=dtype, device=dev())
    M, H, G, hd, cap, dt = 9, 2, 1, 128, 64, DT[dtype]
    g = torch.Generator(device=dev()).manual_seed(3)
    qkv = torch.randn(M, (H + 2 * G) * hd, device=dev(), generator=g)
    layer = [i for i in range(2) if dm.t["layers"][i].get("ve") is None][0]
    kc, vc = (torch.zeros(2, 1, G, cap, hd, device=dev(), dtype=dt) for _ in range(2))
    h = torch.zeros(16 * 256, device=dev(), dtype=dt)
    pos = up(np.arange(20, 20 + M))
    q = OPS.attn_prologue(ctypes.addressof(dm.desc), layer, kc, vc, qkv, h, up([0] * M), up([0] * M), pos)
    kp, vp = torch.zeros(1, G, cap, hd, device=dev(), dtype=dt), torch.zeros(1, G, 2, hd, 32, device=dev(), dtype=dt)
    x = qkv.view(M, H + 2 * G, hd)
    got = OPS.rope_append(x[:, :H], x[:, H:H + G], x[:, H + G:], pos, pos, dm.t["rope_cos"], dm.t["rope_sin"], kp, vp,
                          False, 1.2)
    # two fp32 evaluations of one formula: each within hd / 2 + 16 half steps (2^-24) of it, and a bf16 step where
    # they round apart
    tol = 2 * (hd / 2 + 16) * 2.0 ** -24 * 4 + (2.0 ** -7 if dtype == "bf16" else 0) * 4
    assert (got.float() - q.float()).abs().max() <= tol
    assert (kp.float().view(-1) - kc[layer].float().view(-1)).abs().max() <= tol
    assert torch.equal(vp.view(-1), vc[layer].view(-1))


# ---------------------------------------------------------------- tree_attention
def _run(c, q, window, a=None, most=None, qt=None, junk=False):
    a = a or c.tree_device(dev(), len(q), junk)
    qt = torch.from_numpy(q).to(dev(), c.dtype) if qt is None else qt
    return OPS.tree_attention(qt, a["k"], a["v"], a["tables"], a["row_off"], a["start"], a["mask"], a["tok_pos"],
                              most or c.most, window, a["pre"] if c.P else None, c.P)


def _check(got, ref, tol, what=""):
    got = got.double().cpu().numpy()
    bad = ~(np.abs(got - ref) <= tol)
    assert not bad.any(), (f"{what}: {bad.sum()} of {bad.size} outputs off, worst {np.nanmax(np.abs(got - ref) / tol)} "
                           f"of the bound, {np.isnan(got).sum()} NaN, first at {np.argwhere(bad)[0]}")


RAGGED = [3, 0, 1, 9, 5]
SHAPES = [
    # ctx, n, prefix, H, G, hd, page, window
    ([0], [1], 0, 1, 1, 128, 32, 0),                           # one key: its own
    ([0], [1], 1, 4, 4, 128, 32, 0),
    ([0, 0], [9, 40], 0, 2, 2, 128, 32, 0),                    # nothing but the tree
    ([640], [16], 0, 6, 6, 128, 64, 0),
    ([31, 32, 33, 0, 95], [7] * 5, 31, 6, 2, 128, 32, 0),      # borders of a tile inside the tree
    ([5, 200, 0, 64, 131], RAGGED, 100, 12, 4, 128, 64, 0),
    ([5, 200, 0, 64, 131], RAGGED, 0, 12, 12, 128, 96, 0),
    ([5, 200, 0, 64, 131], RAGGED, 333, 8, 1, 128, 32, 0),     # 8 heads on one
    ([5, 200, 0, 64, 700], RAGGED, 333, 12, 4, 128, 32, 150),  # windows that end in the prefix and past it
    ([5, 2000, 0, 64, 700], RAGGED, 1000, 6, 6, 128, 256, 1),  # a window shorter than the trees are deep
    ([300, 0, 17], [64, 30, 0], 250, 6, 6, 128, 64, 0),
    ([300, 0, 17], [64, 20, 33], 0, 12, 4, 128, 128, 77),
    ([300, 20, 63, 64], [65, 200, 130, 1], 0, 4, 2, 128, 64, 0),   # masks of several words
    ([10, 450], [100, 2], 1500, 6, 2, 128, 64, 600),
    ([5, 200, 0, 64, 131], RAGGED, 100, 24, 8, 64, 32, 0),
    ([300, 0, 17], [64, 200, 0], 250, 3, 3, 64, 64, 190),
    ([5, 200, 0, 64, 131], RAGGED, 70, 6, 2, 96, 32, 0),
    ([5, 100], [2, 70], 70, 2, 2, 40, 32, 33),
    ([5, 100], [2, 5], 70, 2, 1, 256, 32, 0),
    ([3000], [5], 0, 2, 2, 128, 32, 0),                        # a long row, cut into splits
    ([3000, 5], [60, 64], 0, 2, 2, 128, 32, 0),
    ([40] * 70, [4] * 70, 600, 2, 2, 128, 32, 0),              # many rows
    ([0, 0], [0, 0], 10, 2, 2, 128, 32, 0),                    # no node at all
    ([300, 0, 17, 64], [45, 64, 0, 33], 0, 2, 2, 128, 64, 0),  # 33 to 64 columns: two waves on either tile of a step
    ([300, 0, 17, 96], [20, 9, 0, 16], 0, 6, 2, 128, 32, 100),
    ([300, 0, 17, 95], [45, 64, 1, 33], 333, 2, 2, 128, 96, 0),
    ([300, 0, 17, 64], [45, 64, 0, 33], 0, 2, 2, 64, 32, 0),
    ([300, 0, 17, 64], [20, 30, 2, 9], 70, 4, 2, 64, 64, 50),
    ([3000, 40], [40, 64], 100, 2, 2, 128, 32, 0),             # such rows, cut
    ([5000, 40], [40, 64], 0, 1, 1, 64, 32, 1500),
    ([200] * 64, [40] * 64, 0, 4, 4, 128, 32, 0),              # rows that fill the card
    ([700], [512], 0, 1, 1, 128, 64, 0),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("case", range(len(SHAPES)))
def test_tree_attention(dtype, case):
    """Against the softmax in 64 bits; every slot that no row holds is NaN, bits past a row's nodes are set, and
    tokens behind the last row come back as 0."""
    ctx, n, P, H, G, hd, page, window = SHAPES[case]
    _say(f"tree_attention {dtype} case {case}: {SHAPES[case]}")
    c = Tree(case, ctx, n, P, G, hd, page, DT[dtype])
    q = c.queries(H, tail=2)
    got = _run(c, q, window, junk=True)
    torch.cuda.synchronize()
    ref, tol = c.tree_reference(q, window)
    _check(got, ref, tol)
    assert torch.all(got[int(c.off[-1]):] == 0)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("hd", [128, 64, 96])
@pytest.mark.parametrize("n,P,window", [([6, 3], 40, 0), ([45, 20], 40, 0), ([6, 3], 0, 9), ([150, 20], 0, 0),
                                        ([45, 130], 70, 25)])
def test_any_mask(dtype, hd, n, P, window):
    """Masks that are no tree's: nodes that see none, later nodes, all of them; positions before the row's start,
    and far behind it."""
    _say(f"tree_attention {dtype} hd={hd} n={n} prefix={P} window={window}: any mask")
    rng = np.random.default_rng(sum(n))
    seen = [rng.random((m, m)) < 0.4 for m in n]
    depth = [rng.integers(0, 30, m) for m in n]
    for s, d in zip(seen, depth):
        s[1], s[2] = False, True
        d[0], d[1] = -40, 10 ** 6
    c = Tree(3, [0, 50], n, P, 2, hd, 32, DT[dtype], seen=seen, depth=depth)
    q = c.queries(4)
    got = _run(c, q, window, junk=True)
    ref, tol = c.tree_reference(q, window)
    _check(got, ref, tol)
    if P == 0 and window == 0:
        assert torch.all(got[1] == 0)  # row 0 holds nothing before its nodes


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("hd", [128, 64, 96])
@pytest.mark.parametrize("n", [[3, 5, 2, 4], [45, 33, 60, 40]])
def test_rows_without_pages(dtype, hd, n):
    """Table and prefix entries that are no page hold no keys, a tree's own nodes included."""
    _say(f"tree_attention {dtype} hd={hd}: entries that are no page")
    c = Tree(5, [70, 10, 0, 126], n, 90, 2, hd, 32, DT[dtype])
    gone = [(0, 1), (1, 0), (2, 0), (3, 4), (-1, 1)]
    a = c.tree_device(dev(), int(c.off[-1]))
    a["tables"][0, 1], a["tables"][1, 0], a["tables"][2, 0], a["tables"][3, 4] = -1, c.N, 2 ** 31 - 1, -2 ** 31
    a["pre"][1] = c.N + 1
    q = c.queries(4)
    for window in (0, 8):
        got = _run(c, q, window, a)
        ref, tol = c.tree_reference(q, window, gone)
        _check(got, ref, tol, f"window {window}")


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("hd", [128, 64, 96])
@pytest.mark.parametrize("n", [6, 45, 150])
@pytest.mark.parametrize("junk", [NAN, INF])
def test_values_of_unseen_nodes(dtype, hd, n, junk):
    """K and V of a node that only its descendants see (here not finite) do not reach the others."""
    _say(f"tree_attention {dtype} hd={hd} n={n}: {junk} at a node")
    c = Tree(7, [37, 3], [n, 2], 50, 2, hd, 32, DT[dtype], kinds=["4", "chain"])
    node = n // 2
    hit = np.concatenate([c.seen[0][:, node], [False, False]])
    assert hit.any() and not hit.all()
    q = c.queries(4)
    ref, tol = c.tree_reference(q, 0)
    at = 37 + node
    for pool in (c.K, c.V):
        pool[c.tables[0, at // 32], :, at % 32] = junk
    got = _run(c, q, 0)
    _check(got[torch.from_numpy(~hit)], ref[~hit], tol[~hit])


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_rows_that_start_inside_the_prefix(dtype):
    """Such a row sees the prefix up to its start; nodes whose positions lie in the prefix hold no key."""
    _say(f"tree_attention {dtype}: positions inside the prefix")
    for n in ([4, 3, 6], [40, 33, 50]):
        c = Tree(9, [40, 0, 3], n, 100, 2, 128, 32, DT[dtype])
        c.start = np.array([140, 37, 98], np.int32)
        c.tok_pos = np.concatenate([c.start[b] + c.depth[b] for b in range(3)])
        for window in (0, 30):
            q = c.queries(4)
            got = _run(c, q, window)
            ref, tol = c.tree_reference(q, window)
            _check(got, ref, tol, f"n={n} window={window}")


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("n", [[2, 30, 3], [20, 64, 33]])
def test_bad_rows_and_tail(dtype, n):
    """A row with more nodes than max_per_row is treated as empty; the C entry leaves the tokens behind the last row."""
    _say(f"tree_attention {dtype}: bad rows")
    from flaxchat_amd import _lib
    c = Tree(11, [40, 7, 90], n, 50, 2, 128, 32, DT[dtype])
    q = c.queries(4, tail=4)
    T = len(q)
    ref, tol = c.tree_reference(q, 0)
    got = _run(c, q, 0, most=n[2])
    for s in (slice(0, n[0]), slice(n[0] + n[1], sum(n))):
        _check(got[s], ref[s], tol[s], "the other rows")
    a = c.tree_device(dev(), T)
    a["row_off"][3] = 1000
    got = _run(c, q, 0, a)
    _check(got[:n[0] + n[1]], ref[:n[0] + n[1]], tol[:n[0] + n[1]], "the rows before")
    a = c.tree_device(dev(), T)
    qt = torch.from_numpy(q).to(dev(), DT[dtype])
    y = torch.full((T, 4 * 128), 7.0, device=dev(), dtype=DT[dtype])
    N, G, page, hd = a["k"].shape
    p = _lib.FcPages(a["k"].data_ptr(), a["v"].data_ptr(), G * page * hd, G * page * hd, N, G, page, hd,
                     1 if dtype == "bf16" else 0)
    L = _lib.lib()
    nb = L.fc_tree_attention_workspace_bytes(p, 3, T, c.most, 4, c.W, c.P, 0)
    ws = torch.empty(max(nb, 1), dtype=torch.uint8, device=dev())
    _lib.check(L.fc_tree_attention(p, qt.data_ptr(), 512, 128, y.data_ptr(), 3, T, c.most, 4, a["tables"].data_ptr(),
                                   c.W, a["row_off"].data_ptr(), a["start"].data_ptr(), a["mask"].data_ptr(),
                                   a["tok_pos"].data_ptr(), a["pre"].data_ptr(), c.P, 0, 0, ws.data_ptr(), nb,
                                   torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    _check(y[:sum(n)], ref[:sum(n)], tol[:sum(n)])
    assert torch.all(y[sum(n):] == 7.0)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("hd", [128, 64])
def test_strided_and_unaligned(dtype, hd):
    """Pages of one layer of a pool of three, queries cut out of a fused projection, arrays off the 16-byte
    boundary."""
    _say(f"tree_attention {dtype} hd={hd}: strides")
    for n in ([3, 6], [40, 33]):
        c = Tree(13, [70, 10], n, 40, 2, hd, 32, DT[dtype])
        q = c.queries(4)
        ref, tol = c.tree_reference(q, 0)
        a = c.tree_device(dev(), len(q))
        for what in ("k", "v"):
            t = torch.full((c.N, 3, *a[what].shape[1:]), NAN, device=dev(), dtype=DT[dtype])
            t[:, 1] = a[what]
            a[what] = t[:, 1]
        qt = torch.from_numpy(q).to(dev(), DT[dtype])
        wide = torch.full((len(q), 8, hd), NAN, device=dev(), dtype=DT[dtype])
        wide[:, 2:6] = qt
        _check(_run(c, q, 0, a, qt=wide[:, 2:6]), ref, tol, "strided")
        buf = torch.empty(qt.numel() + 1, device=dev(), dtype=DT[dtype])
        odd = buf[1:].view_as(qt)
        odd.copy_(qt)
        _check(_run(c, q, 0, a, qt=odd), ref, tol, "unaligned")
        t = torch.empty(len(q), hd, 4, device=dev(), dtype=DT[dtype])
        t.copy_(qt.transpose(1, 2))
        _check(_run(c, q, 0, a, qt=t.transpose(1, 2)), ref, tol, "dims apart")


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("B,most,P,window", [(300, 3, 0, 0), (300, 20, 40, 50), (1000, 2, 10, 0), (257, 40, 0, 0),
                                             (260, 25, 0, 0), (260, 25, 33, 70)])
def test_many_rows(dtype, B, most, P, window):
    _say(f"tree_attention {dtype}: {B} rows")
    rng = np.random.default_rng(B)
    c = Tree(B, rng.integers(0, 90, B), rng.integers(0, most + 1, B), P, 1, 64, 32, DT[dtype])
    q = c.queries(2, tail=1)
    got = _run(c, q, window, most=most)
    ref, tol = c.tree_reference(q, window)
    _check(got, ref, tol)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("P", [0, 333])
def test_chains_are_paged_attention(dtype, P):
    """Chains of nodes: the result of paged_attention, within both bounds."""
    _say(f"tree_attention {dtype}: chains behind {P}")
    for n in ([3, 1, 9], [40, 64, 10]):
        c = Tree(15, [100, 2000, 31], n, P, 2, 128, 64, DT[dtype], kinds=["chain"])
        q = c.queries(6)
        a = c.tree_device(dev(), len(q))
        qt = torch.from_numpy(q).to(dev(), DT[dtype])
        for window in (0, 1000):
            want = OPS.paged_attention(qt, a["k"], a["v"], a["tables"], a["row_off"], a["start"], c.most, window,
                                       a["pre"] if P else None, P)
            tol = c.tree_reference(q, window)[1]
            _check(_run(c, q, window, a), want.double().cpu().numpy(), 2 * tol, f"n={n} window={window}")


def test_pool_past_32_bits():
    """A pool of more than 2^31 elements, pages at its end."""
    _say("a pool past 32 bits")
    N, G, page, hd, B, n = 66000, 4, 64, 128, 3, 40
    k = torch.zeros(N, G, page, hd, dtype=torch.bfloat16, device=dev())
    v = torch.zeros(N, G, page // 32, hd, 32, dtype=torch.bfloat16, device=dev())
    assert k.numel() > 2 ** 31
    tables = up([[N - 1, N - 5], [N - 2, N - 6], [0, N - 7]])
    start, off = up([20, 64, 30]), up([0, n, 2 * n, 3 * n])
    rng = np.random.default_rng(0)
    par = np.concatenate([np.maximum(np.arange(n) - 1 - rng.integers(0, 4, n), 0) for _ in range(B)])
    par[::n] = -1
    mask, pos = OPS.tree_tables(up(par), off, start, n)
    row = np.repeat(np.arange(B), n)
    at = start.cpu().numpy()[row] + np.tile(np.arange(n), B)
    slots = tables.cpu().numpy()[row, at // page] * page + at % page
    x = torch.randn(B * n, 3 * G, hd, device=dev(), generator=torch.Generator(device=dev()).manual_seed(1))
    cos, sin = torch.ones(200, 64, device=dev()), torch.zeros(200, 64, device=dev())
    q = OPS.rope_append(x[:, :G], x[:, G:2 * G], x[:, 2 * G:], pos, up(slots), cos, sin, k, v)
    assert torch.equal(q, x[:, :G].bfloat16())  # (no turn, no norm)
    # the same rows in a small pool
    small = torch.tensor([N - 1, N - 5, N - 2, N - 6, 0, N - 7], device=dev())
    y = OPS.tree_attention(q, k, v, tables, off, start, mask, pos, n, 0)
    kk, vv = k[small].contiguous(), v[small].contiguous()
    few = up([[0, 1], [2, 3], [4, 5]])
    assert torch.equal(y, OPS.tree_attention(q, kk, vv, few, off, start, mask, pos, n, 0)) and y.abs().max() > 0
    path = np.full(B * n, -1)
    path[:3], path[n:n + 2], path[2 * n:2 * n + 3] = (0, 5, 39), (0, 9), (0, 2, 38)
    in_small = few.cpu().numpy()[row, at // page] * page + at % page
    OPS.tree_commit(up(path), up(slots), off, n, k, v)
    OPS.tree_commit(up(path), up(in_small), off, n, kk, vv)
    assert torch.equal(k[small], kk) and torch.equal(v[small], vv)


def test_side_stream_and_graph():
    """On a stream of its own, and the whole step captured into a graph that is replayed on new contents, eager work
    between the replays; two graphs of the same inputs hold workspaces of their own."""
    _say("a step on a side stream and in graphs")
    n, P, dt = [20, 7, 33, 64], 150, torch.bfloat16
    c = Tree(17, [300, 60, 1000, 5], n, P, 2, 128, 32, dt, junk=0.0)
    H, T, layers = 6, sum(n), 2
    rng = np.random.default_rng(2)
    off = up(c.off)
    row = np.repeat(np.arange(4), n)
    at = c.ctx[row] + np.arange(T) - c.off[row]
    slots = up(c.tables[row, at // 32] * 32 + at % 32)
    a = c.device(dev())
    k0, v0 = torch.stack([a["k"]] * layers), torch.stack([a["v"]] * layers)
    cos, sin = torch.rand(2000, 64, device=dev()), torch.rand(2000, 64, device=dev())

    def inputs(seed):
        r = np.random.default_rng(seed)
        _, par, _ = packed(r, n, ["4", "chain", "8"])
        g = torch.Generator(device=dev()).manual_seed(seed)
        return [up(par), up(r.integers(0, 3, T)), up(r.integers(0, 3, T)),
                torch.randn(T, H + 4, 128, device=dev(), generator=g)]

    def step(parent, tokens, target, qkv, k, v):
        mask, pos = OPS.tree_tables(parent, off, a["start"], 64)
        ys = []
        for i in range(layers):
            q = OPS.rope_append(qkv[:, :H], qkv[:, H:H + 2], qkv[:, H + 2:], pos, slots, cos, sin, k[i], v[i], False,
                                1.2)
            ys.append(OPS.tree_attention(q, k[i], v[i], a["tables"], off, a["start"], mask, pos, 64, 0, a["pre"], P))
        n_acc, nxt, path = OPS.tree_accept(parent, tokens, target, off, 64)
        OPS.tree_commit(path, slots, off, 64, k, v)
        return [mask, pos, *ys, n_acc, nxt, path]

    def eager(x):
        k, v = k0.clone(), v0.clone()
        return step(*x, k, v) + [k, v]

    want = {s: eager(inputs(s)) for s in (1, 2, 3)}
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = eager(inputs(2))
    side.synchronize()
    for g, w in zip(got, want[2]):
        assert torch.equal(g, w)
    bufs, k, v = inputs(1), k0.clone(), v0.clone()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(*bufs, k, v))
        graphs.append(g)
    for turn, seed in enumerate((3, 1, 2, 3)):
        for b, x in zip(bufs, inputs(seed)):
            b.copy_(x)
        k.copy_(k0)
        v.copy_(v0)
        eager(inputs(1))  # other work in between
        graphs[turn % 2].replay()
        torch.cuda.synchronize()
        for i, (g, w) in enumerate(zip(outs[turn % 2] + [k, v], want[seed])):
            assert torch.equal(g, w), (turn, i)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_two_calls_at_once(dtype):
    """Calls on two streams at once, each with its own workspace and results."""
    _say(f"tree_attention {dtype}: two streams")
    cs = [Tree(19 + i, [3000, 900], n, 0, 2, 128, 32, DT[dtype]) for i, n in enumerate(([30, 60], [5, 8]))]
    qs = [c.queries(4) for c in cs]
    dv = [(c.tree_device(dev(), len(q)), torch.from_numpy(q).to(dev(), DT[dtype])) for c, q in zip(cs, qs)]
    want = [_run(c, q, 0, a, qt=qt) for c, q, (a, qt) in zip(cs, qs, dv)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(_run(cs[i], qs[i], 0, dv[i][0], qt=dv[i][1]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


# ---------------------------------------------------------------- together
@pytest.mark.parametrize("interleaved", [False, True])
def test_decode_with_trees(interleaved):
    """Greedy decoding of a small attention model, trees of drafted tokens a step, gives the tokens that one-by-one
    decoding in 64 bits on the host gives, and takes fewer steps."""
    _say(f"a decode loop with trees, interleaved={interleaved}")
    rng = np.random.default_rng(4)
    V, D, H, G, hd, page, B, want_n, layers, window = 50, 64, 4, 2, 64, 32, 3, 40, 2, 37
    E = rng.standard_normal((V, D))
    Wq, Wk, Wv = (rng.standard_normal((layers, D, h * hd)) * 0.3 for h in (H, G, G))
    Wo = rng.standard_normal((layers, H * hd, D)) * 0.3
    prompts = [rng.integers(0, V, m).tolist() for m in (5, 33, 1)]
    rot = 32
    ang = np.outer(np.arange(400), 100.0 ** (-np.arange(rot // 2) / (rot // 2)))
    cos, sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)

    def host_logits(seq):
        x, L = E[seq], len(seq)
        for i in range(layers):
            q, k = (rope_plain((x @ W[i]).reshape(L, h, hd), np.arange(L), cos, sin, interleaved, 1.2)[0]
                    for W, h in ((Wq, H), (Wk, G)))
            v = (x @ Wv[i]).reshape(L, G, hd)
            y = np.zeros((L, H, hd))
            d = np.arange(L)[:, None] - np.arange(L)
            for h in range(H):
                s = np.where((d >= 0) & (d <= window), q[:, h] @ k[:, h // 2].T / hd ** 0.5, -np.inf)
                p = np.exp(s - s.max(1, keepdims=True))
                y[:, h] = p / p.sum(1, keepdims=True) @ v[:, h // 2]
            x = x + y.reshape(L, H * hd) @ Wo[i]
        return x[-1] @ E.T

    truth = []
    for p in prompts:
        seq = list(p)
        for _ in range(want_n + 12):
            lg = np.sort(host_logits(seq))
            assert lg[-1] - lg[-2] > 1e-3  # no tie that fp32 could break otherwise
            seq.append(int(np.argmax(host_logits(seq))))
        truth.append(seq[len(p):])
    f = lambda a: torch.from_numpy(np.asarray(a, np.float32)).to(dev())  # noqa: E731
    dE, dWq, dWk, dWv, dWo, dcos, dsin = (f(a) for a in (E, Wq, Wk, Wv, Wo, cos, sin))
    W, N = 6, 3 * 6
    k = torch.full((layers, N, G, page, hd), NAN, device=dev())
    v = torch.full((layers, N, G, page // 32, hd, 32), NAN, device=dev())
    tables, held = torch.full((B, W), -1, dtype=torch.int32, device=dev()), up([0] * B)
    free, n_free, length = up(rng.permutation(N)), up([N]), up([0] * B)

    def forward(toks, parents, n_new):
        T, most = len(toks), int(max(n_new))
        z = lambda m: torch.zeros(m, dtype=torch.int32, device=dev())  # noqa: E731
        row_off, start, tok_row, tok_pos, slots = z(B + 1), z(B), z(T), z(T), z(T)
        OPS.page_tables(tables, held, free, n_free, length, up(n_new), row_off, start, tok_row, tok_pos, slots, page)
        parent = up(parents)
        mask, pos = OPS.tree_tables(parent, row_off, start, most)
        x = dE[up(toks).long()]
        for i in range(layers):
            q = OPS.rope_append((x @ dWq[i]).view(T, H, hd), (x @ dWk[i]).view(T, G, hd), (x @ dWv[i]).view(T, G, hd),
                                pos, slots, dcos, dsin, k[i], v[i], interleaved, 1.2)
            y = OPS.tree_attention(q, k[i], v[i], tables, row_off, start, mask, pos, most, window)
            x = x + y @ dWo[i]
        target = (x @ dE.T).argmax(-1).to(torch.int32)
        n_acc, nxt, path = OPS.tree_accept(parent, up(toks), target, row_off, most)
        OPS.tree_commit(path, slots, row_off, most, k, v)
        length.add_(n_acc)
        return n_acc.tolist(), nxt.tolist(), path.tolist(), row_off.tolist()

    # the prompts, a token of each row a step: a root each, which is accepted as it is
    out, pend = [[] for _ in range(B)], [p[0] for p in prompts]
    for b_pos in range(max(len(p) for p in prompts)):
        rows = [[p[b_pos]] if b_pos < len(p) else [] for p in prompts]
        n_acc, nxt, _, _ = forward(sum(rows, []), [-1] * len(sum(rows, [])), [len(r) for r in rows])
        for b, p in enumerate(prompts):
            if b_pos == len(p) - 1:
                pend[b] = nxt[b]
    for b in range(B):
        out[b].append(pend[b])
    steps = 0
    while min(len(o) for o in out) < want_n:
        toks, parents, n_new = [], [], []
        for b in range(B):
            m = int(rng.integers(1, 14))
            par = np.maximum(np.arange(m) - 1 - rng.integers(0, 3, m), 0)
            par[0] = -1
            tk = rng.integers(0, V, m)
            tk[0] = pend[b]
            done = len(out[b])
            good = {0: 0}  # nodes on the true continuation, with their depth
            for i in range(1, m):
                p = int(par[i])
                if p in good and rng.random() < 0.8 and done + good[p] < len(truth[b]):
                    tk[i], good[i] = truth[b][done + good[p]], good[p] + 1
            if len(out[b]) >= want_n:
                tk, par, m = tk[:0], par[:0], 0  # finished
            toks += tk.tolist()
            parents += par.tolist()
            n_new.append(m)
        n_acc, nxt, path, off = forward(toks, parents, n_new)
        steps += 1
        for b in range(B):
            if n_new[b]:
                on = path[off[b]:off[b] + n_acc[b]]
                out[b] += [toks[off[b] + i] for i in on[1:]] + [nxt[b]]
                pend[b] = nxt[b]
    for b in range(B):
        m = min(len(out[b]), len(truth[b]))
        assert out[b][:m] == truth[b][:m], b
    assert steps < want_n * 0.8
