"""Trees of drafted tokens at their limits, on the GPU: windows shorter than a tree is deep; rows of 17 to 32 and of 33
to 64 query columns (nodes times heads a KV head), which have kernels of their own, where masks, pages or values go
wrong; rotation by workgroups of several heads."""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import flaxchat_amd.torch_ops  # noqa: E402,F401
from tests.test_gpu_kernels import _say  # noqa: E402
from tests.test_gpu_tree import DT, OPS, ROWS, _check, _run, dev, same, up  # noqa: E402
from tests.test_tree_limits import narrowed  # noqa: E402
from tests.tree_cases import Tree, line_of, packed, rope_plain  # noqa: E402

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- a layer's window among a row's nodes
@pytest.mark.parametrize("window", [1, 2, 30, 63, 64, 100, 511, 2 ** 31 - 1])
@pytest.mark.parametrize("case", range(len(ROWS)))
def test_tables_of_a_window(case, window):
    """The mask of a window: each node and the last `window` of its ancestors, walked on the host; positions do not
    change."""
    ns, kinds, most, tail = ROWS[case]
    _say(f"tree_tables case {case}, window {window}")
    rng = np.random.default_rng(case)
    off, parent, par = packed(rng, ns, kinds)
    T, most = int(off[-1]) + tail, most or max(1, max(ns))
    parent = np.concatenate([parent, rng.integers(-1, 9, tail)])
    start = rng.integers(0, 1000, len(ns))
    mask, pos = OPS.tree_tables(up(parent), up(off), up(start), most, window)
    want = np.zeros((T, -(-most // 64)), np.uint64)
    for b, n in enumerate(ns):
        for i in range(n if n <= most else 0):
            for j in line_of(par[b], i)[-min(window, 512) - 1:]:
                want[off[b] + i, j // 64] |= np.uint64(1) << np.uint64(j % 64)
    same(mask, want.view(np.int64), "mask")
    same(pos, OPS.tree_tables(up(parent), up(off), up(start), most)[1].cpu().numpy(), "tok_pos")


def _parents(c):
    """Each row's parents of a Tree, from what its nodes see: the nearest ancestor."""
    out = []
    for s in c.seen:
        above = s & ~np.eye(len(s), dtype=bool)
        out += [int(np.flatnonzero(r)[-1]) if r.any() else -1 for r in above]
    return np.array(out, np.int64)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("ctx,n,P,H,G,hd,window,kinds", [
    ([40], [200], 0, 2, 2, 128, 128, ["chain"]),
    ([40, 3], [40, 25], 0, 4, 2, 128, 16, ["chain", "3"]),
    ([5, 200, 0, 64], [9, 33, 14, 64], 100, 6, 2, 128, 3, ["chain", "2", "3"]),
    ([5, 200, 0, 64], [9, 33, 14, 64], 100, 2, 2, 64, 1, ["chain", "2", "3"]),
    ([300, 2000], [70, 150], 0, 4, 4, 128, 20, ["chain", "2"]),
    ([30, 31], [20, 12], 0, 2, 1, 96, 5, ["chain", "2"]),
])
def test_a_windowed_layer_is_token_by_token_decoding(dtype, ctx, n, P, H, G, hd, window, kinds):
    """tree_tables with a layer's window, tree_attention with its mask: the 64-bit attention of each node's own path,
    and, for rows that are chains, paged_attention's result. The mask of all ancestors gives neither."""
    _say(f"tree_attention {dtype} n={n} prefix={P} hd={hd}: a window of {window} among the nodes")
    c = Tree(21, ctx, n, P, G, hd, 32, DT[dtype], kinds=kinds)
    q = c.queries(H)
    a = c.tree_device(dev(), len(q))
    parent = up(_parents(c))
    a["mask"], a["tok_pos"] = OPS.tree_tables(parent, a["row_off"], a["start"], c.most, window)
    everything = c.tree_reference(q, window)[0]
    got = _run(c, q, window, a)
    ref, tol = narrowed(c, window).tree_reference(q, window)
    _check(got, ref, tol)
    assert (np.abs(everything - ref) > 2 * tol).any()
    chains = np.concatenate([np.full(m, kinds[b % len(kinds)] == "chain") for b, m in enumerate(n)])
    qt = torch.from_numpy(q).to(dev(), DT[dtype])
    plain = OPS.paged_attention(qt, a["k"], a["v"], a["tables"], a["row_off"], a["start"], c.most, window,
                                a["pre"] if P else None, P)
    _check(got[torch.from_numpy(chains)], plain.double().cpu().numpy()[chains], 2 * tol[chains])


@pytest.mark.parametrize("pattern", [(5, 0), (2, 9), (1, 1)])
def test_decode_with_windowed_layers(pattern):
    """A model of layers with and without a window shorter than the drafted trees are deep: greedy decoding in trees
    gives the tokens that decoding one by one in 64 bits on the host gives."""
    _say(f"a decode loop with trees, layers' windows {pattern}")
    rng = np.random.default_rng(6)
    V, D, H, G, hd, page, B, want_n, layers, m = 50, 64, 2, 1, 64, 32, 2, 36, 2, 18
    E = rng.standard_normal((V, D))
    Wq, Wk, Wv = (rng.standard_normal((layers, D, h * hd)) * 0.3 for h in (H, G, G))
    Wo = rng.standard_normal((layers, H * hd, D)) * 0.3
    ang = np.outer(np.arange(200), 100.0 ** (-np.arange(hd // 2) / (hd // 2)))
    cos, sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)

    def host_next(seq):
        x, L = E[seq], len(seq)
        d = np.arange(L)[:, None] - np.arange(L)
        for i, window in enumerate(pattern):
            q, k = (rope_plain((x @ W[i]).reshape(L, h, hd), np.arange(L), cos, sin, False, 1.2)[0]
                    for W, h in ((Wq, H), (Wk, G)))
            v, y = x @ Wv[i], np.zeros((L, H, hd))
            for h in range(H):
                s = np.where((d >= 0) & ((d <= window) | (window == 0)), q[:, h] @ k[:, 0].T / hd ** 0.5, -np.inf)
                p = np.exp(s - s.max(1, keepdims=True))
                y[:, h] = p / p.sum(1, keepdims=True) @ v
            x = x + y.reshape(L, H * hd) @ Wo[i]
        lg = x[-1] @ E.T
        top = np.sort(lg)
        assert top[-1] - top[-2] > 1e-3  # no tie that fp32 could break otherwise
        return int(np.argmax(lg))

    first = [3, 17]
    truth = []
    for t in first:
        seq = [t]
        while len(seq) < want_n + m + 2:
            seq.append(host_next(seq))
        truth.append(seq[1:])
    f = lambda a: torch.from_numpy(np.asarray(a, np.float32)).to(dev())  # noqa: E731
    dE, dWq, dWk, dWv, dWo, dcos, dsin = (f(a) for a in (E, Wq, Wk, Wv, Wo, cos, sin))
    W = 4
    k = torch.full((layers, B * W, G, page, hd), float("nan"), device=dev())
    v = torch.full((layers, B * W, G, page // 32, hd, 32), float("nan"), device=dev())
    tables = up(rng.permutation(B * W).reshape(B, W))
    length, out, steps = [0] * B, [[] for _ in range(B)], 0
    while min(len(o) for o in out) < want_n:
        toks, parents, slots = [], [], []
        for b in range(B):
            par = np.maximum(np.arange(m) - 1 - (rng.random(m) < 0.2) * rng.integers(0, 3, m), 0)
            par[0] = -1
            tk, good = rng.integers(0, V, m), {0: 0}
            tk[0] = (first[b:b + 1] + out[b])[-1]
            for i in range(1, m):  # most of them on the true continuation
                p = int(par[i])
                if p in good and rng.random() < 0.9:
                    tk[i], good[i] = truth[b][len(out[b]) + good[p]], good[p] + 1
            toks += tk.tolist()
            parents += par.tolist()
            at = length[b] + np.arange(m)
            slots += (tables[b].cpu().numpy()[at // page] * page + at % page).tolist()
        off, start, parent, slots = up(np.arange(B + 1) * m), up(length), up(parents), up(slots)
        masks = {w: OPS.tree_tables(parent, off, start, m, w) for w in set(pattern)}
        x = dE[up(toks).long()]
        T = len(toks)
        for i, window in enumerate(pattern):
            mask, pos = masks[window]
            q = OPS.rope_append((x @ dWq[i]).view(T, H, hd), (x @ dWk[i]).view(T, G, hd), (x @ dWv[i]).view(T, G, hd),
                                pos, slots, dcos, dsin, k[i], v[i], False, 1.2)
            x = x + OPS.tree_attention(q, k[i], v[i], tables, off, start, mask, pos, m, window) @ dWo[i]
        target = (x @ dE.T).argmax(-1).to(torch.int32)
        n_acc, nxt, path = OPS.tree_accept(parent, up(toks), target, off, m)
        OPS.tree_commit(path, slots, off, m, k, v)
        for b in range(B):
            on = path[b * m:b * m + int(n_acc[b])].tolist()
            out[b] += [toks[b * m + i] for i in on[1:]] + [int(nxt[b])]
            length[b] += len(on)
            w = min(len(out[b]), len(truth[b]))
            assert out[b][:w] == truth[b][:w], (steps, b)
            out[b] = out[b][:want_n + 1]
            length[b] = min(length[b], len(out[b]))
        steps += 1
    assert steps < want_n / 3


# ---------------------------------------------------------------- 24 and 50 columns a row
COLUMNS = [[12, 3], [25, 8]]  # two heads a KV head


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("hd", [128, 64])
@pytest.mark.parametrize("P", [0, 50])
@pytest.mark.parametrize("n", COLUMNS)
@pytest.mark.parametrize("junk", [float("nan"), float("inf")])
def test_values_of_unseen_nodes(dtype, hd, P, n, junk):
    """What is not finite at a node that only its descendants see does not reach the others; it reaches those that see
    it (every weight is positive)."""
    _say(f"tree_attention {dtype} hd={hd} n={n} prefix={P}: {junk} at a node")
    c = Tree(7, [37, 3], n, P, 2, hd, 32, DT[dtype], kinds=["4", "chain"])
    q = c.queries(4)
    ref, tol = c.tree_reference(q, 0)
    for node in (n[0] // 2, 1, n[0] - 1):
        hit = np.concatenate([c.seen[0][:, node], np.zeros(n[1], bool)])
        assert hit.any() and not hit.all()
        at = 37 + node
        K, V = c.K.copy(), c.V.copy()
        for both in (False, True):
            c.V[c.tables[0, at // 32], :, at % 32] = junk
            if both:
                c.K[c.tables[0, at // 32], :, at % 32] = junk
            got = _run(c, q, 0)
            _check(got[torch.from_numpy(~hit)], ref[~hit], tol[~hit], f"node {node}, K too: {both}")
            assert both or not torch.isfinite(got[torch.from_numpy(hit)]).any()
        c.K, c.V = K, V


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("hd", [128, 64])
@pytest.mark.parametrize("n,P,window", [([12, 3], 40, 0), ([12, 3], 0, 9), ([25, 20], 0, 0), ([25, 20], 40, 0),
                                        ([25, 32], 70, 25), ([32, 9], 0, 8)])
def test_any_mask(dtype, hd, n, P, window):
    """Masks that are no tree's: nodes that see none, later nodes, all of them; columns of one wave that see nothing."""
    _say(f"tree_attention {dtype} hd={hd} n={n} prefix={P} window={window}: any mask")
    rng = np.random.default_rng(sum(n))
    seen = [rng.random((m, m)) < 0.4 for m in n]
    depth = [rng.integers(0, 30, m) for m in n]
    for s, d in zip(seen, depth):
        s[1], s[2] = False, True
        d[0], d[1] = -40, 10 ** 6
    seen[0][:16] = False  # (32 columns, all of a wave's)
    c = Tree(3, [0, 50], n, P, 2, hd, 32, DT[dtype], seen=seen, depth=depth)
    q = c.queries(4)
    got = _run(c, q, window, junk=True)
    ref, tol = c.tree_reference(q, window)
    _check(got, ref, tol)
    if P == 0 and window == 0:
        assert torch.all(got[:min(16, n[0])] == 0)  # row 0 holds nothing before its nodes


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("hd", [128, 64])
@pytest.mark.parametrize("P", [0, 90])
@pytest.mark.parametrize("n", [[12, 9, 16, 10], [25, 17, 32, 20]])
def test_rows_without_pages(dtype, hd, P, n):
    """Entries that are no page: of one of a step's two tiles, of all of a row's, of the tree's own nodes."""
    _say(f"tree_attention {dtype} hd={hd} n={n} prefix={P}: entries that are no page")
    c = Tree(5, [70, 10, 0, 126], n, P, 2, hd, 32, DT[dtype])
    gone = [(0, 1), (1, 0), (2, 0), (3, 4)] + ([(-1, 1)] if P else [])
    a = c.tree_device(dev(), int(c.off[-1]))
    a["tables"][0, 1], a["tables"][1, 0], a["tables"][2, 0], a["tables"][3, 4] = -1, c.N, 2 ** 31 - 1, -2 ** 31
    if P:
        a["pre"][1] = c.N + 1
    q = c.queries(4)
    for window in (0, 8):
        got = _run(c, q, window, a)
        ref, tol = c.tree_reference(q, window, gone)
        _check(got, ref, tol, f"window {window}")


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("n", [[12, 3, 16], [25, 17, 32]])
def test_rows_that_start_inside_the_prefix(dtype, n):
    _say(f"tree_attention {dtype} n={n}: positions inside the prefix")
    c = Tree(9, [40, 0, 3], n, 100, 2, 128, 32, DT[dtype])
    c.start = np.array([140, 37, 98], np.int32)
    c.tok_pos = np.concatenate([c.start[b] + c.depth[b] for b in range(3)])
    q = c.queries(4)
    for window in (0, 30):
        got = _run(c, q, window)
        ref, tol = c.tree_reference(q, window)
        _check(got, ref, tol, f"window={window}")


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("n", [[12, 16, 3], [25, 32, 17]])
def test_rows_of_too_many_nodes(dtype, n):
    """A row of more nodes than max_per_row is treated as empty, and the others are as they are without it."""
    _say(f"tree_attention {dtype} n={n}: bad rows")
    c = Tree(11, [40, 7, 90], n, 50, 2, 128, 32, DT[dtype])
    q = c.queries(4)
    ref, tol = c.tree_reference(q, 0)
    got = _run(c, q, 0, most=n[0])
    for s in (slice(0, n[0]), slice(n[0] + n[1], sum(n))):
        _check(got[s], ref[s], tol[s])


# ---------------------------------------------------------------- rope_append, several heads a workgroup
@pytest.mark.parametrize("dtype,src", [("bf16", "bf16"), ("bf16", "fp32"), ("fp32", "fp32")])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [0.0, 1.2])
@pytest.mark.parametrize("M,H,G,hd,rot", [(14000, 10, 5, 128, 128), (10001, 10, 5, 128, 32), (13999, 20, 10, 64, 64)])
def test_rope_append_of_many_tokens(M, H, G, hd, rot, interleaved, norm, dtype, src):
    """Workgroups of 2 to 4 heads, q's and K's in one of them: a sample of the tokens, those at the tiles' borders and at
    both ends among them, against the formula in 64 bits."""
    _say(f"rope_append {src} -> {dtype}: {M} tokens of {H} and {G} heads of {hd}, {rot} rotated, interleaved="
         f"{interleaved}, norm={norm}")
    rng = np.random.default_rng(M + rot)
    page, length = 64, 3000
    N = -(-M // page) + 1
    slots, pos = rng.permutation(N * page)[:M], rng.integers(0, length, M)
    angle = np.outer(np.arange(length) * 25.0, 100000.0 ** (-np.arange(rot // 2) / (rot // 2)))
    cos, sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
    g = torch.Generator(device=dev()).manual_seed(M)
    qkv = (2 * torch.randn(M, H + 2 * G, hd, device=dev(), generator=g)).to(DT[src])
    k = torch.zeros(N, G, page, hd, device=dev(), dtype=DT[dtype])
    v = torch.zeros(N, G, page // 32, hd, 32, device=dev(), dtype=DT[dtype])
    q = OPS.rope_append(qkv[:, :H], qkv[:, H:H + G], qkv[:, H + G:], up(pos), up(slots), torch.from_numpy(cos).to(dev()),
                        torch.from_numpy(sin).to(dev()), k, v, interleaved, norm)
    some = np.unique(np.concatenate([np.arange(70), np.arange(M - 70, M), rng.integers(0, M, 300)]))
    x = qkv[torch.from_numpy(some).to(dev())].float().cpu().numpy()
    blk, at = slots[some] // page, slots[some] % page
    if dtype == "bf16" and hd == 128:  # positions' order: see the block layout
        from tests.paged_cases import k_blocks
        number = k_blocks(np.arange(32 * hd).reshape(32, hd)).reshape(-1)
        kk = k.view(N, G, page // 32, 32 * hd)[..., torch.from_numpy(np.argsort(number)).to(dev())]
        kk = kk.view(N, G, page, hd)
    else:
        kk = k
    sel = [torch.from_numpy(z).to(dev()) for z in (blk, at, at // 32, at % 32)]
    got = [("q", q[torch.from_numpy(some).to(dev())], x[:, :H]), ("K", kk[sel[0], :, sel[1]], x[:, H:H + G])]
    for what, t, heads in got:
        y, tol = rope_plain(heads, pos[some], cos, sin, interleaved, norm)
        if dtype == "bf16":  # half a step of the result's rounding: 2^-8 of it
            tol = tol + 2.0 ** -8 * (abs(y) + tol)
        bad = ~(abs(t.double().cpu().numpy() - y) <= tol)
        assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, first at {np.argwhere(bad)[0]}"
    vv = v[sel[0], :, sel[2], :, sel[3]]
    assert torch.equal(vv, qkv[torch.from_numpy(some).to(dev()), H + G:].to(DT[dtype]))


@pytest.mark.parametrize("hd,rot", [(128, 128), (64, 32), (96, 40)])
def test_rope_append_of_zeros(hd, rot):
    """Heads of zeros, and tokens without a position, stay 0 under the largest norm."""
    _say(f"rope_append: zeros, heads of {hd}")
    x = torch.zeros(5, 3, hd, device=dev())
    x[0] = 1.0
    cos, sin = torch.ones(9, rot // 2, device=dev()), torch.ones(9, rot // 2, device=dev())
    k, v = torch.full((1, 1, 32, hd), 7.0, device=dev()), torch.full((1, 1, 1, hd, 32), 7.0, device=dev())
    q = OPS.rope_append(x[:, :1], x[:, 1:2], x[:, 2:], up([-1, 0, 8, 9, 3]), up([0, 1, 2, 3, 4]), cos, sin, k, v, False, 3e35)
    assert torch.all(q == 0) and torch.all(k[0, 0, [1, 2, 4]] == 0) and torch.all(k[0, 0, [0, 3, 5]] == 7)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("hd", [128, 96])
def test_paged_attention_of_any_max_per_row(dtype, hd):
    """A plain chunk's max_per_row may be as large as its type: no word of bits is counted from it."""
    _say(f"paged_attention {dtype} hd={hd}: max_per_row up to 2^31 - 1")
    c = Tree(2, [70, 3], [5, 2], 40, 2, hd, 32, DT[dtype])
    q = c.queries(4)
    a = c.device(dev())
    qt = torch.from_numpy(q).to(dev(), DT[dtype])
    ref, tol = c.reference(q, 9)
    for most in (2 ** 31 - 1, 2 ** 31 - 63, 2 ** 31 - 64, 7):
        y = OPS.paged_attention(qt, a["k"], a["v"], a["tables"], a["row_off"], a["start"], most, 9, a["pre"], 40)
        _check(y, ref, tol, f"max_per_row {most}")


# ---------------------------------------------------------------- one long row among finished or short ones
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("n", [5, 25, 64])
@pytest.mark.parametrize("others", [0, 2])
def test_a_long_row_among_others(dtype, n, others):
    """A row of 3000 keys and 63 slots whose rows have ended, or hold a few keys."""
    _say(f"tree_attention {dtype}: one row of {n} nodes at 3000 keys, 63 of {others}")
    ctx = np.zeros(64, np.int64)
    ctx[40], ctx[3::7] = 3000, 50 * others
    ns = np.full(64, others)
    ns[40] = n
    c = Tree(4, ctx, ns, 0, 4, 128, 64, DT[dtype])
    q = c.queries(4, tail=3)
    got = _run(c, q, 0, most=n)
    ref, tol = c.tree_reference(q, 0)
    _check(got, ref, tol)
    assert torch.all(got[int(c.off[-1]):] == 0)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("n", [3, 25, 40])
@pytest.mark.parametrize("last", [1100, 20, 4200])
def test_rows_of_one_length(dtype, n, last):
    """As many rows as leave a workgroup for every CU, longer than those that no call cuts: whole beside a place for
    partials, and with a last row that is shorter, or cut."""
    _say(f"tree_attention {dtype}: 29 rows of {n} nodes at 1100 keys, one at {last}")
    c = Tree(6, [1100] * 29 + [last], [n] * 30, 0, 9, 64, 64, DT[dtype])
    q = c.queries(9, tail=1)
    got = _run(c, q, 0)
    ref, tol = c.tree_reference(q, 0)
    _check(got, ref, tol)
    assert torch.all(got[int(c.off[-1]):] == 0)
