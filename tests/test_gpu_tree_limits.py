"""Trees of drafted tokens at their limits, on the GPU: windows shorter than a tree is deep."""

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
