"""Plain implementations, in 64 bits, of the operators that decode with trees
of drafted tokens, and the trees and chunks their tests use."""

import numpy as np
import torch

from tests.paged_cases import Paged, rounded


def line_of(parent, i):
    """Node i and the nodes above it, from the root; a parent outside [0, i) makes a root."""
    out = [i]
    while 0 <= parent[out[-1]] < out[-1]:
        out.append(int(parent[out[-1]]))
    return out[::-1]


def trees(rng, n, kind):
    """Parents of a row of n nodes."""
    i = np.arange(n)
    if kind == "chain":
        return i - 1
    if kind == "star":
        return np.where(i > 0, 0, -1)
    if kind == "roots":
        return np.full(n, -1)
    if kind == "odd":  # what no caller should pass: such nodes are roots
        p = np.maximum(i - 1 - rng.integers(0, 4, n), 0)
        p[rng.random(n) < 0.3] = rng.choice([-2 ** 31, -2, 2 ** 31 - 1, n])
        p[n // 2:n // 2 + 1] = n // 2
        return p
    p = np.maximum(i - 1 - rng.integers(0, int(kind), n), 0)
    p[rng.random(n) < 0.03] = -1
    if n:
        p[0] = -1
    return p


def packed(rng, ns, kinds):
    """(row_off, parent) of rows of ns nodes."""
    par = [trees(rng, n, kinds[b % len(kinds)]) for b, n in enumerate(ns)]
    return np.concatenate([[0], np.cumsum(ns)]), np.concatenate(par + [np.zeros(0, np.int64)]).astype(np.int64), par


def tables_plain(off, parent, start, T, most):
    """tree_tables, node by node: (mask as uint64 [T][words], tok_pos)."""
    W = -(-most // 64)
    mask, pos = np.zeros((T, W), np.uint64), np.full(T, -1, np.int64)
    for b in range(len(off) - 1):
        n = off[b + 1] - off[b]
        if n > most or off[b + 1] > T:
            continue
        for i in range(n):
            on = line_of(parent[off[b]:off[b + 1]], i)
            for j in on:
                mask[off[b] + i, j // 64] |= np.uint64(1) << np.uint64(j % 64)
            pos[off[b] + i] = start[b] + len(on) - 1
    return mask, pos


def accept_plain(off, parent, tokens, target, T, most):
    """tree_accept by every node's line from its root."""
    B = len(off) - 1
    count, nxt, path = np.zeros(B, np.int64), np.full(B, -1, np.int64), np.full(T, -1, np.int64)
    for b in range(B):
        n = off[b + 1] - off[b]
        if n > most or off[b + 1] > T:
            continue
        tk, tg = tokens[off[b]:off[b + 1]], target[off[b]:off[b + 1]]
        best = []
        for i in range(n):
            on = line_of(parent[off[b]:off[b + 1]], i)
            if len(on) > len(best) and all(tk[y] == tg[x] for x, y in zip(on, on[1:])):
                best = on
        if best:
            count[b], nxt[b] = len(best), tg[best[-1]]
            path[off[b]:off[b] + len(best)] = best
    return count, nxt, path


def moves_plain(off, path, slots, pool, most, T):
    """(source, destination) slots of tree_commit, row by row."""
    out = []
    for b in range(len(off) - 1):
        n = off[b + 1] - off[b]
        if n > most or off[b + 1] > T:
            continue
        for j in range(n):
            p = path[off[b] + j]
            if j < p < n:
                s, d = slots[off[b] + p], slots[off[b] + j]
                if 0 <= s < pool and 0 <= d < pool:
                    out.append((int(s), int(d)))
    return out


def rope_plain(x, pos, cos, sin, interleaved, norm):
    """(y, bound) of the rotated heads x [M][heads][hd] in 64 bits. The bound of an fp32 result: each of a pair's
    products and their sum rounds once (3 half steps of |x1 c| + |x2 s|); the sum of hd squares is off by hd + 3
    half steps and by what the pairs' errors make of it (6 sqrt(2) of them at most, the rotation keeping lengths),
    of which its root takes half; mean, root, quotient and product round 5 times."""
    M, H, hd = x.shape
    rot, x = 2 * cos.shape[1], x.astype(np.float64)
    there = (pos >= 0) & (pos < len(cos))
    at = np.where(there, pos, 0)
    c, s = cos[at].astype(np.float64)[:, None], sin[at].astype(np.float64)[:, None]
    a = slice(0, rot, 2) if interleaved else slice(0, rot // 2)
    b = slice(1, rot, 2) if interleaved else slice(rot // 2, rot)
    y, tol = x.copy(), np.zeros_like(x)
    y[..., a], y[..., b] = x[..., a] * c + x[..., b] * s, x[..., b] * c - x[..., a] * s
    tol[..., a] = 3 * 2.0 ** -24 * (abs(x[..., a] * c) + abs(x[..., b] * s))
    tol[..., b] = 3 * 2.0 ** -24 * (abs(x[..., b] * c) + abs(x[..., a] * s))
    if norm > 0:
        f = norm / np.sqrt((y * y).mean(-1, keepdims=True) + 1e-6)
        y = y * f
        tol = tol * f + abs(y) * ((hd + 3 + 9) / 2 + 5) * 2.0 ** -24
    return np.where(there[:, None, None], y, 0), np.where(there[:, None, None], tol, 0)


class Tree(Paged):
    """A pool whose rows' last n positions are a chunk of nodes: `parents` a list of each row's, or `seen` a list of
    [n][n] truth values (which nodes a node sees) with each token's position."""

    def __init__(self, seed, ctx, n, prefix, G, hd, page, dtype, kinds=("4", "chain"), seen=None, depth=None, **kw):
        super().__init__(seed, ctx, n, prefix, G, hd, page, dtype, **kw)
        rng = np.random.default_rng(seed + 1)
        if seen is None:
            seen, depth = [], []
            for b, m in enumerate(self.n):
                par = trees(rng, int(m), kinds[b % len(kinds)])
                ok = np.zeros((m, m), bool)
                for i in range(m):
                    ok[i, line_of(par, i)] = True
                seen.append(ok)
                depth.append(ok.sum(1) - 1)
        self.seen, self.depth = seen, depth
        self.most = int(max(1, self.n.max()))
        self.tok_pos = np.concatenate([self.start[b] + np.asarray(depth[b]) for b in range(self.B)]
                                      + [np.zeros(0)]).astype(np.int64)

    def words(self, T, junk=False):
        """The mask of T tokens, int64 [T][words]; junk: bits past each row's nodes set."""
        W = -(-self.most // 64)
        bits = np.full((T, 64 * W), junk, bool)
        for b in range(self.B):
            m = int(self.n[b])
            bits[self.off[b]:self.off[b] + m, :m] = self.seen[b]
        return np.packbits(bits, axis=-1, bitorder="little").view(np.int64)

    def tree_device(self, dev, T, junk=False):
        a = self.device(dev)
        a["mask"] = torch.from_numpy(self.words(T, junk)).to(dev)
        pos = np.concatenate([self.tok_pos, np.full(T - len(self.tok_pos), -1)])
        a["tok_pos"] = torch.from_numpy(pos.astype(np.int32)).to(dev)
        return a

    def visible(self, b, window):
        """[n][keys of row b] truth values."""
        m, first = int(self.n[b]), int(self.start[b])
        L = self.P + len(self.rows[b][0])
        pos = np.maximum(self.tok_pos[self.off[b]:self.off[b] + m], first)[:, None]
        key = np.arange(L)[None]
        ok = (key < first) & ((pos - key <= window) if window > 0 else np.ones((m, 1), bool))
        for j in range(m):  # nodes whose positions lie in the prefix, or past the row's own keys, hold none
            if self.P <= first + j < L:
                ok[:, first + j] = self.seen[b][:, j]
        return ok

    def tree_reference(self, q, window, gone=()):
        """(y, bound): Paged.reference with the nodes' own visibility."""
        T, H, hd = q.shape
        rep, page = H // self.G, self.page
        y, tol = np.zeros((T, H, hd)), np.zeros((T, H, hd))
        for b in range(self.B):
            m = int(self.n[b])
            if m == 0:
                continue
            k = torch.from_numpy(np.concatenate([self.pre[0], self.rows[b][0]])).double()
            v = torch.from_numpy(np.concatenate([self.pre[1], self.rows[b][1]])).double()
            there = torch.ones(len(k), dtype=torch.bool)
            for r, j in gone:
                if r == b:
                    there[self.P + j * page:self.P + (j + 1) * page] = False
                elif r == -1:
                    there[j * page:min(self.P, (j + 1) * page)] = False
            ok = torch.from_numpy(self.visible(b, window)) & there
            qb = torch.from_numpy(q[self.off[b]:self.off[b] + m]).double()
            for h in range(H):
                kh, vh, qh = k[:, h // rep], v[:, h // rep], qb[:, h]
                x = (qh @ kh.T / hd ** 0.5).masked_fill(~ok, -torch.inf)
                S = ((qh.abs() @ kh.abs().T) / hd ** 0.5).masked_fill(~ok, 0).amax(1, keepdim=True)
                mx = x.amax(1, keepdim=True)
                e = (x - mx.masked_fill(mx == -torch.inf, 0)).exp()
                s = e.sum(1, keepdim=True)
                p = torch.where(s > 0, e / s, 0)
                yh = torch.stack([p[i, ok[i]] @ vh[ok[i]] for i in range(m)])
                A = torch.stack([p[i, ok[i]] @ vh[ok[i]].abs() for i in range(m)])
                nk = ok.sum(1, keepdim=True)
                t = A * (2 * (hd + 4) * 2.0 ** -24 * S + 2.0 ** -20 + (nk + 16) * 2.0 ** -23)
                if self.dtype == torch.bfloat16:
                    t = t + 2.0 ** -8 * (A + yh.abs() + 2.0 ** -8 * A)
                y[self.off[b]:self.off[b] + m, h] = yh.numpy()
                tol[self.off[b]:self.off[b] + m, h] = t.numpy()
        return y.reshape(T, H * hd), tol.reshape(T, H * hd)


__all__ = ["Tree", "rounded", "trees", "packed", "line_of", "tables_plain", "accept_plain", "moves_plain", "rope_plain"]
