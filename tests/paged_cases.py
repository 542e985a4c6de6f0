"""Plain implementations of the paged-cache operators in 64 bits (numpy and
torch on the CPU), and the layouts their tests write pages in."""

import numpy as np
import torch


def k_blocks(K):
    """[..][page][hd] keys in the matrix-core order of bf16 heads of 128: position kk and dim d of a 32-position
    block at ((2*(d//32) + (kk//4)%2)*64 + 4*(kk//8) + kk%4 + 16*((d//8)%4))*8 + d%8."""
    kk, d = np.arange(32)[:, None], np.arange(128)[None]
    at = ((2 * (d // 32) + (kk // 4) % 2) * 64 + 4 * (kk // 8) + kk % 4 + 16 * ((d // 8) % 4)) * 8 + d % 8
    blocks = K.reshape(*K.shape[:-2], K.shape[-2] // 32, 4096)
    out = np.empty_like(blocks)
    out[..., at.reshape(-1)] = blocks
    return out.reshape(K.shape)


def v_blocks(V):
    """[..][page][hd] values as [..][page / 32][hd][32]."""
    *lead, page, hd = V.shape
    return np.ascontiguousarray(V.reshape(*lead, page // 32, 32, hd).swapaxes(-1, -2))


def in_pages(K, V, dtype):
    """Pools [N][G][page][hd] in position order -> (k_pages, v_pages) CPU tensors of `dtype`."""
    frag = dtype == torch.bfloat16 and K.shape[-1] == 128
    return (torch.from_numpy(k_blocks(K) if frag else K).to(dtype), torch.from_numpy(v_blocks(V)).to(dtype))


def rounded(x, dtype):
    return torch.from_numpy(np.asarray(x, np.float32)).to(dtype).float().numpy()


def tables_reference(tables, held, free, n_free, length, n_new, page, prefix, T):
    """fc_page_tables row by row (numpy int64 arrays; the state is changed in place)."""
    B, W = tables.shape
    F = len(free)
    top = min(max(int(n_free[0]), 0), F)
    stack = free[:top].tolist()
    for b in range(B):
        if n_new[b] < 0:
            stack += tables[b, :min(max(int(held[b]), 0), W)].tolist()
    stack = stack[:F]
    free[:len(stack)] = stack
    avail, asked, used, full = len(stack), 0, 0, False
    off, start, tok = [0], [], []
    for b in range(B):
        n, c, h = int(n_new[b]), int(length[b]), int(held[b])
        start.append(prefix + (0 if n < 0 else c))
        took = 0
        if n < 0:
            held[b] = 0
        elif n > 0 and c >= 0 and c + n <= W * page and -(-c // page) <= h <= W:
            need = max(0, -(-(c + n) // page) - h)
            asked += need
            if need == 0 or asked <= avail:
                full = full or used + n > T
                if not full:
                    for j in range(need):
                        tables[b, h + j] = stack.pop()
                    held[b] += need
                    used += n
                    took = n
                    for p in range(c, c + n):
                        pid = int(tables[b, p // page])
                        ok = pid >= 0 and (pid + 1) * page <= 0x7fffffff
                        tok.append((b, prefix + p, pid * page + p % page if ok else -1))
        off.append(off[-1] + took)
    n_free[0] = len(stack)
    tok += [(-1, -1, -1)] * (T - len(tok))
    tok = np.array(tok, np.int64)
    return np.array(off), np.array(start), tok[:, 0], tok[:, 1], tok[:, 2]


class Paged:
    """A pool with rows and a shared prefix: logical K / V per row and for the
    prefix (values of `dtype`), laid out in shuffled pages; every slot that
    belongs to no position holds `junk`."""

    def __init__(self, seed, ctx, n, prefix, G, hd, page, dtype, junk=float("nan"), width=None, extra=2):
        rng = self.rng = np.random.default_rng(seed)
        self.ctx, self.n = np.asarray(ctx), np.asarray(n)
        self.P, self.G, self.hd, self.page, self.dtype = prefix, G, hd, page, dtype
        B = self.B = len(self.n)
        mk = lambda m: rounded(rng.standard_normal((m, G, hd)), dtype)  # noqa: E731
        self.pre = (mk(prefix) * np.float32(1), mk(prefix))
        self.rows = [(mk(c + m), mk(c + m)) for c, m in zip(self.ctx, self.n)]
        npre = -(-prefix // page)
        np_row = [-(-int(c + m) // page) for c, m in zip(self.ctx, self.n)]
        N = self.N = npre + sum(np_row) + extra
        ids = rng.permutation(N)
        self.pre_ids = ids[:npre]
        W = self.W = width or max(1, max(np_row))
        self.tables = np.full((B, W), -1, np.int32)
        K = np.full((N, G, page, hd), junk, np.float32)
        V = K.copy()
        at = npre
        jobs = [(self.pre_ids, self.pre)]
        for b in range(B):
            self.tables[b, :np_row[b]] = ids[at:at + np_row[b]]
            jobs.append((ids[at:at + np_row[b]], self.rows[b]))
            at += np_row[b]
        for pid, (k, v) in jobs:
            for j, i in enumerate(pid):
                k1, v1 = k[j * page:(j + 1) * page], v[j * page:(j + 1) * page]
                K[i, :, :len(k1)] = k1.swapaxes(0, 1)
                V[i, :, :len(v1)] = v1.swapaxes(0, 1)
        self.K, self.V = K, V
        self.off = np.concatenate([[0], np.cumsum(self.n)]).astype(np.int32)
        self.start = (prefix + self.ctx).astype(np.int32)

    def device(self, dev):
        t = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(dev)  # noqa: E731
        k, v = in_pages(self.K, self.V, self.dtype)
        return dict(k=k.to(dev), v=v.to(dev), tables=t(self.tables), row_off=t(self.off), start=t(self.start),
                    pre=t(self.pre_ids))

    def queries(self, H, tail=0):
        return rounded(self.rng.standard_normal((int(self.off[-1]) + tail, H, self.hd)), self.dtype)

    def reference(self, q, window, gone=()):
        """(y, bound) in 64 bits: the attention of q [T][H][hd] and how far a kernel's result may be off. gone:
        (row, table entry) pairs whose keys are not there (row -1: the prefix).

        The bound, per output: with S >= sum_d |q_d k_d| / sqrt(hd) over the row's keys, an fp32 score is off by
        at most (hd + 4) 2^-24 S, so a softmax weight by twice that relatively, plus 2^-20 for its exponential
        and the running rescalings; the sums over n keys add (n + 16) 2^-23 of A = sum_j p_j |v_j|. bf16 rounds
        each weight (half a step: 2^-8 of A) and the result (2^-8 of it)."""
        T, H, hd = q.shape
        rep, G, page = H // self.G, self.G, self.page
        y, tol = np.zeros((T, H, hd)), np.zeros((T, H, hd))
        for b in range(self.B):
            m, pos0 = int(self.n[b]), int(self.start[b])
            if m == 0:
                continue
            k = torch.from_numpy(np.concatenate([self.pre[0], self.rows[b][0]])).double()
            v = torch.from_numpy(np.concatenate([self.pre[1], self.rows[b][1]])).double()
            L = len(k)
            there = torch.ones(L, dtype=torch.bool)
            for r, j in gone:
                if r == b:
                    there[self.P + j * page:self.P + (j + 1) * page] = False
                elif r == -1:
                    there[j * page:min(self.P, (j + 1) * page)] = False
            qb = torch.from_numpy(q[self.off[b]:self.off[b] + m]).double()
            pos, key = pos0 + torch.arange(m)[:, None], torch.arange(L)[None]
            ok = (key <= pos) & there
            if window > 0:
                ok &= pos - key <= window
            for h in range(H):
                kh, vh, qh = k[:, h // rep], v[:, h // rep], qb[:, h]
                x = (qh @ kh.T / hd ** 0.5).masked_fill(~ok, -torch.inf)
                S = ((qh.abs() @ kh.abs().T) / hd ** 0.5).masked_fill(~ok, 0).amax(1, keepdim=True)
                mx = x.amax(1, keepdim=True)
                e = (x - mx.masked_fill(mx == -torch.inf, 0)).exp()
                s = e.sum(1, keepdim=True)
                p = torch.where(s > 0, e / s, 0)
                # a key that a query does not see has no part in its sum, whatever its value
                yh = torch.stack([p[i, ok[i]] @ vh[ok[i]] for i in range(m)])
                A = torch.stack([p[i, ok[i]] @ vh[ok[i]].abs() for i in range(m)])
                nk = ok.sum(1, keepdim=True)
                t = A * (2 * (hd + 4) * 2.0 ** -24 * S + 2.0 ** -20 + (nk + 16) * 2.0 ** -23)
                if self.dtype == torch.bfloat16:
                    t = t + 2.0 ** -8 * (A + yh.abs() + 2.0 ** -8 * A)
                y[self.off[b]:self.off[b] + m, h] = yh.numpy()
                tol[self.off[b]:self.off[b] + m, h] = t.numpy()
        return y.reshape(T, H * hd), tol.reshape(T, H * hd)
