"""page_tables, page_append and paged_attention on the GPU against 64-bit
references (tests/paged_cases.py), at the sizes and masks where they can go
wrong, and a run of the three together as a decode loop uses them."""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import flaxchat_amd.torch_ops  # noqa: E402,F401
from tests.paged_cases import Paged, in_pages, rounded, tables_reference  # noqa: E402
from tests.test_gpu_kernels import _say  # noqa: E402

pytestmark = pytest.mark.gpu
OPS = torch.ops.flaxchat_mi355x
DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
NAN, INF = float("nan"), float("inf")


def dev():
    return torch.device("cuda", 0)


def up(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(dev())


# ---------------------------------------------------------------- page_tables
def _table_state(seed, B, W, page, q, ends=0.1, pool=1.0, odd=False):
    rng = np.random.default_rng(seed)
    length = rng.integers(0, max(1, W * page - 2 * q), B)
    n_new = rng.integers(0, q + 1, B)
    n_new[rng.random(B) < ends] = -1
    held = np.minimum(-(-length // page) + (rng.random(B) < 0.2), W)
    spare = int(pool * (np.maximum(n_new, 0) // page + 1).sum())
    ids = rng.permutation(int(held.sum()) + spare)
    tables = np.full((B, W), -1, np.int64)
    at = 0
    for b in range(B):
        tables[b, :held[b]] = ids[at:at + held[b]]
        at += held[b]
    free = np.full(len(ids) + 1, -7, np.int64)
    free[:spare] = ids[at:]
    if odd:  # what no caller should pass: such rows are left out
        k = rng.permutation(B)
        n = max(1, B // 12)
        length[k[:n]] = -5
        n_new[k[n:2 * n]] = 2 ** 31 - 1
        held[k[2 * n:3 * n]] = W + 3
        held[k[3 * n:4 * n]] = -2
        length[k[4 * n:5 * n]] = 2 ** 31 - 10
        tables[k[5 * n:6 * n]] = 2 ** 30
    return tables, held, free, np.array([spare]), length, n_new


@pytest.mark.parametrize("B,W,page,q,T,prefix,kw", [
    (1, 1, 32, 1, 1, 0, {}),
    (1, 40, 32, 900, 5000, 77, {}),
    (5, 4, 64, 3, 7, 100, {}),                       # tokens that pass the chunk
    (64, 33, 64, 1, 64, 1000, dict(ends=0.3)),
    (65, 9, 96, 17, 2000, 0, dict(pool=0.3)),        # a pool that runs short
    (300, 20, 32, 100, 2048, 5, dict(pool=0.6)),     # the last size one workgroup fills, cut short
    (300, 20, 32, 100, 2049, 5, dict(pool=0.0)),     # the first of two launches; no free page
    (1000, 12, 128, 300, 200000, 6144, dict(ends=0.5)),
    (1025, 3, 32, 7, 9000, 0, dict(odd=True)),
    (4096, 5, 32, 2, 9000, 0, dict(odd=True, pool=0.5)),
    (4095, 5, 64, 9, 1500, 0, dict(ends=0.9)),
    (37, 6, 64, 30, 600, 0, dict(odd=True, ends=0.4)),
])
def test_page_tables(B, W, page, q, T, prefix, kw):
    _say(f"page_tables B={B} W={W} page={page} q={q} T={T} {kw}")
    tables, held, free, n_free, length, n_new = _table_state(B + W, B, W, page, q, **kw)
    state = [up(a) for a in (tables, held, free, n_free)]
    rows = [up(length), up(n_new)]
    out = [torch.full((k,), 99, dtype=torch.int32, device=dev()) for k in (B + 1, B, T, T, T)]
    for again in range(2):  # a second call changes nothing
        OPS.page_tables(*state, *rows, *out, page, prefix)
        torch.cuda.synchronize()
        if again == 0:
            want = tables_reference(tables, held, free, n_free, length, n_new, page, prefix, T)
        top = int(n_free[0])
        for name, g, w in zip(("row_off", "start", "tok_row", "tok_pos", "slots"), out, want):
            w = w.astype(np.int64).astype(np.int32) if name == "start" else w
            np.testing.assert_array_equal(g.cpu().numpy(), w, err_msg=f"{name}, call {again}")
        for name, g, w in zip(("tables", "held", "n_free"), (state[0], state[1], state[3]), (tables, held, n_free)):
            np.testing.assert_array_equal(g.cpu().numpy(), w, err_msg=f"{name}, call {again}")
        np.testing.assert_array_equal(state[2].cpu().numpy()[:top], free[:top], err_msg=f"free_pages, call {again}")


def test_page_tables_small_stack():
    """Pages given back past the stack's end, n_free outside it, and a pool
    whose slots would pass 31 bits (slot -1)."""
    _say("page_tables: stack bounds")
    for n_free in (-3, 100):
        tables = np.array([[2 ** 27, 3], [4, 5], [6, 7]])
        held, free = np.array([2, 2, 2]), np.array([10, 11, 12])
        length, n_new = np.array([5, 40, 64]), np.array([2, -1, -1])
        state = [up(a) for a in (tables, held, free, [n_free])]
        out = [torch.zeros(k, dtype=torch.int32, device=dev()) for k in (4, 3, 3, 3, 3)]
        nf = np.array([n_free])
        OPS.page_tables(*state, up(length), up(n_new), *out, 32, 0)
        torch.cuda.synchronize()
        want = tables_reference(tables, held, free, nf, length, n_new, 32, 0, 3)
        assert want[4].tolist() == [-1, -1, -1]
        for g, w in zip(out + state, list(want) + [tables, held, free, nf]):
            np.testing.assert_array_equal(g.cpu().numpy(), w)


# ---------------------------------------------------------------- page_append
def test_page_tables_no_pages():
    """A stack without room: rows that need no page are taken in, others not."""
    _say("page_tables: an empty stack")
    B, W, page, T = 4, 3, 32, 12
    tables = np.array([[5, -1, -1], [6, 7, -1], [-1, -1, -1], [8, -1, -1]])
    held, length, n_new = np.array([1, 2, 0, 1]), np.array([30, 40, 0, 32]), np.array([2, 5, 1, 1])
    t = [tables, held, np.zeros(0), np.array([0]), length, n_new, np.zeros(B + 1), np.zeros(B)]
    d = [up(x) for x in t + 3 * [np.zeros(T)]]
    OPS.page_tables(*d, page, 10)
    want = tables_reference(tables, held, np.zeros(0, np.int64), np.array([0]), length, n_new, page, 10, T)
    for got, w in zip(d[6:], want):
        assert np.array_equal(got.cpu().numpy(), w)
    assert np.array_equal(d[0].cpu().numpy(), tables) and d[6].tolist() == [0, 2, 7, 7, 7] and d[3].item() == 0


@pytest.mark.parametrize("dtype,src", [("bf16", "bf16"), ("bf16", "fp32"), ("fp32", "fp32")])
@pytest.mark.parametrize("G,hd,page,runs,strided", [
    (1, 128, 32, [1], False),
    (12, 128, 64, [7, 1, 40, 130, 3], True),
    (4, 128, 96, [200, 31, 33, 64], True),
    (3, 64, 32, [5, 77, 1, 1, 1], True),
    (2, 96, 64, [50, 2], False),
    (2, 40, 32, [35, 9], True),
    (1, 256, 128, [129], False),
    (5, 7, 32, [40, 1], True),
])
def test_page_append(dtype, src, G, hd, page, runs, strided):
    _say(f"page_append {src} -> {dtype} G={G} hd={hd} page={page} runs={runs} strided={strided}")
    rng = np.random.default_rng(G * hd)
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
    if M > 3:
        slots[1], slots[2] = N * page, 2 ** 31 - 1  # outside the pool
    H = 3
    qkv = torch.from_numpy(rng.standard_normal((M, H + 2 * G, hd)).astype(np.float32)).to(dev(), DT[src])
    k, v = (qkv[:, H:H + G], qkv[:, H + G:]) if strided else (qkv[:, H:H + G].contiguous(),
                                                              qkv[:, H + G:].contiguous())
    # a pool of two layers: pages of this one are strided where `strided`
    old = rng.standard_normal((2, N, 2, G, page, hd)).astype(np.float32)
    pools = [in_pages(old[0][:, i], old[1][:, i], DT[dtype]) for i in range(2)]
    kp, vp = (torch.stack([p[j] for p in pools], 1).to(dev()) for j in range(2))
    kl, vl = (kp[:, 1], vp[:, 1]) if strided else (kp[:, 1].contiguous(), vp[:, 1].contiguous())
    OPS.page_append(k, v, up(slots), kl, vl)
    torch.cuda.synchronize()
    K, V = (rounded(old[j][:, 1], DT[dtype]).copy() for j in range(2))
    for m, s in enumerate(slots):
        if 0 <= s < N * page:
            K[s // page, :, s % page] = rounded(k[m].float().cpu().numpy(), DT[dtype])
            V[s // page, :, s % page] = rounded(v[m].float().cpu().numpy(), DT[dtype])
    wk, wv = in_pages(K, V, DT[dtype])
    assert torch.equal(kl.cpu(), wk) and torch.equal(vl.cpu(), wv)
    if strided:  # the other layer is as it was
        assert torch.equal(kp[:, 0].cpu(), pools[0][0]) and torch.equal(vp[:, 0].cpu(), pools[0][1])


# ---------------------------------------------------------------- paged_attention
def _run(c, q, window, a=None, max_per_row=None, qt=None):
    a = a or c.device(dev())
    qt = torch.from_numpy(q).to(dev(), c.dtype) if qt is None else qt
    return OPS.paged_attention(qt, a["k"], a["v"], a["tables"], a["row_off"], a["start"],
                               max_per_row or int(max(1, c.n.max())), window, a["pre"] if c.P else None, c.P)


def _check(got, ref, tol, what=""):
    got = got.double().cpu().numpy()
    bad = ~(np.abs(got - ref) <= tol)
    assert not bad.any(), (f"{what}: {bad.sum()} of {bad.size} outputs off, worst {np.nanmax(np.abs(got - ref) / tol)} "
                           f"of the bound, {np.isnan(got).sum()} NaN, first at {np.argwhere(bad)[0]}")


RAGGED = [3, 0, 1, 9, 5]
SHAPES = [
    # ctx, n, prefix, H, G, hd, page, window
    ([0], [1], 0, 1, 1, 128, 32, 0),                           # one key
    ([0], [1], 1, 4, 4, 128, 32, 0),                           # a prefix of one position
    ([640], [1], 0, 6, 6, 128, 64, 0),
    ([31, 32, 33, 0, 95], [1] * 5, 31, 6, 2, 128, 32, 0),      # borders of a tile
    ([5, 200, 0, 64, 131], RAGGED, 100, 12, 4, 128, 64, 0),
    ([5, 200, 0, 64, 131], RAGGED, 0, 12, 12, 128, 96, 0),
    ([5, 200, 0, 64, 131], RAGGED, 333, 8, 1, 128, 32, 0),     # 8 heads on one
    ([5, 200, 0, 64, 700], RAGGED, 333, 12, 4, 128, 32, 150),  # windows that end in the prefix and past it
    ([5, 2000, 0, 64, 700], RAGGED, 1000, 6, 6, 128, 256, 1),
    ([300, 0, 17], [40, 200, 0], 250, 6, 6, 128, 64, 0),       # prompt chunks
    ([300, 0, 17], [40, 200, 130], 0, 12, 4, 128, 128, 77),
    ([10, 450], [33, 2], 1500, 6, 2, 128, 64, 600),
    ([5, 200, 0, 64, 131], RAGGED, 100, 24, 8, 64, 32, 0),
    ([300, 0, 17], [40, 200, 0], 250, 3, 3, 64, 64, 190),
    ([5, 200, 0, 64, 131], RAGGED, 70, 6, 2, 96, 32, 0),
    ([5, 100], [2, 5], 70, 2, 2, 40, 32, 33),
    ([5, 100], [2, 5], 70, 2, 1, 256, 32, 0),
    ([3000], [1], 0, 2, 2, 128, 32, 0),                        # a long row, cut into splits
    ([40] * 70, [1] * 70, 600, 2, 2, 128, 32, 0),              # many rows
    ([0, 0], [0, 0], 10, 2, 2, 128, 32, 0),                    # no query at all
]


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("case", range(len(SHAPES)))
def test_paged_attention(dtype, case):
    """Against the softmax in 64 bits; every slot that no row holds is NaN,
    and tokens behind the last row come back as 0."""
    ctx, n, P, H, G, hd, page, window = SHAPES[case]
    _say(f"paged_attention {dtype} case {case}: {SHAPES[case]}")
    c = Paged(case, ctx, n, P, G, hd, page, DT[dtype])
    q = c.queries(H, tail=2)
    got = _run(c, q, window)
    torch.cuda.synchronize()
    ref, tol = c.reference(q, window)
    _check(got, ref, tol)
    assert torch.all(got[int(c.off[-1]):] == 0)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("hd", [128, 64, 96])
def test_rows_without_pages(dtype, hd):
    """Table and prefix entries that are no page (negative, past the pool)
    hold no keys; a query that sees none gets 0; the slots of the rows' own
    later positions, infinite here, stay out of earlier queries."""
    _say(f"paged_attention {dtype} hd={hd}: entries that are no page")
    c = Paged(5, [70, 10, 0, 130], [3, 5, 2, 4], 90, 2, hd, 32, DT[dtype])
    gone = [(0, 1), (1, 0), (2, 0), (3, 4), (-1, 1)]
    a = c.device(dev())
    a["tables"][0, 1], a["tables"][1, 0], a["tables"][2, 0], a["tables"][3, 4] = -1, c.N, 2 ** 31 - 1, -2 ** 31
    a["pre"][1] = c.N + 1
    q = c.queries(4)
    got = _run(c, q, 0, a)
    ref, tol = c.reference(q, 0, gone)
    _check(got, ref, tol, "no window")
    got = _run(c, q, 8, a)  # rows 1 and 2 see a window without keys in part
    ref, tol = c.reference(q, 8, gone)
    _check(got, ref, tol, "window")


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("hd", [128, 64])
@pytest.mark.parametrize("n", [6, 45, 150])
@pytest.mark.parametrize("junk", [NAN, INF])
def test_masked_values_of_later_queries(dtype, hd, n, junk):
    """K and V that only later queries of the same chunk see (here not finite)
    do not reach the earlier ones; nor do those behind a window."""
    _say(f"paged_attention {dtype} hd={hd} n={n}: {junk} at a later position")
    c = Paged(7, [37, 3], [n, 2], 50, 2, hd, 32, DT[dtype])
    q = c.queries(4)
    ref, tol = c.reference(q, 0)
    refw, tolw = c.reference(q, 20)
    clean = c.K.copy(), c.V.copy()
    at = 37 + n - 2  # row 0's last position but one
    for pool in (c.K, c.V):
        pool[c.tables[0, at // 32], :, at % 32] = junk
    got = _run(c, q, 0)
    _check(got[:n - 2], ref[:n - 2], tol[:n - 2], "causal")
    _check(got[n:], ref[n:], tol[n:], "the other row")
    c.K, c.V = clean
    for pool in (c.K, c.V):
        pool[c.pre_ids[1], :, 40 - 32] = junk  # prefix position 40: behind the windows of positions past 60
    got = _run(c, q, 20)
    _check(got[:n], refw[:n], tolw[:n], "window")  # (row 1, at positions 53 and 54, does see position 40)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_rows_that_start_inside_the_prefix(dtype):
    """A row's positions may begin before the prefix ends: it sees the prefix
    up to itself and none of its own pages."""
    _say(f"paged_attention {dtype}: positions inside the prefix")
    c = Paged(9, [40, 0, 3], [4, 3, 6], 100, 2, 128, 32, DT[dtype])
    c.start = np.array([140, 37, 98], np.int32)  # row 1: 37 .. 39; row 2: 98 .. 103
    q = c.queries(4)
    got = _run(c, q, 0)
    ref, tol = c.reference(q, 0)
    _check(got, ref, tol)


def test_bad_rows_and_tail():
    """A row with more tokens than max_per_row, or past the chunk's capacity,
    is treated as empty; the C entry leaves the tokens behind the last row."""
    _say("paged_attention: bad rows")
    from flaxchat_amd import _lib
    for dtype in (torch.bfloat16, torch.float32):
        c = Paged(11, [40, 7, 90], [2, 30, 3], 50, 2, 128, 32, dtype)
        q = c.queries(4, tail=4)
        ref, tol = c.reference(q, 0)
        got = _run(c, q, 0, max_per_row=5)
        for s in (slice(0, 2), slice(32, 35)):
            _check(got[s], ref[s], tol[s], "the other rows")
        a = c.device(dev())
        a["row_off"][3] = 1000
        got = _run(c, q, 0, a)
        _check(got[:32], ref[:32], tol[:32], "the rows before")
        a = c.device(dev())
        qt = torch.from_numpy(q).to(dev(), dtype)
        y = torch.full((39, 4 * 128), 7.0, device=dev(), dtype=dtype)
        N, G, page, hd = a["k"].shape
        p = _lib.FcPages(a["k"].data_ptr(), a["v"].data_ptr(), G * page * hd, G * page * hd, N, G, page, hd,
                         1 if dtype == torch.bfloat16 else 0)
        L = _lib.lib()
        nb = L.fc_paged_attention_workspace_bytes(p, 3, 39, 30, 4, c.W, c.P, 0)
        ws = torch.empty(max(nb, 1), dtype=torch.uint8, device=dev())
        _lib.check(L.fc_paged_attention(p, qt.data_ptr(), 512, 128, y.data_ptr(), 3, 39, 30, 4,
                                        a["tables"].data_ptr(), c.W, a["row_off"].data_ptr(), a["start"].data_ptr(),
                                        a["pre"].data_ptr(), c.P, 0, 0, ws.data_ptr(), nb,
                                        torch.cuda.current_stream().cuda_stream))
        torch.cuda.synchronize()
        _check(y[:35], ref[:35], tol[:35])
        assert torch.all(y[35:] == 7.0)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("hd", [128, 64])
def test_strided_and_unaligned(dtype, hd):
    """Pages of one layer of a pool of three, queries cut out of a fused
    projection, and arrays off the 16-byte boundary."""
    _say(f"paged_attention {dtype} hd={hd}: strides")
    c = Paged(13, [40, 7, 900], [2, 30, 3], 150, 2, hd, 32, DT[dtype])
    q = c.queries(6)
    ref, tol = c.reference(q, 0)
    a = c.device(dev())
    T = len(q)
    qkv = torch.full((T, 10, hd), NAN, device=dev(), dtype=c.dtype)
    qkv[:, 2:8] = torch.from_numpy(q).to(dev(), c.dtype)
    pool = {x: torch.full((c.N, 3, *a[x].shape[1:]), NAN, device=dev(), dtype=c.dtype) for x in "kv"}
    for x in "kv":
        pool[x][:, 1] = a[x]
    b = dict(a, k=pool["k"][:, 1], v=pool["v"][:, 1])
    _check(_run(c, q, 0, b, qt=qkv[:, 2:8]), ref, tol, "strided")
    qt = torch.from_numpy(q).to(dev(), c.dtype)
    _check(_run(c, q, 0, a, qt=qt.transpose(0, 1).contiguous().transpose(0, 1)), ref, tol, "heads first")
    _check(_run(c, q, 0, a, qt=qt.transpose(1, 2).contiguous().transpose(1, 2)), ref, tol, "dims not contiguous")
    off1 = lambda t: torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape)  # noqa: E731
    _check(_run(c, q, 0, a, qt=off1(qt)), ref, tol, "q off the boundary")
    _check(_run(c, q, 0, dict(a, k=off1(a["k"])), qt=qt), ref, tol, "K off the boundary")
    _check(_run(c, q, 0, dict(a, v=off1(a["v"])), qt=qt), ref, tol, "V off the boundary")
    odd = torch.full((c.N, a["k"][0].numel() + 1), NAN, device=dev(), dtype=c.dtype)
    kk = odd[:, :-1].unflatten(1, a["k"].shape[1:])
    kk.copy_(a["k"])
    _check(_run(c, q, 0, dict(a, k=kk), qt=qt), ref, tol, "an odd page stride")


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_prefix_equals_copies(dtype):
    """The same keys once as a shared prefix and once in every row's own
    pages give the same attention (both within the bound)."""
    _say(f"paged_attention {dtype}: prefix against copies")
    c = Paged(17, [20, 33, 0, 250], [7, 1, 4, 2], 320, 3, 128, 64, DT[dtype])
    q = c.queries(6)
    ref, tol = c.reference(q, 0)
    _check(_run(c, q, 0), ref, tol, "prefix")
    a = c.device(dev())
    tables = np.concatenate([np.tile(c.pre_ids, (4, 1)), c.tables], 1)  # 320 = 5 pages of 64
    got = OPS.paged_attention(torch.from_numpy(q).to(dev(), c.dtype), a["k"], a["v"], up(tables), a["row_off"],
                              a["start"], 7, 0)
    _check(got, ref, tol, "copies")


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_same_as_the_contiguous_operator(dtype):
    """A layer of a contiguous cache is a pool whose rows are its pages."""
    _say(f"paged_attention {dtype}: on a contiguous cache")
    rng = np.random.default_rng(3)
    B, G, H, cap = 3, 2, 4, 160
    kc = torch.from_numpy(rng.standard_normal((B, G, cap, 128)).astype(np.float32)).to(dev(), DT[dtype])
    vc = torch.from_numpy(rng.standard_normal((B, G, cap // 32, 128, 32)).astype(np.float32)).to(dev(), DT[dtype])
    off, start = up([0, 3, 4, 9]), up([90, 3, 151])
    q = torch.from_numpy(rng.standard_normal((9, H, 128)).astype(np.float32)).to(dev(), DT[dtype])
    want = OPS.attention(q, kc, vc, off, start, 5, 0).double()
    got = OPS.paged_attention(q, kc, vc, up([[0], [1], [2]]), off, start, 5, 0).double()
    # two results of the same kind: each within 2^-8 (A + |y|) of the truth in bf16, with A <= max |v| ~ 4.5
    tol = 2 * 2.0 ** -8 * 9 if dtype == "bf16" else 1e-5
    assert (got - want).abs().max() <= tol


def test_side_stream_and_graph():
    """On another stream than the default one, and captured: the whole step
    (tables, append, attention) replayed with new lengths between replays and
    eager work in between equals the eager step on the same state."""
    _say("paged ops: side stream and graph")
    rng = np.random.default_rng(21)
    B, G, H, hd, page, W, P, T = 6, 2, 6, 128, 32, 12, 70, 24
    N = 90
    mk = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32)).to(dev(), torch.bfloat16)  # noqa: E731

    def fresh():
        r = np.random.default_rng(5)
        return dict(tables=up(np.full((B, W), -1)), held=up([0] * B), free=up(r.permutation(N - 3)), nf=up([N - 3]),
                    off=up([0] * (B + 1)), start=up([0] * B), row=up([0] * T), pos=up([0] * T), slots=up([0] * T))

    pools = mk(N, G, page, hd), mk(N, G, page // 32, hd, 32)
    pre = up([N - 3, N - 2, N - 1])
    qkv = mk(T, H + 2 * G, hd)
    length, n_new = up([0] * B), up([0] * B)

    def step(s, kp, vp):
        OPS.page_tables(s["tables"], s["held"], s["free"], s["nf"], length, n_new, s["off"], s["start"], s["row"],
                        s["pos"], s["slots"], page, P)
        OPS.page_append(qkv[:, H:H + G], qkv[:, H + G:], s["slots"], kp, vp)
        return OPS.paged_attention(qkv[:, :H], kp, vp, s["tables"], s["off"], s["start"], T, 0, pre, P)

    a, b = fresh(), fresh()
    ka, va = (p.clone() for p in pools)
    kb, vb = (p.clone() for p in pools)
    side = torch.cuda.Stream(device=dev())
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm = fresh()
        step(warm, ka.clone(), va.clone())
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        y = step(a, ka, va)
    lens = np.zeros(B, np.int64)
    for rep in range(5):
        n = rng.integers(0, 5, B)
        n[rep % B] = -1 if rep > 1 else 3
        length.copy_(up(lens))
        n_new.copy_(up(n))
        qkv.copy_(mk(T, H + 2 * G, hd))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        ref = step(b, kb, vb)
        torch.cuda.synchronize()
        assert torch.equal(y, ref), f"replay {rep}"
        for x in a:
            assert torch.equal(a[x], b[x]), f"replay {rep}: {x}"
        assert torch.equal(ka, kb) and torch.equal(va, vb)
        assert int(b["off"][-1]) == int(np.maximum(n, 0).sum())
        lens = np.where(n < 0, 0, lens + np.maximum(n, 0))


def test_pool_past_32_bits():
    """Pages whose elements lie past 2^31 (bf16) of the pool."""
    _say("paged ops: a pool of more than 2^31 elements")
    G, hd, page = 8, 128, 256
    N = (2 ** 31 // (G * hd * page)) + 40
    k = torch.empty(N, G, page, hd, device=dev(), dtype=torch.bfloat16)
    v = torch.empty(N, G, page // 32, hd, 32, device=dev(), dtype=torch.bfloat16)
    c = Paged(31, [500, 90], [3, 1], 300, G, hd, page, torch.bfloat16, extra=0)
    shift = N - c.N  # the pages of the small pool sit at the large one's end
    a = c.device(dev())
    k[shift:], v[shift:] = a["k"], a["v"]
    new = torch.from_numpy(c.rng.standard_normal((2, 4, G, hd)).astype(np.float32)).to(dev())
    slots = []
    for b, (cx, m) in enumerate(zip(c.ctx, c.n)):
        p = np.arange(cx, cx + m)
        slots += (c.tables[b][p // page].astype(np.int64) * page + p % page + shift * page).tolist()
    OPS.page_append(new[0], new[1], up(slots), k, v)
    for j in range(2):
        x = rounded(new[j].cpu().numpy(), torch.bfloat16)
        c.rows[0][j][500:], c.rows[1][j][90:] = x[:3], x[3:]
    q = c.queries(16)
    ref, tol = c.reference(q, 0)
    b = dict(a, k=k, v=v, tables=a["tables"] + shift, pre=a["pre"] + shift)
    b["tables"][a["tables"] < 0] = -1
    _check(_run(c, q, 0, b), ref, tol)


# ---------------------------------------------------------------- together
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_decode_loop(dtype):
    """A batch of continuations of one prompt over several steps, as a server
    runs them: rows of unequal progress, a rollback, a row that ends and whose
    pages another takes; every step's attention against the softmax in 64
    bits over the rows' whole history."""
    _say(f"paged ops: decode loop {dtype}")
    rng = np.random.default_rng(41)
    B, G, H, hd, page, W, P = 4, 2, 4, 128, 32, 6, 75
    dt = DT[dtype]
    N = 3 + 9  # the rows' 9 pages run short in the end
    c = Paged(2, [0] * B, [0] * B, P, G, hd, page, dt, extra=N - 3)
    a = c.device(dev())
    kp, vp = a["k"], a["v"]
    others = [i for i in range(N) if i not in c.pre_ids]
    T = 200
    s = dict(tables=up(np.full((B, W), -1)), held=up([0] * B), free=up(others), nf=up([len(others)]),
             off=up([0] * (B + 1)), start=up([0] * B), row=up([0] * T), pos=up([0] * T), slots=up([0] * T))
    hist = [(np.zeros((0, G, hd), np.float32),) * 2 for _ in range(B)]
    plan = [([60, 20, 1, 31], None), ([1, 7, 1, 1], None), ([5, 7, 5, 5], (1, 4)), ([-1, 7, 40, 0], None),
            ([30, 9, 1, 1], None), ([90, 10, 90, 20], None)]  # 2 free pages at the end: rows 0 and 2 need 3 each
    for step, (n, back) in enumerate(plan):
        lens = np.array([len(h[0]) for h in hist])
        qkv = rounded(rng.standard_normal((T, H + 2 * G, hd)), dt)
        dq = torch.from_numpy(qkv).to(dev(), dt)
        OPS.page_tables(s["tables"], s["held"], s["free"], s["nf"], up(lens), up(n), s["off"], s["start"], s["row"],
                        s["pos"], s["slots"], page, P)
        OPS.page_append(dq[:, H:H + G], dq[:, H + G:], s["slots"], kp, vp)
        got = OPS.paged_attention(dq[:, :H], kp, vp, s["tables"], s["off"], s["start"], T, 0, a["pre"], P)
        off = s["off"].cpu().numpy()
        took = np.diff(off)
        assert took.tolist() == ([max(x, 0) for x in n] if step < 5 else [0, 10, 0, 20]), f"step {step}"
        for b in range(B):
            if n[b] < 0:
                hist[b] = (np.zeros((0, G, hd), np.float32),) * 2
            sl = slice(off[b], off[b + 1])
            hist[b] = tuple(np.concatenate([hist[b][j], qkv[sl, H + j * G:H + (j + 1) * G]]) for j in range(2))
        r = Paged.__new__(Paged)
        r.P, r.G, r.hd, r.page, r.dtype, r.B, r.pre, r.rows = P, G, hd, page, dt, B, c.pre, hist
        r.n, r.off = took, off
        r.start = np.array([P + len(h[0]) - m for h, m in zip(hist, took)])
        ref, tol = r.reference(qkv[:, :H], 0)
        _check(got, ref, tol, f"step {step}")
        if back:
            hist[back[0]] = tuple(x[:-back[1]] for x in hist[back[0]])


@pytest.mark.parametrize("hd,H,G", [(128, 4, 2), (64, 6, 2)])
@pytest.mark.parametrize("P,window", [(0, 0), (0, 100), (1, 0), (33, 0), (96, 40), (500, 333), (1500, 1024)])
@pytest.mark.parametrize("ctx,n", [
    ([0, 5, 31, 200], [130, 1, 64, 0]),          # short rows: each one's keys are one piece
    ([1500, 0, 700], [90, 20, 150]),             # pieces of long rows beside a short one's whole
    ([40] * 40, [66, 0, 1, 130] * 10),           # more column blocks than workgroups at once
])
def test_prompts_behind_a_prefix(hd, H, G, P, window, ctx, n):
    """Rows of many query columns: prefixes that end inside a block of 32 keys,
    windows that reach back over their end, and rows that are cut into pieces
    beside rows that are not."""
    _say(f"paged_attention hd={hd} prefix {P} window {window}: rows of {n[:4]} tokens at {ctx[:4]}")
    c = Paged(23, ctx, n, P, G, hd, 64, torch.bfloat16)
    q = c.queries(H, tail=3)
    got = _run(c, q, window)
    ref, tol = c.reference(q, window)
    _check(got, ref, tol)
    assert torch.all(got[int(c.off[-1]):] == 0)
    # a V that is not finite at a position that only the row's last two queries see
    if window == 0:
        b = int(np.argmax(c.n))
        at = int(c.ctx[b] + c.n[b]) - 2
        c.V[c.tables[b, at // 64], :, at % 64] = INF
        got = _run(c, q, window)
        keep = np.ones(len(q), bool)
        keep[c.off[b + 1] - 2:c.off[b + 1]] = False
        _check(got[keep], ref[keep], tol[keep], "a later position's V")


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("B,most,P,window", [
    (70, 3, 0, 0), (256, 9, 40, 0), (257, 3, 0, 0), (300, 20, 33, 0), (300, 70, 0, 25), (1030, 2, 10, 0),
    (4096, 1, 0, 0),  # the most there may be
])
def test_many_rows(dtype, B, most, P, window):
    """Rows by the hundred, a few of them long and many without a token, in
    blocks of 16, 32 and 128 columns."""
    _say(f"paged_attention {dtype}: {B} rows of up to {most} tokens, prefix {P}, window {window}")
    r = np.random.default_rng(B)
    ctx, n = r.integers(0, 40, B), r.integers(0, most + 1, B)
    ctx[r.integers(0, B, 3)] = 700
    n[[0, B - 1]] = most
    c = Paged(29, ctx, n, P, 1, 128, 32, DT[dtype])
    q = c.queries(2, tail=1)
    got = _run(c, q, window)
    ref, tol = c.reference(q, window)
    _check(got, ref, tol)
    assert torch.all(got[int(c.off[-1]):] == 0)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("n,window", [(3, 40), (3, 0), (45, 40)])
def test_last_positions(dtype, n, window):
    """A table of 2^31 - 32 positions, all but the last two pages without an
    entry: the arithmetic of positions and pieces at the end of its range."""
    _say(f"paged_attention {dtype}: {n} tokens at the last positions, window {window}")
    W, N = 2 ** 26 - 1, 4
    c = Paged(31, [64 - n], [n], 0, 2, 128, 32, DT[dtype], extra=2)  # 64 positions: the last two pages
    assert c.N == N
    a = c.device(dev())
    tables = torch.full((1, W), -1, dtype=torch.int32, device=dev())
    tables[0, -2:] = a["tables"][0]
    q = c.queries(4)
    got = _run(c, q, window, dict(a, tables=tables, start=up([32 * W - n])))
    ref, tol = c.reference(q, window)
    _check(got, ref, tol)


@pytest.mark.parametrize("hd", [128, 64])
@pytest.mark.parametrize("window", [0, 30])
def test_many_rows_and_a_long_one(hd, window):
    """300 rows of few tokens and one of column blocks, behind 40 keys."""
    _say(f"paged_attention hd={hd} window {window}: 300 rows, one long")
    n = np.arange(300) % 4
    n[150] = 130
    c = Paged(37, np.arange(300) * 7 % 50, n, 40, 2, hd, 32, torch.bfloat16)
    q = c.queries(2, tail=1)
    ref, tol = c.reference(q, window)
    _check(_run(c, q, window), ref, tol)


@pytest.mark.parametrize("hd,window", [(128, 1000), (64, 0)])
def test_many_blocks_behind_a_long_prefix(hd, window):
    """Full column blocks for several rounds of workgroups, which then walk a
    prefix past 1024 keys themselves."""
    _say(f"paged_attention hd={hd} window {window}: many blocks behind 1100 keys")
    n = [16] * 97
    n[3], n[90] = 15, 0
    c = Paged(41, np.arange(97) * 7 % 50, n, 1100, 16, hd, 32, torch.bfloat16)
    q = c.queries(128, tail=1)
    got = _run(c, q, window)
    rows = [2, 3, 4, 90, 91, 96]  # of which the result is looked at
    sub = Paged.__new__(Paged)
    sub.__dict__.update(c.__dict__)
    sub.n = np.where(np.isin(np.arange(97), rows), c.n, 0)
    ref, tol = sub.reference(q, window)
    at = np.concatenate([np.arange(c.off[b], c.off[b + 1]) for b in rows])
    _check(got[at], ref[at], tol[at])
    whole = got[:int(c.off[-1])]
    assert torch.isfinite(whole).all() and (whole != 0).any(1).all()


@pytest.mark.parametrize("fill", [(-INF, 0.0), (NAN, NAN), (0.0, -1.0)])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("ctx,n,P", [([3000, 5, 700], [1, 3, 2], 0), ([3000, 5, 700], [1, 3, 2], 40),
                                     ([2500, 5, 0], [140, 3, 20], 33)])
def test_workspace_holds_anything(fill, dtype, ctx, n, P):
    """What an earlier call left in the workspace (marks of pieces without
    keys, of whole ones) decides nothing, for tokens behind the last row
    either."""
    from flaxchat_amd import _lib
    _say(f"paged_attention {dtype}: workspace full of {fill}, prefix {P}")
    c = Paged(43, ctx, n, P, 2, 128, 32, DT[dtype])
    q = c.queries(4, tail=5)
    ref, tol = c.reference(q, 0)
    a, T, most = c.device(dev()), len(q), int(max(n))
    qt = torch.from_numpy(q).to(dev(), c.dtype)
    N, G, page, hd = a["k"].shape
    p = _lib.FcPages(a["k"].data_ptr(), a["v"].data_ptr(), G * page * hd, G * page * hd, N, G, page, hd,
                     1 if dtype == "bf16" else 0)
    L = _lib.lib()
    nb = L.fc_paged_attention_workspace_bytes(p, 3, T, most, 4, c.W, P, 0)
    assert nb > 0
    room = torch.tensor(fill, device=dev()).repeat(nb // 4 + 1024)  # the middle half is the call's
    at = (room.numel() - nb // 4) // 2 // 64 * 64
    ws = room[at:at + nb // 4]
    y = torch.full((T, 4 * 128), 7.0, device=dev(), dtype=c.dtype)
    _lib.check(L.fc_paged_attention(p, qt.data_ptr(), 512, 128, y.data_ptr(), 3, T, most, 4, a["tables"].data_ptr(),
                                    c.W, a["row_off"].data_ptr(), a["start"].data_ptr(), a["pre"].data_ptr() or None,
                                    P, 0, 1, ws.data_ptr(), nb, torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    _check(y, ref, tol)
    assert torch.all(y[int(c.off[-1]):] == 0)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("n", [3, 45])
@pytest.mark.parametrize("window", [70, 300])
def test_windows_far_apart_in_the_prefix(dtype, n, window):
    """Rows that begin within the prefix, a thousand positions from each
    other: one column block's windows lie all over it."""
    _say(f"paged_attention {dtype}: rows of {n} at 100, 1000, 1990 and 2050, window {window}")
    c = Paged(47, [0, 0, 0, 50], [n] * 4, 2000, 2, 128, 32, DT[dtype])
    c.start = np.array([100, 1000, 1990, 2050], np.int32)
    q = c.queries(4)
    ref, tol = c.reference(q, window)
    _check(_run(c, q, window), ref, tol)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_two_calls_at_once_and_replays(dtype):
    """A captured call over many rows replayed on one stream while others of
    other shapes run on a second one: each as it is alone, bit for bit."""
    _say(f"paged_attention {dtype}: two streams, a graph of 300 rows")
    n = np.arange(300) % 4
    n[150] = 130
    big = Paged(37, np.arange(300) * 7 % 50, n, 40, 2, 128, 32, DT[dtype])
    small = Paged(53, [3000, 5, 700], [1, 3, 2], 333, 2, 128, 32, DT[dtype])
    calls = []
    for c in (big, small):
        a, q = c.device(dev()), torch.from_numpy(c.queries(4, tail=1)).to(dev(), c.dtype)
        calls.append(lambda c=c, a=a, q=q: _run(c, None, 100, a, qt=q))
    alone = [f().clone() for f in calls]
    torch.cuda.synchronize()
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(one):
        calls[0]()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=one):
        y = calls[0]()
    for _ in range(4):
        y.fill_(7.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(one):
            graph.replay()
        with torch.cuda.stream(two):
            got = [calls[1]() for _ in range(3)] + [calls[0]()]
        torch.cuda.synchronize()
        assert torch.equal(y, alone[0]) and torch.equal(got[3], alone[0])
        assert all(torch.equal(g, alone[1]) for g in got[:3])
