"""paged_attention at the ends of what it accepts, and where the tests of
tests/test_gpu_paged.py cannot tell: against the softmax in 64 bits, and
against whole numbers that one key more or less changes."""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from tests.paged_cases import Paged  # noqa: E402
from tests.test_gpu_kernels import _say  # noqa: E402
from tests.test_gpu_paged import DT, INF, OPS, _check, _run, dev, up  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("n,window", [(3, 20), (3, 90), (3, 0), (45, 5), (45, 20)])
def test_last_positions_with_values_not_finite(dtype, n, window):
    """The last positions of a table of 2^31 - 32, whose last two V are infinite: the
    queries ahead of those go over their keys in the plain form, whose
    arithmetic has to end at the last position."""
    _say(f"paged_attention {dtype}: {n} tokens at the last positions, window {window}, V not finite")
    W = 2 ** 26 - 1
    c = Paged(31, [64 - n], [n], 0, 2, 128, 32, DT[dtype], extra=2)  # 64 positions: the last two pages
    q = c.queries(4)
    ref, tol = c.reference(q, window)
    c.V[c.tables[0, 1], :, 30:] = INF
    a = c.device(dev())
    tables = torch.full((1, W), -1, dtype=torch.int32, device=dev())
    tables[0, -2:] = a["tables"][0]
    got = _run(c, q, window, dict(a, tables=tables, start=up([32 * W - n])))
    _check(got[:n - 2], ref[:n - 2], tol[:n - 2])
    assert not torch.isfinite(got[n - 2:]).any()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("B,n", [(1, 3), (2, 9)])
@pytest.mark.parametrize("inside,window", [(False, 0), (False, 40), (True, 0), (True, 17)])
def test_longest_prefix(dtype, B, n, inside, window):
    """A prefix of 2^31 - 33 positions, of which the last 63 are held: rows
    behind it, and rows that begin in it ahead of a V that is infinite."""
    P = 2 ** 31 - 33
    _say(f"paged_attention {dtype}: {B} rows of {n} {'within' if inside else 'behind'} the longest prefix, {window}")
    c = Paged(59, [10 + b for b in range(B)], [n] * B, 63, 2, 128, 32, DT[dtype])
    c.start = np.array([63 - n if inside else 63 + 10 + b for b in range(B)], np.int32)
    q = c.queries(4)
    ref, tol = c.reference(q, window)
    if inside:  # the last position is a row's last query's alone
        c.V[c.pre_ids[1], :, 30] = INF
    a = c.device(dev())
    pre = torch.full((2 ** 26 - 1,), -1, dtype=torch.int32, device=dev())
    pre[-2:] = a["pre"]
    got = OPS.paged_attention(torch.from_numpy(q).to(dev(), c.dtype), a["k"], a["v"], a["tables"], a["row_off"],
                              up(c.start.astype(np.int64) + (P - 63)), n, window, pre, P)
    keep = np.arange(len(q)) % n < (n - 1 if inside else n)
    _check(got[keep], ref[keep], tol[keep])
    assert not torch.isfinite(got[~keep]).any()


def test_written_tensors_are_seen_by_autograd():
    """A pool that autograd keeps for a backward pass and that page_append then
    writes to is noticed there, as are the tables that page_tables writes."""
    _say("page_append, page_tables: versions")
    f = dict(device=dev(), dtype=torch.float32)
    kp, vp = torch.ones(2, 1, 32, 128, **f), torch.ones(2, 1, 1, 128, 32, **f)
    x = torch.ones_like(kp, requires_grad=True)
    y = (x * kp).sum()
    k = torch.ones(1, 1, 128, **f)
    OPS.page_append(k, k, up([3]), kp, vp)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with pytest.raises(ValueError, match="backward"):
        OPS.page_append(k, k.clone().requires_grad_(), up([3]), kp, vp)
    s = [up(a) for a in ([[-1, -1]], [0], [0, 1], [2], [0], [1], [0, 0], [0], [0], [0], [0])]
    OPS.page_tables(*s, 32, 0)
    assert [t._version for t in s] == [1, 1, 1, 1, 0, 0, 1, 1, 1, 1, 1]
    with torch.inference_mode():  # tensors made here have no version
        kp, vp, k = torch.ones(2, 1, 32, 128, **f), torch.ones(2, 1, 1, 128, 32, **f), torch.zeros(1, 1, 128, **f)
        OPS.page_append(k, k, up([3]), kp, vp)
        assert int((kp == 0).sum()) == 128 and int((vp == 0).sum()) == 128


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("n", [1, 30])
def test_a_row_of_one_key_more_than_a_piece(dtype, n):
    """Beside a row of 1.69e9 positions, of which a 64th is a piece, one of one
    key more than that: float has no room for the one, the sums have to."""
    piece = 26433600
    _say(f"paged_attention {dtype}: {n} tokens up to key {piece}")
    c = Paged(61, [0, 97 - n], [1, n], 0, 2, 128, 32, DT[dtype])
    q = c.queries(4)
    ref, tol = c.reference(q, 0, gone=[(0, 0)])  # the long row holds no page at all
    a = c.device(dev())
    tables = torch.full((2, piece * 64 // 32), -1, dtype=torch.int32, device=dev())
    tables[1, piece // 32 - 3:piece // 32 + 1] = a["tables"][1, :4]
    got = _run(c, q, 0, dict(a, tables=tables, start=up([64 * piece - 1, piece + 1 - n])))
    _check(got, ref, tol)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("B,W,most", [(64, 2 ** 22, 1), (64, 2 ** 22, 20), (300, 2 ** 20, 1)])
def test_short_rows_in_wide_tables(dtype, B, W, most):
    """Rows of up to a few hundred positions in tables of 2^25 and 2^27, in
    front of which the table's own length would ask for 2^24 workgroups."""
    _say(f"paged_attention {dtype}: {B} rows of up to {most} tokens, tables of {W} pages")
    r = np.random.default_rng(B)
    n = r.integers(0, most + 1, B) if most > 1 else np.ones(B, int)
    c = Paged(67, r.integers(0, 200, B), n, 0, 8, 64, 32, DT[dtype])
    q = c.queries(8)
    ref, tol = c.reference(q, 0)
    a = c.device(dev())
    tables = torch.full((B, W), -1, dtype=torch.int32, device=dev())
    tables[:, :c.W] = a["tables"]
    _check(_run(c, q, 0, dict(a, tables=tables)), ref, tol)


def test_append_of_very_many_tokens():
    """More tokens than a launch has room for at 32 a workgroup, nearly all of
    them without a slot."""
    M = 2 ** 29 + 5
    _say(f"page_append: {M} tokens")
    one = torch.arange(1, 9, device=dev(), dtype=torch.bfloat16).view(1, 1, 8)
    k = one.expand(M, 1, 8)
    slots = torch.full((M,), -1, dtype=torch.int32, device=dev())
    slots[[0, 2 ** 28, M - 1]] = up([5, 40, 63])
    kp = torch.zeros(2, 1, 32, 8, device=dev(), dtype=torch.bfloat16)
    vp = torch.zeros(2, 1, 1, 8, 32, device=dev(), dtype=torch.bfloat16)
    OPS.page_append(k, k, slots, kp, vp)
    rows = torch.zeros(64, 8)
    rows[[5, 40, 63]] = torch.arange(1.0, 9.0)
    assert torch.equal(kp.float().cpu().view(64, 8), rows)
    assert torch.equal(vp.float().cpu().view(2, 8, 32).transpose(1, 2).reshape(64, 8), rows)


def test_pages_given_back_past_the_stack():
    """Pages that the stack has no room for are not on it, and the ended row's
    table still names them: put back by the caller, they are handed out."""
    _say("page_tables: a stack of two for three pages")
    s = [up(a) for a in ([[4, 5, 6], [-1] * 3], [3, 0], [-1, -1], [0], [70, 0], [-1, 0], [0] * 3, [0] * 2, [0] * 70,
                         [0] * 70, [0] * 70)]
    OPS.page_tables(*s, 32, 0)
    assert s[2].tolist() == [4, 5] and s[3].item() == 2 and s[1].tolist() == [0, 0]
    assert s[0][0].tolist() == [4, 5, 6]
    s[2] = up([4, 5, 6])  # a stack with room
    s[3].fill_(3)
    s[4:6] = up([0, 0]), up([0, 70])
    OPS.page_tables(*s, 32, 0)
    assert s[0][1].tolist() == [6, 5, 4] and s[1].tolist() == [0, 3] and s[3].item() == 0


# ---------------------------------------------------------------- every key counted once
def _counted(c, H, window, div, gone=()):
    """With queries of 0 every visible key weighs 1, and with V of one 1 at dim (position // div + 17 head) % head_dim
    the output times the number of keys is how many visible keys have that dim: whole numbers, exact in the
    sums, and off by at most 2^-8 of themselves in a bf16 result, so by less than a half up to 127. Writes those V
    into c; returns (counts [T][H][hd], keys [T])."""
    P, page, hd, G = c.P, c.page, c.hd, c.G
    counts, keys = np.zeros((int(c.off[-1]), H, hd), np.int64), np.zeros(int(c.off[-1]), np.int64)
    for b in range(c.B):
        L = P + int(c.ctx[b] + c.n[b])
        at, there = np.arange(L), np.ones(L, bool)
        for r, j in gone:
            if r == b:
                there[P + j * page:P + (j + 1) * page] = False
            elif r == -1:
                there[j * page:min(P, (j + 1) * page)] = False
        for first, last, table in ((0, P, c.pre_ids), (P, L, c.tables[b])):
            i = np.arange(first, last) - first
            pid = np.asarray(table)[i // page]
            for g in range(G):
                c.V[pid, g, i % page] = (at[first:last, None] // div + 17 * g) % hd == np.arange(hd)
        hot = ((at[:, None, None] // div + 17 * np.arange(G)[:, None]) % hd == np.arange(hd)) & there[:, None, None]
        upto = np.concatenate([np.zeros((1, G, hd), np.int64), hot.cumsum(0)])
        n_upto = np.concatenate([[0], there.cumsum()])
        pos = c.start[b] + np.arange(c.n[b])
        lo = np.maximum(0, pos - window) if window > 0 else 0 * pos
        seen = np.s_[c.off[b]:c.off[b] + c.n[b]]
        counts[seen] = (upto[pos + 1] - upto[lo]).repeat(H // G, 1)
        keys[seen] = n_upto[pos + 1] - n_upto[lo]
    assert counts.max() < 128
    return counts, keys


COUNTED = [
    # ctx, n, prefix, start (None: behind the prefix), H, G, hd, page, window
    ([5, 700, 0, 64, 131], [3, 0, 1, 9, 5], 7003, None, 12, 4, 128, 64, 0),     # a long prefix, few tokens
    ([10, 450, 90], [33, 2, 60], 6001, None, 6, 2, 128, 96, 0),                 # and many
    ([10, 450, 90], [33, 2, 60], 6001, None, 6, 2, 128, 32, 3000),
    ([10, 450, 90], [33, 2, 60], 5000, None, 4, 4, 64, 64, 0),
    ([300, 0, 17], [140, 200, 130], 250, None, 6, 6, 128, 64, 0),               # prompts that walk a short prefix
    ([300, 0, 17], [140, 200, 130], 999, None, 4, 2, 64, 32, 700),              # themselves
    ([300, 0, 17, 0], [140, 200, 130, 20], 1023, [1323, 900, 500, 1010], 4, 2, 128, 32, 0),  # rows that begin in it
    ([300, 0, 17, 0], [140, 200, 130, 20], 1023, [1323, 900, 500, 1010], 4, 2, 128, 64, 300),
    ([7000, 3, 2500], [1, 1, 1], 0, None, 6, 6, 128, 64, 0),                    # long rows, cut into pieces
    ([7000, 3, 2500], [1, 1, 1], 2000, None, 16, 2, 128, 32, 0),
    ([7000, 3, 2500], [12, 1, 7], 0, None, 4, 2, 128, 256, 0),
    ([7000, 3, 2500], [90, 120, 7], 0, None, 4, 2, 128, 96, 0),
    ([7000, 3, 2500], [90, 120, 7], 0, None, 4, 2, 64, 32, 4000),
    ([5000, 40, 3000], [200, 129, 64], 500, None, 4, 2, 128, 64, 0),            # pieces that begin in the prefix
    ([50 * (i % 40) for i in range(300)], [i % 3 for i in range(300)], 777, None, 2, 2, 128, 32, 0),
    ([50 * (i % 40) for i in range(300)], [i % 3 for i in range(300)], 0, None, 2, 1, 64, 32, 900),
    ([7 * i % 50 for i in range(97)], [16] * 97, 1100, None, 128, 16, 128, 32, 0),  # rounds of blocks behind 1100 keys
    ([9 * i % 70 for i in range(30)], [40] * 30, 1500, [1500 - 40 * (i % 9) for i in range(30)], 4, 4, 128, 32, 0),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("case", range(len(COUNTED)))
def test_every_key_counts_once(dtype, case):
    """No key left out or taken twice at a border of tiles, pages, pieces,
    splits or of the prefix, however many keys there are."""
    ctx, n, P, start, H, G, hd, page, window = COUNTED[case]
    _say(f"paged_attention {dtype} counted case {case}: {len(n)} rows, prefix {P}, window {window}")
    c = Paged(case, ctx, n, P, G, hd, page, DT[dtype])
    if start is not None:
        c.start = np.array(start, np.int32)
    q = np.zeros((int(c.off[-1]), H, hd), np.float32)
    for div in (1, 32):
        counts, keys = _counted(c, H, window, div)
        got = _run(c, q, window).double().cpu().numpy().reshape(counts.shape) * keys[:, None, None]
        assert np.abs(got - counts).max() < 0.5, f"div {div}: {np.argwhere(np.abs(got - counts) >= 0.5)[:4].tolist()}"


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("hd", [128, 64, 96])
@pytest.mark.parametrize("n", [[3, 5, 2], [45, 20, 9], [150, 130, 3]])
def test_counted_keys_without_pages(dtype, hd, n):
    """The same where entries of the tables and of the prefix are no page, and
    where a position that only a row's last two queries see holds an infinity."""
    _say(f"paged_attention {dtype} hd={hd}: rows of {n} tokens, entries that are no page, an infinity")
    c = Paged(71, [170, 10, 600], n, 290, 2, hd, 32, DT[dtype])
    gone = [(0, 1), (2, 0), (2, 18), (-1, 3), (-1, 9)]
    q = np.zeros((int(c.off[-1]), 4, hd), np.float32)
    for window in (0, 250):
        counts, keys = _counted(c, 4, window, 1, gone)
        at = 170 + n[0] - 2
        assert at // 32 != 1
        c.V[c.tables[0, at // 32], :, at % 32] = INF
        a = c.device(dev())
        a["tables"][0, 1], a["tables"][2, 0], a["tables"][2, 18] = -1, c.N, 2 ** 31 - 1
        a["pre"][3], a["pre"][9] = -2 ** 31, c.N + 1
        got = _run(c, q, window, a).double().cpu().numpy().reshape(counts.shape) * keys[:, None, None]
        keep = np.ones(len(q), bool)
        keep[n[0] - 2:n[0]] = False
        assert np.abs(got - counts)[keep].max() < 0.5, f"window {window}"
        assert not np.isfinite(got[~keep]).any()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("window", [0, 60])
def test_contiguous_and_paged_within_the_bound(dtype, window):
    """attention on a contiguous cache and paged_attention on the same cache as
    a pool of one page a row: both as near the softmax as the bound of each
    output says."""
    _say(f"attention and paged_attention {dtype}, window {window}")
    c = Paged(73, [90, 3, 151, 0], [5, 1, 9, 40], 0, 2, 128, 160, DT[dtype], junk=0.0)
    q = c.queries(4)
    ref, tol = c.reference(q, window)
    a = c.device(dev())
    _check(_run(c, q, window, a), ref, tol, "paged")
    ids = a["tables"][:, 0].long()
    qt = torch.from_numpy(q).to(dev(), c.dtype)
    got = OPS.attention(qt, a["k"][ids], a["v"][ids], a["row_off"], a["start"], 40, window)
    _check(got, ref, tol, "contiguous")
    as_pool = dict(a, k=a["k"][ids], v=a["v"][ids], tables=up(np.arange(4)[:, None]))
    _check(_run(c, q, window, as_pool), ref, tol, "the cache as a pool")
