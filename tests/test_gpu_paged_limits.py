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
