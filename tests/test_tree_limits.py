"""Trees of drafted tokens at their limits, without a GPU: windows shorter than a tree is deep, norms past fp32."""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import flaxchat_amd.torch_ops  # noqa: E402,F401
from flaxchat_amd import _lib  # noqa: E402
from tests.test_tree import OPS, rope_args, tables_args  # noqa: E402
from tests.tree_cases import Tree, line_of, trees  # noqa: E402


def within(seen, depth, window):
    """Of the nodes that each of a row's nodes sees ([n][n]) those at most `window` positions above it (0: all)."""
    d = np.asarray(depth)
    return seen & (d[:, None] - d[None] <= window) if window > 0 else seen


def narrowed(c, window):
    """The rows, keys and nodes of c; its nodes see their ancestors as far as the window reaches."""
    c.seen = [within(s, d, window) for s, d in zip(c.seen, c.depth)]
    return c


@pytest.mark.parametrize("n,ctx,window", [(200, 40, 128), (40, 40, 16), (9, 0, 1), (5, 100, 4), (5, 100, 3)])
def test_a_chain_behind_a_window_is_plain_decoding(n, ctx, window):
    """Two 64-bit references of one thing: a chain of nodes with the windowed mask, and a plain chunk."""
    c = Tree(3, [ctx, 7], [n, 3], 10, 1, 8, 32, torch.float32, kinds=["chain"])
    q = c.queries(1)
    want = c.reference(q, window)[0]
    deeper = np.abs(c.tree_reference(q, window)[0] - want).max()
    assert (deeper > 1e-3) == (n > window + 1)  # the mask of all ancestors is another one exactly there
    np.testing.assert_allclose(narrowed(c, window).tree_reference(q, window)[0], want, atol=1e-12)


def test_each_node_is_its_path_decoded_token_by_token():
    """The same for trees: every node against a row that holds its path and nothing else."""
    rng = np.random.default_rng(8)
    n, ctx, window = 40, 6, 4
    par = trees(rng, n, "4")
    seen = np.zeros((n, n), bool)
    for i in range(n):
        seen[i, line_of(par, i)] = True
    depth = seen.sum(1) - 1
    assert depth.max() > window + 2
    c = narrowed(Tree(4, [ctx], [n], 0, 1, 8, 32, torch.float32, seen=[seen], depth=[depth]), window)
    q = c.queries(1)
    got = c.tree_reference(q, window)[0]
    for i in range(n):
        on = line_of(par, i)
        one = Tree(4, [ctx + len(on) - 1], [1], 0, 1, 8, 32, torch.float32)
        one.rows = [tuple(x[list(range(ctx)) + [ctx + j for j in on]] for x in c.rows[0])]
        np.testing.assert_allclose(got[i], one.reference(q[i:i + 1], window)[0][0], atol=1e-12)


def test_tree_tables_takes_a_window():
    mask, pos = OPS.tree_tables(*[t.to("meta") if torch.is_tensor(t) else t for t in tables_args(max_per_row=65)], 7)
    assert mask.shape == (7, 2) and pos.shape == (7,)
    for window in (-1, 1 << 31):
        with pytest.raises(ValueError, match="window"):
            OPS.tree_tables(*tables_args(), window)
    with pytest.raises(ValueError, match="CUDA"):
        OPS.tree_tables(*tables_args(), 7)
    L, p = _lib.lib(), 0x1000
    good = [p] * 5 + [2, 7, 5, 3, None]
    for at, value in [(i, None) for i in range(5)] + [(5, 0), (6, 0), (7, 513), (8, -1)]:
        a = list(good)
        a[at] = value
        assert L.fc_tree_tables_window(*a) == -1, (at, value)


def test_norms_whose_quotient_is_no_fp32_value():
    """norm / sqrt(1e-6) is what a head of zeros is multiplied by: past fp32's largest value it would come back as NaN."""
    assert np.float32(3e35) / np.sqrt(np.float32(1e-6)) < np.float32(np.inf)
    for norm in (4e35, 3e38):
        with pytest.raises(ValueError, match="norm"):
            OPS.rope_append(*rope_args(norm=norm))
    with pytest.raises(ValueError, match="CUDA"):
        OPS.rope_append(*rope_args(norm=3e35))
    L, p = _lib.lib(), 0x1000
    pages = _lib.FcPages(k=p, v=p, k_stride=64 * 3 * 128, v_stride=64 * 3 * 128, n_pages=4, n_kv_head=3, page=64,
                         head_dim=128, dtype=1)
    for norm, rc in ((4e35, -1), (3e35, 0)):  # (no token: nothing is launched)
        assert L.fc_rope_append(pages, p, p, p, 768, 128, 384, 128, 384, 128, 1, p, p, p, p, 9, 128, 0, norm, p, 6, 0,
                                None) == rc


@pytest.mark.parametrize("slots,most,G", [(64, 8, 12), (64, 64, 12), (128, 25, 4), (32, 32, 12)])
@pytest.mark.parametrize("width", [20, 33, 64])
def test_rows_may_be_cut_whatever_the_batch_has_room_for(slots, most, G, width):
    """How many key splits a row may have does not hang on how many rows the call has slots for: a batch whose other rows
    have ended, or are short, cuts its long one (tables of 1280 to 4096 keys; partials of two splits at least)."""
    L, p = _lib.lib(), 0x1000
    pages = _lib.FcPages(k=p, v=p, k_stride=64 * G * 128, v_stride=64 * G * 128, n_pages=4, n_kv_head=G, page=64,
                         head_dim=128, dtype=1)
    T = slots * most
    nb = L.fc_tree_attention_workspace_bytes(pages, slots, T, most, 12, width, 0, 0)
    assert nb >= 2 * T * 12 * (128 + 2) * 4
