"""The operators for trees of drafted tokens without a GPU: registration,
shape propagation and every refusal (nothing is launched), and the 64-bit
references of the GPU tests against second statements of the same."""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import flaxchat_amd.torch_ops  # noqa: E402,F401
from flaxchat_amd import _lib  # noqa: E402
from tests.tree_cases import Tree, accept_plain, line_of, moves_plain, packed, rope_plain, tables_plain  # noqa: E402

OPS = torch.ops.flaxchat_mi355x


def i32(*s):
    return torch.zeros(*s, dtype=torch.int32)


def i64(*s):
    return torch.zeros(*s, dtype=torch.int64)


def args(base, kw):
    assert set(kw) <= set(base)
    return list({**base, **kw}.values())


def pool(L=None):
    lead = () if L is None else (L,)
    return dict(k_pages=torch.zeros(*lead, 4, 3, 64, 128), v_pages=torch.zeros(*lead, 4, 3, 2, 128, 32))


def tables_args(**kw):
    return args(dict(parent=i32(7), row_off=i32(3), start=i32(2), max_per_row=5), kw)


def accept_args(**kw):
    return args(dict(parent=i32(7), tokens=i32(7), target=i32(7), row_off=i32(3), max_per_row=5), kw)


def commit_args(**kw):
    return args(dict(path=i32(7), slots=i32(7), row_off=i32(3), max_per_row=5, **pool()), kw)


def attention_args(**kw):
    return args(dict(q=torch.zeros(7, 6, 128), **pool(), tables=i32(2, 3), row_off=i32(3), start=i32(2),
                     mask=i64(7, 1), tok_pos=i32(7), max_per_row=4, window=0, prefix_pages=i32(2), prefix_len=100), kw)


def rope_args(**kw):
    return args(dict(q=torch.zeros(5, 6, 128), k=torch.zeros(5, 3, 128), v=torch.zeros(5, 3, 128), tok_pos=i32(5),
                     slots=i32(5), cos=torch.zeros(9, 64), sin=torch.zeros(9, 64), **pool(), interleaved=False,
                     norm=1.2), kw)


def test_registered_and_shapes():
    m = lambda a: [t.to("meta") if torch.is_tensor(t) else t for t in a]  # noqa: E731
    mask, pos = OPS.tree_tables(*m(tables_args(max_per_row=65)))
    assert mask.shape == (7, 2) and mask.dtype == torch.int64 and pos.shape == (7,) and pos.dtype == torch.int32
    n, nxt, path = OPS.tree_accept(*m(accept_args()))
    assert n.shape == nxt.shape == (2,) and path.shape == (7,) and path.dtype == torch.int32
    y = OPS.tree_attention(*m(attention_args()))
    assert y.shape == (7, 768) and y.dtype == torch.float32
    assert OPS.tree_commit(*m(commit_args())) is None and OPS.tree_commit(*m(commit_args(**pool(2)))) is None
    q = OPS.rope_append(*m(rope_args(k_pages=pool()["k_pages"].bfloat16(), v_pages=pool()["v_pages"].bfloat16())))
    assert q.shape == (5, 6, 128) and q.dtype == torch.bfloat16


@pytest.mark.parametrize("kw,match", [
    (dict(), "CUDA"),
    (dict(max_per_row=0), "max_per_row"),
    (dict(max_per_row=513), "512"),
    (dict(parent=i64(7)), "int32"),
    (dict(parent=i32(14)[::2]), "contiguous"),
    (dict(row_off=i32(0)), "row_off"),
    (dict(row_off=i32(1)), "row_off"),
    (dict(row_off=i32(4098), start=i32(4097)), "4097"),
    (dict(start=i32(3)), "start"),
])
def test_tables_refusals(kw, match):
    with pytest.raises(ValueError, match=match):
        OPS.tree_tables(*tables_args(**kw))


@pytest.mark.parametrize("kw,match", [
    (dict(), "CUDA"),
    (dict(max_per_row=513), "512"),
    (dict(tokens=i32(6)), "tokens"),
    (dict(target=i64(7)), "int32"),
    (dict(row_off=i32(1)), "row_off"),
])
def test_accept_refusals(kw, match):
    with pytest.raises(ValueError, match=match):
        OPS.tree_accept(*accept_args(**kw))


@pytest.mark.parametrize("kw,match", [
    (dict(), "CUDA"),
    (pool(2), "CUDA"),
    (dict(max_per_row=0), "max_per_row"),
    (dict(slots=i32(6)), "slots"),
    (dict(path=i64(7)), "int32"),
    (dict(k_pages=torch.zeros(4, 3, 48, 128)), "multiple of 32"),
    (dict(k_pages=torch.zeros(2, 4, 3, 64, 128)), "layers"),
    (dict(pool(3), k_pages=torch.zeros(2, 4, 3, 64, 128)), "layers"),
    (dict(k_pages=torch.zeros(1, 4, 3, 64, 128).expand(2, 4, 3, 64, 128),
          v_pages=torch.zeros(2, 4, 3, 2, 128, 32)), "overlap"),
    (dict(k_pages=torch.zeros(4, 3, 64, 128, requires_grad=True)), "backward"),
])
def test_commit_refusals(kw, match):
    with pytest.raises(ValueError, match=match):
        OPS.tree_commit(*commit_args(**kw))


def test_layers_of_a_pool_page_by_page():
    """[n_pages][n_layer] pools seen as [n_layer][n_pages]: neither overlaps."""
    k, v = torch.zeros(4, 2, 3, 64, 128).transpose(0, 1), torch.zeros(4, 2, 3, 2, 128, 32).transpose(0, 1)
    with pytest.raises(ValueError, match="CUDA"):
        OPS.tree_commit(*commit_args(k_pages=k, v_pages=v))


@pytest.mark.parametrize("kw,match", [
    (dict(), "CUDA"),
    (dict(max_per_row=513, mask=i64(7, 9)), "512"),
    (dict(mask=i64(7, 2)), "mask"),
    (dict(mask=i64(6, 1)), "mask"),
    (dict(mask=i32(7, 1)), "mask"),
    (dict(mask=i64(1, 7).t()[:, :1].expand(7, 1)[::1]), "CUDA"),
    (dict(mask=i64(7, 2)[:, :1]), "mask"),
    (dict(tok_pos=i32(6)), "tok_pos"),
    (dict(tok_pos=i64(7)), "int32"),
    (dict(q=torch.zeros(7, 4, 128)), "tree_attention: q"),
    (dict(q=torch.zeros(7, 6, 128, requires_grad=True)), "backward"),
    (dict(tables=i32(3, 2).t()), "contiguous"),
    (dict(start=i32(3)), "start"),
    (dict(window=-1), "window"),
    (dict(prefix_len=129), "prefix_pages"),
    (dict(prefix_len=(1 << 31) - 100), "2\\^31"),
])
def test_attention_refusals(kw, match):
    with pytest.raises(ValueError, match=match):
        OPS.tree_attention(*attention_args(**kw))


BF = dict(k=torch.zeros(5, 3, 128).bfloat16(), v=torch.zeros(5, 3, 128).bfloat16(), q=torch.zeros(5, 6, 128).bfloat16())


@pytest.mark.parametrize("kw,match", [
    (dict(), "CUDA"),
    (dict(q=torch.zeros(5, 6, 64)), "q "),
    (dict(q=torch.zeros(5, 0, 128)), "q "),
    (dict(k=torch.zeros(4, 3, 128)), "k and v"),
    (dict(v=torch.zeros(5, 3, 64)), "k and v"),
    (BF, "dtype"),
    (dict(q=torch.zeros(5, 6, 128).bfloat16()), "dtype"),
    (dict(cos=torch.zeros(9, 65), sin=torch.zeros(9, 65)), "pairs"),
    (dict(cos=torch.zeros(9, 0), sin=torch.zeros(9, 0)), "pairs"),
    (dict(cos=torch.zeros(0, 4), sin=torch.zeros(0, 4)), "pairs"),
    (dict(cos=torch.zeros(8, 64)), "cos and sin"),
    (dict(cos=torch.zeros(9, 64).bfloat16()), "fp32"),
    (dict(cos=torch.zeros(64, 9).t()), "contiguous"),
    (dict(norm=-1.0), "norm"),
    (dict(norm=float("nan")), "norm"),
    (dict(norm=float("inf")), "norm"),
    (dict(tok_pos=i32(4)), "tok_pos"),
    (dict(slots=i64(5)), "int32"),
    (dict(sin=torch.zeros(9, 64, requires_grad=True)), "backward"),
    (dict(k=torch.zeros(5, 3, 128, requires_grad=True)), "backward"),
])
def test_rope_refusals(kw, match):
    with pytest.raises(ValueError, match=match):
        OPS.rope_append(*rope_args(**kw))


def test_c_abi_refusals():
    """Status codes before any GPU call."""
    L, p = _lib.lib(), 0x1000

    def each(call, good, bad):
        for at, value in bad:
            a = list(good)
            a[at] = value
            assert call(*a) == -1, (at, value)

    sizes = [(0, 0), (0, 4097), (1, 0), (1, 1 << 30), (2, 0), (2, 513)]
    each(L.fc_tree_tables, [p] * 5 + [2, 7, 5, None], [(i, None) for i in range(5)] + [(5 + i, v) for i, v in sizes])
    each(L.fc_tree_accept, [p] * 7 + [2, 7, 5, None], [(i, None) for i in range(7)] + [(7 + i, v) for i, v in sizes])
    good = dict(k=p, v=p, k_stride=64 * 3 * 128, v_stride=64 * 3 * 128, n_pages=4, n_kv_head=3, page=64, head_dim=128,
                dtype=1)
    pages = _lib.FcPages(**good)
    commit = [pages, 2, 1 << 20, 1 << 20, p, p, p, 2, 7, 5, None]
    each(L.fc_tree_commit, commit, [(i, None) for i in (4, 5, 6)] + [(1, 0), (1, 65536)] +
         [(7 + i, v) for i, v in sizes])
    att = [pages, p, 768, 128, p, 2, 7, 4, 6, p, 3, p, p, p, p, p, 100, 0, 0, p, 1 << 40, None]
    each(L.fc_tree_attention, att, [(i, None) for i in (1, 4, 9, 11, 12, 13, 14, 15)] +
         [(5, 0), (5, 4097), (6, 0), (7, 0), (7, 513), (8, 4), (10, 0), (16, -1), (17, -1)])
    assert L.fc_tree_attention_workspace_bytes(pages, 2, 7, 513, 6, 3, 100, 0) == -1
    assert L.fc_tree_attention_workspace_bytes(pages, 2, 7, 4, 6, 3, 100, 0) >= 0
    rope = [pages, p, p, p, 768, 128, 384, 128, 384, 128, 1, p, p, p, p, 9, 128, 0, 1.2, p, 6, 5, None]
    each(L.fc_rope_append, rope, [(i, None) for i in (1, 2, 3, 11, 12, 13, 14, 19)] +
         [(10, 2), (15, 0), (16, 0), (16, 3), (16, 130), (18, -1.0), (18, float("nan")), (20, 0), (21, -1)])
    assert L.fc_rope_append(*rope[:21], 0, None) == 0  # no token: nothing is launched
    for bad in (dict(k=None), dict(page=33), dict(head_dim=257), dict(dtype=2), dict(k_stride=100)):
        q = _lib.FcPages(**{**good, **bad})
        assert L.fc_tree_commit(q, *commit[1:]) == -1 and L.fc_rope_append(q, *rope[1:]) == -1
        assert L.fc_tree_attention(q, *att[1:]) == -1
    f32 = _lib.FcPages(**{**good, "dtype": 0})
    assert L.fc_rope_append(f32, *rope[1:]) == -1 and b"bf16" in L.fc_last_error()


def test_plain_forms_agree():
    """The 64-bit references on trees small enough to write out."""
    rng = np.random.default_rng(0)
    #      0
    #    1   2      6 (a second root)
    #   3 4   5     7
    par = np.array([-1, 0, 0, 1, 1, 2, -1, 6])
    off = np.array([0, 8])
    mask, pos = tables_plain(off, par, [100], 9, 8)
    assert [int(m) for m in mask[:, 0]] == [1, 3, 5, 11, 19, 37, 64, 192, 0]
    assert pos.tolist() == [100, 101, 101, 102, 102, 102, 100, 101, -1]
    tokens = np.array([9, 1, 2, 3, 4, 5, 6, 7])
    target = np.array([2, 4, 5, 8, 8, 8, 0, 8])  # 0 -> 2 -> 5; 1 is not chosen, so 4 is out; 7 is not
    n, nxt, path = accept_plain(off, par, tokens, target, 8, 8)
    assert n.tolist() == [3] and nxt.tolist() == [8] and path.tolist() == [0, 2, 5] + [-1] * 5
    assert line_of(par, 4) == [0, 1, 4] and line_of([-1, 0, 2], 2) == [2]
    assert moves_plain(off, path, np.arange(40, 48), 46, 8, 8) == [(42, 41), (45, 42)]
    x = rng.standard_normal((2, 1, 8))
    ang = np.array([[0.3, 1.1], [0.7, 2.0]])
    y, tol = rope_plain(x, np.array([1, 5]), np.cos(ang), np.sin(ang), False, 0.0)
    z = (x[0, 0, 0] + 1j * x[0, 0, 2]) * np.exp(-0.7j)
    np.testing.assert_allclose([y[0, 0, 0], y[0, 0, 2]], [z.real, z.imag])
    assert np.all(y[1] == 0) and np.array_equal(y[0, 0, 4:], x[0, 0, 4:]) and tol[0, 0, 4] == 0 < tol[0, 0, 0]
    # a chain of nodes is what paged_attention computes
    c = Tree(1, [40, 0], [3, 4], 10, 1, 64, 32, torch.float32, kinds=["chain"])
    q = c.queries(2)
    for window in (0, 12, 2):
        a, b = c.reference(q, window)[0], c.tree_reference(q, window)[0]
        if window != 2:  # (a window shorter than the chain: the mask alone decides among nodes)
            np.testing.assert_allclose(a, b, atol=1e-12)
    assert packed(rng, [2, 0, 3], ["chain"])[0].tolist() == [0, 2, 2, 5]
