"""The paged-cache operators at the ends of what they accept, without a GPU:
how a call is cut (its workspace) and what is refused. Nothing is launched."""

import pytest

torch = pytest.importorskip("torch")

import flaxchat_amd.torch_ops  # noqa: E402,F401
from flaxchat_amd import _lib  # noqa: E402

P_MOST = 2 ** 31 - 1 - 32  # with a table of one page of 32 positions: the longest prefix accepted


def pages(G=1, hd=128, page=32, n_pages=4, dtype=_lib.FC_BF16):
    each = G * page * hd
    return _lib.FcPages(0x1000, 0x1000, each, each, n_pages, G, page, hd, dtype)


def workspace(p, B, T, most, H, W, P, window=0):
    return _lib.lib().fc_paged_attention_workspace_bytes(p, B, T, most, H, W, P, window)


@pytest.mark.parametrize("dtype", [_lib.FC_BF16, _lib.FC_F32])
@pytest.mark.parametrize("B,T,most,G,H,window", [
    (1, 1, 1, 1, 1, 0), (1, 1, 1, 8, 8, 0), (64, 64, 1, 12, 12, 0), (40, 4096, 100, 12, 12, 0), (4, 8, 2, 2, 8, 0),
    (1, 1, 1, 1, 1, 2 ** 31 - 1), (300, 4000, 40, 4, 12, 2 ** 31 - 40),
])
def test_workspace_of_long_prefixes(dtype, B, T, most, G, H, window):
    """A prefix has at least one split, the own keys another: room for both
    whatever the prefix's length, up to the last one accepted."""
    p = pages(G, dtype=dtype)
    two = 2 * T * H * (128 + 2) * 4
    lengths = [1, 127, 128, 129, 10 ** 6, 1908874305, 2130836481, 2 ** 31 - 200, 2 ** 31 - 129, 2 ** 31 - 97,
               P_MOST - 1, P_MOST]
    lengths += range(2 ** 31 - 40 * 10 ** 6, P_MOST, 1234567)
    for P in lengths:
        nb = workspace(p, B, T, most, H, 1, P, window)
        assert nb >= two, (P, nb)


def test_workspace_refuses_what_the_call_does():
    p = pages()
    assert workspace(p, 1, 1, 1, 1, 1, P_MOST) > 0
    for bad in (dict(P=P_MOST + 1), dict(W=2 ** 26), dict(B=4097), dict(H=65536), dict(T=1 << 24), dict(window=-1),
                dict(T=1 << 22, H=60000)):
        assert workspace(p, **{**dict(B=1, T=1, most=1, H=1, W=1, P=0), **bad}) < 0, bad


# ---------------------------------------------------------------- autograd
OPS = torch.ops.flaxchat_mi355x


def append_args(**kw):
    a = dict(k=torch.zeros(5, 3, 128), v=torch.zeros(5, 3, 128), slots=torch.zeros(5, dtype=torch.int32),
             k_pages=torch.zeros(4, 3, 64, 128), v_pages=torch.zeros(4, 3, 2, 128, 32))
    a.update(kw)
    return a


@pytest.mark.parametrize("name", ["k", "v", "k_pages", "v_pages"])
def test_append_refuses_gradients(name):
    """There is no backward pass, so a gradient is refused, not dropped; where
    none is recorded the call goes on (here to the check of the device)."""
    a = append_args()
    a[name] = a[name].requires_grad_()
    with pytest.raises(ValueError, match="backward"):
        OPS.page_append(*a.values())
    for off in (torch.no_grad, torch.inference_mode):
        with off(), pytest.raises(ValueError, match="CUDA"):
            OPS.page_append(*a.values())


def test_versions_of_what_is_written():
    """Autograd finds a tensor that it kept and that the operators then wrote to."""
    m = lambda *s: torch.zeros(*s, dtype=torch.int32, device="meta")  # noqa: E731
    a = {k: t.to("meta") for k, t in append_args().items()}
    OPS.page_append(*a.values())
    assert {k: t._version for k, t in a.items()} == dict(k=0, v=0, slots=0, k_pages=1, v_pages=1)
    t = [m(3, 4), m(3), m(9), m(1), m(3), m(3), m(4), m(3), m(6), m(6), m(6)]
    OPS.page_tables(*t, 64, 0)
    assert [x._version for x in t] == [1, 1, 1, 1, 0, 0, 1, 1, 1, 1, 1]
    with torch.inference_mode():  # which has no versions
        a = {k: t.to("meta") for k, t in append_args().items()}
        OPS.page_append(*a.values())


# ---------------------------------------------------------------- wide tables
@pytest.mark.parametrize("B,G,H,W,P,most", [
    (64, 8, 8, 2 ** 26 - 2, 0, 1), (64, 8, 64, 2 ** 26 - 2, 0, 4), (4096, 8, 8, 2 ** 26 - 1, 0, 1),
    (300, 32, 32, 2 ** 25, 2 ** 30 - 64, 1), (64, 8, 8, 2 ** 26 - 2, 0, 40),
])
@pytest.mark.parametrize("dtype", [_lib.FC_BF16, _lib.FC_F32])
def test_wide_tables_are_taken(dtype, B, G, H, W, P, most):
    """Positions up to 2^31 are accepted whatever the number of rows: how many
    workgroups a call takes is bounded by its pieces, not by the table. (With
    no workspace the call ends at that check, the one behind the sizes'.)"""
    p, L = pages(G, dtype=dtype), _lib.lib()
    T, x = B * most, 0x1000
    assert workspace(p, B, T, most, H, W, P) > 0
    rc = L.fc_paged_attention(p, x, H * 128, 128, x, B, T, most, H, x, W, x, x, x, P, 0, 0, None, 0, None)
    assert rc == -1 and b"workspace" in L.fc_last_error()


# ---------------------------------------------------------------- counts past 31 bits
def test_counts_past_31_bits_are_refused():
    """The C entries count in 32 bits: what does not fit is refused, not cut
    off. (Shapes alone: tensors without memory, given to the operators' own
    functions.)"""
    def m(*s, dtype=torch.bfloat16):
        return torch.empty(s, dtype=dtype, device="meta")

    def i(*s):
        return m(*s, dtype=torch.int32)

    ops, T = flaxchat_amd.torch_ops, 2 ** 32 + 1
    kp, vp = m(4, 1, 32, 8), m(4, 1, 1, 8, 32)
    with pytest.raises(ValueError, match="tokens below"):
        ops.page_append(m(T, 1, 8), m(T, 1, 8), i(T), kp, vp)
    with pytest.raises(ValueError, match="tokens below"):
        ops.paged_attention(m(T, 1, 8), kp, vp, i(1, 1), i(2), i(1), 1, 0)
    for N, page in ((2 ** 32 + 1, 32), (1, 2 ** 32 + 32)):
        with pytest.raises(ValueError, match="below 2\\^31"):
            ops.page_append(m(1, 1, 1), m(1, 1, 1), i(1), m(N, 1, page, 1), m(N, 1, page // 32, 1, 32))
