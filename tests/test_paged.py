"""The paged-cache operators without a GPU: registration, shape propagation,
the C structure, and every refusal (nothing is launched)."""

import ctypes
import subprocess

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import flaxchat_amd.torch_ops  # noqa: E402,F401
from flaxchat_amd import _lib  # noqa: E402
from tests.paged_cases import Paged, k_blocks, tables_reference  # noqa: E402
from tests.test_abi import HEADER  # noqa: E402

OPS = torch.ops.flaxchat_mi355x


def i32(*s, device="cpu"):
    return torch.zeros(*s, dtype=torch.int32, device=device)


def attention_args(device="cpu", **kw):
    a = dict(q=torch.zeros(7, 6, 128, device=device), k_pages=torch.zeros(4, 3, 64, 128, device=device),
             v_pages=torch.zeros(4, 3, 2, 128, 32, device=device), tables=i32(2, 3, device=device),
             row_off=i32(3, device=device), start=i32(2, device=device), max_per_row=4, window=0,
             prefix_pages=i32(2, device=device), prefix_len=100)
    a.update(kw)
    return list(a.values())


def append_args(**kw):
    a = dict(k=torch.zeros(5, 3, 128), v=torch.zeros(5, 3, 128), slots=i32(5), k_pages=torch.zeros(4, 3, 64, 128),
             v_pages=torch.zeros(4, 3, 2, 128, 32))
    a.update(kw)
    return list(a.values())


def table_args(**kw):
    a = dict(tables=i32(3, 4), held=i32(3), free_pages=i32(9), n_free=i32(1), length=i32(3), n_new=i32(3),
             row_off=i32(4), start=i32(3), tok_row=i32(6), tok_pos=i32(6), slots=i32(6), page=64, prefix_len=0)
    a.update(kw)
    return list(a.values())


def test_registered_and_shapes():
    for name in ("page_tables", "page_append", "paged_attention"):
        assert hasattr(OPS, name)
    m = lambda t: t.to("meta") if torch.is_tensor(t) else t  # noqa: E731
    y = OPS.paged_attention(*[m(a) for a in attention_args()])
    assert y.shape == (7, 768) and y.dtype == torch.float32 and y.device.type == "meta"
    assert OPS.page_append(*[m(a) for a in append_args()]) is None
    assert OPS.page_tables(*[m(a) for a in table_args()]) is None


BIG = torch.zeros(1).expand(4, 3, 64, 128)  # pages that overlap


@pytest.mark.parametrize("kw,match", [
    (dict(), "CUDA"),
    (dict(k_pages=torch.zeros(4, 3, 48, 128)), "multiple of 32"),
    (dict(k_pages=torch.zeros(4, 3, 128)), "k_pages"),
    (dict(k_pages=torch.zeros(4, 3, 64, 288)), "head_dim"),
    (dict(v_pages=torch.zeros(4, 3, 64, 128)), "v_pages"),
    (dict(v_pages=torch.zeros(4, 3, 2, 128, 32).double()), "dtype"),
    (dict(k_pages=BIG), "contiguous"),
    (dict(k_pages=torch.zeros(4, 3, 128, 64).transpose(2, 3)), "contiguous"),
    (dict(q=torch.zeros(7, 6, 64)), "q "),
    (dict(q=torch.zeros(7, 4, 128)), "n_head"),
    (dict(q=torch.zeros(7, 6, 128).bfloat16()), "dtype"),
    (dict(q=torch.zeros(7, 6, 128, requires_grad=True)), "backward"),
    (dict(tables=i32(6)), "tables"),
    (dict(tables=torch.zeros(2, 3, dtype=torch.int64)), "int32"),
    (dict(tables=i32(3, 2).t()), "contiguous"),
    (dict(row_off=i32(2)), "row_off"),
    (dict(start=i32(3)), "start"),
    (dict(max_per_row=0), "max_per_row"),
    (dict(window=-1), "window"),
    (dict(window=1 << 31), "window"),
    (dict(prefix_len=129), "prefix_pages"),
    (dict(prefix_pages=None), "prefix_pages"),
    (dict(prefix_len=-1), "prefix_len"),
    (dict(prefix_len=(1 << 31) - 100), "2\\^31"),
    (dict(tables=i32(4097, 1), row_off=i32(4098), start=i32(4097)), "4096"),
])
def test_attention_refusals(kw, match):
    with pytest.raises(ValueError, match=match):
        OPS.paged_attention(*attention_args(**kw))


@pytest.mark.parametrize("kw,match", [
    (dict(), "CUDA"),
    (dict(k=torch.zeros(5, 2, 128)), "k and v"),
    (dict(v=torch.zeros(4, 3, 128)), "k and v"),
    (dict(k=torch.zeros(5, 3, 128).bfloat16(), v=torch.zeros(5, 3, 128).bfloat16()), "dtype"),
    (dict(v=torch.zeros(5, 3, 128).bfloat16()), "dtype"),
    (dict(slots=i32(4)), "slots"),
    (dict(slots=torch.zeros(5, dtype=torch.int64)), "int32"),
    (dict(k_pages=BIG), "contiguous"),
])
def test_append_refusals(kw, match):
    with pytest.raises(ValueError, match=match):
        OPS.page_append(*append_args(**kw))


@pytest.mark.parametrize("kw,match", [
    (dict(), "CUDA"),
    (dict(page=48), "multiple of 32"),
    (dict(page=0), "multiple of 32"),
    (dict(prefix_len=-1), "prefix_len"),
    (dict(prefix_len=(1 << 31) - 256), "2\\^31"),
    (dict(tables=i32(12)), "tables"),
    (dict(held=i32(4)), "held"),
    (dict(n_free=i32(2)), "n_free"),
    (dict(row_off=i32(3)), "row_off"),
    (dict(slots=i32(5)), "tok_row"),
    (dict(n_new=torch.zeros(3, dtype=torch.int64)), "int32"),
    (dict(length=i32(6)[::2]), "contiguous"),
    (dict(free_pages=i32(0)), "CUDA"),  # a stack without room is none to refuse
    (dict(free_pages=torch.zeros(9, dtype=torch.int64)), "free"),
])
def test_tables_refusals(kw, match):
    with pytest.raises(ValueError, match=match):
        OPS.page_tables(*table_args(**kw))


def test_c_abi_refusals():
    """Status codes before any GPU call: null pointers, sizes, dtypes."""
    L = _lib.lib()
    p = 0x1000
    t = [p] * 11 + [3, 4, 9, 6, 64, 0, None]
    for at, bad in ((0, None), (10, None), (11, 0), (11, 4097), (12, 0), (13, 1 << 30), (14, 0), (15, 40), (16, -1),
                    (16, 0x7fffffff)):
        a = list(t)
        a[at] = bad
        assert L.fc_page_tables(*a) == -1, (at, bad)
    good = dict(k=p, v=p, k_stride=64 * 3 * 128, v_stride=64 * 3 * 128, n_pages=4, n_kv_head=3, page=64, head_dim=128,
                dtype=1)
    bad_pages = [dict(k=None), dict(page=33), dict(page=0), dict(head_dim=257), dict(n_pages=0), dict(dtype=2),
                 dict(k_stride=100), dict(v_stride=0)]
    att = [p, 768, 128, p, 2, 7, 4, 6, p, 3, p, p, p, 100, 0, 0, p, 1 << 40, None]
    app = [p, p, 384, 128, 384, 128, 1, p, 5, None]
    for bad in bad_pages:
        pages = _lib.FcPages(**{**good, **bad})
        assert L.fc_paged_attention(pages, *att) == -1
        assert L.fc_page_append(pages, *app) == -1
    pages = _lib.FcPages(**good)
    for at, bad in ((0, None), (3, None), (4, 0), (4, 4097), (5, 0), (6, 0), (7, 4), (8, None), (9, 0), (10, None),
                    (11, None), (12, None), (13, -1), (14, -1), (13, 0x7fffffff)):
        a = list(att)
        a[at] = bad
        assert L.fc_paged_attention(pages, *a) == -1, (at, bad)
    for at, bad in ((0, None), (1, None), (6, 2), (7, None), (8, -1)):
        a = list(app)
        a[at] = bad
        assert L.fc_page_append(pages, *a) == -1, (at, bad)
    f32 = _lib.FcPages(**{**good, "dtype": 0})
    assert L.fc_page_append(f32, *app) == -1 and b"bf16" in L.fc_last_error()
    assert L.fc_page_append(pages, *app[:8], 0, None) == 0  # no token: nothing is launched


def test_struct_layout(tmp_path):
    lines = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{HEADER}"', 'int main(void){',
             'printf("%zu", sizeof(fc_pages));']
    lines += [f'printf(" %zu", offsetof(fc_pages, {f}));' for f, _ in _lib.FcPages._fields_]
    c = tmp_path / "p.c"
    c.write_text("\n".join(lines + ["return 0;}"]))
    subprocess.run(["gcc", str(c), "-o", str(tmp_path / "p")], check=True)
    got = subprocess.run([str(tmp_path / "p")], capture_output=True, text=True, check=True).stdout.split()
    assert [int(x) for x in got] == [ctypes.sizeof(_lib.FcPages)] + [getattr(_lib.FcPages, f).offset
                                                                      for f, _ in _lib.FcPages._fields_]


def test_plain_forms_agree():
    """The 64-bit references of the GPU tests against a second statement of
    the same: tables on a case small enough to write out, blocks element by
    element, attention of one row against a dense softmax."""
    tables = np.array([[5, 9, -1], [7, -1, -1], [3, 4, 8]])
    held, n_free = np.array([2, 1, 3]), np.array([2])
    free = np.array([1, 2, 0, 0, 0, 0])
    off, start, row, pos, slot = tables_reference(tables, held, free, n_free, np.array([63, 0, 90]),
                                                  np.array([2, -1, 6]), 32, 10, 12)
    # row 1 gives page 7: stack 1 2 7; row 0 takes one page for positions 63, 64; row 2 has its pages
    assert off.tolist() == [0, 2, 2, 8] and start.tolist() == [73, 10, 100] and held.tolist() == [3, 0, 3]
    assert tables[0].tolist() == [5, 9, 7] and free[:3].tolist() == [1, 2, 7] and n_free[0] == 2
    assert row.tolist() == [0] * 2 + [2] * 6 + [-1] * 4 and pos[:3].tolist() == [73, 74, 100]
    assert slot[:3].tolist() == [9 * 32 + 31, 7 * 32, 8 * 32 + 26] and slot[8:].tolist() == [-1] * 4
    rng = np.random.default_rng(0)
    K = rng.standard_normal((1, 32, 128)).astype(np.float32)
    B = k_blocks(K).reshape(-1)
    for kk, d in ((0, 0), (5, 37), (31, 127), (12, 64)):
        assert B[((2 * (d // 32) + (kk // 4) % 2) * 64 + 4 * (kk // 8) + kk % 4 + 16 * ((d // 8) % 4)) * 8 + d % 8] \
            == K[0, kk, d]
    c = Paged(1, [40], [3], 10, 1, 64, 32, torch.float32)
    q = c.queries(2)
    y, tol = c.reference(q, 0)
    k = np.concatenate([c.pre[0], c.rows[0][0]])[:, 0].astype(np.float64)
    v = np.concatenate([c.pre[1], c.rows[0][1]])[:, 0].astype(np.float64)
    for i in range(3):
        for h in range(2):
            e = np.exp(k[:51 + i] @ q[i, h] / 8)
            np.testing.assert_allclose(y[i, 64 * h:64 * h + 64], e @ v[:51 + i] / e.sum(), rtol=1e-12)
    assert np.all(tol > 0) and tol.max() < 1e-4
