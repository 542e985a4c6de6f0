"""The C-ABI kernels as PyTorch operators: ``torch.ops.flaxchat_mi355x.*``.

Importing this module registers the namespace (``torch.library.custom_op``),
so code that composes torch tensors can call the hot kernels directly, and
shape propagation (meta / fake tensors) works without a GPU. Each operator
is a thin call of one C-ABI entry point on the current stream of the input's
device; the engine itself (``SpecSession``, ``Engine``) calls the C-ABI
directly and does not go through here.

Operators:
  pack_operand(src)                  bf16 [R][K] row-major -> fragment order [round16(R)][K]
  linear(x, w, softcap=False)        fp32 x @ w^T (nnx.Linear, flaxchat/gpt.py:93-99); softcap applies
                                     15 tanh(z / 15) (flaxchat/engine.py:173-174)
  attention(q, k_cache, v_cache, row_off, start, max_per_row, window)
                                     decode / verify attention over one cache layer
                                     (flaxchat/engine.py:128-156)
  cross_entropy(logits, targets)     per-row logsumexp(z) - z[t], 0 where t < 0
                                     (flaxchat/gpt.py:446-452)

The engine entry points take a model as the address of its fc_model
descriptor (`DeviceModel.desc`, read-only weights that stay alive with the
DeviceModel) and everything they write as tensors, declared mutated:
  forward(model, k_cache, v_cache, hist, tokens, row_off, start, max_per_row, n_out, logits,
          workspace, typ_tokens=0, flags=0)
                                     one packed chunk through the model (fc_forward;
                                     flaxchat/engine.py:51-177, 396-407)
  attn_prologue(model, layer, k_cache, v_cache, qkv, h, tokens, tok_row, tok_pos) -> q
                                     RoPE, QK-norm, VE gate, cache append (engine.py:96-126)
  attn_qkv(model, layer, k_cache, v_cache, h, tokens, tok_row, tok_pos, typ_tokens=0) -> q
                                     the QKV projection with that prologue fused
  row_stats(logits, temperature, top_k) -> (mx, sum, tau, tie_idx, argmax)
                                     top-k keep set and softmax statistics (engine.py:461-476)
  spec_accept(buffers, batch, k, max_tokens, gen_cap, vocab, temperature, top_k, seed)
                                     accept / reject / bonus and the rollback bookkeeping
                                     (engine.py:525-606) on a round's logits
  spec_round(target, draft, t_k, t_v, t_hist, d_k, d_v, d_hist, buffers, batch, k, max_tokens,
             gen_cap, vocab, temperature, top_k, seed, workspace)
                                     one whole speculative round (engine.py:484-606)

The paged KV cache (one layer unless said; k_pages [n_pages][n_kv_head][page][head_dim]
and v_pages [n_pages][n_kv_head][page / 32][head_dim][32] in the caches' block
order, whose pages may be strided, as those of one layer of a pool of all
layers are; every index tensor int32). None has a backward pass: tensors that require a gradient are refused
where gradients are recorded, and what a call writes counts as modified in place:
  page_tables(tables, held, free_pages, n_free, length, n_new, row_off, start, tok_row, tok_pos, slots,
              page, prefix_len=0)
                                     block tables, packed chunk and slot map of a step from the rows'
                                     lengths, on the GPU (fc_page_tables); all but length and n_new mutated
  page_append(k, v, slots, k_pages, v_pages)
                                     new K and V [tokens][n_kv_head][head_dim], strided views of a fused
                                     projection included, into their slots (engine.py:119-126)
  paged_attention(q, k_pages, v_pages, tables, row_off, start, max_per_row, window, prefix_pages=None,
                  prefix_len=0)      attention over the pages, the shared prefix computed once for all rows
                                     (engine.py:128-156) -> [tokens][n_head * head_dim]; inference only
Decoding with trees of drafted tokens over that cache: row b's chunk is a tree or a forest whose node i, token
row_off[b] + i, continues node parent[row_off[b] + i] < i of its row (any other value: a root), lies in the cache at
start[b] + i and counts as position start[b] + its depth; at most 512 nodes a row (max_per_row):
  tree_tables(parent, row_off, start, max_per_row, window=0) -> (mask, tok_pos)
                                     each node's ancestors and itself as bits, int64 [tokens][words of 64], and its
                                     position (fc_tree_tables_window); of the ancestors those at most `window`
                                     positions above: the mask of the layers with that window
  rope_append(q, k, v, tok_pos, slots, cos, sin, k_pages, v_pages, interleaved=False, norm=0.0) -> q
                                     page_append with the rotation of q and k at tok_pos and the QK norm
                                     (gpt.py:52-71, engine.py:108-126); trees or not
  tree_attention(q, k_pages, v_pages, tables, row_off, start, mask, tok_pos, max_per_row, window,
                 prefix_pages=None, prefix_len=0)
                                     paged_attention where a node sees what its row holds, as far as the window
                                     reaches, and the nodes of its mask, whatever the window
  tree_accept(parent, tokens, target, row_off, max_per_row) -> (n_accepted, next_token, path)
                                     the deepest path on which the target's choices are the drafted tokens
  tree_commit(path, slots, row_off, max_per_row, k_pages, v_pages)
                                     that path's K and V to the front of its row's chunk, in one layer, or in all of
                                     [n_layer] of them
`buffers` is the speculative state's device arrays in fc_spec_state order
(`SPEC_BUFFERS`: t_len .. p_stats, then the partials buffer `part`).
"""

from __future__ import annotations

import torch

from . import _lib
from ._lib import check, lib

__all__ = ["pack_operand", "linear", "attention", "cross_entropy", "frag_to_rows", "forward", "attn_prologue",
           "attn_qkv", "row_stats", "spec_accept", "spec_round", "SPEC_BUFFERS", "page_tables", "page_append",
           "paged_attention", "tree_tables", "tree_attention", "tree_accept", "tree_commit", "rope_append"]

NS = "flaxchat_mi355x"


def _stream(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


def _dtype_code(t: torch.Tensor) -> int:
    if t.dtype == torch.bfloat16:
        return _lib.FC_BF16
    if t.dtype == torch.float32:
        return _lib.FC_F32
    raise ValueError(f"flaxchat_mi355x operators take bf16 or fp32 tensors (got {t.dtype})")


def frag_to_rows(t: torch.Tensor, rows: int) -> torch.Tensor:
    """Row-major [rows][K] view of a fragment-order [round16(rows)][K]
    tensor: 16-row x 32-column blocks of 512 elements, element (r, k) of a
    block at ((k % 32) // 8 * 16 + r) * 8 + k % 8."""
    R, K = t.shape
    blk = t.reshape(R // 16, K // 32, 4, 16, 8)          # [row block][k block][k group][row][k % 8]
    return blk.permute(0, 3, 1, 2, 4).reshape(R, K)[:rows]


# ---------------------------------------------------------------- pack_operand
@torch.library.custom_op(f"{NS}::pack_operand", mutates_args=())
def pack_operand(src: torch.Tensor) -> torch.Tensor:
    if src.dtype != torch.bfloat16 or src.dim() != 2 or src.shape[1] % 64 != 0:
        raise ValueError("pack_operand takes a bf16 [R][K] matrix with K % 64 == 0")
    src = src.contiguous()
    R, K = src.shape
    out = torch.empty(((R + 15) // 16 * 16, K), dtype=src.dtype, device=src.device)
    check(lib().fc_pack_operand(src.data_ptr(), out.data_ptr(), R, K, _stream(src)), "fc_pack_operand")
    return out


@pack_operand.register_fake
def _(src):
    return src.new_empty(((src.shape[0] + 15) // 16 * 16, src.shape[1]))


# ---------------------------------------------------------------- linear
@torch.library.custom_op(f"{NS}::linear", mutates_args=())
def linear(x: torch.Tensor, w: torch.Tensor, softcap: bool = False) -> torch.Tensor:
    if x.dim() != 2 or w.dim() != 2 or x.shape[1] != w.shape[1] or x.dtype != w.dtype:
        raise ValueError("linear takes x [M][K] and w [N][K] of one dtype")
    code = _dtype_code(x)
    M, K = x.shape
    N = w.shape[0]
    if code == _lib.FC_BF16:
        if K % 64 != 0 or N % 32 != 0:
            raise ValueError(f"bf16 linear needs K % 64 == 0 and N % 32 == 0 (got K={K}, N={N})")
        a, b = pack_operand(x), pack_operand(w)
    else:
        a, b = x.contiguous(), w.contiguous()
    out = torch.empty((M, N), dtype=torch.float32, device=x.device)
    check(lib().fc_gemm(a.data_ptr(), b.data_ptr(), out.data_ptr(), M, N, K, code, 4 if softcap else 0,
                        _stream(x)), "fc_gemm")
    return out


@linear.register_fake
def _(x, w, softcap=False):
    return x.new_empty((x.shape[0], w.shape[0]), dtype=torch.float32)


# ---------------------------------------------------------------- attention
@torch.library.custom_op(f"{NS}::attention", mutates_args=())
def attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, row_off: torch.Tensor,
              start: torch.Tensor, max_per_row: int, window: int) -> torch.Tensor:
    """q [tokens][H][128] packed by row (row b's queries at row_off[b] ..
    row_off[b+1], at positions start[b] ..); k_cache / v_cache one layer of
    the engine's cache in its layout: k_cache shaped [B][G][cap][128] (bf16:
    32-key blocks in S^T fragment order; fp32: row-major), v_cache with as
    many elements, [B][G][cap / 32][128][32] (any shape of that size);
    window 0 = full causal, else keys with pos - j <= window. Returns
    [tokens][H * 128] in q's dtype, row-major."""
    code = _dtype_code(q)
    if q.dim() != 3 or k_cache.dim() != 4 or v_cache.numel() != k_cache.numel():
        raise ValueError("attention takes q [T][H][hd], k_cache [B][G][cap][hd] and a v_cache of the same size")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("attention: the caches must be contiguous")
    tot, H, hd = q.shape
    B, G, cap, hd2 = k_cache.shape
    if hd != hd2 or H % G != 0 or row_off.numel() != B + 1 or start.numel() != B:
        raise ValueError("attention: head_dim, GQA grouping or row_off / start sizes do not match")
    if k_cache.dtype != q.dtype or v_cache.dtype != q.dtype:
        raise ValueError("attention: q and the caches share one dtype")
    if row_off.dtype != torch.int32 or start.dtype != torch.int32:
        raise ValueError("attention: row_off and start are int32")
    max_keys = min(cap, window + max_per_row) if window > 0 else cap
    nb = lib().fc_attention_workspace_bytes(B, max_per_row, H, G, hd, max_keys)
    ws = torch.empty(max(nb, 1), dtype=torch.uint8, device=q.device)
    y = torch.empty((max(tot, 1), H * hd), dtype=q.dtype, device=q.device)
    qc = q.contiguous()
    check(lib().fc_attention_rows(qc.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), y.data_ptr(), B, tot,
                             max_per_row, H, G, hd, cap, row_off.data_ptr(), start.data_ptr(), window, max_keys,
                             code, ws.data_ptr(), ws.numel(), _stream(q)), "fc_attention_rows")
    return y[:tot]


@attention.register_fake
def _(q, k_cache, v_cache, row_off, start, max_per_row, window):
    return q.new_empty((q.shape[0], q.shape[1] * q.shape[2]))


# ---------------------------------------------------------------- cross_entropy
@torch.library.custom_op(f"{NS}::cross_entropy", mutates_args=())
def cross_entropy(logits: torch.Tensor, targets: torch.Tensor) -> torch.Tensor:
    if logits.dtype != torch.float32 or logits.dim() != 2 or logits.stride(1) != 1:
        raise ValueError("cross_entropy takes fp32 logits [rows][V] with unit column stride")
    rows, V = logits.shape
    t = targets.to(torch.int32).contiguous()
    if t.numel() != rows:
        raise ValueError("cross_entropy: one target per logits row")
    if rows and int(t.max()) >= V:
        raise ValueError("cross_entropy: target id >= vocabulary size")
    loss = torch.empty(rows, dtype=torch.float32, device=logits.device)
    check(lib().fc_cross_entropy(logits.data_ptr(), logits.stride(0), t.data_ptr(), rows, V, loss.data_ptr(),
                                 _stream(logits)), "fc_cross_entropy")
    return loss


@cross_entropy.register_fake
def _(logits, targets):
    return logits.new_empty((logits.shape[0],))


# ---------------------------------------------------------------- engine entry points
import ctypes  # noqa: E402
from typing import List, Tuple  # noqa: E402

SPEC_BUFFERS = list(_lib._SPEC_PTRS) + ["part"]


def _model(addr: int):
    """(descriptor pointer, DeviceModel) of the live DeviceModel whose
    fc_model descriptor sits at host address `addr`. Any other integer (a
    stale address of a collected model, a hand-built descriptor) is refused:
    the kernels would dereference its weight pointers."""
    from .runtime import live_model
    dm = live_model(addr) if addr else None
    if dm is None:
        raise ValueError("model: the descriptor address of a live DeviceModel (ctypes.addressof(DeviceModel.desc))")
    return ctypes.pointer(dm.desc), dm


def _tdt(dm) -> torch.dtype:
    return torch.bfloat16 if dm.dtype == _lib.FC_BF16 else torch.float32


def _same_device(dm, *ts):
    """Every tensor on the model's device (meta / fake tensors carry no
    memory and are checked for shape only)."""
    for t in ts:
        if t is not None and t.device.type != "meta" and t.device != dm.device:
            raise ValueError(f"tensor on {t.device}, the model's weights are on {dm.device}")


def _cache(dm, k_cache: torch.Tensor, v_cache: torch.Tensor, hist: torch.Tensor = None) -> _lib.FcCache:
    """fc_cache over one model's cache tensors, checked against the model:
    k [n_layer][batch][n_kv_head][cap][head_dim] in the model dtype, v of as
    many elements, hist [batch][cap][n_embd] fp32 (or absent)."""
    if k_cache.dim() != 5 or (k_cache.shape[0], k_cache.shape[2], k_cache.shape[4]) != (dm.L, dm.G, dm.hd):
        raise ValueError(f"k_cache [n_layer={dm.L}][batch][n_kv_head={dm.G}][cap][head_dim={dm.hd}] "
                         f"(got {tuple(k_cache.shape)})")
    if v_cache.numel() != k_cache.numel():
        raise ValueError("v_cache must hold as many elements as k_cache")
    if k_cache.dtype != _tdt(dm) or v_cache.dtype != _tdt(dm):
        raise ValueError(f"the caches are {_tdt(dm)} like the model (got {k_cache.dtype} / {v_cache.dtype})")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("the caches must be contiguous")
    B, cap = k_cache.shape[1], k_cache.shape[3]
    if B < 1 or cap % 32 != 0:
        raise ValueError("cache capacity must be a multiple of 32")
    if hist is not None and (hist.dtype != torch.float32 or tuple(hist.shape) != (B, cap, dm.D)
                             or not hist.is_contiguous()):
        raise ValueError(f"hist: contiguous fp32 [batch={B}][cap={cap}][n_embd={dm.D}]")
    _same_device(dm, k_cache, v_cache, hist)
    return _lib.FcCache(k_cache.data_ptr(), v_cache.data_ptr(), hist.data_ptr() if hist is not None else 0, B, cap)


def _i32(*ts):
    for t in ts:
        if t.dtype != torch.int32 or not t.is_contiguous():
            raise ValueError("index arrays are contiguous int32 tensors")


def _gemm_input(dm, h: torch.Tensor, M: int, name: str):
    """h: the RMS-normed GEMM input of M tokens: bf16 in fragment order
    ([round16(M)][n_embd], as the forward writes it) or fp32 row-major."""
    rows = (M + 15) // 16 * 16 if dm.dtype == _lib.FC_BF16 else M
    if h.dtype != _tdt(dm) or h.numel() < rows * dm.D or not h.is_contiguous():
        raise ValueError(f"{name}: h is contiguous {_tdt(dm)} with at least {rows} x {dm.D} elements")


@torch.library.custom_op(f"{NS}::forward", mutates_args=("k_cache", "v_cache", "hist", "logits", "workspace"))
def forward(model: int, k_cache: torch.Tensor, v_cache: torch.Tensor, hist: torch.Tensor, tokens: torch.Tensor,
            row_off: torch.Tensor, start: torch.Tensor, max_per_row: int, n_out: int, logits: torch.Tensor,
            workspace: torch.Tensor, typ_tokens: int = 0, flags: int = 0) -> None:
    m, dm = _model(model)
    c = _cache(dm, k_cache, v_cache, hist)
    _i32(tokens, row_off, start)
    _same_device(dm, tokens, row_off, start, logits, workspace)
    B = c.batch
    if row_off.numel() != B + 1 or start.numel() != B:
        raise ValueError("forward: row_off has batch + 1 entries and start batch")
    V = dm.V
    if n_out > 0 and (logits.dtype != torch.float32 or logits.numel() < B * n_out * V or not logits.is_contiguous()):
        raise ValueError("forward: logits is contiguous fp32 with at least batch * n_out * vocab elements")
    need = lib().fc_forward_workspace_bytes(m, B, tokens.numel(), max_per_row, typ_tokens)
    if need < 0 or workspace.numel() < need:
        raise ValueError(f"forward: workspace of {workspace.numel()} bytes, {need} needed")
    ch = _lib.FcChunk(tokens.numel(), max_per_row, typ_tokens, tokens.data_ptr(), row_off.data_ptr(),
                      start.data_ptr(), n_out, logits.data_ptr() if n_out > 0 else 0, n_out * V, flags)
    check(lib().fc_forward(m, ctypes.byref(c), ctypes.byref(ch), workspace.data_ptr(), workspace.numel(),
                           _stream(tokens)), "fc_forward")


@forward.register_fake
def _(model, k_cache, v_cache, hist, tokens, row_off, start, max_per_row, n_out, logits, workspace, typ_tokens=0,
      flags=0):
    return None


def _q_out(dm, M: int, like: torch.Tensor) -> torch.Tensor:
    return torch.empty((M, dm.H, dm.hd), dtype=_tdt(dm), device=like.device)


@torch.library.custom_op(f"{NS}::attn_prologue", mutates_args=("k_cache", "v_cache"))
def attn_prologue(model: int, layer: int, k_cache: torch.Tensor, v_cache: torch.Tensor, qkv: torch.Tensor,
                  h: torch.Tensor, tokens: torch.Tensor, tok_row: torch.Tensor, tok_pos: torch.Tensor) -> torch.Tensor:
    _i32(tokens, tok_row, tok_pos)
    m, dm = _model(model)
    M = tokens.numel()
    if not 0 <= layer < dm.L:
        raise ValueError(f"attn_prologue: layer {layer} outside [0, {dm.L})")
    nqkv = (dm.H + 2 * dm.G) * dm.hd
    if (qkv.dtype != torch.float32 or qkv.dim() != 2 or qkv.shape[0] < M or qkv.shape[1] != nqkv
            or not qkv.is_contiguous()):
        raise ValueError(f"attn_prologue: qkv is contiguous fp32 [M][{nqkv}]")
    if tok_row.numel() < M or tok_pos.numel() < M:
        raise ValueError("attn_prologue: tok_row / tok_pos hold one entry per token")
    _gemm_input(dm, h, M, "attn_prologue")
    c = _cache(dm, k_cache, v_cache)
    _same_device(dm, qkv, h, tokens, tok_row, tok_pos)
    q = _q_out(dm, M, qkv)
    check(lib().fc_attn_prologue(m, layer, ctypes.byref(c), qkv.data_ptr(), h.data_ptr(),
                                 tokens.data_ptr(), tok_row.data_ptr(), tok_pos.data_ptr(), M, q.data_ptr(),
                                 _stream(qkv)), "fc_attn_prologue")
    return q


def _q_fake(model: int, M, like: torch.Tensor, cache: torch.Tensor) -> torch.Tensor:
    _, dm = _model(model)  # the descriptor is host memory: readable while tracing
    return like.new_empty((M, dm.H, dm.hd), dtype=cache.dtype)


@attn_prologue.register_fake
def _(model, layer, k_cache, v_cache, qkv, h, tokens, tok_row, tok_pos):
    return _q_fake(model, tokens.shape[0], qkv, k_cache)


@torch.library.custom_op(f"{NS}::attn_qkv", mutates_args=("k_cache", "v_cache"))
def attn_qkv(model: int, layer: int, k_cache: torch.Tensor, v_cache: torch.Tensor, h: torch.Tensor,
             tokens: torch.Tensor, tok_row: torch.Tensor, tok_pos: torch.Tensor, typ_tokens: int = 0) -> torch.Tensor:
    _i32(tokens, tok_row, tok_pos)
    M = tokens.numel()
    m, dm = _model(model)
    if not 0 <= layer < dm.L:
        raise ValueError(f"attn_qkv: layer {layer} outside [0, {dm.L})")
    if tok_row.numel() < M or tok_pos.numel() < M:
        raise ValueError("attn_qkv: tok_row / tok_pos hold one entry per token")
    _gemm_input(dm, h, M, "attn_qkv")
    c = _cache(dm, k_cache, v_cache)
    _same_device(dm, h, tokens, tok_row, tok_pos)
    q = _q_out(dm, M, h)
    need = lib().fc_attn_qkv_workspace_bytes(m, M, typ_tokens)
    ws = torch.empty(max(need, 1), dtype=torch.uint8, device=h.device)
    check(lib().fc_attn_qkv(m, layer, ctypes.byref(c), h.data_ptr(), tokens.data_ptr(), tok_row.data_ptr(),
                            tok_pos.data_ptr(), M, typ_tokens, q.data_ptr(), ws.data_ptr(), ws.numel(), _stream(h)),
          "fc_attn_qkv")
    return q


@attn_qkv.register_fake
def _(model, layer, k_cache, v_cache, h, tokens, tok_row, tok_pos, typ_tokens=0):
    return _q_fake(model, tokens.shape[0], h, k_cache)


@torch.library.custom_op(f"{NS}::row_stats", mutates_args=())
def row_stats(logits: torch.Tensor, temperature: float, top_k: int) -> Tuple[torch.Tensor, torch.Tensor,
                                                                             torch.Tensor, torch.Tensor,
                                                                             torch.Tensor]:
    if logits.dtype != torch.float32 or logits.dim() != 2 or not logits.is_contiguous():
        raise ValueError("row_stats takes contiguous fp32 logits [rows][V]")
    rows, V = logits.shape
    f = [torch.empty(rows, dtype=torch.float32, device=logits.device) for _ in range(3)]
    i = [torch.empty(rows, dtype=torch.int32, device=logits.device) for _ in range(2)]
    check(lib().fc_row_stats_fields(logits.data_ptr(), rows, V, temperature, top_k, *[t.data_ptr() for t in f + i],
                                    _stream(logits)), "fc_row_stats_fields")
    return f[0], f[1], f[2], i[0], i[1]


@row_stats.register_fake
def _(logits, temperature, top_k):
    r = logits.shape[0]
    f = lambda: logits.new_empty((r,))  # noqa: E731
    i = lambda: logits.new_empty((r,), dtype=torch.int32)  # noqa: E731
    return f(), f(), f(), i(), i()


_PMAX, _RES_STRIDE, _ROWSTAT = 16, 40, ctypes.sizeof(_lib.FcRowstat)


def _spec_bytes(batch: int, k: int, gen_cap: int, vocab: int) -> dict:
    """Bytes each fc_spec_state array needs (include/flaxchat_amd.h)."""
    B = batch
    n = dict(t_len=B, d_len=B, t_pend=B * _PMAX, d_pend=B * _PMAX, t_pend_n=B, d_pend_n=B, t_dirty=B, d_dirty=B,
             gen=B * gen_cap, gen_n=B, prompt_len=B, round=B, stall=B, result=B * _RES_STRIDE, tok_d0=B * _PMAX,
             off_d0=B + 1, start_d=k * B, tok_ds=k * B, off_ds=B + 1, tok_v=B * (_PMAX + k), off_v=B + 1,
             start_v=B, drafts=B * k, q_logits=B * k * vocab, p_logits=B * (k + 1) * vocab)
    out = {name: 4 * v for name, v in n.items()}
    out["q_stats"] = B * k * _ROWSTAT
    out["p_stats"] = B * (k + 1) * _ROWSTAT
    out["part"] = int(lib().fc_spec_part_bytes(B, k, vocab))
    return out


def _spec_state(buffers: List[torch.Tensor], batch, k, max_tokens, gen_cap, vocab, temperature, top_k, seed,
                device=None):
    if len(buffers) != len(SPEC_BUFFERS):
        raise ValueError(f"buffers: the {len(SPEC_BUFFERS)} arrays of SPEC_BUFFERS in order")
    if batch < 1 or k < 1 or vocab < 1 or gen_cap < 1:
        raise ValueError("batch, k, gen_cap and vocab must be positive")
    need = _spec_bytes(batch, k, gen_cap, vocab)
    dev = device if device is not None else buffers[0].device
    for name, t in zip(SPEC_BUFFERS, buffers):
        if not t.is_contiguous():
            raise ValueError(f"buffer {name} must be contiguous")
        if t.numel() * t.element_size() < need[name]:
            raise ValueError(f"buffer {name}: {t.numel() * t.element_size()} bytes, {need[name]} needed "
                             f"for batch {batch}, k {k}, gen_cap {gen_cap}, vocab {vocab}")
        if t.device != dev:
            raise ValueError(f"buffer {name} is on {t.device}, not {dev}")
    part = buffers[-1]
    return _lib.FcSpecState(batch, k, max_tokens, gen_cap, vocab, temperature, top_k, seed,
                            *[t.data_ptr() for t in buffers[:-1]], part.data_ptr(), part.numel())


@torch.library.custom_op(f"{NS}::spec_accept", mutates_args=("buffers",))
def spec_accept(buffers: List[torch.Tensor], batch: int, k: int, max_tokens: int, gen_cap: int, vocab: int,
                temperature: float, top_k: int, seed: int) -> None:
    if buffers and buffers[0].device.type != "cuda":
        raise ValueError("spec_accept: the state buffers live on a CUDA device")
    st = _spec_state(buffers, batch, k, max_tokens, gen_cap, vocab, temperature, top_k, seed)
    check(lib().fc_spec_accept(ctypes.byref(st), _stream(buffers[0])), "fc_spec_accept")


@spec_accept.register_fake
def _(buffers, batch, k, max_tokens, gen_cap, vocab, temperature, top_k, seed):
    return None


@torch.library.custom_op(f"{NS}::spec_round",
                         mutates_args=("t_k", "t_v", "t_hist", "d_k", "d_v", "d_hist", "buffers", "workspace"))
def spec_round(target: int, draft: int, t_k: torch.Tensor, t_v: torch.Tensor, t_hist: torch.Tensor,
               d_k: torch.Tensor, d_v: torch.Tensor, d_hist: torch.Tensor, buffers: List[torch.Tensor], batch: int,
               k: int, max_tokens: int, gen_cap: int, vocab: int, temperature: float, top_k: int, seed: int,
               workspace: torch.Tensor) -> None:
    (mt, tdm), (md, ddm) = _model(target), _model(draft)
    if tdm.V != vocab or ddm.V != vocab:
        raise ValueError(f"spec_round: vocab {vocab}, the models have {tdm.V} / {ddm.V}")
    if tdm.device != ddm.device:
        raise ValueError("spec_round: target and draft on different devices")
    tc, dc = _cache(tdm, t_k, t_v, t_hist), _cache(ddm, d_k, d_v, d_hist)
    if tc.batch != batch or dc.batch != batch:
        raise ValueError(f"spec_round: the caches hold {tc.batch} / {dc.batch} rows, batch is {batch}")
    _same_device(tdm, workspace)
    st = _spec_state(buffers, batch, k, max_tokens, gen_cap, vocab, temperature, top_k, seed, device=tdm.device)
    need = lib().fc_spec_workspace_bytes(mt, md, batch, k)
    if need < 0 or workspace.numel() < need:
        raise ValueError(f"spec_round: workspace of {workspace.numel()} bytes, {need} needed")
    check(lib().fc_spec_round(mt, ctypes.byref(tc), md, ctypes.byref(dc), ctypes.byref(st), workspace.data_ptr(),
                              workspace.numel(), _stream(workspace)), "fc_spec_round")


@spec_round.register_fake
def _(target, draft, t_k, t_v, t_hist, d_k, d_v, d_hist, buffers, batch, k, max_tokens, gen_cap, vocab, temperature,
      top_k, seed, workspace):
    return None


# ---------------------------------------------------------------- paged KV cache
# Registered below custom_op, which costs about 12 us a call: a decode step's kernels take less.
from typing import Optional  # noqa: E402

_PAGED = torch.library.Library(NS, "FRAGMENT")


def _op(schema: str):
    """Defines operator `schema` with the decorated function as its implementation on every device (which
    itself refuses tensors off the GPU)."""
    def deco(fn):
        _PAGED.define(schema)
        _PAGED.impl(schema[:schema.index("(")], fn, "CompositeExplicitAutograd")
        return fn
    return deco


def _on_gpu(name: str, first: torch.Tensor, *rest: torch.Tensor) -> int:
    """The index of the CUDA device that all tensors are on."""
    d = first.get_device()
    for t in rest:
        if t.get_device() != d:
            raise ValueError(f"{name}: tensors on {first.device} and {t.device}")
    if d < 0:
        raise ValueError(f"{name}: tensors live on a CUDA device (got {first.device})")
    return d


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)  # the handle alone: a tenth of current_stream's time


def _launch(name: str, device: int, fn, *args):
    """fn(*args, stream) on `device`'s current stream, with that device current."""
    s = _raw_stream(device) if _raw_stream else torch.cuda.current_stream(device).cuda_stream
    if device == torch.cuda.current_device():
        rc = fn(*args, s)
    else:
        with torch.cuda.device(device):
            rc = fn(*args, s)
    if rc != 0:
        check(rc, name)


# Takes what an operator writes, so that autograd notices if it had kept one of them: nothing else does below custom_op.
_written = torch.autograd.graph.increment_version


def _inner_contiguous(t: torch.Tensor) -> bool:
    """Whether t[0] is contiguous."""
    want = 1
    for n, st in zip(reversed(t.shape[1:]), reversed(t.stride()[1:])):
        if n != 1 and st != want:
            return False
        want *= n
    return True


def _pages(name: str, k_pages: torch.Tensor, v_pages: torch.Tensor):
    """(fc_pages, n_kv_head, page, head_dim) of a pool."""
    if k_pages.dim() != 4:
        raise ValueError(f"{name}: k_pages [n_pages][n_kv_head][page][head_dim] (got {tuple(k_pages.shape)})")
    N, G, page, hd = k_pages.shape
    if page == 0 or page % 32 != 0:
        raise ValueError(f"{name}: page must be a multiple of 32 (got {page})")
    if N < 1 or G < 1 or not 1 <= hd <= 256 or max(N, G, page) > 0x7fffffff:
        raise ValueError(f"{name}: n_pages, n_kv_head and head_dim (at most 256) must be positive, and below 2^31")
    if v_pages.shape != (N, G, page // 32, hd, 32):
        raise ValueError(f"{name}: v_pages {[N, G, page // 32, hd, 32]} (got {tuple(v_pages.shape)})")
    dt = k_pages.dtype
    if v_pages.dtype != dt:
        raise ValueError(f"{name}: k_pages and v_pages share one dtype")
    ks = vs = G * page * hd
    if not (k_pages.is_contiguous() and v_pages.is_contiguous()):
        if N > 1:
            ks, vs = k_pages.stride(0), v_pages.stride(0)
        if min(ks, vs) < G * page * hd or not (_inner_contiguous(k_pages) and _inner_contiguous(v_pages)):
            raise ValueError(f"{name}: each page must be contiguous, and pages must not overlap")
    code = _lib.FC_BF16 if dt == torch.bfloat16 else _dtype_code(k_pages)
    return _lib.FcPages(k_pages.data_ptr(), v_pages.data_ptr(), ks, vs, N, G, page, hd, code), G, page, hd


def _index(name: str, what: str, t: torch.Tensor, n: int):
    if t.dtype != torch.int32 or t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{name}: {what} is a contiguous int32 tensor of {n} entries "
                         f"(got {t.dtype}, {tuple(t.shape)})")


@_op("page_tables(Tensor(a!) tables, Tensor(b!) held, Tensor(c!) free_pages, Tensor(d!) n_free, Tensor length, "
     "Tensor n_new, Tensor(e!) row_off, Tensor(f!) start, Tensor(g!) tok_row, Tensor(h!) tok_pos, Tensor(i!) slots, "
     "int page, int prefix_len=0) -> ()")
def page_tables(tables, held, free_pages, n_free, length, n_new, row_off, start, tok_row, tok_pos, slots, page,
                prefix_len=0):
    if tables.dim() != 2:
        raise ValueError(f"page_tables: tables [batch][width] (got {tuple(tables.shape)})")
    B, W = tables.shape
    T, F = slots.numel(), free_pages.numel()
    if not 1 <= B <= 4096 or W < 1 or not 1 <= T < 1 << 30 or F >= 1 << 30:
        raise ValueError("page_tables: batch in [1, 4096], width and tokens not empty, both and free_pages below 2^30")
    if page < 32 or page % 32 != 0 or prefix_len < 0 or W * page + prefix_len > 0x7fffffff:
        raise ValueError("page_tables: page a multiple of 32, prefix_len >= 0, positions below 2^31")
    ts = (tables, held, free_pages, n_free, length, n_new, row_off, start, tok_row, tok_pos, slots)
    sizes = (B * W, B, F, 1, B, B, B + 1, B, T, T, T)
    i32, d = torch.int32, tables.get_device()
    for t, n in zip(ts, sizes):  # (one walk over the arrays: their checks are most of a call's time)
        if t.dtype is not i32 or t.numel() != n or not t.is_contiguous() or t.get_device() != d or d < 0:
            for what, t, n in zip(("tables", "held", "free_pages", "n_free", "length", "n_new", "row_off", "start",
                                   "tok_row", "tok_pos", "slots"), ts, sizes):
                _index("page_tables", what, t, n)
            _on_gpu("page_tables", *ts)
    _written((tables, held, free_pages, n_free, row_off, start, tok_row, tok_pos, slots))
    _launch("fc_page_tables", d, lib().fc_page_tables, *[t.data_ptr() for t in ts], B, W, F, T, page, prefix_len)


@_op("page_append(Tensor k, Tensor v, Tensor slots, Tensor(a!) k_pages, Tensor(b!) v_pages) -> ()")
def page_append(k, v, slots, k_pages, v_pages):
    p, G, _, hd = _pages("page_append", k_pages, v_pages)
    if k.dim() != 3 or k.shape[1:] != (G, hd) or v.shape != k.shape:
        raise ValueError(f"page_append: k and v [tokens][{G}][{hd}] (got {tuple(k.shape)} and {tuple(v.shape)})")
    if k.dtype != v.dtype or (k.dtype != k_pages.dtype and k.dtype != torch.float32):
        raise ValueError(f"page_append: k and v in the pages' dtype or fp32 (got {k.dtype} and {v.dtype})")
    if (k.requires_grad or v.requires_grad or k_pages.requires_grad or v_pages.requires_grad) and \
            torch.is_grad_enabled():
        raise ValueError("page_append has no backward pass")
    M = k.shape[0]
    if M > 0x7fffffff:
        raise ValueError("page_append: tokens below 2^31")
    _index("page_append", "slots", slots, M)
    d = _on_gpu("page_append", k_pages, v_pages, k, v, slots)
    if M == 0:
        return
    _written((k_pages, v_pages))
    kt, kh, kd = k.stride()
    vt, vh, vd = v.stride()
    if hd != 1 and (kd != 1 or vd != 1):
        k, v = k.contiguous(), v.contiguous()
        (kt, kh, _), (vt, vh, _) = k.stride(), v.stride()
    _launch("fc_page_append", d, lib().fc_page_append, p, k.data_ptr(), v.data_ptr(), kt, kh, vt, vh, _dtype_code(k),
            slots.data_ptr(), M)


@_op("paged_attention(Tensor q, Tensor k_pages, Tensor v_pages, Tensor tables, Tensor row_off, Tensor start, "
     "int max_per_row, int window, Tensor? prefix_pages=None, int prefix_len=0) -> Tensor")
def paged_attention(q, k_pages, v_pages, tables, row_off, start, max_per_row, window, prefix_pages=None,
                    prefix_len=0):
    return _attend("paged_attention", q, k_pages, v_pages, tables, row_off, start, (), max_per_row, window,
                   prefix_pages, prefix_len)


def _attend(name, q, k_pages, v_pages, tables, row_off, start, tree, max_per_row, window, prefix_pages, prefix_len):
    """paged_attention, or with tree = (mask, tok_pos) tree_attention."""
    p, G, page, hd = _pages(name, k_pages, v_pages)
    if q.dim() != 3 or q.shape[2] != hd or q.shape[1] == 0 or q.shape[1] % G != 0:
        raise ValueError(f"{name}: q [tokens][n_head][{hd}], n_head a multiple of {G} "
                         f"(got {tuple(q.shape)})")
    if q.dtype != k_pages.dtype:
        raise ValueError(f"{name}: q and the pages share one dtype")
    if (q.requires_grad or k_pages.requires_grad or v_pages.requires_grad) and torch.is_grad_enabled():
        raise ValueError(f"{name} has no backward pass")
    if tables.dim() != 2:
        raise ValueError(f"{name}: tables [batch][width] (got {tuple(tables.shape)})")
    B, W = tables.shape
    T, H, _ = q.shape
    if not 1 <= B <= 4096 or W < 1 or H > 65535 or not 1 <= max_per_row <= 0x7fffffff:
        raise ValueError(f"{name}: batch in [1, 4096], width and max_per_row at least 1 and below 2^31")
    if not 0 <= window <= 0x7fffffff or T > 0x7fffffff:
        raise ValueError(f"{name}: window in [0, 2^31), tokens below 2^31")
    if prefix_len < 0 or W * page + prefix_len > 0x7fffffff:
        raise ValueError(f"{name}: prefix_len >= 0, positions below 2^31")
    _index(name, "tables", tables, B * W)
    _index(name, "row_off", row_off, B + 1)
    _index(name, "start", start, B)
    if tree:
        _tree_rows(name, max_per_row)
        mask, tok_pos = tree
        if mask.dtype is not torch.int64 or mask.shape != (T, (max_per_row + 63) // 64) or not mask.is_contiguous():
            raise ValueError(f"{name}: mask is a contiguous int64 tensor [{T}][{(max_per_row + 63) // 64}] "
                             f"(got {mask.dtype}, {tuple(mask.shape)})")
        _index(name, "tok_pos", tok_pos, T)
    pre = 0
    if prefix_len > 0:
        if prefix_pages is None or prefix_pages.numel() * page < prefix_len:
            raise ValueError(f"{name}: prefix_pages holds the pages of {prefix_len} positions")
        _index(name, "prefix_pages", prefix_pages, prefix_pages.numel())
        pre = prefix_pages.data_ptr()
        d = _on_gpu(name, q, k_pages, v_pages, tables, row_off, start, prefix_pages, *tree)
    else:
        d = _on_gpu(name, q, k_pages, v_pages, tables, row_off, start, *tree)
    y = q.new_empty((T, H * hd))
    if T == 0:
        return y
    qt, qh, qd = q.stride()
    if hd != 1 and qd != 1:
        q = q.contiguous()
        qt, qh, _ = q.stride()
    L = lib()
    query, call = (L.fc_tree_attention_workspace_bytes, L.fc_tree_attention) if tree else \
        (L.fc_paged_attention_workspace_bytes, L.fc_paged_attention)
    nb = query(p, B, T, max_per_row, H, W, prefix_len, window)
    if nb < 0:
        check(nb, f"fc_{name}_workspace_bytes")
    ws = torch.empty(nb, dtype=torch.uint8, device=q.device) if nb else None  # held until the launch is queued
    _launch(f"fc_{name}", d, call, p, q.data_ptr(), qt, qh, y.data_ptr(), B, T, max_per_row, H, tables.data_ptr(), W,
            row_off.data_ptr(), start.data_ptr(), *[t.data_ptr() for t in tree], pre, prefix_len, window,
            _lib.FC_PAGED_ZERO_TAIL, ws.data_ptr() if nb else 0, nb)
    return y


@torch.library.register_fake(f"{NS}::page_tables", lib=_PAGED)
def _(tables, held, free_pages, n_free, length, n_new, row_off, start, tok_row, tok_pos, slots, page, prefix_len=0):
    _written((tables, held, free_pages, n_free, row_off, start, tok_row, tok_pos, slots))


@torch.library.register_fake(f"{NS}::page_append", lib=_PAGED)
def _(k, v, slots, k_pages, v_pages):
    _written((k_pages, v_pages))


@torch.library.register_fake(f"{NS}::paged_attention", lib=_PAGED)
def _(q, k_pages, v_pages, tables, row_off, start, max_per_row, window, prefix_pages=None, prefix_len=0):
    return q.new_empty((q.shape[0], q.shape[1] * q.shape[2]))


# ---------------------------------------------------------------- trees of drafted tokens
def _tree_rows(name: str, max_per_row: int):
    if not 1 <= max_per_row <= _lib.FC_TREE_MOST:
        raise ValueError(f"{name}: max_per_row in [1, {_lib.FC_TREE_MOST}]")


def _tree_chunk(name: str, names: str, row_off: torch.Tensor, max_per_row: int, per_token, per_row=()):
    """(batch, tokens, device) of a chunk, its arrays checked; `names`: those of the arrays."""
    _tree_rows(name, max_per_row)
    n, T, i32, d = row_off.numel(), per_token[0].numel(), torch.int32, row_off.get_device()
    if not 2 <= n <= 4097 or T >= 1 << 30:
        raise ValueError(f"{name}: row_off of 2 to 4097 entries, tokens below 2^30")
    ok = row_off.dtype is i32 and row_off.is_contiguous() and d >= 0
    for t in per_token:  # (one walk over the arrays: their checks are most of a call's time)
        ok = ok and t.dtype is i32 and t.numel() == T and t.is_contiguous() and t.get_device() == d
    for t in per_row:
        ok = ok and t.dtype is i32 and t.numel() == n - 1 and t.is_contiguous() and t.get_device() == d
    if not ok:
        sizes = [n] + [T] * len(per_token) + [n - 1] * len(per_row)
        for what, t, k in zip(names.split(), (row_off, *per_token, *per_row), sizes):
            _index(name, what, t, k)
        _on_gpu(name, row_off, *per_token, *per_row)
    return n - 1, T, d


@_op("tree_tables(Tensor parent, Tensor row_off, Tensor start, int max_per_row, int window=0) -> (Tensor, Tensor)")
def tree_tables(parent, row_off, start, max_per_row, window=0):
    if not 0 <= window <= 0x7fffffff:
        raise ValueError("tree_tables: window in [0, 2^31)")
    B, T, d = _tree_chunk("tree_tables", "row_off parent start", row_off, max_per_row, (parent,), (start,))
    mask = parent.new_empty((T, (max_per_row + 63) // 64), dtype=torch.int64)
    tok_pos = parent.new_empty((T,))
    if T > 0:
        _launch("fc_tree_tables_window", d, lib().fc_tree_tables_window, parent.data_ptr(), row_off.data_ptr(),
                start.data_ptr(), mask.data_ptr(), tok_pos.data_ptr(), B, T, max_per_row, window)
    return mask, tok_pos


@_op("tree_attention(Tensor q, Tensor k_pages, Tensor v_pages, Tensor tables, Tensor row_off, Tensor start, "
     "Tensor mask, Tensor tok_pos, int max_per_row, int window, Tensor? prefix_pages=None, int prefix_len=0) "
     "-> Tensor")
def tree_attention(q, k_pages, v_pages, tables, row_off, start, mask, tok_pos, max_per_row, window,
                   prefix_pages=None, prefix_len=0):
    return _attend("tree_attention", q, k_pages, v_pages, tables, row_off, start, (mask, tok_pos), max_per_row, window,
                   prefix_pages, prefix_len)


@_op("tree_accept(Tensor parent, Tensor tokens, Tensor target, Tensor row_off, int max_per_row) "
     "-> (Tensor, Tensor, Tensor)")
def tree_accept(parent, tokens, target, row_off, max_per_row):
    B, T, d = _tree_chunk("tree_accept", "row_off parent tokens target", row_off, max_per_row,
                          (parent, tokens, target))
    n_accepted, next_token, path = (parent.new_empty((n,)) for n in (B, B, T))
    if T == 0:
        n_accepted.fill_(0)
        next_token.fill_(-1)
    else:
        _launch("fc_tree_accept", d, lib().fc_tree_accept, parent.data_ptr(), tokens.data_ptr(), target.data_ptr(),
                row_off.data_ptr(), n_accepted.data_ptr(), next_token.data_ptr(), path.data_ptr(), B, T, max_per_row)
    return n_accepted, next_token, path


@_op("tree_commit(Tensor path, Tensor slots, Tensor row_off, int max_per_row, Tensor(a!) k_pages, "
     "Tensor(b!) v_pages) -> ()")
def tree_commit(path, slots, row_off, max_per_row, k_pages, v_pages):
    L, ks, vs = 1, 0, 0
    if k_pages.dim() == 5:  # all layers
        if v_pages.dim() != 6 or v_pages.shape[0] != k_pages.shape[0] or not 1 <= k_pages.shape[0] <= 65535:
            raise ValueError(f"tree_commit: k_pages and v_pages of as many layers, 1 to 65535 (got "
                             f"{tuple(k_pages.shape)} and {tuple(v_pages.shape)})")
        L = k_pages.shape[0]
        kl, vl = k_pages[0], v_pages[0]
        if L > 1:
            ks, vs = k_pages.stride(0), v_pages.stride(0)
    else:
        kl, vl = k_pages, v_pages
    p, G, page, hd = _pages("tree_commit", kl, vl)
    if L > 1 and not (_layers_apart(k_pages) and _layers_apart(v_pages)):
        raise ValueError("tree_commit: layers must not overlap")
    if G > 65535:
        raise ValueError("tree_commit: n_kv_head at most 65535")
    if (k_pages.requires_grad or v_pages.requires_grad) and torch.is_grad_enabled():
        raise ValueError("tree_commit has no backward pass")
    B, T, d = _tree_chunk("tree_commit", "row_off path slots", row_off, max_per_row, (path, slots))
    if k_pages.get_device() != d or v_pages.get_device() != d:
        _on_gpu("tree_commit", path, k_pages, v_pages)
    if T == 0:
        return
    _written((k_pages, v_pages))
    _launch("fc_tree_commit", d, lib().fc_tree_commit, p, L, ks, vs, path.data_ptr(), slots.data_ptr(),
            row_off.data_ptr(), B, T, max_per_row)


def _layers_apart(t: torch.Tensor) -> bool:
    """Whether layers [n_layer][n_pages].. share no element: one behind the other, or page by page."""
    one = t[0, 0].numel()
    ls, ps, L, N = t.stride(0), t.stride(1) if t.shape[1] > 1 else one, t.shape[0], t.shape[1]
    return ls >= ps * (N - 1) + one or (ls >= one and ps >= ls * (L - 1) + one)


@_op("rope_append(Tensor q, Tensor k, Tensor v, Tensor tok_pos, Tensor slots, Tensor cos, Tensor sin, "
     "Tensor(a!) k_pages, Tensor(b!) v_pages, bool interleaved=False, float norm=0.0) -> Tensor")
def rope_append(q, k, v, tok_pos, slots, cos, sin, k_pages, v_pages, interleaved=False, norm=0.0):
    p, G, _, hd = _pages("rope_append", k_pages, v_pages)
    qs, cs, dt = q.shape, cos.shape, k.dtype
    if len(qs) != 3 or qs[2] != hd or not 1 <= qs[1] <= 65535 or G > 65535:
        raise ValueError(f"rope_append: q [tokens][n_head][{hd}], at most 65535 heads (got {tuple(qs)})")
    M, H, _ = qs
    if k.shape != (M, G, hd) or v.shape != (M, G, hd):
        raise ValueError(f"rope_append: k and v [{M}][{G}][{hd}] (got {tuple(k.shape)} and {tuple(v.shape)})")
    if q.dtype is not dt or v.dtype is not dt or (dt is not k_pages.dtype and dt is not torch.float32):
        raise ValueError(f"rope_append: q, k and v in the pages' dtype or fp32 (got {q.dtype}, {dt} and {v.dtype})")
    if (q.requires_grad or k.requires_grad or v.requires_grad or cos.requires_grad or sin.requires_grad or
            k_pages.requires_grad or v_pages.requires_grad) and torch.is_grad_enabled():
        raise ValueError("rope_append has no backward pass")
    if len(cs) != 2 or sin.shape != cs or not 1 <= cs[1] <= hd // 2 or not 1 <= cs[0] <= 0x7fffffff:
        raise ValueError(f"rope_append: cos and sin [positions][pairs], up to {hd // 2} pairs of a head (got "
                         f"{tuple(cs)} and {tuple(sin.shape)})")
    if cos.dtype is not torch.float32 or sin.dtype is not torch.float32 or \
            not (cos.is_contiguous() and sin.is_contiguous()):
        raise ValueError("rope_append: cos and sin are contiguous fp32 tensors")
    if not 0.0 <= norm <= 3e35:
        raise ValueError(f"rope_append: norm in [0, 3e35] (got {norm})")
    if M > 0x7fffffff:
        raise ValueError("rope_append: tokens below 2^31")
    _index("rope_append", "tok_pos", tok_pos, M)
    _index("rope_append", "slots", slots, M)
    d = _on_gpu("rope_append", q, k, v, tok_pos, slots, cos, sin, k_pages, v_pages)
    out = q.new_empty(qs) if dt is k_pages.dtype else q.new_empty(qs, dtype=k_pages.dtype)
    if M == 0:
        return out
    _written((k_pages, v_pages))
    (qt, qh, qd), (kt, kh, kd), (vt, vh, vd) = q.stride(), k.stride(), v.stride()
    if hd != 1 and (qd != 1 or kd != 1 or vd != 1):
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
        (qt, qh, _), (kt, kh, _), (vt, vh, _) = q.stride(), k.stride(), v.stride()
    _launch("fc_rope_append", d, lib().fc_rope_append, p, q.data_ptr(), k.data_ptr(), v.data_ptr(), qt, qh, kt, kh, vt,
            vh, _dtype_code(k), tok_pos.data_ptr(), slots.data_ptr(), cos.data_ptr(), sin.data_ptr(), cs[0], 2 * cs[1],
            interleaved, norm, out.data_ptr(), H, M)
    return out


@torch.library.register_fake(f"{NS}::tree_tables", lib=_PAGED)
def _(parent, row_off, start, max_per_row, window=0):
    T = parent.numel()
    return parent.new_empty((T, (max_per_row + 63) // 64), dtype=torch.int64), parent.new_empty((T,))


@torch.library.register_fake(f"{NS}::tree_attention", lib=_PAGED)
def _(q, k_pages, v_pages, tables, row_off, start, mask, tok_pos, max_per_row, window, prefix_pages=None,
      prefix_len=0):
    return q.new_empty((q.shape[0], q.shape[1] * q.shape[2]))


@torch.library.register_fake(f"{NS}::tree_accept", lib=_PAGED)
def _(parent, tokens, target, row_off, max_per_row):
    B, T = row_off.numel() - 1, parent.numel()
    return parent.new_empty((B,)), parent.new_empty((B,)), parent.new_empty((T,))


@torch.library.register_fake(f"{NS}::tree_commit", lib=_PAGED)
def _(path, slots, row_off, max_per_row, k_pages, v_pages):
    _written((k_pages, v_pages))


@torch.library.register_fake(f"{NS}::rope_append", lib=_PAGED)
def _(q, k, v, tok_pos, slots, cos, sin, k_pages, v_pages, interleaved=False, norm=0.0):
    _written((k_pages, v_pages))
    return q.new_empty(q.shape, dtype=k_pages.dtype)
