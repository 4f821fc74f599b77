"""A cache in pages for several streams at once, and its attentions, on hand-written gfx950 HIP kernels: what a server
needs to step many Talkers (or the thinker's MLA layers) together, where the reference decodes one stream over a static
cache (fast_talker.py:165-212, engine.py:537-548).

  paged_append   the new tokens' keys (rotated by their positions) and values into their pages, and the rotated queries,
                 in one kernel
  paged_attn     new tokens over the paged cache: one token a stream in decode, a piece of a prompt, or both in one batch
  prompt_attn    whole prompts of different lengths packed one behind the other, causal, over their own rows

The pool: k_pages [n_pages, nkv, page, dqk], v_pages [n_pages, nkv, page, dv], bf16 or fp16, any strides with a contiguous
last dim (a permuted [n_pages, page, nkv, d] tensor too). The batch: stream b's new tokens are rows cu_seqlens[b] ..
cu_seqlens[b + 1] - 1 of the packed tensors, kv_lens[b] counts its cached rows, the new ones the last of them, and position
p lies in row p % page of page page_table[b, p // page]. cu_seqlens, kv_lens and page_table are device tensors of one
dtype (int32 or int64) that the kernels read when they run, so one captured graph serves every length; a padded batch has
streams of no tokens, and output rows behind cu_seqlens[-1] are left as they were. One layer's step is

    q = paged_append(q, k, v, k_pages, v_pages, page_table, cu_seqlens, kv_lens, inv_freq)
    o = paged_attn(q, k_pages, v_pages, page_table, cu_seqlens, kv_lens)

and for prompts that start from nothing prompt_attn(q, k, v, cu_seqlens) with the rotated keys (k_out) in the second
call's place. Every call enqueues on torch's current stream of its tensors' device and can be captured in a hipGraph;
there is no CPU path.
"""
import torch

import _mingmoe as _mm

__all__ = ["paged_append", "paged_attn", "paged_attn_workspace", "prompt_attn", "prompt_attn_workspace"]


def _rows(t, name, what, heads=None, width=None, dtype=None):
    """(pointer, token stride, head stride) of a [tokens, heads, width] tensor with a contiguous last dim; the stride of a
    dim of one is any number in torch and 0 here."""
    if t.dim() != 3 or t.stride(2) != 1 or (heads is not None and t.shape[1] != heads) or \
            (width is not None and t.shape[2] != width):
        raise ValueError(f"{what}: {name} must be [tokens, {heads or 'heads'}, {width or 'd'}] with a contiguous last dim "
                         f"(got {tuple(t.shape)}, strides {t.stride()})")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{what}: {name} must be {dtype} (got {t.dtype})")
    return t.data_ptr(), t.stride(0) if t.shape[0] > 1 else 0, t.stride(1) if t.shape[1] > 1 else 0


def _pages(k_pages, v_pages, what):
    if k_pages.dim() != 4 or v_pages.dim() != 4 or k_pages.shape[:3] != v_pages.shape[:3] or k_pages.stride(3) != 1 or \
            v_pages.stride(3) != 1:
        raise ValueError(f"{what}: k_pages and v_pages must be [n_pages, nkv, page, d] with one n_pages, nkv and page and "
                         f"contiguous rows (got {tuple(k_pages.shape)}, {tuple(v_pages.shape)})")
    if k_pages.dtype != v_pages.dtype or k_pages.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"{what}: k_pages and v_pages must both be bf16 or fp16 (got {k_pages.dtype}, {v_pages.dtype})")
    n, nkv, page, dqk = k_pages.shape
    ks, vs = ([s if m > 1 else 0 for s, m in zip(t.stride(), t.shape)] for t in (k_pages, v_pages))
    return _mm.Pages(k_pages.data_ptr(), v_pages.data_ptr(), _mm.dtype_code(k_pages), nkv, dqk, v_pages.shape[3], n, page,
                     ks[0], ks[1], ks[2], vs[0], vs[1], vs[2])


def _cu(cu_seqlens, what):
    if cu_seqlens.dim() != 1 or not cu_seqlens.is_contiguous() or cu_seqlens.shape[0] < 1 or \
            cu_seqlens.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{what}: cu_seqlens must be a contiguous int32 or int64 [streams + 1] tensor")
    return cu_seqlens.shape[0] - 1


def _batch(page_table, cu_seqlens, kv_lens, tokens, what):
    B = _cu(cu_seqlens, what)
    if kv_lens.shape != (B,) or not kv_lens.is_contiguous():
        raise ValueError(f"{what}: kv_lens must be a contiguous [{B}] tensor (got {tuple(kv_lens.shape)})")
    if page_table.dim() != 2 or page_table.shape[0] != B or (page_table.stride(1) != 1 and page_table.shape[1] > 1):
        raise ValueError(f"{what}: page_table must be [{B}, pages] with contiguous rows (got {tuple(page_table.shape)})")
    if not cu_seqlens.dtype == kv_lens.dtype == page_table.dtype:
        raise ValueError(f"{what}: cu_seqlens, kv_lens and page_table must have one dtype (got {cu_seqlens.dtype}, "
                         f"{kv_lens.dtype}, {page_table.dtype})")
    return _mm.Batch(cu_seqlens.data_ptr(), kv_lens.data_ptr(), page_table.data_ptr(), page_table.stride(0),
                     page_table.shape[1], B, tokens, _mm.dtype_code(cu_seqlens))


def paged_append(q, k, v, k_pages, v_pages, page_table, cu_seqlens, kv_lens, inv_freq=None, *, rot_offset=0,
                 interleaved=False, q_out=None, k_out=None):
    """Stores the new tokens' keys and values into their pages, rotating queries and keys by their positions on the way;
    returns the rotated queries [tokens, nh, dqk] (q_out when given; q itself is allowed).

    q [tokens, nh, dqk], k [tokens, nkv, dqk], v [tokens, nkv, dv] of the pool's dtype (column slices of one projection
    are fine; rows 16-byte aligned). inv_freq: fp32 [pairs] (a multiple of 8), the angle of pair j at position p being
    p * inv_freq[j], exact for far positions too; dims rot_offset .. rot_offset + 2 * pairs - 1 turn, first half against
    second half (as the Talker's Qwen2, fast_talker.py:176-187), or neighbours with interleaved=True. None: no rotation.
    k_out (k itself is allowed): also receives the rotated keys, for prompt_attn. A token whose position or page does not
    exist (kv_lens outside the table, a page id outside the pool) stores nothing. Streams that share pages must not
    append to the same rows."""
    what = "paged_append"
    _mm.require_gpu(q, k, v, k_pages, v_pages, page_table, cu_seqlens, kv_lens, inv_freq, q_out, k_out)
    g = _pages(k_pages, v_pages, what)
    dt = k_pages.dtype
    qr = _rows(q, "q", what, None, g.dqk, dt)
    N, nh = q.shape[0], q.shape[1]
    kr, vr = _rows(k, "k", what, g.nkv, g.dqk, dt), _rows(v, "v", what, g.nkv, g.dv, dt)
    if k.shape[0] != N or v.shape[0] != N:
        raise ValueError(f"{what}: q, k and v must hold the same tokens (got {N}, {k.shape[0]}, {v.shape[0]})")
    b = _batch(page_table, cu_seqlens, kv_lens, N, what)
    if inv_freq is not None and (inv_freq.dtype != torch.float32 or inv_freq.dim() != 1 or not inv_freq.is_contiguous()):
        raise ValueError(f"{what}: inv_freq must be a contiguous fp32 [pairs] tensor")
    if q_out is None:
        q_out = torch.empty(N, nh, g.dqk, device=q.device, dtype=dt)
    elif q_out.shape[0] != N:
        raise ValueError(f"{what}: q_out must hold {N} tokens (got {q_out.shape[0]})")
    qo = _rows(q_out, "q_out", what, nh, g.dqk, dt)
    if k_out is not None and k_out.shape[0] != N:
        raise ValueError(f"{what}: k_out must hold {N} tokens (got {k_out.shape[0]})")
    ko = (None, 0, 0) if k_out is None else _rows(k_out, "k_out", what, g.nkv, g.dqk, dt)
    with _mm.on_device(q):
        _mm.check(_mm.load().mm_paged_append(*qr, *kr, *vr, nh, g, b, _mm.ptr(inv_freq),
                                             inv_freq.shape[0] if inv_freq is not None else 0, int(rot_offset),
                                             1 if interleaved else 0, *qo, *ko, _mm.stream_of(q)), what)
    return q_out


def _workspace(n, device, what, workspace):
    """The workspace of n bytes: the caller's, or a new one; None where none is needed."""
    if n < 0:
        raise ValueError(f"{what}: {_mm.last_error()}")
    if workspace is None:
        return torch.empty(n, dtype=torch.uint8, device=device) if n else None
    return workspace


def paged_attn_workspace(tokens, streams, max_keys, nh, nkv, dqk, dv, device="cuda"):
    """The workspace paged_attn needs for a batch of up to `tokens` tokens in `streams` streams behind a table of max_keys
    = pages * page positions (no initialisation); calls that share it must not overlap in time."""
    n = _mm.load().mm_paged_attn_workspace(tokens, streams, max_keys, nh, nkv, dqk, dv)
    return _workspace(max(n, 16) if n >= 0 else n, device, "paged_attn_workspace", None)


def paged_attn(q, k_pages, v_pages, page_table, cu_seqlens, kv_lens, scale=None, out=None, workspace=None):
    """Attention of the new tokens over the paged cache, which holds their own rows already (paged_append): token i of
    stream b stands at position p = kv_lens[b] - n_b + i (n_b its new tokens) and takes softmax(scale * q . K[0..p]^T) .
    V[0..p], query head h on key / value head h // (nh // nkv). q [tokens, nh, dqk]; returns out [tokens, nh, dv] (scale
    defaults to dqk ** -0.5). Scores, statistics and sums in fp32; the weights meet the values in the cache's dtype. A page
    id outside [0, n_pages) leaves its positions out; a token with no position left gets zeros; kv_lens outside the table
    gives NaN. Rows past a token's position never reach it, whatever they hold. out must not overlap q or the pool.
    workspace: from paged_attn_workspace (allocated when None)."""
    what = "paged_attn"
    _mm.require_gpu(q, k_pages, v_pages, page_table, cu_seqlens, kv_lens, out, workspace)
    g = _pages(k_pages, v_pages, what)
    dt = k_pages.dtype
    qr = _rows(q, "q", what, None, g.dqk, dt)
    N, nh = q.shape[0], q.shape[1]
    b = _batch(page_table, cu_seqlens, kv_lens, N, what)
    if out is None:
        out = torch.empty(N, nh, g.dv, device=q.device, dtype=dt)
    elif out.shape[0] != N:
        raise ValueError(f"{what}: out must hold {N} tokens (got {out.shape[0]})")
    o = _rows(out, "out", what, nh, g.dv, dt)
    lib = _mm.load()
    with _mm.on_device(q):
        ws = _workspace(lib.mm_paged_attn_workspace(N, b.seqs, b.max_pages * g.page, nh, g.nkv, g.dqk, g.dv), q.device, what,
                        workspace)
        _mm.check(lib.mm_paged_attn(*qr, nh, g, b, float(scale) if scale is not None else g.dqk ** -0.5, *o, _mm.ptr(ws),
                                    ws.numel() * ws.element_size() if ws is not None else 0, _mm.stream_of(q)), what)
    return out


def prompt_attn_workspace(tokens, prompts, nh, nkv, dqk, dv, device="cuda"):
    """The workspace prompt_attn needs for up to `tokens` tokens in `prompts` prompts (no initialisation); calls that
    share it must not overlap in time."""
    n = _mm.load().mm_prompt_attn_workspace(tokens, prompts, nh, nkv, dqk, dv)
    return _workspace(max(n, 16) if n >= 0 else n, device, "prompt_attn_workspace", None)


def prompt_attn(q, k, v, cu_seqlens, scale=None, out=None, workspace=None):
    """Causal attention over whole prompts packed one behind the other: token i of prompt b (rows cu_seqlens[b] ..
    cu_seqlens[b + 1] - 1) takes softmax(scale * q . K[0..i]^T) . V[0..i] over its own prompt's rows. q [tokens, nh, dqk],
    k [tokens, nkv, dqk], v [tokens, nkv, dv] (bf16 or fp16; column slices of one projection are fine); returns out
    [tokens, nh, dv] (scale defaults to dqk ** -0.5). Rounding, rows behind the last prompt and workspace (from
    prompt_attn_workspace) as for paged_attn. out must not overlap q, k or v."""
    what = "prompt_attn"
    _mm.require_gpu(q, k, v, cu_seqlens, out, workspace)
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"{what}: q must be bf16 or fp16 (got {q.dtype})")
    dt = q.dtype
    qr = _rows(q, "q", what)
    N, nh, dqk = q.shape
    kr, vr = _rows(k, "k", what, None, dqk, dt), _rows(v, "v", what, k.shape[1], None, dt)
    nkv, dv = v.shape[1:]
    if k.shape[0] != N or v.shape[0] != N:
        raise ValueError(f"{what}: q, k and v must hold the same tokens (got {N}, {k.shape[0]}, {v.shape[0]})")
    B = _cu(cu_seqlens, what)
    if out is None:
        out = torch.empty(N, nh, dv, device=q.device, dtype=dt)
    elif out.shape[0] != N:
        raise ValueError(f"{what}: out must hold {N} tokens (got {out.shape[0]})")
    o = _rows(out, "out", what, nh, dv, dt)
    lib = _mm.load()
    with _mm.on_device(q):
        ws = _workspace(lib.mm_prompt_attn_workspace(N, B, nh, nkv, dqk, dv), q.device, what, workspace)
        _mm.check(lib.mm_prompt_attn(*qr, *kr, *vr, _mm.dtype_code(q), nh, nkv, dqk, dv, _mm.ptr(cu_seqlens),
                                     _mm.dtype_code(cu_seqlens), B, N, float(scale) if scale is not None else dqk ** -0.5,
                                     *o, _mm.ptr(ws), ws.numel() * ws.element_size() if ws is not None else 0,
                                     _mm.stream_of(q)), what)
    return out
