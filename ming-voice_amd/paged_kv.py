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

# The argument blocks as bytes and the current stream by its raw handle: a decode step calls these wrappers once a layer, and
# building ctypes arguments and stream objects took longer than the kernels (a call of paged_append 19.6 -> 10.8 us, 9.4 where
# it makes no output; 3.8 of them are the C entry with its launch).
_APPEND, _PAGED, _PROMPT = (_mm.packer(s) for s in (_mm.PagedAppendArgs, _mm.PagedAttnArgs, _mm.PromptAttnArgs))
_HALF = (torch.bfloat16, torch.float16)
_CODES = {torch.bfloat16: _mm.MM_BF16, torch.float16: _mm.MM_FP16, torch.int32: _mm.MM_INT32, torch.int64: _mm.MM_INT64}
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda device: torch.cuda.current_stream(device).cuda_stream)


def _device(what, *tensors):
    """The index of the GPU that holds every tensor."""
    dev = tensors[0].get_device()
    for t in tensors:
        if t is not None and (t.get_device() != dev or dev < 0):
            _mm.require_gpu(*tensors)
    return dev


def _rows(what, name, t, shape, dtype):
    """(pointer, token stride, head stride) of a [tokens, heads, width] tensor with a contiguous last dim."""
    s = t.stride()
    if t.shape != shape or t.dtype is not dtype or s[-1] != 1:
        raise ValueError(f"{what}: {name} must be a {dtype} {list(shape)} tensor with a contiguous last dim (got {t.dtype} "
                         f"{list(t.shape)}, strides {s})")
    return t.data_ptr(), s[0], s[1]


def _queries(what, q, width, dtype):
    """(tokens, heads, pointer, token stride, head stride) of q."""
    shape, s = q.shape, q.stride()
    if len(shape) != 3 or shape[2] != width or q.dtype is not dtype or s[2] != 1:
        raise ValueError(f"{what}: q must be a {dtype} [tokens, heads, {width}] tensor with a contiguous last dim (got "
                         f"{q.dtype} {list(shape)}, strides {s})")
    return shape[0], shape[1], q.data_ptr(), s[0], s[1]


def _pool(what, k_pages, v_pages):
    """(mm_pages, nkv, page, dqk, dv, dtype) of the pool."""
    dt = k_pages.dtype
    if k_pages.dim() != 4 or v_pages.dim() != 4 or v_pages.dtype is not dt or dt not in _HALF:
        raise ValueError(f"{what}: k_pages and v_pages must both be bf16 or fp16 [n_pages, nkv, page, d] (got {k_pages.dtype} "
                         f"{list(k_pages.shape)}, {v_pages.dtype} {list(v_pages.shape)})")
    n, nkv, page, dqk = k_pages.shape
    m, vkv, vpage, dv = v_pages.shape
    k0, k1, k2, k3 = k_pages.stride()
    v0, v1, v2, v3 = v_pages.stride()
    if n != m or nkv != vkv or page != vpage or k3 != 1 or v3 != 1:
        raise ValueError(f"{what}: k_pages and v_pages must be [n_pages, nkv, page, d] with one n_pages, nkv and page and "
                         f"contiguous rows (got {list(k_pages.shape)}, {list(v_pages.shape)})")
    return ((k_pages.data_ptr(), v_pages.data_ptr(), _CODES[dt], nkv, dqk, dv, n, page, k0, k1, k2, v0, v1, v2),
            nkv, page, dqk, dv, dt)


def _cu(what, cu_seqlens):
    """(streams, dtype code) of cu_seqlens."""
    shape, code = cu_seqlens.shape, _CODES.get(cu_seqlens.dtype)
    if len(shape) != 1 or code not in (_mm.MM_INT32, _mm.MM_INT64) or shape[0] < 1 or not cu_seqlens.is_contiguous():
        raise ValueError(f"{what}: cu_seqlens must be a contiguous int32 or int64 [streams + 1] tensor (got "
                         f"{cu_seqlens.dtype} {list(shape)})")
    return shape[0] - 1, code


def _batch(what, page_table, cu_seqlens, kv_lens, tokens):
    """(mm_batch, streams, pages of a row of the table)."""
    B, code = _cu(what, cu_seqlens)
    it = cu_seqlens.dtype
    if kv_lens.dtype is not it or page_table.dtype is not it:
        raise ValueError(f"{what}: cu_seqlens, kv_lens and page_table must have one dtype (got {it}, {kv_lens.dtype}, "
                         f"{page_table.dtype})")
    if kv_lens.shape != (B,) or not kv_lens.is_contiguous():
        raise ValueError(f"{what}: kv_lens must be a contiguous [{B}] tensor (got {list(kv_lens.shape)})")
    shape, s = page_table.shape, page_table.stride()
    if len(shape) != 2 or shape[0] != B or (s[1] != 1 and shape[1] > 1):
        raise ValueError(f"{what}: page_table must be [{B}, pages] with contiguous rows (got {list(shape)}, strides {s})")
    pages = shape[1]
    return ((cu_seqlens.data_ptr(), kv_lens.data_ptr(), page_table.data_ptr(), s[0], pages, B, tokens, code), B, pages)


def _on(dev, fn, *args):
    """fn(*args) with device dev current."""
    if torch.cuda.current_device() == dev:
        return fn(*args)
    with torch.cuda.device(dev):
        return fn(*args)


def _call(what, dev, fn, args):
    """fn(args, stream) on device dev's current stream."""
    rc = _on(dev, fn, args, _raw_stream(dev))
    if rc:
        _mm.check(rc, what)


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
    dev = _device(what, q, k, v, k_pages, v_pages, page_table, cu_seqlens, kv_lens, inv_freq, q_out, k_out)
    pool, nkv, _, dqk, dv, dt = _pool(what, k_pages, v_pages)
    N, nh, *qr = _queries(what, q, dqk, dt)
    kr, vr = _rows(what, "k", k, (N, nkv, dqk), dt), _rows(what, "v", v, (N, nkv, dv), dt)
    batch, _, _ = _batch(what, page_table, cu_seqlens, kv_lens, N)
    if not 0 <= rot_offset <= dqk:
        raise ValueError(f"{what}: rot_offset={rot_offset} lies outside a head of {dqk}")
    inv, pairs = 0, 0
    if inv_freq is not None:
        if inv_freq.dtype is not torch.float32 or inv_freq.dim() != 1 or not inv_freq.is_contiguous():
            raise ValueError(f"{what}: inv_freq must be a contiguous fp32 [pairs] tensor (got {inv_freq.dtype} "
                             f"{list(inv_freq.shape)})")
        inv, pairs = inv_freq.data_ptr(), inv_freq.shape[0]
    if q_out is None:
        q_out = torch.empty(N, nh, dqk, device=q.device, dtype=dt)
    qo = _rows(what, "q_out", q_out, (N, nh, dqk), dt)
    ko = (0, 0, 0) if k_out is None else _rows(what, "k_out", k_out, (N, nkv, dqk), dt)
    args = _APPEND.pack(*pool, *batch, *qr, *kr, *vr, *qo, *ko, inv, pairs, nh, int(rot_offset), 1 if interleaved else 0)
    _call(what, dev, _mm.load().mm_paged_append, args)
    return q_out


def _workspace(n, like, workspace):
    """The workspace of n bytes: the caller's, or a new one where one is needed. A new one lives until its call's kernels
    are enqueued; what the allocator then hands out of it comes behind them on the stream."""
    if workspace is None and n > 0:  # else none is needed, or the call itself refuses the sizes
        workspace = torch.empty(n, dtype=torch.uint8, device=like.device)
    return workspace


def _bytes(what, workspace):
    if workspace is None:
        return 0, 0
    if not workspace.is_contiguous():
        raise ValueError(f"{what}: workspace must be contiguous (got {list(workspace.shape)}, strides {workspace.stride()})")
    return workspace.data_ptr(), workspace.numel() * workspace.element_size()


def _new_workspace(what, device, size, *args):
    with torch.cuda.device(device):  # sizes go by its compute units
        n = size(*args, 1)
    if n < 0:
        raise ValueError(f"{what}: {_mm.last_error()}")
    return torch.empty(max(n, 16), dtype=torch.uint8, device=device)


def paged_attn_workspace(tokens, streams, max_keys, nh, nkv, dqk, dv, device="cuda"):
    """A workspace for paged_attn over every batch of at most `tokens` tokens in `streams` streams behind tables of at most
    max_keys = pages * page positions (no initialisation); calls that share it must not overlap in time."""
    return _new_workspace("paged_attn_workspace", device, _mm.load().mm_paged_attn_workspace, tokens, streams, max_keys, nh,
                          nkv, dqk, dv)


def paged_attn(q, k_pages, v_pages, page_table, cu_seqlens, kv_lens, scale=None, out=None, workspace=None):
    """Attention of the new tokens over the paged cache, which holds their own rows already (paged_append): token i of
    stream b stands at position p = kv_lens[b] - n_b + i (n_b its new tokens) and takes softmax(scale * q . K[0..p]^T) .
    V[0..p], query head h on key / value head h // (nh // nkv). q [tokens, nh, dqk]; returns out [tokens, nh, dv] (scale
    defaults to dqk ** -0.5). Scores, statistics and sums in fp32; the weights meet the values in the cache's dtype. A page
    id outside [0, n_pages) leaves its positions out; a token with no position left gets zeros; kv_lens outside the table
    gives NaN. Rows past a token's position never reach it, whatever they hold. out must not overlap q or the pool.
    workspace: from paged_attn_workspace (allocated when None)."""
    what = "paged_attn"
    dev = _device(what, q, k_pages, v_pages, page_table, cu_seqlens, kv_lens, out, workspace)
    pool, nkv, page, dqk, dv, dt = _pool(what, k_pages, v_pages)
    N, nh, *qr = _queries(what, q, dqk, dt)
    batch, B, pages = _batch(what, page_table, cu_seqlens, kv_lens, N)
    if out is None:
        out = torch.empty(N, nh, dv, device=q.device, dtype=dt)
    o = _rows(what, "out", out, (N, nh, dv), dt)
    lib = _mm.load()
    ws = _workspace(_on(dev, lib.mm_paged_attn_workspace, N, B, pages * page, nh, nkv, dqk, dv, 0), q, workspace)
    args = _PAGED.pack(*pool, *batch, *qr, *o, *_bytes(what, ws), nh, dqk ** -0.5 if scale is None else scale)
    _call(what, dev, lib.mm_paged_attn, args)
    return out


def prompt_attn_workspace(tokens, prompts, nh, nkv, dqk, dv, device="cuda"):
    """A workspace for prompt_attn over at most `tokens` tokens in at most `prompts` prompts (no initialisation); calls
    that share it must not overlap in time."""
    return _new_workspace("prompt_attn_workspace", device, _mm.load().mm_prompt_attn_workspace, tokens, prompts, nh, nkv,
                          dqk, dv)


def prompt_attn(q, k, v, cu_seqlens, scale=None, out=None, workspace=None):
    """Causal attention over whole prompts packed one behind the other: token i of prompt b (rows cu_seqlens[b] ..
    cu_seqlens[b + 1] - 1) takes softmax(scale * q . K[0..i]^T) . V[0..i] over its own prompt's rows. q [tokens, nh, dqk],
    k [tokens, nkv, dqk], v [tokens, nkv, dv] (bf16 or fp16; column slices of one projection are fine); returns out
    [tokens, nh, dv] (scale defaults to dqk ** -0.5). Rounding, rows behind the last prompt and workspace (from
    prompt_attn_workspace) as for paged_attn. out must not overlap q, k or v."""
    what = "prompt_attn"
    dev = _device(what, q, k, v, cu_seqlens, out, workspace)
    dt = q.dtype
    if dt not in _HALF:
        raise ValueError(f"{what}: q must be bf16 or fp16 (got {dt})")
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise ValueError(f"{what}: q, k and v must be [tokens, heads, d] (got {list(q.shape)}, {list(k.shape)}, "
                         f"{list(v.shape)})")
    nkv, dqk, dv = k.shape[1], k.shape[2], v.shape[2]
    N, nh, *qr = _queries(what, q, dqk, dt)
    kr, vr = _rows(what, "k", k, (N, nkv, dqk), dt), _rows(what, "v", v, (N, nkv, dv), dt)
    B, code = _cu(what, cu_seqlens)
    if out is None:
        out = torch.empty(N, nh, dv, device=q.device, dtype=dt)
    o = _rows(what, "out", out, (N, nh, dv), dt)
    lib = _mm.load()
    ws = _workspace(_on(dev, lib.mm_prompt_attn_workspace, N, B, nh, nkv, dqk, dv, 0), q, workspace)
    args = _PROMPT.pack(*qr, *kr, *vr, *o, cu_seqlens.data_ptr(), B, N, *_bytes(what, ws), code, _CODES[dt], nh, nkv, dqk, dv,
                        dqk ** -0.5 if scale is None else scale)
    _call(what, dev, lib.mm_prompt_attn, args)
    return out
