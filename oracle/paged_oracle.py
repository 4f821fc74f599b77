"""The paged cache and its attentions from their formulas, in 64 bits, stream by stream and head by head; runs on any
device. Used by the tests only."""
import math

import torch


def streams(cu, kv_lens):
    """[(first token, tokens, cached rows)] of each stream."""
    cu = cu.tolist()
    return [(a, b - a, n) for a, b, n in zip(cu, cu[1:], kv_lens.tolist())]


def rows_of(table, page, n_pages, b, kv):
    """(page ids, rows) of positions 0 .. kv - 1 of stream b, and which of them exist."""
    p = torch.arange(kv, device=table.device)
    ids = table[b].long()[p // page] if kv else p
    return ids, p % page, (ids >= 0) & (ids < n_pages)


def rotate(x, pos, inv_freq, rot_offset=0, interleaved=False):
    """x [n, heads, d] at positions pos [n], rotated: float64."""
    x, P = x.double().clone(), inv_freq.numel()
    i0 = torch.arange(P, device=x.device) * (2 if interleaved else 1) + rot_offset
    i1 = i0 + (1 if interleaved else P)
    ang = (pos.double()[:, None] * inv_freq.double())[:, None]
    a, b = x[..., i0], x[..., i1]
    x[..., i0] = a * ang.cos() - b * ang.sin()
    x[..., i1] = b * ang.cos() + a * ang.sin()
    return x


def append(q, k, v, k_pages, v_pages, table, cu, kv_lens, inv_freq=None, rot_offset=0, interleaved=False):
    """(rotated q, rotated k, k pages, v pages) in float64; rows of no stream are those of q and k."""
    q, k = q.double().clone(), k.double().clone()
    kp, vp = k_pages.double().clone(), v_pages.double().clone()
    n_pages, _, page, _ = k_pages.shape
    for b, (first, n, kv) in enumerate(streams(cu, kv_lens)):
        ok = 0 <= kv <= table.shape[1] * page
        rows = slice(first, first + n)
        pos = torch.arange(n, device=q.device) + (kv - n if ok else 0)
        if not ok:
            pos = torch.zeros_like(pos)
        if inv_freq is not None:
            q[rows], k[rows] = (rotate(x[rows], pos, inv_freq, rot_offset, interleaved) for x in (q, k))
        if not ok:
            continue
        for i, p in enumerate(pos.tolist()):
            if p < 0:
                continue
            at = int(table[b, p // page])
            if 0 <= at < n_pages:
                kp[at, :, p % page] = k[first + i]
                vp[at, :, p % page] = v[first + i].double()
    return q, k, kp, vp


def _attend(q, k, v, seen, scale):
    """q [n, d], k [m, d], v [m, dv], seen [n, m]: (out, sum of the weights times |v|, the largest sum of |q_d k_d| a seen
    key has, in scaled units), rows that see nothing zero. Keys that no row sees may hold anything."""
    any_row = seen.any(0)
    k, v = (torch.where(any_row[:, None], t.double(), 0.0) for t in (k, v))
    q = q.double()
    s = (q @ k.t() * scale).masked_fill(~seen, -math.inf)
    some = seen.any(1)[:, None]
    p = torch.softmax(torch.where(some, s, 0.0), -1)
    p = torch.where(seen & some, p, 0.0)
    mag = ((q.abs() @ k.abs().t()) * abs(scale)).masked_fill(~seen, 0.0)
    return p @ v, p @ v.abs(), mag.amax(1) if mag.shape[1] else mag.new_zeros(len(q))


def attn(q, fetch, cu, kv_lens, nkv, dv, scale):
    """Attention of packed tokens; fetch(b, kv, head) gives (keys, values, which exist) of stream b. Returns (out, weighted
    |v|, the largest score's magnitude) for the tolerance, and which tokens belong to a stream with a valid length."""
    N, nh, _ = q.shape
    out = torch.zeros(N, nh, dv, dtype=torch.float64, device=q.device)
    wv, mag = torch.zeros_like(out), torch.zeros(N, nh, 1, dtype=torch.float64, device=q.device)
    G = nh // nkv
    for b, (first, n, kv) in enumerate(streams(cu, kv_lens)):
        rows = slice(first, first + n)
        for h in range(nkv):
            k, v, ok = fetch(b, kv, h)
            pos = torch.arange(kv - n, kv, device=q.device)
            seen = (torch.arange(kv, device=q.device) <= pos[:, None]) & ok
            for j in range(h * G, h * G + G):
                out[rows, j], wv[rows, j], mag[rows, j, 0] = _attend(q[rows, j], k, v, seen, scale)
    return out, wv, mag


def paged_attn(q, k_pages, v_pages, table, cu, kv_lens, scale):
    n_pages, nkv, page, _ = k_pages.shape

    def fetch(b, kv, h):
        ids, rows, ok = rows_of(table, page, n_pages, b, kv)
        at = torch.where(ok, ids, 0)
        return k_pages[at, h, rows], v_pages[at, h, rows], ok
    return attn(q, fetch, cu, kv_lens, nkv, v_pages.shape[3], scale)


def prompt_attn(q, k, v, cu, scale):
    def fetch(b, kv, h):
        rows = slice(int(cu[b]), int(cu[b + 1]))
        return k[rows, h], v[rows, h], torch.ones(kv, dtype=torch.bool, device=q.device)
    return attn(q, fetch, cu, cu[1:] - cu[:-1], k.shape[1], v.shape[2], scale)


def attn_tolerance(out, wv, mag, keys, dqk, dtype):
    """How far an attention that keeps scores, statistics and sums in fp32 and rounds the weights (where they meet the
    values) and the output to dtype may be from `out`, element by element. With u the half step of dtype and e that of
    fp32: a score of magnitude `mag` is off by at most (dqk + 4) e mag (products, their sum, scale, the shift by the
    maximum), a weight relatively by that, its exponential's 4 e and, in the numerator, u; numerator and denominator are
    sums of `keys` terms (keys e each); the quotient is rounded once to dtype (u)."""
    u, e = torch.finfo(dtype).eps / 2, 2.0 ** -24
    w = 2 * ((dqk + 4) * e * mag + (4 + keys) * e)
    err = (u + w) * wv
    tiny = torch.finfo(dtype).smallest_normal
    return err + u * (out.abs() + err) + tiny
