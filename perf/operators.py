"""What is measured of the operators that serve several streams at once (paged_kv): a cache held in pages, its append and
the attentions that go with it.

  append  paged_kv.paged_append: the new tokens' keys (rotated by their positions) and values into their pages, and the
          rotated queries
  paged   paged_kv.paged_attn: new tokens (one a stream in decode, a chunk in a prompt) over the paged cache that holds
          them and what came before
  prompt  paged_kv.prompt_attn: whole prompts of different lengths packed one behind the other, causal

Tokens are packed: stream b's are rows cu[b] .. cu[b + 1] - 1, and kv_lens[b] rows of its cache count, the new ones the
last of them. Heads are (query heads, key / value heads, width of queries and keys, width of values).
"""
import math
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ming-voice_amd"))

DEV = "cuda"
F32, F64 = torch.float32, torch.float64
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}

own = False

TALKER = dict(heads=14, kv_heads=2, dqk=64, dv=64)      # the Talker's Qwen2
THINKER = dict(heads=16, kv_heads=16, dqk=192, dv=128)  # an MLA layer of the thinker, its last 64 dims rotated
GROUPED = dict(heads=32, kv_heads=8, dqk=128, dv=128)
WIDE = dict(heads=16, kv_heads=2, dqk=256, dv=256)
ODD = dict(heads=15, kv_heads=3, dqk=80, dv=80)
ONE_KV = dict(heads=20, kv_heads=1, dqk=64, dv=64)
HALF = dict(rot="half", rot_offset=0)                   # the whole head, first half against second half


def _rotation(shape):
    return dict(rot="pairs", rot_offset=128, rot_dims=64) if shape is THINKER else dict(HALF, rot_dims=shape["dqk"])


def listed():
    return [
        # one Talker stream's next token: the smallest call, once a layer and token
        dict(name="append_1", op="append", type="bf16", page=16, seqs=1, new=1, new_most=1, ctx=300, ctx_most=300,
             **TALKER, **_rotation(TALKER)),
        # the prompts of 16 Talker streams that start together
        dict(name="append_talker_prompts", op="append", type="bf16", page=16, seqs=16, new=9, new_most=700, ctx=0,
             ctx_most=0, **TALKER, **_rotation(TALKER)),
        # a long prompt's piece behind a long context, rotated in its last dims
        dict(name="append_thinker_4000", op="append", type="bf16", page=64, seqs=2, new=1999, new_most=2001, ctx=30000,
             ctx_most=100000, **THINKER, **_rotation(THINKER)),
        # one Talker stream's next token
        dict(name="decode_1", op="paged", type="bf16", page=16, seqs=1, new=1, new_most=1, ctx=700, ctx_most=700, **TALKER),
        # a server's decode step: 64 streams at different places of their speech
        dict(name="decode_64", op="paged", type="bf16", page=16, seqs=64, new=1, new_most=1, ctx=3, ctx_most=1000, **TALKER),
        # decode behind long contexts: the largest read of the cache
        dict(name="decode_16_long", op="paged", type="fp16", page=64, seqs=16, new=1, new_most=1, ctx=4000,
             ctx_most=40000, **GROUPED),
        # a user's next turn: pieces of prompts behind what was said before
        dict(name="chunk_500", op="paged", type="bf16", page=16, seqs=4, new=100, new_most=500, ctx=611, ctx_most=5000,
             **GROUPED),
        # the thinker's heads: streams that decode among others that read their prompts
        dict(name="chunk_mixed", op="paged", type="bf16", page=32, seqs=9, new=1, new_most=300, ctx=100, ctx_most=2000,
             **THINKER),
        # one short spoken prompt
        dict(name="prompt_37", op="prompt", type="bf16", seqs=1, new=37, new_most=37, **TALKER),
        # a batch of Talker prompts of all lengths
        dict(name="prompt_12_ragged", op="prompt", type="bf16", seqs=12, new=5, new_most=2000, **TALKER),
        # the thinker's heads over two prompts
        dict(name="prompt_thinker_2", op="prompt", type="bf16", seqs=2, new=900, new_most=2048, **THINKER),
        # a whole document
        dict(name="prompt_8192", op="prompt", type="fp16", seqs=1, new=8192, new_most=8192, **GROUPED),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "paged", "paged", "prompt"])
    shape = rng.choice([TALKER, TALKER, THINKER, GROUPED, WIDE, ODD, ONE_KV])
    c = dict(op=op, type=rng.choice(["bf16", "bf16", "fp16"]), **shape)
    if op != "prompt":
        c["page"] = rng.choice([1, 8, 16, 16, 24, 64, 100, 256])
    if op == "prompt":
        seqs = _log_int(rng, 1, 40)
        most = _log_int(rng, 1, 6000 // seqs if seqs > 1 else 6000)
        return dict(c, seqs=seqs, new=rng.randint(1, most), new_most=most)
    decode = op == "paged" and rng.random() < 0.5
    if decode:
        seqs = _log_int(rng, 1, 128)
        ctx = _log_int(rng, 1, 200000 // seqs)
        return dict(c, seqs=seqs, new=1, new_most=1, ctx=rng.randint(0, ctx), ctx_most=ctx)
    seqs = _log_int(rng, 1, 24)
    most = _log_int(rng, 1, 3000 // seqs)
    ctx = _log_int(rng, 1, min(12000, 40000 // seqs))
    c = dict(c, seqs=seqs, new=rng.randint(1, most), new_most=most, ctx=rng.randint(0, ctx), ctx_most=ctx)
    return dict(c, **_rotation(shape)) if op == "append" else c


# ------------------------------------------------------------------------------------------------ inputs from a seed

def _spread(count, least, most, turn):
    """`count` lengths from `least` to `most`, even over their logarithm, in an order that is not sorted."""
    if count == 1:
        return [most]
    at = [(i * 0.6180339887498949 + turn) % 1.0 for i in range(count)]
    lo, hi = min(at), max(at)
    return [round((least + 1) * ((most + 1) / (least + 1)) ** ((x - lo) / (hi - lo))) - 1 for x in at]


def _lengths(case):
    """(new tokens of each stream, rows of its cache that count)."""
    new = _spread(case["seqs"], case["new"], case["new_most"], 0.0)
    ctx = _spread(case["seqs"], case["ctx"], case["ctx_most"], 0.37) if "ctx" in case else [0] * len(new)
    return new, [n + c for n, c in zip(new, ctx)]


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    dt = TYPES[case["type"]]
    new, kv = _lengths(case)
    N, B = sum(new), len(new)
    nh, nkv, dqk, dv = (case[n] for n in ("heads", "kv_heads", "dqk", "dv"))

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEV).to(dt)

    s = dict(op=case["op"], scale=dqk ** -0.5, most_new=max(new), most_kv=max(kv), new=new, kv=kv,
             cu=torch.tensor([0] + new, device=DEV).cumsum(0).to(torch.int32),
             kv_lens=torch.tensor(kv, dtype=torch.int32, device=DEV))
    # one projection's output holds queries, keys and values
    row = normal(N, nh * dqk + nkv * (dqk + dv))
    s["q"] = row[:, :nh * dqk].view(N, nh, dqk)
    s["k"] = row[:, nh * dqk:(nh + nkv) * dqk].view(N, nkv, dqk)
    s["v"] = row[:, (nh + nkv) * dqk:].view(N, nkv, dv)
    if case["op"] != "prompt":
        page = case["page"]
        pages = [-(-n // page) for n in kv]
        if case["op"] == "append":  # the pool holds the pages that the new tokens fall into; those before are elsewhere
            first = [(n - m) // page for n, m in zip(kv, new)]
        else:
            first = [0] * B
        used = sum(p - f for p, f in zip(pages, first))
        order = torch.randperm(used + 3, generator=g, device=DEV).to(torch.int32)
        table = torch.full((B, max(pages)), -1, dtype=torch.int32, device=DEV)
        at = 0
        for b, (f, p) in enumerate(zip(first, pages)):
            table[b, f:p] = order[at:at + p - f]
            at += p - f
        s.update(page=page, table=table, k_pages=normal(used + 3, nkv, page, dqk), v_pages=normal(used + 3, nkv, page, dv))
    if case["op"] == "append":
        r = case["rot_dims"]
        s.update(rot=case["rot"], rot_offset=case["rot_offset"],
                 inv_freq=(1e6 ** (-torch.arange(0, r, 2, dtype=F64) / r)).to(F32).to(DEV))
    return s


# ------------------------------------------------------------------------------------------------------ the operators

def _tokens(cu, kv_lens, N):
    """For each packed token: its stream, and its position in it."""
    i = torch.arange(N, device=DEV)
    b = torch.searchsorted(cu[1:].contiguous(), i.to(torch.int32), right=True)
    return b, i - cu[b + 1] + kv_lens[b]


def _rotate(x, ang, s):
    """x [N, heads, d] in 32 bits, its dims rot_offset .. turned by ang [N, pairs]."""
    r = 2 * ang.shape[1]
    cos, sin = ang.cos().float()[:, None], ang.sin().float()[:, None]
    part = x[..., s["rot_offset"]:s["rot_offset"] + r]
    if s["rot"] == "half":
        a, b = part[..., :r // 2], part[..., r // 2:]
        part = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = part[..., 0::2], part[..., 1::2]
        part = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([x[..., :s["rot_offset"]], part, x[..., s["rot_offset"] + r:]], -1)


def _append_plain(s):
    dt = s["q"].dtype
    b, pos = _tokens(s["cu"], s["kv_lens"], s["q"].shape[0])
    ang = pos.to(F64)[:, None] * s["inv_freq"].to(F64)
    at = s["table"][b, pos // s["page"]].long()
    s["k_pages"][at, :, pos % s["page"]] = _rotate(s["k"].float(), ang, s).to(dt)
    s["v_pages"][at, :, pos % s["page"]] = s["v"]
    return _rotate(s["q"].float(), ang, s).to(dt), s["k_pages"], s["v_pages"]


def _attend(s, k, v):
    """Queries s["q"] over k [B, most_kv, kv_heads, dqk] and v [B, most_kv, kv_heads, dv] in 32 bits, padded."""
    N, nh, dqk = s["q"].shape
    B, L, nkv, dv = v.shape
    M, G = s["most_new"], nh // nkv
    start, lens = s["cu"][:-1].long(), s["cu"].diff().long()
    i = torch.arange(M, device=DEV)
    q = s["q"].float()[(start[:, None] + i).clamp(max=N - 1)]  # [B, M, nh, dqk]
    q = q.view(B, M, nkv, G, dqk).permute(0, 2, 3, 1, 4).reshape(B, nkv, G * M, dqk)
    score = (q @ k.permute(0, 2, 3, 1)).mul_(s["scale"]).view(B, nkv, G, M, L)
    pos = (s["kv_lens"].long() - lens)[:, None] + i  # [B, M]
    score.masked_fill_((torch.arange(L, device=DEV) > pos[:, :, None])[:, None, None], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    p = (p / p.sum(-1, keepdim=True)).view(B, nkv, G * M, L)
    o = (p @ v.permute(0, 2, 1, 3)).view(B, nkv, G, M, dv).permute(0, 3, 1, 2, 4)  # [B, M, nkv, G, dv]
    b, at = _tokens(s["cu"], lens, N)
    return o[b, at].reshape(N, nh, dv).to(s["q"].dtype)


def _paged_plain(s):
    """The cached rows gathered from their pages, then attention over them; rows past a stream's end are zero."""
    pos = torch.arange(s["most_kv"], device=DEV)
    at = s["table"][:, pos // s["page"]].long().clamp(min=0)  # [B, most_kv]
    live = (pos < s["kv_lens"][:, None])[..., None, None]
    k = s["k_pages"][at, :, pos % s["page"]].float().masked_fill_(~live, 0)
    return _attend(s, k, s["v_pages"][at, :, pos % s["page"]].float().masked_fill_(~live, 0))


def _prompt_plain(s):
    at = s["cu"][:-1, None].long() + torch.arange(s["most_kv"], device=DEV)
    live = (at < s["cu"][1:, None])[..., None, None]
    at = at.clamp(max=s["q"].shape[0] - 1)
    return _attend(s, s["k"].float()[at].masked_fill_(~live, 0), s["v"].float()[at].masked_fill_(~live, 0))


def run(s):
    if own:
        import paged_kv
        if s["op"] == "append":
            q = paged_kv.paged_append(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["cu"], s["kv_lens"],
                                      s["inv_freq"], rot_offset=s["rot_offset"], interleaved=s["rot"] == "pairs")
            return q, s["k_pages"], s["v_pages"]
        if s["op"] == "paged":
            return paged_kv.paged_attn(s["q"], s["k_pages"], s["v_pages"], s["table"], s["cu"], s["kv_lens"], s["scale"])
        return paged_kv.prompt_attn(s["q"], s["k"], s["v"], s["cu"], s["scale"])
    return {"append": _append_plain, "paged": _paged_plain, "prompt": _prompt_plain}[s["op"]](s)


def work(case):
    new, kv = _lengths(case)
    nh, nkv, dqk, dv = (case[n] for n in ("heads", "kv_heads", "dqk", "dv"))
    N = sum(new)
    if case["op"] == "append":
        return dict(bytes=2 * 2 * N * (nh * dqk + nkv * (dqk + dv)), flops=3 * N * (nh + nkv) * case["rot_dims"])
    pairs = sum(n * (m - n) + n * (n + 1) // 2 for n, m in zip(new, kv))
    return dict(bytes=2 * (N * nh * (dqk + dv) + sum(kv) * nkv * (dqk + dv)), flops=2 * pairs * nh * (dqk + dv))


# ---------------------------------------------------------------------------------------------------- in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    new, kv, nkv = s["new"], s["kv"], case["kv_heads"]
    G = case["heads"] // nkv
    if case["op"] == "append":
        inv = s["inv_freq"].double()
        q, pages = s["q"].double(), [s["k_pages"].double(), s["v_pages"].double()]
        o, P = s["rot_offset"], inv.numel()
        # the two dims of each pair
        x0 = torch.arange(P, device=DEV) * (2 if s["rot"] == "pairs" else 1) + o
        x1 = x0 + (1 if s["rot"] == "pairs" else P)
        first = 0
        for b, (n, m) in enumerate(zip(new, kv)):
            pos = torch.arange(m - n, m, device=DEV)
            turn = torch.polar(torch.ones(n, P, dtype=F64, device=DEV), pos[:, None] * inv[None])[:, None]
            k = s["k"][first:first + n].double()
            for x in (q[first:first + n], k):
                z = torch.complex(x[..., x0], x[..., x1]) * turn
                x[..., x0], x[..., x1] = z.real, z.imag
            page, slot = s["table"][b].long()[pos // s["page"]], pos % s["page"]
            for h in range(nkv):
                pages[0][page, h, slot] = k[:, h]
                pages[1][page, h, slot] = s["v"][first:first + n, h].double()
            first += n
        return q, pages[0], pages[1]
    out, first = torch.empty(sum(new), case["heads"], case["dv"], dtype=F64, device=DEV), 0
    for b, (n, m) in enumerate(zip(new, kv)):
        rows = slice(first, first + n)
        first += n
        if case["op"] == "paged":
            mine = s["table"][b, :-(-m // s["page"])].long()
        for h in range(nkv):
            if case["op"] == "paged":
                k, v = (s[t][mine, h].flatten(0, 1)[:m].double() for t in ("k_pages", "v_pages"))
            else:
                k, v = (s[t][rows, h].double() for t in ("k", "v"))
            later = torch.ones(n, m, dtype=torch.bool, device=DEV).triu(m - n + 1)
            for j in range(h * G, h * G + G):
                w = torch.softmax((s["q"][rows, j].double() @ k.t() * s["scale"]).masked_fill_(later, -math.inf), -1)
                out[rows, j] = w @ v
    return out
