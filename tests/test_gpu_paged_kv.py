"""GPU parity of the paged cache (append, attention over pages, packed prompts) with the 64-bit oracle, at the sizes and
masks where they can go wrong. Tolerances are the oracle's (attn_tolerance), element by element; of the append, one
rounding of the type plus (|x0| + |x1|) 6e-7: the angle's fraction of a turn rounded to fp32 (1e-7 of an angle), cosine and
sine (2.4e-7), two products and their sum (1.8e-7)."""
import pytest
import torch

import paged_kv as PK
from oracle import paged_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, FP = torch.bfloat16, torch.float16


class Streams:
    """Streams of `new` tokens behind `ctx` cached rows: packed q, k, v as column slices of one projection, a pool whose
    pages lie in no order, the table. Every pool row that no stream holds is NaN, and so are the packed rows behind the
    last stream (`spare` of them)."""

    def __init__(self, new, ctx, nh=14, nkv=2, dqk=64, dv=64, page=16, dtype=BF, idx=torch.int32, seed=0, spare=0,
                 layout="hnd", more_pages=2, std=1.0):
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.new, self.kv = list(new), [n + c for n, c in zip(new, ctx)]
        N = self.N = sum(new)
        self.nh, self.nkv, self.dqk, self.dv, self.page, self.dtype = nh, nkv, dqk, dv, page, dtype
        row = (torch.randn(N + spare, nh * dqk + nkv * (dqk + dv), generator=g, device=DEV) * std).to(dtype)
        row[N:] = float("nan")
        self.q = row[:, :nh * dqk].view(-1, nh, dqk)
        self.k = row[:, nh * dqk:(nh + nkv) * dqk].view(-1, nkv, dqk)
        self.v = row[:, (nh + nkv) * dqk:].view(-1, nkv, dv)
        self.cu = torch.tensor([0] + self.new, device=DEV).cumsum(0).to(idx)
        self.lens = torch.tensor(self.kv, device=DEV, dtype=idx)
        need = [-(-n // page) for n in self.kv]
        n_pages = sum(need) + 3
        order = torch.randperm(n_pages, generator=g, device=DEV)
        self.table = torch.full((len(new), max(need) + more_pages), -7, dtype=idx, device=DEV)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n].to(idx)
            at += n
        shapes = [(n_pages, nkv, page, dqk), (n_pages, nkv, page, dv)]
        if layout == "hnd":
            pools = [torch.full(s, float("nan"), dtype=dtype, device=DEV) for s in shapes]
        else:  # rows of all heads side by side
            pools = [torch.full((s[0], s[2], s[1], s[3]), float("nan"), dtype=dtype, device=DEV).transpose(1, 2)
                     for s in shapes]
        self.kp, self.vp = pools
        for b, kv in enumerate(self.kv):
            p = torch.arange(kv, device=DEV)
            ids = self.table[b].long()[p // page]
            for pool in pools:
                pool[ids, :, p % page] = (torch.randn(kv, nkv, pool.shape[3], generator=g, device=DEV) * std).to(dtype)

    def attn(self, **kw):
        return PK.paged_attn(self.q, self.kp, self.vp, self.table, self.cu, self.lens, **kw)

    def oracle(self, scale=None):
        return O.paged_attn(self.q[:self.N], self.kp, self.vp, self.table, self.cu, self.lens, scale or self.dqk ** -0.5)


# The host chooses the kernel by the sizes alone: blocks of 16 rows where these would read few keys, of 128 rows (in one or
# two groups of waves) where many. The same small batch goes through each of them by a table that allows long contexts, and
# by rows behind the last prompt.
WIDE_TABLE = 400000  # positions


def many_pages(kind, page):
    return 2 if kind == "few" else WIDE_TABLE // page


def spare_rows(kind, nh, dqk, dv):
    if kind == "few":
        return 3
    return 300 + (131072 // nh if kind == "one group" else int(((64 << 20) * 16 / (nh * (dqk + dv) * 2)) ** 0.5))


BOTH = pytest.mark.parametrize("kind", ["few", "many"])
ALL = pytest.mark.parametrize("kind", ["few", "one group", "two groups"])


def check(got, want, keys, dqk, dtype):
    out, wv, mag = want
    tol = O.attn_tolerance(out, wv, mag, keys, dqk, dtype)
    off = (got.double() - out).abs()
    assert bool((off <= tol).all()), f"off by {float((off / tol).max()):.3f} of the tolerance"


HEADS = [(14, 2, 64, 64), (16, 16, 192, 128), (32, 8, 128, 128), (5, 1, 256, 256), (6, 2, 80, 80), (20, 1, 64, 64),
         (3, 3, 8, 8), (2, 1, 40, 136), (33, 1, 96, 24), (4, 2, 256, 64), (4, 2, 64, 200)]


# ------------------------------------------------------------------------------------------------ append

def run_append(s, inv, off=0, inter=False, **kw):
    want = O.append(s.q[:s.N], s.k[:s.N], s.v[:s.N], s.kp, s.vp, s.table, s.cu, s.lens, inv, off, inter)
    before = s.q.clone(), s.k.clone()
    q = PK.paged_append(s.q, s.k, s.v, s.kp, s.vp, s.table, s.cu, s.lens, inv, rot_offset=off, interleaved=inter, **kw)
    torch.cuda.synchronize()
    return q, want, before


def near(got, want, x, dtype):
    """got against want, float64: NaN where want has it; one rounding, and the rotation's error in units of the head's
    largest value."""
    nan = want.isnan()
    assert torch.equal(got.isnan(), nan)
    got, want = got.double().masked_fill(nan, 0), want.masked_fill(nan, 0)
    u = torch.finfo(dtype).eps / 2
    assert bool(((got - want).abs() <= u * want.abs() + 2 * x * 6e-7 + torch.finfo(dtype).smallest_normal).all())


@pytest.mark.parametrize("nh,nkv,dqk,dv,off,pairs,inter", [
    (14, 2, 64, 64, 0, 32, False), (16, 16, 192, 128, 128, 32, True), (32, 8, 128, 128, 0, 64, False),
    (5, 1, 256, 256, 0, 128, False), (6, 2, 80, 80, 0, 40, False), (6, 2, 80, 80, 16, 16, True), (3, 3, 16, 8, 0, 8, False),
    (4, 2, 96, 40, 8, 24, False), (2, 1, 64, 64, 0, 32, True), (3, 1, 8, 8, 0, 0, False)])
@pytest.mark.parametrize("dtype,idx,page,layout", [(BF, torch.int32, 16, "hnd"), (FP, torch.int64, 5, "nhd")])
def test_append(nh, nkv, dqk, dv, off, pairs, inter, dtype, idx, page, layout):
    s = Streams([1, 9, 0, 33, 2], [0, 3, 50, 700, 99998], nh, nkv, dqk, dv, page, dtype, idx, seed=nh, layout=layout)
    inv = (1e6 ** (-torch.arange(pairs, device=DEV) / max(pairs, 1))).float() if pairs else None
    q, (wq, wk, wkp, wvp), before = run_append(s, inv, off, inter)
    near(q, wq, float(s.q.abs().max()), dtype)
    near(s.kp, wkp, float(s.q.abs().max()), dtype)
    assert torch.equal(s.vp.double().nan_to_num(7.0), wvp.nan_to_num(7.0))
    assert torch.equal(s.q, before[0]) and torch.equal(s.k, before[1])
    # only the new rows changed
    fresh = Streams([1, 9, 0, 33, 2], [0, 3, 50, 700, 99998], nh, nkv, dqk, dv, page, dtype, idx, seed=nh, layout=layout)
    changed = (s.kp.double().nan_to_num(7.0) != fresh.kp.double().nan_to_num(7.0)).any(-1).any(1)  # [pages, rows]
    assert int(changed.sum()) <= s.N
    # a head whose dims do not turn is copied bit for bit
    if inv is None:
        assert torch.equal(q, s.q)


@pytest.mark.parametrize("off,pairs,inter", [(0, 32, False), (16, 16, True), (0, 0, False)])
def test_append_in_place_gives_the_same(off, pairs, inter):
    inv = (1e6 ** (-torch.arange(pairs, device=DEV) / max(pairs, 1))).float() if pairs else None
    a, b = (Streams([3, 40, 1], [5, 0, 1000], seed=3) for _ in range(2))
    k_out = torch.empty(a.N, a.nkv, a.dqk, device=DEV, dtype=BF)
    q, (_, wk, _, _), _ = run_append(a, inv, off, inter, k_out=k_out)
    got = PK.paged_append(b.q, b.k, b.v, b.kp, b.vp, b.table, b.cu, b.lens, inv, rot_offset=off, interleaved=inter, q_out=b.q,
                          k_out=b.k)
    assert got is b.q and torch.equal(b.q, q) and torch.equal(b.k, k_out) and torch.equal(b.v, a.v)
    assert torch.equal(a.kp.view(torch.int16), b.kp.view(torch.int16))
    near(k_out, wk, float(a.k.abs().max()), BF)
    # the cached rows are the rotated keys bit for bit
    p = torch.arange(5, 8, device=DEV)
    assert torch.equal(a.kp[a.table[0].long()[p // 16], :, p % 16], k_out[:3])


def test_append_stores_nothing_where_nothing_exists():
    s = Streams([4, 3, 2, 5, 3], [30, 6, 20, 1, 0], seed=5, spare=3)
    cap = s.table.shape[1] * s.page
    s.table[0, 2] = s.kp.shape[0]       # positions 32, 33 of stream 0 lie in no page
    s.lens[1] = cap + 1                 # outside the table
    s.lens[2] = -1
    s.lens[3] = 2                       # fewer rows than new tokens: three stand before position 0
    s.table[4, 0] = -5
    inv = (1e6 ** (-torch.arange(32, device=DEV) / 32)).float()
    kp, vp = s.kp.clone(), s.vp.clone()
    q_out = torch.full_like(s.q, 3.0)
    q, (wq, _, wkp, wvp), _ = run_append(s, inv, q_out=q_out)
    near(s.kp, wkp, float(s.k[:s.N].abs().max()), BF)
    assert torch.equal(s.vp.double().nan_to_num(7.0), wvp.nan_to_num(7.0))
    near(q[:s.N], wq, float(s.q[:s.N].abs().max()), BF)
    assert (q[s.N:] == 3.0).all()       # behind the last stream
    stored = (s.vp.nan_to_num(7.0) != vp.nan_to_num(7.0)).any(-1).any(1).sum()
    assert int(stored) == 2 + 2         # positions 30, 31 of stream 0; 0, 1 of stream 3


# ------------------------------------------------------------------------------------------------ attention over pages

@pytest.mark.parametrize("nh,nkv,dqk,dv", HEADS)
@pytest.mark.parametrize("dtype,idx,page,layout", [(BF, torch.int32, 16, "hnd"), (FP, torch.int64, 7, "nhd"),
                                                   (BF, torch.int64, 64, "nhd"), (FP, torch.int32, 1, "hnd"),
                                                   (BF, torch.int32, 1000, "hnd")])
@pytest.mark.parametrize("new,ctx", [([1, 1, 1, 1, 1], [0, 1, 63, 64, 300]), ([5, 1, 0, 37, 2], [0, 700, 9, 130, 31]),
                                     ([150], [45]), ([1], [0])])
@BOTH
def test_paged_attn(nh, nkv, dqk, dv, dtype, idx, page, layout, new, ctx, kind):
    print(f"heads {nh}/{nkv} {dqk}/{dv} {dtype} {idx} page {page} {layout} {new} behind {ctx} {kind}", flush=True)
    s = Streams(new, ctx, nh, nkv, dqk, dv, page, dtype, idx, seed=len(new), layout=layout,
                more_pages=many_pages(kind, page))
    got = s.attn()
    check(got, s.oracle(), max(s.kv), dqk, dtype)


@pytest.mark.parametrize("new,ctx", [([1], [5000]), ([1], [70000]), ([2, 1], [9, 40000]), ([1, 1, 1], [20000, 3, 0]), ([3, 1], [9000, 8191]), ([64], [6000]),
                                     ([200, 1, 17], [3000, 40, 2500]), ([700], [2000])])
@pytest.mark.parametrize("nh,nkv,dqk,dv", [(14, 2, 64, 64), (4, 1, 128, 128), (2, 2, 192, 128), (4, 2, 256, 256)])
def test_long_contexts(nh, nkv, dqk, dv, new, ctx):
    print(f"heads {nh}/{nkv} {dqk}/{dv} {new} behind {ctx}", flush=True)
    s = Streams(new, ctx, nh, nkv, dqk, dv, seed=7)
    first = s.attn()
    check(first, s.oracle(), max(s.kv), dqk, BF)
    assert torch.equal(first, s.attn())  # sums are joined in one order


@pytest.mark.parametrize("count", [63, 64, 65, 128, 129, 700, 1100, 4200])
@BOTH
def test_many_streams(count, kind):
    new = [(0, 1, 30)[i % 3] if kind == "many" else i % 3 for i in range(count)]
    s = Streams(new, [(i * 37) % 90 + 700 * (i == 5) for i in range(count)], 4, 2, 64, 64, page=8, seed=count,
                more_pages=many_pages(kind, 8))
    check(s.attn(), s.oracle(), 900, 64, BF)


def test_every_token_a_stream_of_its_own_or_none():
    s = Streams([0, 0, 1, 0, 1, 0], [4, 0, 0, 7, 90, 0], seed=2)
    check(s.attn(), s.oracle(), 100, 64, BF)
    empty = Streams([0, 0], [3, 0], seed=2, spare=2)
    out = torch.full((2, 14, 64), 5.0, device=DEV, dtype=BF)
    empty.attn(out=out)
    assert (out == 5.0).all()


@BOTH
def test_rows_that_see_nothing_are_zero_and_bad_lengths_nan(kind):
    s = Streams([4, 3, 2, 5, 1, 2], [30, 6, 20, 1, 10, 0], seed=11, spare=4, more_pages=many_pages(kind, 16))
    s.lens[0] = 2                                          # tokens 0, 1 stand before position 0
    s.lens[1] = s.table.shape[1] * s.page + 1
    s.lens[2] = -1
    s.table[4, 0] = s.kp.shape[0]                          # every page of stream 4 is missing
    s.lens[5] = 0
    out = torch.full((s.N + 4, s.nh, s.dv), 9.0, device=DEV, dtype=BF)
    got = s.attn(out=out)
    assert got is out and (out[s.N:] == 9.0).all()
    assert (out[:2] == 0).all() and out[4:9].isnan().all() and (out[14] == 0).all() and (out[15:17] == 0).all()
    good = [2, 3, 9, 10, 11, 12, 13]
    s.lens[1] = s.lens[2] = 0
    want = tuple(t[good] for t in s.oracle())
    check(out[good], want, 64, 64, BF)


@pytest.mark.parametrize("page", [4, 32, 100])
@pytest.mark.parametrize("new", [[1, 1], [40, 3], [200, 1]])
@BOTH
def test_missing_pages_are_left_out(page, new, kind):
    s = Streams(new, [400, 77], page=page, seed=13, more_pages=many_pages(kind, page))
    for at in range(0, -(-s.kv[0] // page), 3):
        s.table[0, at] = -1 if at % 2 else 1 << 30
    check(s.attn(), s.oracle(), 700, 64, BF)


@pytest.mark.parametrize("nh,nkv,dqk,dv", [(14, 2, 64, 64), (4, 2, 128, 128), (2, 2, 192, 128), (4, 2, 256, 256), (6, 2, 80, 80)])
@pytest.mark.parametrize("new,ctx", [([7], [0]), ([90, 1], [3, 40]), ([300], [1000])])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@BOTH
def test_later_rows_never_reach_a_token(nh, nkv, dqk, dv, new, ctx, bad, kind):
    """What the last two positions of a stream hold is seen by its last two tokens alone."""
    s = Streams(new, ctx, nh, nkv, dqk, dv, seed=17, more_pages=many_pages(kind, 16))
    want = s.oracle()
    for b, kv in enumerate(s.kv):
        for p in (kv - 2, kv - 1):
            if p >= ctx[b] and p > 0:
                at = s.table[b, p // s.page]
                s.kp[at, :, p % s.page], s.vp[at, :, p % s.page] = bad, bad
    got = s.attn()
    cu = s.cu.tolist()
    fine = [i for a, e in zip(cu, cu[1:]) for i in range(a, e) if i < e - 2]
    check(got[fine], tuple(t[fine] for t in want), max(s.kv), dqk, BF)
    for b, (a, e) in enumerate(zip(cu, cu[1:])):
        if e - a > 2:
            assert not got[a + (e - a) - 1].isfinite().any()


@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0, 1e-6])
@pytest.mark.parametrize("dtype", [BF, FP])
@BOTH
def test_scales(scale, dtype, kind):
    s = Streams([1, 40, 200], [90, 17, 0], dtype=dtype, seed=19, more_pages=many_pages(kind, 16))
    got = s.attn(scale=scale)
    want = O.paged_attn(s.q, s.kp, s.vp, s.table, s.cu, s.lens, scale)
    check(got, want, 300, 64, dtype)


@pytest.mark.parametrize("dtype", [BF, FP])
@BOTH
def test_weights_far_apart(dtype, kind):
    """Scores that rise and fall by hundreds along the keys: the running maximum moves often."""
    s = Streams([1, 64, 130], [1500, 700, 20], dtype=dtype, seed=23, std=4.0, more_pages=many_pages(kind, 16))
    check(s.attn(scale=1.0), s.oracle(1.0), 1600, 64, dtype)


def test_offsets_past_32_bits():
    """A pool whose pages lie 3 GiB apart, and packed rows 0.3 GiB apart."""
    s = Streams([1, 20], [40, 3], nh=2, nkv=1, page=16, seed=29)
    n, gap = s.kp.shape[0], 3 << 29
    raw = torch.empty(n * gap, device=DEV, dtype=BF)
    far = raw.as_strided(s.kp.shape, (gap, 1024, 64, 1))
    far_v = raw.as_strided(s.vp.shape, (gap, 1024, 64, 1), 4096)
    far.copy_(s.kp)
    far_v.copy_(s.vp)
    want = s.attn()
    assert torch.equal(PK.paged_attn(s.q, far, far_v, s.table, s.cu, s.lens), want)
    gap = 0x0A000000
    rows = raw.as_strided((s.N, 2, 64), (gap, 64, 1), 1 << 20)
    out = raw.as_strided((s.N, 2, 64), (gap, 64, 1), 2 << 20)
    rows.copy_(s.q)
    assert torch.equal(PK.paged_attn(rows, s.kp, s.vp, s.table, s.cu, s.lens, out=out), want)
    k, v = (raw.as_strided((s.N, 1, 64), (gap, 64, 1), (3 + i) << 20) for i in range(2))
    k.copy_(s.k)
    v.copy_(s.v)
    want = PK.prompt_attn(s.q, s.k, s.v, s.cu)
    assert torch.equal(PK.prompt_attn(rows, k, v, s.cu, out=out), want)
    inv = torch.ones(32, device=DEV)
    want = PK.paged_append(s.q, s.k, s.v, s.kp, s.vp, s.table, s.cu, s.lens, inv)
    got = PK.paged_append(rows, k, v, far, far_v, s.table, s.cu, s.lens, inv, q_out=out)
    assert torch.equal(got, want) and torch.equal(far.nan_to_num(7.0), s.kp.nan_to_num(7.0))
    assert torch.equal(far_v.nan_to_num(7.0), s.vp.nan_to_num(7.0))


@pytest.mark.parametrize("page,row", [(16, 1024), (56, 1 << 25), (64, 1 << 25)])
def test_far_pages_in_a_block_of_many_rows(page, row):
    """Pages 3 GiB apart, and rows of a page whose last lies before or past 2^32 bytes of its first."""
    s = Streams([1, 20], [40, 3], nh=2, nkv=1, page=page, seed=31, more_pages=many_pages("many", page))
    n, gap = s.kp.shape[0], max(3 << 29, page * row)
    raw = torch.empty(n * gap, device=DEV, dtype=BF)
    far = raw.as_strided(s.kp.shape, (gap, row, row, 1))
    far_v = raw.as_strided(s.vp.shape, (gap, row, row, 1), 512)
    far.copy_(s.kp)
    far_v.copy_(s.vp)
    got = PK.paged_attn(s.q, far, far_v, s.table, s.cu, s.lens)
    assert torch.equal(got, s.attn())
    check(got, s.oracle(), 64, 64, BF)


def test_rows_far_apart_in_a_block_of_many_rows():
    """Keys and values 128 MiB apart, past what one buffer resource spans, at 512 query heads on one."""
    s = Streams([70, 30], [0, 0], nh=512, nkv=1, seed=30)
    gap = 1 << 26
    raw = torch.empty(s.N * gap, device=DEV, dtype=BF)
    k, v = (raw.as_strided((s.N, 1, 64), (gap, 64, 1), 64 * i) for i in range(2))
    k.copy_(s.k)
    v.copy_(s.v)
    got = PK.prompt_attn(s.q, k, v, s.cu)
    assert torch.equal(got, PK.prompt_attn(s.q, s.k, s.v, s.cu))
    check(got, O.prompt_attn(s.q, s.k, s.v, s.cu, 0.125), 70, 64, BF)


# ------------------------------------------------------------------------------------------------ packed prompts

@pytest.mark.parametrize("nh,nkv,dqk,dv", HEADS)
@pytest.mark.parametrize("dtype,idx", [(BF, torch.int32), (FP, torch.int64)])
@pytest.mark.parametrize("new", [[1], [2, 0, 31, 1], [64, 65, 3], [300], [17] * 9])
@ALL
def test_prompt_attn(nh, nkv, dqk, dv, dtype, idx, new, kind):
    print(f"heads {nh}/{nkv} {dqk}/{dv} {dtype} {new} {kind}", flush=True)
    s = Streams(new, [0] * len(new), nh, nkv, dqk, dv, dtype=dtype, idx=idx, seed=31, spare=spare_rows(kind, nh, dqk, dv))
    out = torch.full((len(s.q), nh, dv), 9.0, device=DEV, dtype=dtype)
    assert PK.prompt_attn(s.q, s.k, s.v, s.cu, out=out) is out
    check(out[:s.N], O.prompt_attn(s.q[:s.N], s.k[:s.N], s.v[:s.N], s.cu, dqk ** -0.5), max(new), dqk, dtype)
    assert (out[s.N:] == 9.0).all()


@pytest.mark.parametrize("nh,nkv,dqk,dv,new", [(14, 2, 64, 64, [1500, 3, 700]), (4, 1, 128, 128, [2100]),
                                               (2, 2, 192, 128, [900, 901]), (2, 1, 256, 256, [1030]),
                                               (2, 2, 64, 64, [2300]), (32, 8, 128, 128, [1500, 2600])])
def test_long_prompts(nh, nkv, dqk, dv, new):
    s = Streams(new, [0] * len(new), nh, nkv, dqk, dv, seed=37)
    got = PK.prompt_attn(s.q, s.k, s.v, s.cu)
    check(got, O.prompt_attn(s.q, s.k, s.v, s.cu, dqk ** -0.5), max(new), dqk, BF)
    assert torch.equal(got, PK.prompt_attn(s.q, s.k, s.v, s.cu))


@pytest.mark.parametrize("new", [[9, 40], [300, 77]])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@ALL
def test_other_prompts_and_later_tokens_never_reach_a_token(new, bad, kind):
    s = Streams(new, [0, 0], seed=41, spare=spare_rows(kind, 14, 64, 64))
    want = PK.prompt_attn(s.q, s.k, s.v, s.cu)
    v = s.v.clone()
    v[new[0] - 3:new[0]] = bad  # the first prompt's last three: seen by those tokens alone
    got = PK.prompt_attn(s.q, s.k, v, s.cu)
    check(got[:new[0] - 3], tuple(o[:new[0] - 3] for o in O.prompt_attn(s.q[:s.N], s.k[:s.N], s.v[:s.N], s.cu, 0.125)),
          max(new), 64, BF)
    assert torch.equal(got[new[0]:s.N], want[new[0]:s.N]) and not got[new[0] - 1].isfinite().any()
    for first, count, keep in ((0, new[0], slice(new[0], None)), (new[0], new[1], slice(0, new[0]))):
        k, v = s.k.clone(), s.v.clone()
        k[first:first + count], v[first:first + count] = bad, bad
        assert torch.equal(PK.prompt_attn(s.q, k, v, s.cu)[:s.N][keep], want[:s.N][keep])


def test_broadcast_and_strided_inputs():
    s = Streams([30, 5], [0, 0], 4, 4, 64, 64, seed=43)
    k, v = s.k[:, :1].expand(-1, 4, -1), s.v[:, :1].expand(-1, 4, -1)  # one head for all: a stride of zero
    want = PK.prompt_attn(s.q, k.contiguous(), v.contiguous(), s.cu)
    assert torch.equal(PK.prompt_attn(s.q, k, v, s.cu), want)
    heads_first = s.q.transpose(0, 1).contiguous().transpose(0, 1)
    out = torch.empty(4, 35, 64, device=DEV, dtype=BF).transpose(0, 1)
    assert torch.equal(PK.prompt_attn(heads_first, k, v, s.cu, out=out), want)


@BOTH
def test_streams_that_share_their_first_pages(kind):
    """A common prompt's pages in three streams' tables, one of them only partly filled by it."""
    s = Streams([1, 30, 2], [64, 40, 200], seed=45, more_pages=many_pages(kind, 16))
    s.table[1, :2] = s.table[0, :2]
    s.table[2, :4] = s.table[0, :4]
    check(s.attn(), s.oracle(), 250, 64, BF)


@BOTH
def test_rows_before_the_first_stream_are_left_as_they_were(kind):
    s = Streams([3, 40, 1], [9, 100, 700], seed=46, more_pages=many_pages(kind, 16))
    wide = torch.cat([torch.full((5, *s.q.shape[1:]), float("nan"), device=DEV, dtype=BF), s.q])
    out = torch.full((5 + s.N, s.nh, s.dv), 9.0, device=DEV, dtype=BF)
    PK.paged_attn(wide, s.kp, s.vp, s.table, s.cu + 5, s.lens, out=out)
    assert (out[:5] == 9.0).all()
    check(out[5:], s.oracle(), 800, 64, BF)
    q = torch.full_like(wide, 9.0)
    k, v = (torch.cat([t[:1].expand(5, -1, -1), t]) for t in (s.k, s.v))
    kp = s.kp.clone()
    PK.paged_append(wide, k, v, s.kp, s.vp, s.table, s.cu + 5, s.lens, q_out=q)
    assert (q[:5] == 9.0).all() and torch.equal(q[5:], s.q)
    assert int((s.kp.nan_to_num(7.0) != kp.nan_to_num(7.0)).any(-1).any(1).sum()) <= s.N


def test_a_contiguous_cache_is_one_page():
    """A stream's static cache [nkv, max_len, hd] is a pool of one page."""
    s = Streams([1], [200], page=256, seed=47, more_pages=0)
    s.kp, s.vp = (t[s.table[0, 0]][None].clone() for t in (s.kp, s.vp))
    s.table.zero_()
    check(s.attn(), s.oracle(), 256, 64, BF)


# ------------------------------------------------------------------------------------------------ as they are used

def _step(s, inv, out=None, ws=None):
    q = PK.paged_append(s.q, s.k, s.v, s.kp, s.vp, s.table, s.cu, s.lens, inv)
    return PK.paged_attn(q, s.kp, s.vp, s.table, s.cu, s.lens, out=out, workspace=ws)


def test_prompt_then_pieces_then_tokens_agree():
    """A prompt at once, the same one in pieces, and its last tokens one by one, over the paged cache: every way is the
    oracle's attention over the rotated rows."""
    n, inv = 150, (1e6 ** (-torch.arange(32, device=DEV) / 32)).float()
    s = Streams([n, 40], [0, 0], seed=53)
    k = torch.empty(s.N, s.nkv, 64, device=DEV, dtype=BF)
    q = PK.paged_append(s.q, s.k, s.v, s.kp, s.vp, s.table, s.cu, s.lens, inv, k_out=k)
    want = O.prompt_attn(q, k, s.v, s.cu, 64 ** -0.5)
    check(PK.prompt_attn(q, k, s.v, s.cu), want, n, 64, BF)
    check(PK.paged_attn(q, s.kp, s.vp, s.table, s.cu, s.lens), want, n, 64, BF)
    s.kp.fill_(float("nan"))
    s.vp.fill_(float("nan"))
    done = [0, 0]
    for step in ([100, 1], [20, 0], [28, 38], [1, 0], [1, 1]):
        rows = torch.cat([torch.arange(d, d + m) + (0, n)[b] for b, (d, m) in enumerate(zip(done, step))]).to(DEV)
        done = [d + m for d, m in zip(done, step)]
        cu = torch.tensor([0, step[0], sum(step)], device=DEV, dtype=torch.int32)
        lens = torch.tensor(done, device=DEV, dtype=torch.int32)
        pq = PK.paged_append(s.q[rows], s.k[rows], s.v[rows], s.kp, s.vp, s.table, cu, lens, inv)
        assert torch.equal(pq, q[rows])
        got = PK.paged_attn(pq, s.kp, s.vp, s.table, cu, lens)
        check(got, tuple(t[rows] for t in want), n, 64, BF)


@pytest.mark.parametrize("idx", [torch.int32, torch.int64])
def test_one_graph_serves_every_length(idx):
    """A padded decode step captured once and replayed while lengths, tables and the number of streams change, with eager
    work between the replays."""
    B, inv = 6, (1e6 ** (-torch.arange(32, device=DEV) / 32)).float()
    cases = [Streams([1] * n + [0] * (B - n), ctx, idx=idx, seed=60 + n, spare=B - n)
             for n, ctx in ((4, [0, 700, 3, 90, 5, 0]), (6, [9, 1000, 2500, 1, 16, 15]), (1, [64, 0, 0, 0, 0, 0]),
                            (5, [800, 17, 31, 32, 33, 0]))]
    width, n_pages = max(s.table.shape[1] for s in cases), max(s.kp.shape[0] for s in cases)
    q, k, v = (torch.zeros(B, h, 64, device=DEV, dtype=BF) for h in (14, 2, 2))
    kp, vp = (torch.zeros(n_pages, 2, 16, 64, device=DEV, dtype=BF) for _ in range(2))
    table, cu, lens = (torch.zeros(n, device=DEV, dtype=idx) for n in ((B, width), (B + 1,), (B,)))
    out = torch.zeros(B, 14, 64, device=DEV, dtype=BF)

    def step():
        PK.paged_attn(PK.paged_append(q, k, v, kp, vp, table, cu, lens, inv), kp, vp, table, cu, lens, out=out)

    def load(s):
        for dst, src in ((q, s.q), (k, s.k), (v, s.v), (cu, s.cu), (lens, s.lens)):
            dst.copy_(src)
        table.fill_(-1)
        table[:, :s.table.shape[1]] = s.table
        kp.fill_(float("nan"))
        vp.fill_(float("nan"))
        kp[:s.kp.shape[0]], vp[:s.vp.shape[0]] = s.kp, s.vp
    load(cases[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for s in cases + cases[::-1]:
        load(s)
        out.fill_(5.0)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        n = sum(s.new)
        assert (got[n:] == 5.0).all()
        eager = Streams.__new__(Streams)
        eager.__dict__.update(s.__dict__)
        eager.kp, eager.vp = s.kp.clone(), s.vp.clone()
        want_q = PK.paged_append(s.q, s.k, s.v, eager.kp, eager.vp, s.table, s.cu, s.lens, inv)
        check(got[:n], O.paged_attn(want_q[:n], eager.kp, eager.vp, s.table, s.cu, s.lens, 64 ** -0.5), 2600, 64, BF)


@BOTH
def test_one_graph_serves_every_length_of_many_streams(kind):
    """The same with an index of the streams (more than 128), in one captured call and its workspace."""
    B = 200
    cases = [Streams([(1, 0, 3)[(i * k) % 3] if i < n else 0 for i in range(B)], [(i * k * 61) % 900 for i in range(B)],
                     4, 2, 64, 64, seed=70 + k, spare=600, more_pages=many_pages(kind, 16)) for k, n in ((1, 200), (2, 130), (5, 1))]
    rows = max(len(s.q) for s in cases)
    q = torch.zeros(rows, 4, 64, device=DEV, dtype=BF)
    out = torch.zeros(rows, 4, 64, device=DEV, dtype=BF)
    kp, vp = (torch.zeros(max(s.kp.shape[0] for s in cases), 2, 16, 64, device=DEV, dtype=BF) for _ in range(2))
    table = torch.zeros(B, max(s.table.shape[1] for s in cases), device=DEV, dtype=torch.int32)
    cu, lens = (torch.zeros(n, device=DEV, dtype=torch.int32) for n in (B + 1, B))
    ws = PK.paged_attn_workspace(rows, B, table.shape[1] * 16, 4, 2, 64, 64)
    graph = torch.cuda.CUDAGraph()
    PK.paged_attn(q, kp, vp, table, cu, lens, out=out, workspace=ws)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        PK.paged_attn(q, kp, vp, table, cu, lens, out=out, workspace=ws)
    for s in cases + cases[::-1]:
        table.fill_(-1)
        for dst, src in ((q[:len(s.q)], s.q), (cu, s.cu), (lens, s.lens), (table[:, :s.table.shape[1]], s.table),
                         (kp[:s.kp.shape[0]], s.kp), (vp[:s.vp.shape[0]], s.vp)):
            dst.copy_(src)
        out.fill_(5.0)
        ws.fill_(255)
        graph.replay()
        torch.cuda.synchronize()
        assert (out[s.N:] == 5.0).all()
        check(out[:s.N], s.oracle(), 1000, 64, BF)


def test_another_stream_and_a_shared_workspace():
    s = Streams([1, 1, 5], [6000, 20, 300], seed=71)
    want = s.attn()
    ws = PK.paged_attn_workspace(s.N, 3, s.table.shape[1] * s.page, s.nh, s.nkv, s.dqk, s.dv)
    ws.fill_(255)  # NaN: its content is nobody's input
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [s.attn(workspace=ws) for _ in range(3)]  # calls that share it, one after the other
    side.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    ws = PK.prompt_attn_workspace(s.N, 3, s.nh, s.nkv, s.dqk, s.dv)
    ws.fill_(255)
    assert torch.equal(PK.prompt_attn(s.q, s.k, s.v, s.cu, workspace=ws), PK.prompt_attn(s.q, s.k, s.v, s.cu))


def test_two_streams_at_once():
    """Calls on two streams, each with a workspace of its own, give what they give alone."""
    a, b = Streams([1] * 20, [50 * i for i in range(20)], seed=73), Streams([400, 3], [900, 50], seed=74)
    want = a.attn(), b.attn()
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate((a, b)):
            with torch.cuda.stream(sides[i]):
                got[i].append(s.attn())
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in got[i])


def test_a_small_workspace_is_refused():
    s = Streams([1], [9000], seed=79)
    ws = PK.paged_attn_workspace(1, 1, s.table.shape[1] * s.page, s.nh, s.nkv, s.dqk, s.dv)
    assert torch.equal(s.attn(workspace=ws), s.attn())
    with pytest.raises(ValueError, match="workspace"):
        s.attn(workspace=ws[:-16])
    with pytest.raises(ValueError, match="dv=12"):
        PK.prompt_attn_workspace(8, 2, 4, 2, 64, 12)


def test_no_streams_no_tokens_no_pages():
    e = torch.empty(0, device=DEV, dtype=torch.int32)
    cu = torch.zeros(1, device=DEV, dtype=torch.int32)
    q, k = torch.full((3, 4, 64), 2.0, device=DEV, dtype=BF), torch.zeros(3, 2, 64, device=DEV, dtype=BF)
    pool = torch.zeros(0, 2, 16, 64, device=DEV, dtype=BF)
    out = torch.full_like(q, 7.0)
    assert (PK.paged_attn(q, pool, pool, e.view(0, 5), cu, e, out=out) == 7.0).all()
    assert (PK.prompt_attn(q, k, k, cu, out=out) == 7.0).all()
    assert (PK.paged_append(q, k, k, pool, pool, e.view(0, 5), cu, e, q_out=out) == 7.0).all()
    one = torch.tensor([0, 3], device=DEV, dtype=torch.int32)
    zero = torch.zeros(1, device=DEV, dtype=torch.int32)
    assert (PK.paged_attn(q, pool, pool, zero.view(1, 1)[:, :0], one, zero, out=out) == 0.0).all()  # nothing to see
    assert torch.equal(PK.paged_append(q, k, k, pool, pool, zero.view(1, 1)[:, :0], one, zero), q)
    none = PK.paged_attn(q[:0], pool, pool, zero.view(1, 1), zero.expand(2).contiguous(), zero)
    assert none.shape == (0, 4, 64)


@BOTH
def test_indices_that_make_no_sense_stay_in_bounds(kind):
    """cu_seqlens that falls, starts behind 0 or ends behind the tokens: which rows are computed is open, but every access
    stays inside the tensors (the host-side twin of the work's division: tests/test_paged_kv.py)."""
    s = Streams([5, 60, 3], [100, 900, 0], seed=83, more_pages=many_pages(kind, 16))
    for cu in ([0, 65, 5, 68], [3, 5, 65, 68], [0, 5, 65, 9999], [-7, 5, 65, 68], [68, 0, 68, 0], [0, 68, 0, 68]):
        s.cu = torch.tensor(cu, device=DEV, dtype=torch.int32)
        s.attn()
        PK.prompt_attn(s.q, s.k, s.v, s.cu)
        PK.paged_append(s.q, s.k, s.v, s.kp, s.vp, s.table, s.cu, s.lens)
        torch.cuda.synchronize()


@BOTH
def test_indices_of_many_streams_that_make_no_sense_stay_in_bounds(kind):
    """The same where the streams are indexed first."""
    s = Streams([1] * 150, [(i * 7) % 300 for i in range(150)], seed=84, spare=40, more_pages=many_pages(kind, 16))
    up = torch.arange(151, device=DEV, dtype=torch.int32)
    for cu in (up.flip(0), (up * 73) % 160, up * 5 - 200, torch.where(up % 2 == 0, 0, 190).int()):
        s.cu = cu.contiguous()
        s.attn()
        PK.prompt_attn(s.q, s.k, s.v, s.cu)
        PK.paged_append(s.q, s.k, s.v, s.kp, s.vp, s.table, s.cu, s.lens)
        torch.cuda.synchronize()
