"""CPU checks of the paged cache: the header and its structs, the refusals of the C entries and of the wrappers, the
arithmetic that turns positions into pages, and the oracle against torch's own attention."""
import ctypes
import hashlib
import math
import os
import re
import subprocess

import pytest
import torch

import _mingmoe as mm
import paged_kv as PK
from oracle import paged_oracle as O

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "mingpaged.h")
BF = torch.bfloat16


def _text():
    return re.sub(r"/\*.*?\*/", " ", open(HEADER).read(), flags=re.S)


def test_header_declares_the_entry_points_and_the_library_exports_them():
    names = sorted(set(re.findall(r"^\s*(?:int|int64_t)\s+(mm_\w+)\s*\(", _text(), re.M)))
    assert names == sorted(mm.PAGED_SIGNATURES)
    lib = mm.load()
    assert all(hasattr(lib, n) for n in names)
    assert lib.mm_paged_version() == mm.PAGED_VERSION


# digests of the header's interface (no comments) by version, as tests/test_abi.py keeps them for mingmoe.h
INTERFACES = {1: "4173de86697e9f74", 2: "d6742157bdb42d72"}


def test_the_version_moves_with_the_interface():
    text = _text()
    version = int(re.search(r"#define MM_PAGED_VERSION (\d+)", text).group(1))
    code = " ".join(re.sub(r"#define MM_PAGED_VERSION \d+", "", text).split())
    assert hashlib.sha256(code.encode()).hexdigest()[:16] == INTERFACES[version]
    assert version == mm.PAGED_VERSION == max(INTERFACES)


STRUCTS = [("mm_pages", mm.Pages), ("mm_batch", mm.Batch), ("mm_rows", mm.Rows),
           ("mm_paged_append_args", mm.PagedAppendArgs), ("mm_paged_attn_args", mm.PagedAttnArgs),
           ("mm_prompt_attn_args", mm.PromptAttnArgs)]


@pytest.mark.parametrize("name,struct", STRUCTS)
def test_struct_layout_matches_c(tmp_path, name, struct):
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "mingpaged.h"\n'
                   f'int main(void){{printf("%zu", sizeof({name}));'
                   + "".join(f'printf(" %zu", offsetof({name}, {f}));' for f, _ in struct._fields_) + 'return 0;}\n')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.dirname(HEADER), str(src), "-o", str(exe)], check=True)
    vals = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert vals == [ctypes.sizeof(struct)] + [getattr(struct, f).offset for f, _ in struct._fields_]


@pytest.mark.parametrize("name,struct", STRUCTS)
def test_packed_arguments_lie_as_the_structure_does(name, struct):
    pack = mm.packer(struct)
    assert pack.size == ctypes.sizeof(struct)

    def leaves(s, at=0):
        for f, kind in s._fields_:
            off = at + getattr(s, f).offset
            if issubclass(kind, ctypes.Structure):
                yield from leaves(kind, off)
            else:
                yield kind, off
    places = list(leaves(struct))
    data = pack.pack(*range(1, len(places) + 1))
    assert [kind.from_buffer_copy(data, off).value for kind, off in places] == list(range(1, len(places) + 1))


# ------------------------------------------------------------------------------------------------ refusals, C entries

P = 4096  # an aligned address that no refused call reads


def pages(**kw):
    g = mm.Pages(P, P, mm.MM_BF16, 2, 64, 64, 10, 16, 2 * 16 * 64, 16 * 64, 64, 2 * 16 * 64, 16 * 64, 64)
    for k, v in kw.items():
        setattr(g, k, v)
    return g


def batch(**kw):
    b = mm.Batch(P, P, P, 4, 4, 3, 5, mm.MM_INT32)
    for k, v in kw.items():
        setattr(b, k, v)
    return b


def err(rc):
    assert rc == mm.MM_ERR_ARG
    return mm.last_error()


def append(g=None, b=None, q=P, q_ts=512, q_hs=64, k=P, v=P, nh=14, inv=P, pairs=32, off=0, q_out=P, k_out=None,
           qo_ts=896):
    a = mm.PagedAppendArgs(g or pages(), b or batch(), (q, q_ts, q_hs), (k, 128, 64), (v, 128, 64), (q_out, qo_ts, 64),
                           (k_out, 128, 64), inv, pairs, nh, off, 0)
    return mm.load().mm_paged_append(ctypes.byref(a), None)


def attn(g=None, b=None, q=P, q_ts=896, nh=14, out=P, o_hs=64, ws=P, ws_bytes=1 << 40):
    a = mm.PagedAttnArgs(g or pages(), b or batch(), (q, q_ts, 64), (out, 896, o_hs), ws, ws_bytes, nh, 0.125)
    return mm.load().mm_paged_attn(ctypes.byref(a), None)


def prompt(q=P, k=P, v=P, dtype=mm.MM_BF16, nh=14, nkv=2, dqk=64, dv=64, cu=P, idx=mm.MM_INT32, seqs=3, tokens=5, out=P,
           k_ts=128):
    a = mm.PromptAttnArgs((q, 896, 64), (k, k_ts, 64), (v, 128, 64), (out, 896, 64), cu, seqs, tokens, P, 1 << 40, idx,
                          dtype, nh, nkv, dqk, dv, 0.125)
    return mm.load().mm_prompt_attn(ctypes.byref(a), None)


@pytest.mark.parametrize("call", [append, attn])
@pytest.mark.parametrize("what,g,b", [
    ("bf16 or fp16", dict(dtype=mm.MM_FP32), {}), ("multiple of nkv", dict(nkv=4), {}), ("multiple of nkv", dict(nkv=0), {}),
    ("dqk=60", dict(dqk=60), {}), ("dqk=264", dict(dqk=264), {}), ("dv=0", dict(dv=0), {}), ("dv=260", dict(dv=260), {}),
    ("page or table", dict(page=0), {}), ("page or table", dict(n_pages=-1), {}), ("page or table", {}, dict(max_pages=-1)),
    ("at most 2^30", dict(page=1 << 20), dict(max_pages=1 << 11)), ("tokens -1", {}, dict(tokens=-1)),
    ("tokens", {}, dict(tokens=1 << 23)), ("streams", {}, dict(seqs=-1)), ("streams", {}, dict(seqs=1 << 21)),
    ("int32 or int64", {}, dict(idx_dtype=mm.MM_FP32)), ("null batch", {}, dict(cu=None)),
    ("null batch", {}, dict(kv_lens=None)), ("null batch", {}, dict(table=None)), ("null pool", dict(v=None), {}),
    ("16-byte aligned", dict(k=P + 8), {}), ("multiples of 8", dict(k_row_stride=68), {}),
    ("multiples of 8", dict(v_page_stride=-8), {})])
def test_the_pool_and_the_batch_are_checked(call, what, g, b):
    assert what in err(call(g=pages(**g), b=batch(**b)))


def test_append_refuses():
    assert "pairs" in err(append(pairs=36)) and "pairs" in err(append(pairs=40)) and "pairs" in err(append(off=8))
    assert "pairs" in err(append(pairs=16, off=4)) and "pairs" in err(append(pairs=-8))
    assert "null q" in err(append(q=None)) and "null k" in err(append(k=None)) and "null v" in err(append(v=None))
    assert "null q_out" in err(append(q_out=None))
    assert "q must be 16-byte" in err(append(q=P + 2)) and "k_out must be 16-byte" in err(append(k_out=P + 8))
    assert "on each other" in err(append(g=pages(), q_out=P, qo_ts=0)) and "strides must be" in err(append(g=pages(k_row_stride=0)))
    assert "strides of q" in err(append(q_ts=900)) and "strides of q" in err(append(q_hs=-64))
    for entry in (mm.load().mm_paged_append, mm.load().mm_paged_attn, mm.load().mm_prompt_attn):
        assert "null arguments" in err(entry(None, None))


def test_attn_refuses():
    assert "null q" in err(attn(q=None)) and "null out" in err(attn(out=None))
    assert "strides of q" in err(attn(q_ts=892)) and "out must be 8-byte" in err(attn(out=P + 4))
    assert "strides of out" in err(attn(o_hs=66)) and "on each other" in err(attn(o_hs=0))
    assert "tokens * nh" in err(attn(b=batch(tokens=1 << 22), nh=512))
    need = mm.load().mm_paged_attn_workspace(5, 3, 16 * 1000, 14, 2, 64, 64, 0)  # a table that allows long contexts
    long = batch(max_pages=1000, table_stride=1000)
    assert need > 0 and "workspace" in err(attn(b=long, ws_bytes=need - 1)) and "workspace" in err(attn(b=long, ws=None))
    assert "workspace" in err(attn(b=long, ws=P + 4))


def test_prompt_refuses():
    assert "bf16 or fp16" in err(prompt(dtype=mm.MM_INT8)) and "multiple of nkv" in err(prompt(nh=15))
    assert "dqk=68" in err(prompt(dqk=68)) and "dv=-8" in err(prompt(dv=-8)) and "null cu" in err(prompt(cu=None))
    assert "int32 or int64" in err(prompt(idx=mm.MM_BF16)) and "tokens" in err(prompt(tokens=-3))
    assert "streams" in err(prompt(seqs=-1)) and "null k" in err(prompt(k=None)) and "strides of k" in err(prompt(k_ts=129))
    assert "out must be 8-byte" in err(prompt(out=P + 2))


def test_nothing_to_do_is_done_without_a_gpu():
    for b in (batch(tokens=0), batch(seqs=0)):
        assert append(b=b) == 0 and attn(b=b) == 0
    assert prompt(tokens=0) == 0 and prompt(seqs=0) == 0


def test_no_streams_need_no_arrays():
    assert attn(b=batch(seqs=0, cu=None, kv_lens=None, table=None)) == 0
    assert append(b=batch(seqs=0, cu=None, kv_lens=None, table=None)) == 0 and prompt(seqs=0, cu=None) == 0


def test_more_than_one_launch_holds_is_refused():
    g, b = pages(nkv=16, k_head_stride=64, v_head_stride=64), batch(seqs=1 << 20, tokens=1 << 22)
    assert "one launch" in err(attn(g=g, b=b, nh=64))


def test_workspace_sizes():
    lib = mm.load()
    assert lib.mm_paged_attn_workspace(-1, 1, 64, 14, 2, 64, 64, 0) == -1
    assert lib.mm_paged_attn_workspace(1, 1, 1 << 31, 14, 2, 64, 64, 1) == -1
    assert lib.mm_paged_attn_workspace(1, 1, 64, 14, 4, 64, 64, 0) == -1
    assert lib.mm_prompt_attn_workspace(1, -1, 14, 2, 64, 64, 0) == -1
    assert lib.mm_prompt_attn_workspace(1, 1, 14, 2, 64, 63, 1) == -1
    assert lib.mm_paged_attn_workspace(1, 1, 700, 14, 2, 64, 64, 0) == 0  # a short table is not cut


@pytest.mark.parametrize("nh,nkv,dqk,dv", [(14, 2, 64, 64), (16, 16, 192, 128), (32, 8, 128, 128), (16, 2, 256, 256),
                                           (20, 1, 64, 64)])
def test_a_workspace_for_at_most_these_sizes_serves_every_smaller_batch(nh, nkv, dqk, dv):
    lib = mm.load()
    sizes = [1, 2, 15, 64, 130, 700, 2500, 9000, 40000]
    for tokens in sizes:
        for seqs in (1, 3, 40, 600):
            most = lib.mm_prompt_attn_workspace(tokens, seqs, nh, nkv, dqk, dv, 1)
            assert all(lib.mm_prompt_attn_workspace(t, s, nh, nkv, dqk, dv, 0) <= most
                       for t in sizes if t <= tokens for s in (1, 2, 3, 39, 40, 600) if s <= seqs)
            for keys in (64, 300, 2000, 50000):
                most = lib.mm_paged_attn_workspace(tokens, seqs, keys, nh, nkv, dqk, dv, 1)
                assert all(lib.mm_paged_attn_workspace(t, s, k, nh, nkv, dqk, dv, 0) <= most
                           for t in sizes if t <= tokens for s in (1, 2, 40, 600) if s <= seqs
                           for k in (64, 299, 300, 1100, 2000, 50000) if k <= keys)


# ------------------------------------------------------------------------------------------------ refusals, wrappers

def test_wrappers_take_gpu_tensors_only():
    t, i = torch.zeros(1, 2, 64, dtype=BF), torch.zeros(2, dtype=torch.int32)
    pool = torch.zeros(1, 2, 16, 64, dtype=BF)
    table = torch.zeros(1, 1, dtype=torch.int32)
    for call in (lambda: PK.paged_append(t, t, t, pool, pool, table, i, i[:1]),
                 lambda: PK.paged_attn(t, pool, pool, table, i, i[:1]), lambda: PK.prompt_attn(t, t, t, i)):
        with pytest.raises(ValueError, match="no CPU path"):
            call()


@pytest.fixture
def any_device(monkeypatch):
    """The wrappers' own checks on CPU tensors: none of the refused calls reaches the library."""
    monkeypatch.setattr(mm, "require_gpu", lambda *t: None)
    monkeypatch.setattr(PK, "_on", lambda dev, fn, *a: fn(*a))
    monkeypatch.setattr(PK, "_call", lambda *a: pytest.fail("the call was not refused"))


def _args(N=3, B=2, nh=4, nkv=2, d=16, dv=8, dt=BF, idx=torch.int32):
    return dict(q=torch.zeros(N, nh, d, dtype=dt), k=torch.zeros(N, nkv, d, dtype=dt), v=torch.zeros(N, nkv, dv, dtype=dt),
                k_pages=torch.zeros(5, nkv, 4, d, dtype=dt), v_pages=torch.zeros(5, nkv, 4, dv, dtype=dt),
                page_table=torch.zeros(B, 3, dtype=idx), cu_seqlens=torch.zeros(B + 1, dtype=idx),
                kv_lens=torch.zeros(B, dtype=idx))


@pytest.mark.parametrize("what,change", [
    ("q must be", dict(q=torch.zeros(3, 4, 24, dtype=BF))), ("q must be", dict(q=torch.zeros(3, 64, dtype=BF))),
    ("q must be", dict(q=torch.zeros(3, 4, 16))), ("contiguous last dim", dict(q=torch.zeros(3, 16, 4, dtype=BF).mT)),
    ("k must be", dict(k=torch.zeros(3, 3, 16, dtype=BF))), ("v must be", dict(v=torch.zeros(3, 2, 16, dtype=BF))),
    ("k must be", dict(k=torch.zeros(4, 2, 16, dtype=BF))), ("rot_offset=-8", dict(rot_offset=-8)),
    ("rot_offset", dict(rot_offset=1 << 32)),
    ("k_pages and v_pages must be", dict(k_pages=torch.zeros(5, 2, 8, 16, dtype=BF))),
    ("k_pages and v_pages must both", dict(k_pages=torch.zeros(5, 2, 16, dtype=BF))),
    ("both be bf16 or fp16", dict(k_pages=torch.zeros(5, 2, 4, 16))),
    ("kv_lens must be", dict(kv_lens=torch.zeros(3, dtype=torch.int32))),
    ("one dtype", dict(kv_lens=torch.zeros(2, dtype=torch.int64))), ("cu_seqlens", dict(cu_seqlens=torch.zeros(3))),
    ("cu_seqlens", dict(cu_seqlens=torch.zeros(0, dtype=torch.int32))),
    ("page_table", dict(page_table=torch.zeros(3, 3, dtype=torch.int32))),
    ("page_table", dict(page_table=torch.zeros(3, 2, dtype=torch.int32).t())),
    ("inv_freq", dict(inv_freq=torch.zeros(8, dtype=BF))), ("q_out", dict(q_out=torch.zeros(3, 4, 8, dtype=BF))),
    ("q_out must be", dict(q_out=torch.zeros(2, 4, 16, dtype=BF))),
    ("k_out must be", dict(k_out=torch.zeros(2, 2, 16, dtype=BF)))])
def test_append_wrapper_refuses(any_device, what, change):
    with pytest.raises(ValueError, match=what):
        PK.paged_append(**{**_args(), **change})


@pytest.mark.parametrize("what,change", [
    ("q must be", dict(q=torch.zeros(3, 4, 24, dtype=BF))), ("q must be", dict(q=torch.zeros(3, 4, 16, dtype=torch.float16))),
    ("k_pages and v_pages must be", dict(v_pages=torch.zeros(4, 2, 4, 8, dtype=BF))),
    ("out must be", dict(out=torch.zeros(2, 4, 8, dtype=BF))), ("out must be", dict(out=torch.zeros(3, 4, 16, dtype=BF))),
    ("one dtype", dict(page_table=torch.zeros(2, 3, dtype=torch.int64))),
    ("workspace must be contiguous", dict(workspace=torch.zeros(1).expand(1 << 20)))])
def test_attn_wrapper_refuses(any_device, what, change):
    a = {k: v for k, v in _args().items() if k not in "kv"}
    with pytest.raises(ValueError, match=what):
        PK.paged_attn(**{**a, **change})


@pytest.mark.parametrize("what,change", [
    ("bf16 or fp16", dict(q=torch.zeros(3, 4, 16))), ("q must be", dict(k=torch.zeros(3, 2, 8, dtype=BF))),
    ("k must be", dict(k=torch.zeros(4, 2, 16, dtype=BF))),
    ("v must be", dict(v=torch.zeros(3, 1, 8, dtype=BF))), ("v must be", dict(v=torch.zeros(2, 2, 8, dtype=BF))), ("q, k and v must be", dict(v=torch.zeros(3, 16, dtype=BF))),
    ("cu_seqlens", dict(cu_seqlens=torch.zeros(2, 2, dtype=torch.int32))),
    ("out must be", dict(out=torch.zeros(3, 4, 8))),
    ("workspace must be contiguous", dict(workspace=torch.zeros(1 << 10)[::2]))])
def test_prompt_wrapper_refuses(any_device, what, change):
    a = {k: v for k, v in _args().items() if k in ("q", "k", "v", "cu_seqlens")}
    with pytest.raises(ValueError, match=what):
        PK.prompt_attn(**{**a, **change})


# ------------------------------------------------------------------------------------------------ arithmetic

def test_division_by_a_page_is_exact():
    """The kernels' n / d: umulhi(n, floor(2^(31 + l) / d) + 1) >> (l - 1), l = ceil(log2 d), for n < 2^31."""
    for d in [2, 3, 5, 7, 14, 16, 24, 25, 100, 255, 256, 641, 1000, 4096, 65537, 1 << 20, (1 << 30) + 1, (1 << 31) - 1]:
        length = (d - 1).bit_length()
        m = (1 << (31 + length)) // d + 1
        assert m < 1 << 32
        top = (1 << 31) - 1
        for n in {0, 1, d - 1, d, d + 1, top, top - 1, top // d * d, top // d * d - 1, 12345678, top // 2}:
            if 0 <= n <= top:
                assert ((n * m) >> 32) >> (length - 1) == n // d, (n, d)


def test_oracle_matches_torch_attention():
    torch.manual_seed(0)
    q, k, v = (torch.randn(7, n, 16, dtype=torch.float64) for n in (4, 2, 2))
    cu = torch.tensor([0, 3, 3, 7])
    out, _, _ = O.prompt_attn(q, k, v, cu, 0.3)
    for a, b in ((0, 3), (3, 7)):
        qs, ks, vs = q[a:b].transpose(0, 1), *(t[a:b].repeat_interleave(2, 1).transpose(0, 1) for t in (k, v))
        want = torch.nn.functional.scaled_dot_product_attention(qs, ks, vs, is_causal=True, scale=0.3)
        torch.testing.assert_close(out[a:b], want.transpose(0, 1))
    # the same rows in pages of 2, as a chunk of the last two tokens behind what came before, and a page that is missing
    pool_k, pool_v = (torch.randn(6, 2, 2, 16, dtype=torch.float64) for _ in range(2))
    table = torch.tensor([[4, 1], [9, 9], [0, 3]])
    for b, (a, e) in enumerate(((0, 3), (3, 3), (3, 7))):
        for p in range(e - a):
            pool_k[table[b, p // 2], :, p % 2], pool_v[table[b, p // 2], :, p % 2] = k[a + p], v[a + p]
    part = torch.cat([q[1:3], q[5:7]])
    got, _, _ = O.paged_attn(part, pool_k, pool_v, table, torch.tensor([0, 2, 2, 4]), torch.tensor([3, 0, 4]), 0.3)
    torch.testing.assert_close(got, torch.cat([out[1:3], out[5:7]]))
    table[0, 0] = -1
    got, _, _ = O.paged_attn(part, pool_k, pool_v, table, torch.tensor([0, 2, 2, 4]), torch.tensor([3, 0, 4]), 0.3)
    assert (got[0] == 0).all()  # its only positions lie in the missing page
    torch.testing.assert_close(got[1], v[2].repeat_interleave(2, 0))


# ------------------------------------------------------------------------------------------------ the division of the work

class Division:
    """The kernels' division of an attention's work (csrc/paged_common.h: stream_at, cut_of, find_work, keys_of, pieces_of,
    keys_of_piece), number by number, for blocks of `br` rows and granules of `gr` keys."""

    def __init__(self, cu, lens, tokens, group, max_keys, br, gr, target, min_cut):
        self.br, self.gr, self.group, self.target = br, gr, group, target
        self.streams = []
        for c0, c1, kv in zip(cu, cu[1:], lens):
            first = min(max(c0, 0), tokens)
            self.streams.append((first, min(max(c1, first), tokens) - first, kv if 0 <= kv <= max_keys else -1))
        total = sum(self.blocks(s) * -(-max(s[2], 0) // gr) for s in self.streams)
        self.cut = 0
        if target:
            # the kernel's sum over the lanes is in fp32, rounded up by 1e-5 of it: the least and the most that it can be
            aim = target - min(sum(self.blocks(s) for s in self.streams), target) / 2
            self.cut = min(max(math.ceil(total * 1.00002 / aim), min_cut), (1 << 30) // gr)
            assert self.cut * target >= total or self.cut == (1 << 30) // gr

    def blocks(self, s):
        return -(-s[1] * self.group // self.br)

    def pieces(self, keys):
        return 1 if self.cut == 0 else max(1, -(--(-keys // self.gr) // self.cut))

    def keys(self, s, blk):
        last = min(blk * self.br + self.br, s[1] * self.group) - 1
        return 0 if s[2] < 0 else max(0, s[2] - s[1] + last // self.group + 1)

    def part(self, keys, piece):
        """The keys of a piece."""
        g, n = -(-keys // self.gr), self.pieces(keys)
        first = piece * (g // n) + min(piece, g % n)
        return first * self.gr, min(keys, (first + g // n + (piece < g % n)) * self.gr)

    def find(self, w, cut_blocks=False):
        """(stream, block, piece, first slot) of workgroup w, or None."""
        slots = 0
        for b, s in enumerate(self.streams):
            nb, p = self.blocks(s), self.pieces(max(s[2], 0))
            held = nb * p if p > 1 else 0
            units = (nb if held else 0) if cut_blocks else nb * p
            if w < units:
                at = w if cut_blocks else w // p
                slot = slots + at * p
                if w < 0 or at >= nb or (p > 1 and not 0 <= slot <= 2 * self.target - p):
                    return None
                return b, nb - 1 - at, 0 if cut_blocks else w - at * p, slot
            w -= units
            slots += held
        return None


    def index(self):
        """index_kernel: for each stream the ends of its workgroups and of its cut blocks, and its first state."""
        units = cut = held = 0
        for s in self.streams:
            nb, p = self.blocks(s), self.pieces(max(s[2], 0))
            units, cut, first = units + nb * p, cut + (nb if p > 1 else 0), held
            held += nb * p if p > 1 else 0
            yield units, cut, first

    def find_indexed(self, w, index, cut_blocks=False):
        """find by the index, as the kernels do it for many streams."""
        ends = [e[1 if cut_blocks else 0] for e in index]
        b = count_before(len(ends), lambda i: ends[i] <= w)
        if b >= len(ends):
            return None
        s, nb, p = self.streams[b], self.blocks(self.streams[b]), self.pieces(max(self.streams[b][2], 0))
        units = (nb if p > 1 else 0) if cut_blocks else nb * p
        u = w - (ends[b] - units)
        at = u if cut_blocks else u // max(p, 1)
        slot = index[b][2] + at * p
        if not 0 <= u < units or (p > 1 and not 0 <= slot <= 2 * self.target - p):
            return None
        return b, nb - 1 - at, 0 if cut_blocks else u - at * p, slot


def count_before(n, before):
    """The kernels' search (csrc/paged_common.h: count_before): every probe stays inside the sequence."""
    def probe(i):
        assert 0 <= i < n
        return before(i)
    lo, hi = 0, n
    while hi - lo > 64:
        step = -(-(hi - lo) // 64)
        at = [lo + (lane + 1) * step - 1 for lane in range(64)]
        passed = sum(probe(min(i, hi - 1)) and i < hi for i in at)
        lo = min(lo + passed * step, hi)
        hi = min(lo + step, hi)
    return lo + sum(probe(min(lo + lane, n - 1)) and lo + lane < hi for lane in range(64))


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 127, 128, 129, 4096, 4097, 4225, 100000])
def test_the_search_counts_what_comes_before(n):
    for answer in {0, 1, 2, 62, 63, 64, 65, 66, n // 2, n - 65, n - 64, n - 63, n - 1, n} & set(range(n + 1)):
        assert count_before(n, lambda i: i < answer) == answer
    assert 0 <= count_before(n, lambda i: i % 3 == 1) <= n  # nonsense stays in bounds


def _divisions(seed):
    import random
    r = random.Random(seed)
    for _ in range(8):
        n = r.choice([1, 2, 5, 64, 65, 200])
        new = [r.choice([0, 1, 1, 1, 3, 40, 700]) for _ in range(n)]
        lens = [m + r.choice([0, 0, 5, 900, 30000]) for m in new]
        br, gr, cut = r.choice([(16, 256, 1), (16, 128, 1), (128, 64, 4)])
        yield new, lens, r.choice([1, 2, 7, 20]), br, gr, cut, r.choice([1, 7, 64, 256])


@pytest.mark.parametrize("seed", range(5))
def test_the_work_is_divided_once_and_within_its_bounds(seed):
    for new, lens, group, br, gr, min_cut, target in _divisions(seed):
        cu = [sum(new[:i]) for i in range(len(new) + 1)]
        N, most = cu[-1], max(lens) + 1
        d = Division(cu, lens, N, group, most, br, gr, target, min_cut)
        rows = N * group
        blocks = min(rows // br + len(new), rows)
        grid = blocks + target  # what the host launches for these sizes
        done, slots, index = set(), {}, list(d.index())
        for w in range(grid):
            f = d.find(w)
            if w % 5 == 0 or w < 70:
                assert d.find_indexed(w, index) == f and d.find_indexed(w, index, True) == d.find(w, True)
            if f is None:
                continue
            b, blk, piece, slot = f
            s = d.streams[b]
            pieces = d.pieces(d.keys(s, blk))
            if piece >= pieces:
                continue
            assert (b, blk, piece) not in done
            done.add((b, blk, piece))
            if pieces > 1:
                assert 0 <= slot + piece < 2 * target and slots.setdefault(slot + piece, (b, blk, piece)) == (b, blk, piece)
                parts = [d.part(d.keys(s, blk), p) for p in range(pieces)]
                assert parts[0][0] == 0 and parts[-1][1] == d.keys(s, blk) and all(a < b for a, b in parts)
                assert all(a[1] == b[0] and a[1] % gr == 0 for a, b in zip(parts, parts[1:]))
                assert max(b - a for a, b in parts) <= d.cut * gr
        want = {(b, blk, p) for b, s in enumerate(d.streams) for blk in range(d.blocks(s)) for p in range(d.pieces(d.keys(s, blk)))}
        assert done == want
        cut = {(b, blk) for b, blk, p in want if p}
        joined = [d.find(w, cut_blocks=True) for w in range(min(blocks, target))]
        joined = {f[:2]: f[3] for f in joined if f and d.pieces(d.keys(d.streams[f[0]], f[1])) > 1}
        assert set(joined) == cut and all(slots[joined[c]] == (*c, 0) for c in cut)


@pytest.mark.parametrize("cu", [[0, 65, 5, 68], [3, 5, 65, 68], [0, 5, 65, 9999], [-7, 5, 65, 68], [68, 0, 68, 0],
                                [0, 68, 0, 68], [1 << 40, -(1 << 40), 1 << 62, 0]])
@pytest.mark.parametrize("br,gr,min_cut,target", [(16, 256, 1, 0), (16, 256, 1, 5), (128, 64, 4, 3)])
def test_a_division_of_nonsense_stays_in_bounds(cu, br, gr, min_cut, target):
    N, group, lens, most = 68, 7, [105, 960, 3], 970
    d = Division(cu, lens, N, group, most, br, gr, target, min_cut)
    index = list(d.index())
    for w in range(min(N * group // br + 3, N * group) + target):
        for f in (d.find(w), d.find(w, True), d.find_indexed(w, index), d.find_indexed(w, index, True)):
            if f is None:
                continue
            b, blk, piece, slot = f
            first, n, kv = d.streams[b]
            assert 0 <= blk < d.blocks(d.streams[b]) and 0 <= first and first + n <= N
            last = min(blk * br + br, n * group) - 1
            assert 0 <= last // group < n and d.keys(d.streams[b], blk) <= kv <= most
            if d.pieces(max(kv, 0)) > 1:
                assert 0 <= slot and slot + d.pieces(max(kv, 0)) <= 2 * target
