// The paged cache of several streams: the append of new tokens with their rotation, the attention of new tokens over the
// pages, and the attention over packed prompts (C ABI: mingpaged.h).
//
//   paged_append_kernel   rotation and stores, one pass over q, k and v
//   index_kernel          where each of many streams' work begins (paged_common.h)
//   few_kernel            attention of few rows, and the joins of cut keys (paged_few.hip)
//   many_kernel           attention of many rows (paged_many.hip)
#include <cmath>

#include "paged_common.h"

namespace {

using namespace mmp;

// ------------------------------------------------------------------------------------------ append

struct AppendArgs {
  Rows q, k, v, q_out, k_out;  // k_out.p NULL: not wanted
  Pool kp, vp;
  Batch batch;
  FastDiv page, iph;  // iph: items of a q or k head
  int64_t n_pages;
  const float* inv_freq;
  int nh, nkv, dqk, dv, pairs, rot_offset, interleaved;
  int q_in_place, k_in_place;  // the dims that do not turn are there already
};

constexpr int kAppendWaves = 4;
constexpr int kMaxPairs = 128;

// Bound by the bytes: each is read once and written once, with 16-byte accesses of neighbouring lanes (131 MB at 4000 tokens
// of 16 + 16 heads of 192 and 16 of 128 in 31.8 us: 4.1 TB/s, where a copy of 2 GiB moves 4.9). WPT waves take a token and
// share its heads; no wave waits for another. A lane keeps one place of a head for all the heads
// that it goes through: 16 elements that turn, or 8 that only move; its cosines and sines, shared by all heads, come once,
// from the angles that the wave's lanes turn side by side. The first heads' data, which hang on nothing, are requested
// before the token's stream, position and page are found.
template <class T, int WPT>
__global__ __launch_bounds__(kAppendWaves * kWave) void paged_append_kernel(AppendArgs a) {
  constexpr int AHEAD = WPT == 1 ? 2 : 3;  // heads of a lane in flight
  __shared__ __align__(16) float s_cos[kAppendWaves][kMaxPairs], s_sin[kAppendWaves][kMaxPairs];
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
  const int t = static_cast<int>(blockIdx.x) * (kAppendWaves / WPT) + wave / WPT, part = wave % WPT;
  if (t >= a.batch.tokens) return;
  // the lane's place in a head of q or k
  const int iph = static_cast<int>(a.iph.d), at_once = kWave / iph, sub = static_cast<int>(div_by(lane, a.iph)), c = lane - sub * iph;
  const bool turns = c < a.pairs / 8;
  const int ch = c - a.pairs / 8;
  const int d0 = !turns ? (ch < a.rot_offset / 8 ? 8 * ch : 8 * ch + 2 * a.pairs) : a.rot_offset + (a.interleaved ? 16 * c : 8 * c);
  const int d1 = !turns ? d0 : a.interleaved ? d0 + 8 : d0 + a.pairs;
  const int heads = a.nh + a.nkv, first = part * at_once + sub, step = WPT * at_once;
  const int last = sub < at_once ? heads : 0;  // lanes behind the last whole head have none
  const uint16_t *q = a.q.at(t, 0), *k = a.k.at(t, 0), *v = a.v.at(t, 0);
  auto source = [&](int h) { return h < a.nh ? q + h * a.q.hs : k + (h - a.nh) * a.k.hs; };
  uint4 x0[AHEAD], x1[AHEAD];
  auto request = [&](int h0) {
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const uint16_t* s = source(min(h0 + u * step, heads - 1));
      x0[u] = ld16(s + d0);
      x1[u] = ld16(s + d1);
    }
  };
  request(first);
  const int vc = a.dv / 8, v_once = kWave / vc, v_sub = lane / vc, vd = 8 * (lane - v_sub * vc);
  const int v_first = part * v_once + v_sub, v_step = WPT * v_once, v_last = v_sub < v_once ? a.nkv : 0;
  uint4 xv = ld16(v + min(v_first, a.nkv - 1) * a.v.hs + vd);

  const int b = __builtin_amdgcn_readfirstlane(stream_of_token(a.batch, t));
  if (b >= a.batch.seqs) return;  // no stream owns the token
  const Stream s = stream_at(a.batch, b);
  if (t < s.first || t >= s.first + s.n) return;
  const int pos = s.kv < 0 ? 0 : s.kv - s.n + (t - s.first);
  bool stored = s.kv >= 0 && pos >= 0 && pos < a.batch.max_keys;
  int row = 0;
  int64_t page = 0;
  if (stored) {
    const int pg = static_cast<int>(div_by(pos, a.page));
    page = value_of(index_at(a.batch.table, a.batch.i64, b * a.batch.table_stride + pg), a.batch.i64);
    row = pos - pg * static_cast<int>(a.page.d);
    stored = page >= 0 && page < a.n_pages;
  }
  // angles in 64 bits, reduced to [-1/2, 1/2] turns: a position of 10^6 leaves 2^-33 of a turn, where 32 bits would leave
  // a hundredth of a turn
  for (int p = lane; p < a.pairs; p += kWave) {
    const double turn = static_cast<double>(pos) * static_cast<double>(a.inv_freq[p]) * 0.15915494309189533577;
    float sn, cs;
    sincospif(2.0f * static_cast<float>(turn - rint(turn)), &sn, &cs);
    s_cos[wave][p] = cs;
    s_sin[wave][p] = sn;
  }
  wave_lds_fence();
  float cs[8], sn[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    cs[e] = turns ? s_cos[wave][8 * c + e] : 1.f;
    sn[e] = turns ? s_sin[wave][8 * c + e] : 0.f;
  }
  uint16_t* q_out = a.q_out.at(t, 0);
  uint16_t* k_out = a.k_out.p ? a.k_out.at(t, 0) : nullptr;
  uint16_t* k_row = a.kp.at(stored ? page : 0, 0, row);
  for (int h0 = first; h0 < last; h0 += AHEAD * step) {
    if (h0 != first) request(h0);
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int h = h0 + u * step;
      if (h >= last) break;
      const bool isq = h < a.nh;
      uint16_t* dst = isq ? q_out + h * a.q_out.hs : k_out ? k_out + (h - a.nh) * a.k_out.hs : nullptr;
      uint16_t* pool = !isq && stored ? k_row + (h - a.nh) * a.kp.hs : nullptr;
      uint4 w0 = x0[u], w1 = x1[u];
      if (turns) {
        float a0[8], a1[8], y0[8], y1[8];
        unpack8<T>(w0, a0);
        unpack8<T>(w1, a1);
        if (a.interleaved) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            y0[2 * e] = fmaf(a0[2 * e], cs[e], -a0[2 * e + 1] * sn[e]);
            y0[2 * e + 1] = fmaf(a0[2 * e + 1], cs[e], a0[2 * e] * sn[e]);
            y1[2 * e] = fmaf(a1[2 * e], cs[4 + e], -a1[2 * e + 1] * sn[4 + e]);
            y1[2 * e + 1] = fmaf(a1[2 * e + 1], cs[4 + e], a1[2 * e] * sn[4 + e]);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            y0[e] = fmaf(a0[e], cs[e], -a1[e] * sn[e]);
            y1[e] = fmaf(a1[e], cs[e], a0[e] * sn[e]);
          }
        }
        w0 = pack8<T>(y0);
        w1 = pack8<T>(y1);
      } else if (isq ? a.q_in_place : a.k_in_place) {
        dst = nullptr;
      }
      if (dst) {
        st16(dst + d0, w0);
        if (turns) st16(dst + d1, w1);
      }
      if (pool) {
        st16(pool + d0, w0);
        if (turns) st16(pool + d1, w1);
      }
    }
  }
  if (!stored) return;
  uint16_t* v_row = a.vp.at(page, 0, row);
  for (int h = v_first; h < v_last; h += v_step) {
    st16(v_row + h * a.vp.hs + vd, xv);
    xv = ld16(v + min(h + v_step, a.nkv - 1) * a.v.hs + vd);
  }
}

template <class T, int WPT>
int launch_append(const AppendArgs& a, hipStream_t st) {
  constexpr int PER = kAppendWaves / WPT;  // tokens of a workgroup
  hipLaunchKernelGGL((paged_append_kernel<T, WPT>), dim3(static_cast<unsigned>((a.batch.tokens + PER - 1) / PER)),
                     dim3(kAppendWaves * kWave), 0, st, a);
  return mm::check_launch("paged_append");
}

// One wave to a token, or four where the tokens alone leave the device idle and a token is more than a wave's one round. us
// a call, one wave | four (heads q/k: tokens): 16/16 of 192: 500 tokens 12.9 | 7.8, 4000 31.8 | 34.0; 32/8 of 128: 128 tokens
// 6.8 | 5.4, 2000 12.4 | 14.8; 14/2 of 64: 64 tokens 4.8 | 4.8, 2549 6.5 | 12.0, 20000 23.4 | 68.0 (a token a workgroup
// before that, whose threads all waited for its position: 37.7 at 4000 tokens, 61.6 at 20000).
template <class T>
int launch_append(const AppendArgs& a, hipStream_t st) {
  const int64_t items = (a.nh + a.nkv) * static_cast<int64_t>(a.iph.d);
  return a.batch.tokens < 4 * mm::cu_count() && items > 2 * kWave ? launch_append<T, 4>(a, st) : launch_append<T, 1>(a, st);
}

// ------------------------------------------------------------------------------------------ checks on the host

constexpr int64_t kMaxTokens = 1 << 22, kMaxSeqs = 1 << 20, kMaxPages = (1LL << 31) - 1;
// positions of a stream, and rows (tokens times heads): 32-bit numbers of them stay positive with a tile or a piece added
constexpr int64_t kMaxKeys = 1LL << 30, kMaxRows = 1LL << 30;

// Rows that are written must not lie on each other: no stride of zero.
int check_rows(const char* what, const char* name, const mm_rows& r, int64_t tokens, int heads, int align, bool written = false) {
  const int64_t ts = r.token_stride, hs = r.head_stride;
  MM_REQUIRE(r.p, "%s: null %s", what, name);
  MM_REQUIRE((reinterpret_cast<uintptr_t>(r.p) & static_cast<uintptr_t>(align - 1)) == 0, "%s: %s must be %d-byte aligned",
             what, name, align);
  MM_REQUIRE((tokens == 1 || (ts >= 0 && ts % (align / 2) == 0)) && (heads == 1 || (hs >= 0 && hs % (align / 2) == 0)),
             "%s: strides of %s must keep rows %d-byte aligned", what, name, align);
  MM_REQUIRE(!written || ((tokens == 1 || ts > 0) && (heads == 1 || hs > 0)), "%s: rows of %s lie on each other", what, name);
  return MM_OK;
}

int check_shape(const char* what, int dtype, int nh, int nkv, int dqk, int dv) {
  MM_REQUIRE(dtype == MM_BF16 || dtype == MM_FP16, "%s: bf16 or fp16 tensors", what);
  MM_REQUIRE(nh >= 1 && nkv >= 1 && nh <= 4096 && nh % nkv == 0, "%s: nh=%d must be a multiple of nkv=%d, at most 4096",
             what, nh, nkv);
  MM_REQUIRE(dqk >= 8 && dqk <= 256 && dqk % 8 == 0, "%s: dqk=%d must be a multiple of 8 up to 256", what, dqk);
  MM_REQUIRE(dv >= 8 && dv <= 256 && dv % 8 == 0, "%s: dv=%d must be a multiple of 8 up to 256", what, dv);
  return MM_OK;
}

int check_tokens(const char* what, int64_t tokens, int64_t seqs) {
  MM_REQUIRE(tokens >= 0 && tokens <= kMaxTokens, "%s: bad number of tokens %lld", what, (long long)tokens);
  MM_REQUIRE(seqs >= 0 && seqs <= kMaxSeqs, "%s: bad number of streams %lld", what, (long long)seqs);
  return MM_OK;
}

int check_paged(const char* what, int nh, const mm_pages* g, const mm_batch* b, bool written) {
  int rc = check_shape(what, g->dtype, nh, g->nkv, g->dqk, g->dv);
  if (rc) return rc;
  if ((rc = check_tokens(what, b->tokens, b->seqs))) return rc;
  MM_REQUIRE(b->idx_dtype == MM_INT32 || b->idx_dtype == MM_INT64, "%s: indices must be int32 or int64", what);
  MM_REQUIRE(b->tokens * nh <= kMaxRows, "%s: tokens * nh must be at most 2^30", what);
  MM_REQUIRE(g->page >= 1 && g->n_pages >= 0 && g->n_pages <= kMaxPages && b->max_pages >= 0 && b->table_stride >= 0, "%s: bad page or table sizes", what);
  MM_REQUIRE(b->max_pages <= kMaxKeys / g->page, "%s: max_pages * page must be at most 2^30", what);
  MM_REQUIRE(b->seqs == 0 || (b->cu && b->kv_lens && (b->table || b->max_pages == 0)), "%s: null batch array", what);
  MM_REQUIRE(g->n_pages == 0 || (g->k && g->v), "%s: null pool", what);
  MM_REQUIRE(mm::aligned16(g->k) && mm::aligned16(g->v), "%s: the pool must be 16-byte aligned", what);
  const int64_t st[6] = {g->k_page_stride, g->k_head_stride, g->k_row_stride, g->v_page_stride, g->v_head_stride, g->v_row_stride};
  const int64_t dims[3] = {g->n_pages, g->nkv, g->page};
  for (int i = 0; i < 6; ++i)
    MM_REQUIRE(dims[i % 3] <= 1 || (st[i] >= (written ? 8 : 0) && st[i] % 8 == 0),
               written ? "%s: the pool's strides must be multiples of 8, not 0" : "%s: the pool's strides must be multiples of 8", what);
  return MM_OK;
}

Batch batch_of(const mm_pages& g, const mm_batch& b) {
  return Batch{b.cu, b.kv_lens, b.table, b.table_stride, b.idx_dtype == MM_INT64, static_cast<int>(b.seqs),
               static_cast<int>(b.tokens), static_cast<int>(b.max_pages * g.page)};
}

Rows rows_of(const mm_rows& r) { return Rows{static_cast<uint16_t*>(r.p), r.token_stride, r.head_stride}; }

bool same_rows(const mm_rows& a, const mm_rows& b) {
  return a.p == b.p && a.token_stride == b.token_stride && a.head_stride == b.head_stride;
}

void set_pool(const mm_pages& g, Pool& k, Pool& v) {
  k = Pool{static_cast<uint16_t*>(g.k), g.k_page_stride, g.k_head_stride, g.k_row_stride};
  v = Pool{static_cast<uint16_t*>(g.v), g.v_page_stride, g.v_head_stride, g.v_row_stride};
}

int attend(AttnArgs& a, int dtype, bool paged, float scale, void* workspace, int64_t workspace_bytes, hipStream_t st,
           const char* what) {
  const int64_t max_keys = paged ? a.batch.max_keys : a.batch.tokens;
  // 0 would turn the -infinity of a key that is not seen into NaN; this leaves every finite score at zero
  a.scale = scale == 0.f ? 1e-37f : fabsf(scale);
  a.negative = scale < 0.f;
  const AttnPlan p = plan_attn(paged, a.batch.tokens, a.batch.seqs, max_keys, a.nh, a.nkv, a.dqk, a.dv);
  MM_REQUIRE((p.blocks + p.target) * a.nkv < (1LL << 23), "%s: too many streams and rows for one launch", what);
  MM_REQUIRE(p.workspace == 0 || (workspace && mm::aligned16(workspace) && workspace_bytes >= p.workspace),
             "%s: a 16-byte aligned workspace of %lld bytes is needed", what, (long long)p.workspace);
  a.index = p.indexed ? static_cast<int4*>(workspace) : nullptr;
  a.ws = static_cast<float*>(workspace) + (p.indexed ? 4 * (a.batch.seqs + static_cast<int64_t>(1)) : 0);
  a.target = static_cast<int>(p.target);
  return p.many ? launch_many(a, p, dtype, paged, st, what) : launch_few(a, p, dtype, paged, st, what);
}

}  // namespace

extern "C" int mm_paged_version(void) { return MM_PAGED_VERSION; }

extern "C" int mm_paged_append(const mm_paged_append_args* g, void* stream) {
  const char* what = "paged_append";
  MM_REQUIRE(g, "%s: null arguments", what);
  int rc = check_paged(what, g->nh, &g->pages, &g->batch, true);
  if (rc) return rc;
  const int64_t pairs = g->inv_freq ? g->pairs : 0;
  const int rot_offset = g->inv_freq ? g->rot_offset : 0, nkv = g->pages.nkv;
  MM_REQUIRE(pairs >= 0 && pairs % 8 == 0 && rot_offset >= 0 && rot_offset % 8 == 0 && pairs <= kMaxPairs &&
                 rot_offset + 2 * pairs <= g->pages.dqk,
             "paged_append: %lld pairs from dim %d on do not fit a head of %d (multiples of 8)", (long long)pairs, rot_offset,
             g->pages.dqk);
  const int64_t N = g->batch.tokens;
  if (N == 0 || g->batch.seqs == 0) return MM_OK;
  if ((rc = check_rows(what, "q", g->q, N, g->nh, 16)) || (rc = check_rows(what, "k", g->k, N, nkv, 16)) ||
      (rc = check_rows(what, "v", g->v, N, nkv, 16)) || (rc = check_rows(what, "q_out", g->q_out, N, g->nh, 16, true)))
    return rc;
  if (g->k_out.p && (rc = check_rows(what, "k_out", g->k_out, N, nkv, 16, true))) return rc;
  AppendArgs a{};
  a.q = rows_of(g->q);
  a.k = rows_of(g->k);
  a.v = rows_of(g->v);
  a.q_out = rows_of(g->q_out);
  a.k_out = rows_of(g->k_out);
  set_pool(g->pages, a.kp, a.vp);
  a.batch = batch_of(g->pages, g->batch);
  a.page = fast_div(g->pages.page);
  a.n_pages = g->pages.n_pages;
  a.inv_freq = g->inv_freq;
  a.nh = g->nh;
  a.nkv = nkv;
  a.dqk = g->pages.dqk;
  a.dv = g->pages.dv;
  a.pairs = static_cast<int>(pairs);
  a.rot_offset = rot_offset;
  a.interleaved = g->interleaved != 0;
  a.iph = fast_div(a.pairs / 8 + (a.dqk - 2 * a.pairs) / 8);
  a.q_in_place = same_rows(g->q_out, g->q);
  a.k_in_place = g->k_out.p == nullptr || same_rows(g->k_out, g->k);
  return g->pages.dtype == MM_BF16 ? launch_append<BF16>(a, MM_STREAM(stream)) : launch_append<FP16>(a, MM_STREAM(stream));
}

extern "C" int64_t mm_paged_attn_workspace(int64_t tokens, int64_t seqs, int64_t max_keys, int nh, int nkv, int dqk, int dv,
                                           int at_most) {
  if (check_shape("paged_attn", MM_BF16, nh, nkv, dqk, dv) || check_tokens("paged_attn", tokens, seqs)) return -1;
  if (max_keys < 0 || max_keys > kMaxKeys) {
    mm::set_error(MM_ERR_ARG, "paged_attn: bad max_keys=%lld", (long long)max_keys);
    return -1;
  }
  return workspace_of(true, tokens, seqs, max_keys, nh, nkv, dqk, dv, at_most != 0);
}

extern "C" int mm_paged_attn(const mm_paged_attn_args* g, void* stream) {
  const char* what = "paged_attn";
  MM_REQUIRE(g, "%s: null arguments", what);
  int rc = check_paged(what, g->nh, &g->pages, &g->batch, false);
  if (rc) return rc;
  const int64_t N = g->batch.tokens;
  if (N == 0 || g->batch.seqs == 0) return MM_OK;
  if ((rc = check_rows(what, "q", g->q, N, g->nh, 16)) || (rc = check_rows(what, "out", g->out, N, g->nh, 8, true))) return rc;
  AttnArgs a{};
  a.q = rows_of(g->q);
  a.out = rows_of(g->out);
  set_pool(g->pages, a.kp, a.vp);
  a.batch = batch_of(g->pages, g->batch);
  a.page = fast_div(g->pages.page);
  a.group = fast_div(g->nh / g->pages.nkv);
  a.n_pages = static_cast<int>(g->pages.n_pages);
  a.nh = g->nh;
  a.nkv = g->pages.nkv;
  a.dqk = g->pages.dqk;
  a.dv = g->pages.dv;
  return attend(a, g->pages.dtype, true, g->scale, g->workspace, g->workspace_bytes, MM_STREAM(stream), what);
}

extern "C" int64_t mm_prompt_attn_workspace(int64_t tokens, int64_t seqs, int nh, int nkv, int dqk, int dv, int at_most) {
  if (check_shape("prompt_attn", MM_BF16, nh, nkv, dqk, dv) || check_tokens("prompt_attn", tokens, seqs)) return -1;
  return workspace_of(false, tokens, seqs, tokens, nh, nkv, dqk, dv, at_most != 0);
}

extern "C" int mm_prompt_attn(const mm_prompt_attn_args* g, void* stream) {
  const char* what = "prompt_attn";
  MM_REQUIRE(g, "%s: null arguments", what);
  const int64_t N = g->tokens;
  int rc = check_shape(what, g->dtype, g->nh, g->nkv, g->dqk, g->dv);
  if (rc) return rc;
  if ((rc = check_tokens(what, N, g->seqs))) return rc;
  MM_REQUIRE(g->idx_dtype == MM_INT32 || g->idx_dtype == MM_INT64, "%s: indices must be int32 or int64", what);
  MM_REQUIRE(g->cu || g->seqs == 0, "%s: null cu", what);
  MM_REQUIRE(N * g->nh <= kMaxRows, "%s: tokens * nh must be at most 2^30", what);
  if (N == 0 || g->seqs == 0) return MM_OK;
  if ((rc = check_rows(what, "q", g->q, N, g->nh, 16)) || (rc = check_rows(what, "k", g->k, N, g->nkv, 16)) ||
      (rc = check_rows(what, "v", g->v, N, g->nkv, 16)) || (rc = check_rows(what, "out", g->out, N, g->nh, 8, true)))
    return rc;
  AttnArgs a{};
  a.q = rows_of(g->q);
  a.k = rows_of(g->k);
  a.v = rows_of(g->v);
  a.out = rows_of(g->out);
  a.batch = Batch{g->cu, nullptr, nullptr, 0, g->idx_dtype == MM_INT64, static_cast<int>(g->seqs), static_cast<int>(N), 0};
  a.page = fast_div(1);
  a.group = fast_div(g->nh / g->nkv);
  a.nh = g->nh;
  a.nkv = g->nkv;
  a.dqk = g->dqk;
  a.dv = g->dv;
  return attend(a, g->dtype, false, g->scale, g->workspace, g->workspace_bytes, MM_STREAM(stream), what);
}
