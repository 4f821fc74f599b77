// What the kernels of the paged cache share: the batch on the device, page arithmetic, the arguments of an attention and
// the division of its work over workgroups.
#pragma once

#include "mingpaged.h"
#include "mm_common.h"

namespace mmp {

using namespace mmd;

// n / d for n < 2^31 by a multiplication: m = floor(2^(31 + l) / d) + 1 with l = ceil(log2 d) exceeds 2^(31 + l) / d by at
// most 1 <= 2^l / d, so the product is off by less than 1 / d for every such n.
struct FastDiv {
  uint32_t d, m;
  int s;
};

inline FastDiv fast_div(int64_t d) {
  FastDiv f{static_cast<uint32_t>(d), 0, 0};
  if (d > 1) {
    int l = 0;
    while ((1LL << l) < d) ++l;
    f.m = static_cast<uint32_t>((1ULL << (31 + l)) / static_cast<uint64_t>(d) + 1);
    f.s = l - 1;
  }
  return f;
}

__device__ __forceinline__ uint32_t div_by(uint32_t n, const FastDiv& f) {
  return f.d == 1 ? n : __umulhi(n, f.m) >> f.s;
}

// The batch as the kernels see it: device arrays of one index type, every value clamped before use, so that no content of
// them leads outside a buffer.
struct Batch {
  const void* cu;
  const void* lens;
  const void* table;
  int64_t table_stride;
  int i64;          // the arrays hold 64-bit numbers
  int seqs, tokens;
  int max_keys;     // max_pages * page
};

__device__ __forceinline__ int64_t idx_at(const void* p, int i64, int64_t i) {
  return i64 ? static_cast<const int64_t*>(p)[i] : static_cast<int64_t>(static_cast<const int32_t*>(p)[i]);
}

// An index as it came: both halves of a 64-bit entry, the same word twice of a 32-bit one. Nothing waits for it, or
// branches on its type, before it is used.
struct Index {
  uint32_t lo, hi;
};

__device__ __forceinline__ Index index_at(const void* p, int i64, int64_t i) {
  const uint32_t* w = static_cast<const uint32_t*>(p) + (i64 ? 2 * i : i);
  return Index{w[0], w[i64 ? 1 : 0]};
}

__device__ __forceinline__ int64_t value_of(Index x, int i64) {
  const int hi = static_cast<int>(i64 ? x.hi : static_cast<uint32_t>(static_cast<int>(x.lo) >> 31));
  return static_cast<int64_t>((static_cast<uint64_t>(static_cast<uint32_t>(hi)) << 32) | x.lo);
}

// A stream's first token, the number of its tokens and the rows of its cache that count (-1: outside the table).
struct Stream {
  int first, n, kv;
};

__device__ __forceinline__ Stream stream_at(const Batch& a, int b) {
  const Index i0 = index_at(a.cu, a.i64, b), i1 = index_at(a.cu, a.i64, b + 1);
  const Index ik = index_at(a.lens ? a.lens : a.cu, a.i64, b);
  const int64_t c0 = value_of(i0, a.i64), c1 = value_of(i1, a.i64), kv = value_of(ik, a.i64);
  Stream s;
  s.first = static_cast<int>(min(max(c0, static_cast<int64_t>(0)), static_cast<int64_t>(a.tokens)));
  s.n = static_cast<int>(min(max(c1, static_cast<int64_t>(s.first)), static_cast<int64_t>(a.tokens))) - s.first;
  s.kv = !a.lens ? s.n : kv < 0 || kv > a.max_keys ? -1 : static_cast<int>(kv);  // no lengths: a prompt's own rows
  return s;
}

// How many of the n entries of a rising sequence pass `before`, which the first of them do: 64 probes at a time, by the whole
// wave (of a sequence that does not rise, some number up to n).
template <class Before>
__device__ __forceinline__ int count_before(int n, Before before) {
  int lo = 0, hi = n;  // the answer lies in lo .. hi
  while (hi - lo > kWave) {
    const int step = (hi - lo + kWave - 1) / kWave, i = lo + (lane_id() + 1) * step - 1;
    const int passed = __popcll(__ballot(i < hi && before(min(i, hi - 1))));
    lo = min(lo + passed * step, hi);
    hi = min(lo + step, hi);
  }
  const int i = lo + lane_id();
  return lo + __popcll(__ballot(i < hi && before(min(i, n - 1))));
}

// The stream that token t belongs to (seqs: none), found by the whole wave: the number of streams that end at or before t.
__device__ __forceinline__ int stream_of_token(const Batch& a, int t) {
  return count_before(a.seqs, [&](int i) { return idx_at(a.cu, a.i64, i + 1) <= t; });
}

template <class T>
__device__ __forceinline__ void unpack8(const uint4& v, float (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (T::kBf16) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      x[2 * i] = f16_to_f32(static_cast<uint16_t>(w[i]));
      x[2 * i + 1] = f16_to_f32(static_cast<uint16_t>(w[i] >> 16));
    }
  }
}

typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));

// Two values rounded to nearest even, side by side: one instruction (converted one by one they take four).
template <class T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (T::kBf16) {
    const bf16x2_t v = {(__bf16)lo, (__bf16)hi};
    return __builtin_bit_cast(uint32_t, v);
  } else {
    const f16x2_t v = {(_Float16)lo, (_Float16)hi};
    return __builtin_bit_cast(uint32_t, v);
  }
}

// The larger, NaN where either is: one v_maximum3 for two of them, where fmaxf first quiets each operand that does not
// come out of an arithmetic instruction.
__device__ __forceinline__ float larger(float a, float b) { return __builtin_elementwise_maximum(a, b); }

template <class T>
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  return make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
}

__device__ __forceinline__ uint4 ld16(const uint16_t* p) { return *reinterpret_cast<const uint4*>(p); }
__device__ __forceinline__ void st16(uint16_t* p, const uint4& v) { *reinterpret_cast<uint4*>(p) = v; }

// Rows [tokens, heads, d] of a packed tensor, or one page's: element strides.
struct Rows {
  uint16_t* p;
  int64_t ts, hs;
  __device__ __forceinline__ uint16_t* at(int64_t t, int h) const { return p + t * ts + h * hs; }
};

struct Pool {
  uint16_t* p;
  int64_t ps, hs, rs;
  __device__ __forceinline__ uint16_t* at(int64_t page, int h, int row) const { return p + page * ps + h * hs + row * rs; }
};

// ------------------------------------------------------------------------------------------ attention

struct AttnArgs {
  Rows q, out;
  Rows k, v;    // a prompt's packed rows
  Pool kp, vp;  // the cache
  Batch batch;
  FastDiv page, group;  // group: query heads of a key / value head
  int n_pages;
  int nh, nkv, dqk, dv;
  float scale;       // its size; negative scales turn the queries' sign
  int negative;
  int target;        // pieces of the keys aimed at, 0: every row block takes all its keys at once
  float* ws;         // the pieces' states
  int4* index;       // where each stream's work begins (index_kernel), NULL: found anew by each wave
};

// How the work is divided. A row is one token's query at one of the G heads that share a key / value head (row r of a
// stream: token r / G, head r % G), so that a block of BR rows reads each key once for all of them. A stream of n tokens
// has ceil(n G / BR) row blocks, and where `target` > 0 a block's keys may be cut into pieces of up to `cut` granules of GR
// keys, one cut for the whole batch, so that a long stream among short ones is shared by many workgroups, each block's keys
// dealt evenly to its pieces. cut is at least the sum over all blocks of (granules / target). Only blocks of more than one
// piece keep states: ceil(x) <= 2 x for x > 1, so there are at most 2 target of them, a bound that needs no length on the
// host, as workgroups are at most target + blocks.
struct Work {
  int b, blk;      // stream (-1: none) and row block
  int piece;       // of the block's keys
  int cut;         // granules in a piece (0: all)
  int slot;        // state of the block's first piece
  Stream s;
};

template <int BR>
__device__ __forceinline__ int blocks_of(const Stream& s, int group) {
  return (s.n * group + BR - 1) / BR;
}

// Keys that the rows r0 .. r0 + BR - 1 of a stream see together (its rows end at n G), and the pieces they make.
template <int BR>
__device__ __forceinline__ int keys_of(const Stream& s, int blk, const FastDiv& group) {
  const int last = min(blk * BR + BR, s.n * static_cast<int>(group.d)) - 1;
  return s.kv < 0 ? 0 : max(0, s.kv - s.n + static_cast<int>(div_by(last, group)) + 1);
}

template <int GR>
__device__ __forceinline__ int pieces_of(int keys, int cut) {
  const int g = (keys + GR - 1) / GR;
  return cut == 0 ? 1 : max(1, (g + cut - 1) / cut);
}

// The keys begin .. end - 1 of a piece: the block's granules dealt out evenly, so that no piece is a small rest.
struct Range {
  int begin, end;
};
template <int GR>
__device__ __forceinline__ Range keys_of_piece(int keys, int pieces, int piece) {
  const int g = (keys + GR - 1) / GR, each = g / pieces, more = g - each * pieces;
  const int first = piece * each + min(piece, more);
  return Range{first * GR, min(keys, (first + each + (piece < more ? 1 : 0)) * GR)};
}

// Inclusive prefix sums over the wave: within rows of 16 lanes, then rows 0 and 2 into 1 and 3, then lane 31 into the
// upper half.
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr:1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast:31
  return v;
}

// The granules of a piece: as many pieces as target allows, counting half a piece a block for the rounding up of its own
// number; of many rows (a piece pays for its state of BR rows and the join) kMinCut granules at least. From the batch's
// granules times blocks, and its blocks.
constexpr int kMinCut = 4;

template <int BR, int GR>
__device__ __forceinline__ int cut_for(const AttnArgs& a, float total, float blocks) {
  const float target = static_cast<float>(a.target), aim = target - 0.5f * fminf(blocks, target);
  // rounded up by more than the sum over the lanes can lose, so that no cut gives more pieces than target
  const float cut = ceilf(total * 1.00001f / aim);
  return static_cast<int>(fminf(fmaxf(cut, static_cast<float>(BR < 128 ? 1 : kMinCut)), static_cast<float>((1 << 30) / GR)));
}

// What a stream adds to the two sums.
template <int BR, int GR>
__device__ __forceinline__ void add_stream(const AttnArgs& a, const Stream& s, double& total, float& blocks) {
  const int n = blocks_of<BR>(s, static_cast<int>(a.group.d));
  total += static_cast<double>(n) * ((max(s.kv, 0) + GR - 1) / GR);  // exact in each lane below 2^53
  blocks += static_cast<float>(n);
}

template <int BR, int GR, class Load>
__device__ __forceinline__ int cut_of(const AttnArgs& a, const Stream& mine, Load load) {
  double total = 0.;
  float blocks = 0.f;
  for (int base = 0; base < a.batch.seqs; base += kWave) {
    if (base) load(base);
    add_stream<BR, GR>(a, mine, total, blocks);
  }
  return cut_for<BR, GR>(a, wave_sum(static_cast<float>(total)), wave_sum(blocks));
}

// For many streams, what every wave of every workgroup would find by going through them all is written down first: the cut,
// then behind it for each stream the ends of its workgroups and of its cut blocks among all, and its first state. One
// workgroup, a stream a thread at a time: bound by the launch and two rounds of reads, 2.0 to 2.6 us at 96 to 256 streams.
template <int BR, int GR>
__global__ __launch_bounds__(1024) void index_kernel(AttnArgs a) {
  constexpr int NW = 1024 / kWave;
  __shared__ float s_total[NW], s_blocks[NW];
  __shared__ int s_ends[3][NW];
  const int tid = threadIdx.x, lane = lane_id(), wave = tid / kWave, B = a.batch.seqs;
  int cut = 0;
  if (a.target > 0) {
    double total = 0.;
    float blocks = 0.f;
    for (int b = tid; b < B; b += 1024) add_stream<BR, GR>(a, stream_at(a.batch, b), total, blocks);
    const float t = wave_sum(static_cast<float>(total)), n = wave_sum(blocks);
    if (lane == 0) {
      s_total[wave] = t;
      s_blocks[wave] = n;
    }
    __syncthreads();
    float all = 0.f, count = 0.f;
#pragma unroll
    for (int x = 0; x < NW; ++x) {
      all += s_total[x];
      count += s_blocks[x];
    }
    cut = cut_for<BR, GR>(a, all, count);
  }
  if (tid == 0) a.index[0] = make_int4(cut, 0, 0, 0);
  int before[3] = {0, 0, 0};  // of the streams already done: workgroups, cut blocks, states
  for (int base = 0; base < B; base += 1024) {
    Stream s{0, 0, 0};
    if (base + tid < B) s = stream_at(a.batch, base + tid);
    const int n = blocks_of<BR>(s, static_cast<int>(a.group.d)), p = pieces_of<GR>(max(s.kv, 0), cut);
    const int mine[3] = {n * p, p > 1 ? n : 0, p > 1 ? n * p : 0};
    int ends[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      ends[i] = wave_scan(mine[i]);
      if (lane == kWave - 1) s_ends[i][wave] = ends[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      ends[i] += before[i];
#pragma unroll
      for (int x = 0; x < NW; ++x) {
        const int v = s_ends[i][x];
        before[i] += v;
        if (x < wave) ends[i] += v;
      }
    }
    if (base + tid < B) a.index[base + tid + 1] = make_int4(ends[0], ends[1], ends[2] - mine[2], 0);
    __syncthreads();  // read before the next round writes
  }
}

template <int BR, int GR>
inline int launch_index(const AttnArgs& a, hipStream_t st, const char* what) {
  if (!a.index) return MM_OK;
  hipLaunchKernelGGL((index_kernel<BR, GR>), dim3(1), dim3(1024), 0, st, a);
  return mm::check_launch(what);
}

// The work of workgroup w (CUT: row block w of those that are cut, at most target of them), found by every wave from the
// batch itself, streams 64 at a time, one to a lane, or from the index. Within a stream the last row block, whose rows see
// the most keys, comes first.
template <int BR, int GR, bool CUT>
__device__ __forceinline__ Work find_work(const AttnArgs& a, int w) {
  const int G = static_cast<int>(a.group.d), lane = lane_id(), B = a.batch.seqs;
  Work k{-1, 0, 0, 0, 0, Stream{0, 0, 0}};
  Stream mine{0, 0, 0};
  auto load = [&](int base) {
    mine = Stream{0, 0, 0};
    if (base + lane < B) mine = stream_at(a.batch, base + lane);
  };
  if (a.index) {
    k.cut = a.index[0].x;
    const int b = count_before(B, [&](int i) { return (CUT ? a.index[i + 1].y : a.index[i + 1].x) <= w; });
    if (b >= B) return k;
    const int4 e = a.index[b + 1];
    k.s = stream_at(a.batch, b);
    const int nb = blocks_of<BR>(k.s, G), p = pieces_of<GR>(max(k.s.kv, 0), k.cut), units = CUT ? (p > 1 ? nb : 0) : nb * p;
    const int u = w - ((CUT ? e.y : e.x) - units), at = CUT ? u : u / p;
    k.blk = nb - 1 - at;
    k.piece = CUT ? 0 : u - at * p;
    k.slot = e.z + at * p;
    if (u >= 0 && u < units && (p == 1 || (k.slot >= 0 && k.slot + p <= 2 * a.target))) k.b = b;
    return k;
  }
  load(0);
  if (a.target > 0) {
    k.cut = cut_of<BR, GR>(a, mine, load);
    if (B > kWave) load(0);
  }
  int slots = 0;
  for (int base = 0; base < B; base += kWave) {
    if (base) load(base);
    const int blocks = blocks_of<BR>(mine, G), pieces = pieces_of<GR>(max(mine.kv, 0), k.cut);
    const int held = pieces > 1 ? blocks * pieces : 0, units = !CUT ? blocks * pieces : held ? blocks : 0;
    const int ends = wave_scan(units), last = __builtin_amdgcn_readlane(ends, kWave - 1);
    if (w < last) {
      const int src = __ffsll(static_cast<long long>(__ballot(ends > w))) - 1;
      const int held_before = wave_scan(held) - held;
      const int u = w - (__builtin_amdgcn_readlane(ends, src) - __builtin_amdgcn_readlane(units, src));
      const int p = __builtin_amdgcn_readlane(pieces, src), nb = __builtin_amdgcn_readlane(blocks, src);
      const int at = CUT ? u : u / p;
      k.b = base + src;
      k.s = Stream{__builtin_amdgcn_readlane(mine.first, src), __builtin_amdgcn_readlane(mine.n, src),
                   __builtin_amdgcn_readlane(mine.kv, src)};
      k.blk = nb - 1 - at;
      k.piece = CUT ? 0 : u - at * p;
      k.slot = slots + __builtin_amdgcn_readlane(held_before, src) + at * p;
      // always so for a cu that does not fall; one that does must not lead out of the buffers either
      if (u < 0 || at >= nb || (p > 1 && (k.slot < 0 || k.slot + p > 2 * a.target))) k.b = -1;
      return k;
    }
    w -= last;
    slots += __builtin_amdgcn_readlane(wave_scan(held), kWave - 1);
  }
  return k;
}

// find_work's answer as the scalars that it is: what follows branches on them, and a matrix instruction, which pays no heed
// to the lanes' mask, must stand behind scalar branches only.
__device__ __forceinline__ Work scalars(const Work& w) {
  auto u = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
  return Work{u(w.b), u(w.blk), u(w.piece), u(w.cut), u(w.slot), Stream{u(w.s.first), u(w.s.n), u(w.s.kv)}};
}

// A state: BR rows of dv sums, then the rows' maxima (in units of log2 of the weight), then their sums.
template <int BR>
__device__ __forceinline__ float* state_at(const AttnArgs& a, int slot, int kvh) {
  return a.ws + (static_cast<int64_t>(slot) * a.nkv + kvh) * BR * (a.dv + 2);
}

typedef float floatx16 __attribute__((ext_vector_type(16)));

template <class T>
struct Mfma;
template <>
struct Mfma<BF16> {
  typedef bf16x8_t V;
  static __device__ __forceinline__ floatx4 m16(const uint4& a, const uint4& b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ floatx16 m32(const uint4& a, const uint4& b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b), c, 0, 0, 0);
  }
  static constexpr uint32_t kExp = 0x7f807f80u;  // the exponents of a pair
};
template <>
struct Mfma<FP16> {
  typedef _Float16 V __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ floatx4 m16(const uint4& a, const uint4& b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ floatx16 m32(const uint4& a, const uint4& b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b), c, 0, 0, 0);
  }
  static constexpr uint32_t kExp = 0x7c007c00u;
};

// acc & kNotFinite says whether some pair accumulated by add_exponents held an infinity or a NaN: an exponent
// of ones and no other carries into its half's top bit.
template <class T>
__device__ __forceinline__ uint32_t add_exponents(uint32_t acc, uint32_t w) {
  constexpr uint32_t one = Mfma<T>::kExp & (~Mfma<T>::kExp << 1);  // the exponents' last bits
  return acc | ((w & Mfma<T>::kExp) + one);
}
template <class T>
__device__ __forceinline__ uint32_t add_exponents(uint32_t acc, const uint4& w) {
  return add_exponents<T>(add_exponents<T>(add_exponents<T>(add_exponents<T>(acc, w.x), w.y), w.z), w.w);
}
constexpr uint32_t kNotFinite = 0x80008000u;

// The page number of a key.
__device__ __forceinline__ Index page_id(const AttnArgs& a, int b, int key) {
  return index_at(a.batch.table, a.batch.i64, b * a.batch.table_stride + div_by(key, a.page));
}

__device__ __forceinline__ bool page_ok(const AttnArgs& a, Index id) {
  return static_cast<int>(id.lo) >= 0 && static_cast<int>(id.lo) < a.n_pages && (!a.batch.i64 || id.hi == 0);
}

// What a row that does not exist reads.
static __device__ const uint4 kZeroRow[32] = {};

// One row of a block over the keys k_begin .. k_end - 1 of its stream, key by key, by one wave: what the matrix units cannot
// do where a key that the row must not see holds an infinity or a NaN in its values (0 * inf). Few tiles can hold such a
// key at all (those that some rows of the block see and others do not), the kernels look into these, and rows of a block
// that met one are computed anew here. Lane l ends with the sums of dims l + 64 e.
struct RowSums {
  float acc[4], m, l;  // m in units of log2 of the weight
};

template <class T>
__device__ __forceinline__ RowSums row_by_keys(const AttnArgs& a, const Work& w, int kvh, int row, int k_begin, int k_end) {
  const int lane = lane_id(), i = static_cast<int>(div_by(row, a.group));
  const uint16_t* q = a.q.at(w.s.first + i, kvh * static_cast<int>(a.group.d) + row - i * static_cast<int>(a.group.d));
  const int end = min(k_end, w.s.kv - w.s.n + i + 1);
  const float sc = (a.negative ? -a.scale : a.scale) * 1.4426950408889634f;
  RowSums r{{0.f, 0.f, 0.f, 0.f}, -INFINITY, 0.f};
#pragma unroll 1
  for (int k0 = k_begin; k0 < end; k0 += kWave) {
    const int key = min(k0 + lane, end - 1);
    bool ok = k0 + lane < end;
    const uint16_t *kr, *vr;
    if (a.batch.table) {
      const Index id = page_id(a, w.b, key);
      ok = ok && page_ok(a, id);
      const int at = key - static_cast<int>(div_by(key, a.page)) * static_cast<int>(a.page.d);
      kr = a.kp.at(static_cast<int>(id.lo), kvh, at);
      vr = a.vp.at(static_cast<int>(id.lo), kvh, at);
    } else {
      kr = a.k.at(w.s.first + key, kvh);
      vr = a.v.at(w.s.first + key, kvh);
    }
    float s = 0.f;
    if (ok) {
#pragma unroll 1
      for (int d = 0; d < a.dqk; d += 8) {
        float x[8], y[8];
        unpack8<T>(ld16(kr + d), x);
        unpack8<T>(ld16(q + d), y);
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fmaf(x[e], y[e], s);
      }
    }
    s = ok ? s * sc : -INFINITY;
    const float mn = fmaxf(r.m, wave_max(s)), mu = mn == -INFINITY ? 0.f : mn;
    const float p = ok ? exp2_fast(s - mu) : 0.f, alpha = exp2_fast(r.m - mu);
    r.m = mn;
    r.l = fmaf(r.l, alpha, wave_sum(p));
#pragma unroll
    for (int e = 0; e < 4; ++e) r.acc[e] *= alpha;
    const uint64_t all = __ballot(ok), v = reinterpret_cast<uint64_t>(vr);
#pragma unroll 1
    for (int j = 0; j < kWave; ++j) {
      if (!((all >> j) & 1)) continue;
      const float pj = __shfl(p, j, kWave);
      const auto* vj = reinterpret_cast<const uint16_t*>((static_cast<uint64_t>(__shfl(static_cast<uint32_t>(v >> 32), j, kWave)) << 32) |
                                                         __shfl(static_cast<uint32_t>(v), j, kWave));
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (lane + kWave * e < a.dv) r.acc[e] = fmaf(pj, T::ld(vj, lane + kWave * e), r.acc[e]);
    }
  }
  return r;
}

// The rows first, first + step, .. of a block's `rows` by row_by_keys, into the outputs or, where the block is cut, into
// the piece's state.
template <class T, int BR>
__device__ __forceinline__ void rows_by_keys(const AttnArgs& a, const Work& w, int kvh, int rows, int first, int step, int k_begin,
                                             int k_end, float* state) {
  const int lane = lane_id(), G = static_cast<int>(a.group.d);
#pragma unroll 1
  for (int r = first; r < rows; r += step) {
    const int row = w.blk * BR + r, i = static_cast<int>(div_by(row, a.group));
    const RowSums s = row_by_keys<T>(a, w, kvh, row, k_begin, k_end);
    uint16_t* out = a.out.at(w.s.first + i, kvh * G + row - i * G);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int d = lane + kWave * e;
      if (d >= a.dv) break;
      if (state) state[r * a.dv + d] = s.acc[e];
      else T::st(out, d, s.m == -INFINITY ? 0.f : s.acc[e] / s.l);
    }
    if (state && lane == 0) {
      state[BR * a.dv + r] = s.m;
      state[BR * a.dv + BR + r] = s.l;
    }
  }
}

// What a call launches, a function of its sizes alone. Few rows to a block (16) or many (128); target: pieces of keys aimed
// at for the whole batch and one key / value head (0: no cutting, no join); blocks: the most row blocks that these sizes
// can have.
struct AttnPlan {
  bool many, indexed;
  int groups;  // of four waves in a workgroup of many rows
  int64_t blocks, target, workspace;
};
AttnPlan plan_attn(bool paged, int64_t tokens, int64_t seqs, int64_t max_keys, int nh, int nkv, int dqk, int dv);
// Its workspace, or with at_most the most that any call of at most these tokens, streams and keys takes.
int64_t workspace_of(bool paged, int64_t tokens, int64_t seqs, int64_t max_keys, int nh, int nkv, int dqk, int dv, bool at_most);
int launch_few(const AttnArgs& a, const AttnPlan& p, int dtype, bool paged, hipStream_t st, const char* what);
int launch_many(const AttnArgs& a, const AttnPlan& p, int dtype, bool paged, hipStream_t st, const char* what);
int launch_join_many(const AttnArgs& a, const AttnPlan& p, int dtype, hipStream_t st, const char* what);

}  // namespace mmp
