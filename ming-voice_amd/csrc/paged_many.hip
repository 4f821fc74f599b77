// Attention of many rows (prompts and their pieces): 128 rows to a workgroup whose waves share every key and value tile in
// LDS.
#include "paged_common.h"

namespace mmp {

namespace {

constexpr int kKeys = 64;   // keys per tile
constexpr int kWaves = 4;    // waves of a group: one group shares a tile
constexpr int kRows = 32;   // rows per wave

// The shape of many_kernel: head dims up to 64 KS (q, k) and 64 VS (v). A tile lies in LDS as pieces of 64 keys by 64 dims,
// 8 KB each: every load instruction then fills 8 rows of 128 bytes, whatever the head dims are.
template <int KS, int VS, int NG>
struct Many {
  static constexpr int BR = kWaves * kRows;
  static constexpr int THREADS = NG * kWaves * kWave;
  static constexpr int GR = kKeys;
  static constexpr int PIECE = kKeys * 128;  // bytes
  static constexpr int K_BYTES = KS * PIECE, V_BYTES = VS * PIECE;
  static_assert(2 * NG * (K_BYTES + V_BYTES) <= 160 * 1024, "tile shape");
};

// The chunk of a piece's row held at LDS place c of the row (involutions). Keys: the 16 rows that a fragment reads at one
// chunk fall on the 16 distinct 16-byte columns of the banks; values: the 4 rows of which 32 lanes of a transposing read
// take 64 bytes each fall on distinct quarters.
__device__ __forceinline__ int k_swizzle(int row, int c) { return c ^ ((row >> 1) & 7); }
__device__ __forceinline__ int v_swizzle(int row, int c) { return c ^ (4 * ((row >> 1) & 1)); }

// 8 keys of a 32-dim tile of V^T as the 32x32x16 MFMA takes them: 4 rows from place p on and the 4 rows `hi` bytes on, each
// read transposed (lane layout: lds_tr4x2). By the builtin: the waits are the compiler's.
__device__ __forceinline__ uint4 v_frag(const char* p, int hi) {
  typedef __attribute__((address_space(3))) s16x4_t* lds4_t;
  const s16x4_t a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4_t)(p));
  const s16x4_t b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4_t)(p + hi));
  const uint2 x = __builtin_bit_cast(uint2, a), y = __builtin_bit_cast(uint2, b);
  return make_uint4(x.x, x.y, y.x, y.y);
}

// Max over the two lanes that share lane % 32.
__device__ __forceinline__ float half_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), true, false);
  return larger(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// Where a tile's rows come from, chosen on the host (launch_type).
enum Source { kPacked, kPaged, kAnywhere };

// Softmax attention of 128 rows over a piece of their keys (all of them, where the batch is not cut), one pass with a
// running maximum and sum. Grid (work x key / value heads) x NG groups of 4 waves; a wave holds 32 rows, a group goes
// through 64 keys at a time, which its waves share in LDS, and two groups take every other tile and join their states in LDS
// at the end. Per tile and wave, on the 32x32x16 MFMA (bf16 or fp16, fp32 sums):
//   S^T [64 keys, 32 rows] = K Q^T: key rows as A fragments from LDS, the queries held as B fragments;
//   a lane of S^T holds 32 keys of row lane % 32, so that maximum, exponentials and sum need one exchange, with lane ^ 32;
//   O^T [dv, 32 rows] += V^T P^T: P^T straight from the S^T registers (slot j of step st is the key of S^T register 8 (st % 2)
//     + j, whichever that is, for both operands alike), the weights rounded to the cache's type, the matrix units' operand
//     (half a step, 2^-9 of a weight in bf16); V^T by transposing LDS reads.
// The running maximum follows a tile's only when it rises by more than 2^8 in weight: the sums of a row then stay below 2^8
// times their final size, far inside fp32 and inside fp16's and bf16's weights, and O is seldom rescaled.
// A tile comes by loads straight into LDS while the tile before is computed: one barrier a tile, after which the wave
// requests its part of the next one (8 rows by 128 bytes an instruction). Swizzles keep every LDS read free of bank
// conflicts (SQ_LDS_BANK_CONFLICT 0). All key fragments are read before the first product and all value fragments before
// the softmax, so that neither waits for LDS.
// Bound at 128 dims by how far matrix and vector work of the two workgroups of a CU overlap: 8192 tokens of 32/8 heads (550
// GFLOP of pairs that count) 549 us, 1.0 PFLOP/s, where the 8192^3 product runs at 1.15; the matrix units are busy 55 % of the
// cycles, the vector units 50 %. At 64 dims by the issue of instructions, one a wave in four cycles whatever its kind, of which
// the products are the least: 12 Talker prompts of 5 to 2000 tokens 32 us (353 TFLOP/s), 4000 tokens 50. So a tile's page
// arithmetic is kept short (pieces of 100 to 500 tokens of 32/8 heads behind 611 to 5000 positions 85.6 -> 82.0 us on the GPU).
// On the way there (8192 tokens): 932 us with rows brought by ds_bpermute and fragments read one by one; 673 with 64-dim
// pieces, one page to a load and the not-finite code out of the loop; 616 with the key fragments ahead, 588 with the value
// fragments too; 560 with one instruction to a pair of weights and to two of a maximum. Not kept: s_setprio around the
// products (588 -> 600), exponentials dealt out between the products (627), for 256 dims the value fragments ahead (spills);
// at 64 dims (2000 Talker tokens, 26.8 us) the last tile's value products under this tile's softmax (27.6), the next tile's
// scores as well (33), tiles requested two ahead (28.2), or behind the scores (27.7), the weights summed by a matrix
// instruction (27.1).
template <class T, int KS, int VS, int NG, int SRC>
__global__ __launch_bounds__(NG * kWaves * kWave, KS <= 3 ? 2 : 1) void many_kernel(AttnArgs a) {
  using P = Many<KS, VS, NG>;
  constexpr int BR = P::BR, NK = 4 * KS, ND = 2 * VS;
  // two buffers, each an object of its own: reads of one then need not wait for the loads in flight into the other
  __shared__ __align__(1024) char s_k0[NG * P::K_BYTES], s_v0[NG * P::V_BYTES], s_k1[NG * P::K_BYTES], s_v1[NG * P::V_BYTES];
  const int tid = threadIdx.x, lane = lane_id();
  const int all_wave = __builtin_amdgcn_readfirstlane(tid / kWave), wave = all_wave % kWaves, group = all_wave / kWaves;
  const int lr = lane & 31, lh = lane >> 5, G = static_cast<int>(a.group.d);
  const int unit = static_cast<int>(blockIdx.x) / a.nkv, kvh = static_cast<int>(blockIdx.x) - unit * a.nkv;
  const Work w = scalars(find_work<BR, P::GR, false>(a, unit));
  if (w.b < 0) return;
  const int r0 = w.blk * BR, rows = min(BR, w.s.n * G - r0);
  auto out_at = [&](int r) {  // row r0 + r of the stream
    const int i = static_cast<int>(div_by(r0 + r, a.group));
    return a.out.at(w.s.first + i, kvh * G + (r0 + r - i * G));
  };
  if (w.s.kv < 0) {
    for (int i = tid; i < rows * a.dv; i += P::THREADS) T::st(out_at(i / a.dv), i % a.dv, NAN);
    return;
  }
  const int keys = keys_of<BR>(w.s, w.blk, a.group), pieces = pieces_of<P::GR>(keys, w.cut);
  if (w.piece >= pieces) return;
  const Range part = keys_of_piece<P::GR>(keys, pieces, w.piece);
  const int k_begin = part.begin, k_end = part.end;
  const int tiles = (k_end - k_begin + kKeys - 1) / kKeys;  // group g takes tiles g, g + NG, ..
  const int ctx = w.s.kv - w.s.n;

  // A wave fills rows 8 wave .. + 7 and 32 + 8 wave .. + 7 of each piece, lane l row l / 8 of them at LDS place l % 8.
  const int lrow = lane / 8, kdim = 8 * k_swizzle(8 * wave + lrow, lane % 8), vdim = 8 * v_swizzle(8 * wave + lrow, lane % 8);
  uint64_t there = 0;  // the tile's keys that exist
  // kPacked, kPaged: the 8 rows of a load lie side by side, in one page: a buffer resource from the first of them to the end
  // of the last that exists; dims past the head's end lie past every resource
  const uint32_t krs = static_cast<uint32_t>(SRC == kPacked ? a.k.ts : a.kp.rs) * 2u, vrs = static_cast<uint32_t>(SRC == kPacked ? a.v.ts : a.vp.rs) * 2u;
  const uint32_t koff = lrow * krs + 2u * kdim, voff = lrow * vrs + 2u * vdim;
  // kAnywhere: lane l finds key l's rows and hands them to the loading lanes
  const char* zeros = reinterpret_cast<const char*>(kZeroRow);
  const char *kr = zeros, *vr = zeros;
  auto row_of = [&](const char* p, int r) {
    const uint64_t v = reinterpret_cast<uint64_t>(p);
    const uint32_t lo = static_cast<uint32_t>(__builtin_amdgcn_ds_bpermute(4 * r, static_cast<int>(v)));
    const uint32_t hi = static_cast<uint32_t>(__builtin_amdgcn_ds_bpermute(4 * r, static_cast<int>(v >> 32)));
    return reinterpret_cast<const char*>((static_cast<uint64_t>(hi) << 32) | lo);
  };
  // the page numbers of a tile: of key l (kAnywhere), of keys 8 (l % 8) .. + 7 (kPaged; pages of 8 rows or more, so that the
  // offset in a table's row fits 32 bits and the divisor is not 1)
  auto page_of = [&](int key) { return __umulhi(static_cast<uint32_t>(key), a.page.m) >> a.page.s; };
  const char* pages = SRC == kPaged ? static_cast<const char*>(a.batch.table) + w.b * a.batch.table_stride * (a.batch.i64 ? 8 : 4) : nullptr;
  auto ids_of = [&](int it) {
    const int key = min(k_begin + it * kKeys + (SRC == kAnywhere ? lane : 8 * (lane % 8)), k_end - 1);
    if (SRC == kPacked || (SRC == kAnywhere && !a.batch.table)) return Index{0, 0};
    if (SRC == kAnywhere) return page_id(a, w.b, key);
    const auto* at = reinterpret_cast<const uint32_t*>(pages + (page_of(key) << (a.batch.i64 ? 3 : 2)));
    Index id{at[0], 0};
    if (a.batch.i64) id.hi = at[1];
    return id;
  };
  const char *kpk = nullptr, *vpk = nullptr;  // kPacked: the wave's first row of the tile to load
  if constexpr (SRC == kPacked) {
    kpk = reinterpret_cast<const char*>(a.k.at(w.s.first + k_begin + kKeys * group + 8 * wave, kvh));
    vpk = reinterpret_cast<const char*>(a.v.at(w.s.first + k_begin + kKeys * group + 8 * wave, kvh));
  }
  // kPaged: the head's first page, its rows and 16-byte units from page to page
  const char *kbase = reinterpret_cast<const char*>(a.kp.at(0, kvh, 0)), *vbase = reinterpret_cast<const char*>(a.vp.at(0, kvh, 0));
  const uint32_t kps = static_cast<uint32_t>(a.kp.ps >> 3), vps = static_cast<uint32_t>(a.vp.ps >> 3);
  const uint32_t kfull = 7 * krs + 2 * a.dqk, vfull = 7 * vrs + 2 * a.dv;  // 8 rows
  auto load_tile = [&](int it, Index id, char* kt, char* vt) {
    const int j0 = k_begin + it * kKeys, left = k_end - j0;  // keys of the tile and behind
    if constexpr (SRC == kAnywhere) {
      const int key = min(j0 + lane, k_end - 1);
      bool ok = lane < left;
      if (a.batch.table) {
        ok = ok && page_ok(a, id);
        const int row = key - static_cast<int>(div_by(key, a.page)) * static_cast<int>(a.page.d);
        kr = reinterpret_cast<const char*>(a.kp.at(static_cast<int>(id.lo), kvh, row));
        vr = reinterpret_cast<const char*>(a.vp.at(static_cast<int>(id.lo), kvh, row));
      } else {
        kr = reinterpret_cast<const char*>(a.k.at(w.s.first + key, kvh));
        vr = reinterpret_cast<const char*>(a.v.at(w.s.first + key, kvh));
      }
      if (!ok) kr = vr = zeros;
      there = __ballot(ok);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = 32 * i + 8 * wave;  // the load's first row
        const char *kp = row_of(kr, r + lrow) + 2 * kdim, *vp = row_of(vr, r + lrow) + 2 * vdim;
#pragma unroll
        for (int s = 0; s < KS; ++s) load_lds16(kdim + 64 * s < a.dqk ? kp + 128 * s : zeros, kt + r * 128 + s * P::PIECE);
#pragma unroll
        for (int s = 0; s < VS; ++s) load_lds16(vdim + 64 * s < a.dv ? vp + 128 * s : zeros, vt + r * 128 + s * P::PIECE);
      }
    } else {
      there = left >= kKeys ? ~0ull : (1ull << left) - 1;
      if constexpr (SRC == kPaged) {
        uint32_t bad = static_cast<uint32_t>(__ballot(!page_ok(a, id))) & 0xffu;  // by groups of 8 keys
        while (bad) {
          const int g = __builtin_ctz(bad);
          bad &= bad - 1;
          there &= ~(0xffull << (8 * g));
        }
      }
      // the 8 rows from r on, of which n exist (scalar instructions, as many as the wave's vector ones: a whole tile skips
      // what only the others need)
      auto load_rows = [&](int i, int n, uint32_t kbytes, uint32_t vbytes) {
        const int r = 32 * i + 8 * wave;
        const char *kb, *vb;
        if constexpr (SRC == kPaged) {
          const uint32_t page = n ? __builtin_amdgcn_readlane(id.lo, 4 * i + wave) : 0;
          const uint32_t row = (j0 + r) - page_of(j0 + r) * a.page.d;
          kb = kbase + (static_cast<uint64_t>(page) * kps << 4) + row * krs;
          vb = vbase + (static_cast<uint64_t>(page) * vps << 4) + row * vrs;
        } else {
          kb = kpk + 32 * i * static_cast<int64_t>(krs);
          vb = vpk + 32 * i * static_cast<int64_t>(vrs);
        }
        const rsrc_t kres = make_rsrc(kb, kbytes), vres = make_rsrc(vb, vbytes);
#pragma unroll
        for (int s = 0; s < KS; ++s) buf_lds16(kres, kdim + 64 * s < a.dqk ? koff + 128u * s : kPast, kt + r * 128 + s * P::PIECE);
#pragma unroll
        for (int s = 0; s < VS; ++s) buf_lds16(vres, vdim + 64 * s < a.dv ? voff + 128u * s : kPast, vt + r * 128 + s * P::PIECE);
      };
      if (there == ~0ull) {
#pragma unroll
        for (int i = 0; i < 2; ++i) load_rows(i, 8, kfull, vfull);
      } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int r = 32 * i + 8 * wave, n = (there >> r) & 1 ? min(8, left - r) : 0;
          load_rows(i, n, n ? (n - 1) * krs + 2 * a.dqk : 0, n ? (n - 1) * vrs + 2 * a.dv : 0);
        }
      }
    }
    if constexpr (SRC == kPacked) {
      kpk += NG * kKeys * static_cast<int64_t>(krs);
      vpk += NG * kKeys * static_cast<int64_t>(vrs);
    }
  };

  // this wave's rows and what they see
  const int wr0 = r0 + kRows * wave;                         // the wave's first row
  const int wrows = max(0, min(kRows, rows - kRows * wave));
  const int my_row = min(wr0 + lr, r0 + rows - 1);
  const int my_i = static_cast<int>(div_by(my_row, a.group));
  const int lim = ctx + my_i + 1;
  const int lim_min = ctx + static_cast<int>(div_by(wr0, a.group)) + 1;  // keys that each of the wave's rows sees
  const int lim_max = wrows ? ctx + static_cast<int>(div_by(wr0 + wrows - 1, a.group)) + 1 : 0;
  const int lim_block = ctx + static_cast<int>(div_by(r0, a.group)) + 1;  // each row of the workgroup
  uint4 qf[NK];
  {
    const uint16_t* qrow = a.q.at(w.s.first + my_i, kvh * G + (my_row - my_i * G));
    const uint32_t sign = a.negative ? 0x80008000u : 0u;
#pragma unroll
    for (int ks = 0; ks < NK; ++ks) {
      const int d = 16 * ks + 8 * lh;
      const bool ok = d < a.dqk;
      const uint4 x = and_mask16(ld16(qrow + (ok ? d : 0)), ok);
      qf[ks] = make_uint4(x.x ^ sign, x.y ^ sign, x.z ^ sign, x.w ^ sign);
    }
  }
  // this lane's places in a piece: key row 32 u + lr, chunk 2 (ks % 4) + lh; value rows 16 st + 4 lh + (lane % 16) / 4
  // (+ 8), dims 32 (dt % 2) + 16 ((lane / 16) % 2) + 4 (lane % 4) .. + 3
  const int kplace = lr * 128 + k_swizzle(lr, lh) * 16;
  const int vfr = 4 * lh + (lane & 15) / 4;
  const int vplace = vfr * 128 + v_swizzle(vfr, 2 * ((lane >> 4) & 1) + (lane & 3) / 2) * 16 + (lane & 1) * 8;
  floatx16 o[ND];
  float m = -INFINITY, l = 0.f;
#pragma unroll
  for (int dt = 0; dt < ND; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[dt][i] = 0.f;
  const float sc = a.scale * 1.4426950408889634f;

  uint32_t seen = 0;  // exponents of values that some row must not meet
  Index next{0, 0};
  auto tile = [&](int it, char* kt, char* vt, char* kt_next, char* vt_next) {
    const int j0 = k_begin + it * kKeys;
    const uint64_t mine = there;
    wait_vmcnt<0>();  // this wave's part of the tile
    __syncthreads();  // every wave's part; and the other buffer has been read
    if (it + NG < tiles) {
      const Index id = next;
      next = ids_of(it + 2 * NG);
      load_tile(it + NG, id, kt_next, vt_next);
    }
    if (NG > 1 && it >= tiles) return;  // the other group's last tile
    if (j0 + kKeys > lim_block) {  // some row does not see some key: its value must be finite, or 0 * inf reaches the row
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int s = 0; s < VS; ++s) {
          const uint4 x = *reinterpret_cast<const uint4*>(vt + s * P::PIECE + (32 * i + 8 * wave) * 128 + lane * 16);
          seen = add_exponents<T>(seen, x);
        }
    }
    if (j0 < lim_max) {
      floatx16 s[2];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[u][i] = 0.f;
      constexpr int AHEAD = KS <= 2 ? NK : 4;  // k steps whose fragments are read before the first product
#pragma unroll
      for (int k0 = 0; k0 < NK; k0 += AHEAD) {
        uint4 kx[2][AHEAD];
#pragma unroll
        for (int ks = 0; ks < AHEAD; ++ks)
#pragma unroll
          for (int u = 0; u < 2; ++u)
            kx[u][ks] = *reinterpret_cast<const uint4*>(kt + ((k0 + ks) / 4) * P::PIECE + u * 4096 + (kplace ^ (32 * (ks % 4))));
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int ks = 0; ks < AHEAD; ++ks)
#pragma unroll
          for (int u = 0; u < 2; ++u) s[u] = Mfma<T>::m32(kx[u][ks], qf[k0 + ks], s[u]);
      }
      // the value fragments too, before the softmax (where they fit: 8 KB a tile and 64 dims, 4 registers a fragment)
      constexpr bool EARLY = KS <= 3;
      uint4 vf[4][ND];
      if constexpr (EARLY) {
#pragma unroll
        for (int st = 0; st < 4; ++st)
#pragma unroll
          for (int dt = 0; dt < ND; ++dt)
            vf[st][dt] = v_frag(vt + (dt / 2) * P::PIECE + (vplace ^ (64 * (dt % 2))) + 16 * st * 128, 8 * 128);
        __builtin_amdgcn_sched_barrier(0);
      }
      uint64_t sees = ~0ull;
      if (j0 + kKeys > lim_min || mine != ~0ull) {  // s[u][i]: key 32 u + 8 (i / 4) + 4 lh + i % 4
        const int n = lim - j0;
        sees = n >= kKeys ? mine : n <= 0 ? 0 : mine & ((1ull << n) - 1);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const uint32_t bits = static_cast<uint32_t>(sees >> (32 * u)) >> (4 * lh);
#pragma unroll
          for (int i = 0; i < 16; ++i) s[u][i] = (bits >> (8 * (i / 4) + i % 4)) & 1u ? s[u][i] : -INFINITY;
        }
      }
      float tmax = larger(s[0][0], s[1][0]);
#pragma unroll
      for (int i = 1; i < 16; ++i) tmax = larger(larger(tmax, s[0][i]), s[1][i]);
      tmax = half_max(tmax);
      if (__any((tmax - m) * sc > 8.f)) {  // the sums stay below 2^8 of a weight of one: no need to follow every rise
        const float mn = fmaxf(m, tmax), mu = mn == -INFINITY ? 0.f : mn;
        const float alpha = exp2_fast((m - mu) * sc);
        m = mn;
        l *= alpha;
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) o[dt] *= alpha;
      }
      const float shift = m == -INFINITY ? 0.f : m * sc;
      uint4 pf[4];
#pragma unroll
      for (int st = 0; st < 4; ++st) {
        uint32_t pw[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = 8 * (st & 1) + 2 * e;
          const float p0 = exp2_fast(fmaf(s[st / 2][i], sc, -shift)), p1 = exp2_fast(fmaf(s[st / 2][i + 1], sc, -shift));
          l += p0 + p1;
          pw[e] = pack2<T>(p0, p1);
        }
        pf[st] = make_uint4(pw[0], pw[1], pw[2], pw[3]);
      }
#pragma unroll
      for (int st = 0; st < 4; ++st)
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) {
          if constexpr (!EARLY) vf[st][dt] = v_frag(vt + (dt / 2) * P::PIECE + (vplace ^ (64 * (dt % 2))) + 16 * st * 128, 8 * 128);
          o[dt] = Mfma<T>::m32(vf[st][dt], pf[st], o[dt]);
        }
    }
  };
  char *k0 = s_k0 + group * P::K_BYTES, *v0 = s_v0 + group * P::V_BYTES, *k1 = s_k1 + group * P::K_BYTES, *v1 = s_v1 + group * P::V_BYTES;
  if (group < tiles) {
    const Index id = ids_of(group);
    next = ids_of(group + NG);
    load_tile(group, id, k0, v0);
  }
  for (int it = 0; it < tiles; it += 2 * NG) {
    tile(it + group, k0, v0, k1, v1);
    if (it + NG < tiles) tile(it + NG + group, k1, v1, k0, v0);
  }
  float* state = pieces > 1 ? state_at<BR>(a, w.slot + w.piece, kvh) : nullptr;
  // whether any wave met such a value: in words of the key buffer, which is no longer needed
  __syncthreads();
  int* met = reinterpret_cast<int*>(s_k0);
  const bool mine_met = __any((seen & kNotFinite) != 0);
  if (lane == 0) met[all_wave] = mine_met;
  __syncthreads();
  int any_met = 0;
#pragma unroll
  for (int x = 0; x < NG * kWaves; ++x) any_met |= met[x];
  if (__builtin_amdgcn_readfirstlane(any_met)) {
    rows_by_keys<T, BR>(a, w, kvh, rows, all_wave, NG * kWaves, k_begin, k_end, state);
    return;
  }
  l += __shfl_xor(l, 32, kWave);
  if constexpr (NG == 2) {
    // the second group's state to the first, a fragment's register of all lanes side by side: 16 KB of sums per 32 dims,
    // the first in one buffer, the rest in the other
    constexpr int HALF = ND / 2;
    static_assert(HALF * 16 * 1024 <= NG * P::V_BYTES, "room");
    __syncthreads();
    float* ml = reinterpret_cast<float*>(s_k0) + wave * 2 * kWave + lane;
    auto sums = [&](int dt) {
      return reinterpret_cast<float*>(dt < HALF ? s_v0 : s_v1) + ((dt % HALF) * kWaves + wave) * 16 * kWave + lane;
    };
    if (group == 1) {
      ml[0] = m;
      ml[kWave] = l;
#pragma unroll
      for (int dt = 0; dt < ND; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) sums(dt)[i * kWave] = o[dt][i];
    }
    __syncthreads();
    if (group == 1) return;
    const float m1 = ml[0], mn = fmaxf(m, m1), mu = mn == -INFINITY ? 0.f : mn;
    const float a0 = exp2_fast((m - mu) * sc), a1 = exp2_fast((m1 - mu) * sc);
    m = mn;
    l = l * a0 + ml[kWave] * a1;
#pragma unroll
    for (int dt = 0; dt < ND; ++dt)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[dt][i] = fmaf(sums(dt)[i * kWave], a1, o[dt][i] * a0);
  }
  if (lr >= wrows) return;
  const int r = kRows * wave + lr;  // of the workgroup
  if (state) {
#pragma unroll
    for (int dt = 0; dt < ND; ++dt)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const int d = 32 * dt + 8 * (i / 4) + 4 * lh;
        if (d < a.dv) *reinterpret_cast<floatx4*>(state + r * a.dv + d) = floatx4{o[dt][i], o[dt][i + 1], o[dt][i + 2], o[dt][i + 3]};
      }
    if (lh == 0) {
      state[BR * a.dv + r] = m == -INFINITY ? m : m * sc;
      state[BR * a.dv + BR + r] = l;
    }
    return;
  }
  const float inv = m == -INFINITY ? 0.f : 1.f / l;
  uint16_t* out = out_at(r);
#pragma unroll
  for (int dt = 0; dt < ND; ++dt)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const int d = 32 * dt + 8 * (i / 4) + 4 * lh;
      if (d < a.dv)
        *reinterpret_cast<uint2*>(out + d) = make_uint2(pack2<T>(o[dt][i] * inv, o[dt][i + 1] * inv), pack2<T>(o[dt][i + 2] * inv, o[dt][i + 3] * inv));
    }
}

template <class T, int KS, int VS, int NG, int SRC>
int launch_shape(const AttnArgs& a, const AttnPlan& p, hipStream_t st, const char* what) {
  using P = Many<KS, VS, NG>;
  int rc = launch_index<P::BR, P::GR>(a, st, what);
  if (rc) return rc;
  hipLaunchKernelGGL((many_kernel<T, KS, VS, NG, SRC>), dim3(static_cast<unsigned>((p.blocks + p.target) * a.nkv)),
                     dim3(NG * kWaves * kWave), 0, st, a);
  return mm::check_launch(what);
}

template <class T, int KS, int VS, int SRC>
int launch_groups(const AttnArgs& a, const AttnPlan& p, hipStream_t st, const char* what) {
  return p.groups == 2 ? launch_shape<T, KS, VS, 2, SRC>(a, p, st, what) : launch_shape<T, KS, VS, 1, SRC>(a, p, st, what);
}

template <class T, int SRC>
int launch_source(const AttnArgs& a, const AttnPlan& p, hipStream_t st, const char* what) {
  if (a.dqk <= 64 && a.dv <= 64) return launch_groups<T, 1, 1, SRC>(a, p, st, what);
  if (a.dqk <= 128 && a.dv <= 128) return launch_groups<T, 2, 2, SRC>(a, p, st, what);
  if (a.dqk <= 192 && a.dv <= 128) return launch_groups<T, 3, 2, SRC>(a, p, st, what);
  return launch_shape<T, 4, 4, 1, SRC>(a, p, st, what);
}

// Packed rows, and pages of a multiple of 8 rows, are read 8 rows to an instruction through a resource that ends with them
// (a resource reaches 2^31 bytes, and addresses are counted in 32 bits: bytes within a page's head, 16-byte units from page
// to page); other pages, and rows further apart, row by row from wherever they lie.
template <class T>
int launch_type(const AttnArgs& a, const AttnPlan& p, bool paged, hipStream_t st, const char* what) {
  const int64_t far = 1 << 26;  // elements between rows: 8 of them stay below 2^31 bytes
  auto pool_near = [&](const Pool& x) {
    return x.rs < far && static_cast<int64_t>(a.page.d) * x.rs < (1LL << 31) && (a.n_pages <= 1 || x.ps < (1LL << 35));
  };
  const bool near = paged ? a.page.d % 8 == 0 && pool_near(a.kp) && pool_near(a.vp) : a.k.ts < far && a.v.ts < far;
  if (!near) return launch_source<T, kAnywhere>(a, p, st, what);
  return paged ? launch_source<T, kPaged>(a, p, st, what) : launch_source<T, kPacked>(a, p, st, what);
}

}  // namespace

int launch_many(const AttnArgs& a, const AttnPlan& p, int dtype, bool paged, hipStream_t st, const char* what) {
  int rc = dtype == MM_BF16 ? launch_type<BF16>(a, p, paged, st, what) : launch_type<FP16>(a, p, paged, st, what);
  if (rc || p.target == 0) return rc;
  return launch_join_many(a, p, dtype, st, what);
}

}  // namespace mmp
