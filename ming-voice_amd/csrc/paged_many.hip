// Attention of many rows (prompts and their pieces): 128 rows to a workgroup of four waves that share every key and value
// tile in LDS.
#include "paged_common.h"

namespace mmp {

namespace {

constexpr int kKeys = 64;   // keys per tile
constexpr int kWaves = 4;
constexpr int kRows = 32;   // rows per wave

// The shape of many_kernel: head dims up to 16 NK (q, k) and 32 ND (v).
template <int NK, int ND>
struct Many {
  static constexpr int BR = kWaves * kRows;
  static constexpr int GR = kKeys;
  static constexpr int KC = 2 * NK, VC = 4 * ND;  // 16-byte chunks of a key, value row in LDS
  static constexpr int KI = KC / kWaves, VI = VC / kWaves;  // loads per thread, key and value tile
  static constexpr int K_BYTES = kKeys * KC * 16, V_BYTES = kKeys * VC * 16;
  static_assert(2 * (K_BYTES + V_BYTES) <= 159 * 1024 && KC % kWaves == 0 && VC % kWaves == 0, "tile shape");
};

// The chunk of a value row held at LDS place c of the row: the 4 rows that 32 lanes of a transposing read take 64 bytes
// of fall on distinct banks.
template <int VC>
__device__ __forceinline__ int v_chunk_of(int row, int c) {
  return VC == 8 ? c ^ (4 * ((row >> 1) & 1)) : c ^ (4 * (row & 3));
}

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
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

template <class T, int NK, int ND, bool PAGED>
__global__ __launch_bounds__(kWaves * kWave, NK <= 12 ? 2 : 1) void many_kernel(AttnArgs a) {
  using P = Many<NK, ND>;
  constexpr int BR = P::BR;
  // two buffers, each an object of its own: reads of one then need not wait for the loads in flight into the other
  __shared__ __align__(1024) char s_k0[P::K_BYTES], s_v0[P::V_BYTES], s_k1[P::K_BYTES], s_v1[P::V_BYTES];
  __shared__ int s_flag[2];  // a tile holds a value that is not finite
  const int tid = threadIdx.x, lane = lane_id();
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
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
    for (int i = tid; i < rows * a.dv; i += kWaves * kWave) T::st(out_at(i / a.dv), i % a.dv, NAN);
    return;
  }
  const int keys = keys_of<BR>(w.s, w.blk, a.group), pieces = pieces_of<P::GR>(keys, w.cut);
  if (w.piece >= pieces) return;
  const int k_begin = w.piece * w.cut * P::GR;
  const int k_end = w.cut == 0 ? keys : min(keys, k_begin + w.cut * P::GR);
  const int tiles = (k_end - k_begin + kKeys - 1) / kKeys;
  const int ctx = w.s.kv - w.s.n;

  // load i of a wave fills LDS chunks 64 (4 i + wave) + lane of a tile: row krow[i], dims kdim[i] ..
  int krow[P::KI], kdim[P::KI], vrow[P::VI], vdim[P::VI];
#pragma unroll
  for (int i = 0; i < P::KI; ++i) {
    const int c = kWave * (kWaves * i + wave) + lane;
    krow[i] = c / P::KC;
    kdim[i] = 8 * k_chunk_at<P::KC>(krow[i], c % P::KC);
  }
#pragma unroll
  for (int i = 0; i < P::VI; ++i) {
    const int c = kWave * (kWaves * i + wave) + lane;
    vrow[i] = c / P::VC;
    vdim[i] = 8 * v_chunk_of<P::VC>(vrow[i], c % P::VC);
  }
  const char* zeros = reinterpret_cast<const char*>(kZeroRow);
  auto key_of = [&](int it) { return min(k_begin + it * kKeys + lane, k_end - 1); };
  const char *kr, *vr;  // lane l: key l's rows of the tile being loaded
  uint64_t there = 0;   // and which keys exist
  auto find_rows = [&](int it, PageId id) {
    const int key = k_begin + it * kKeys + lane, kc = min(key, k_end - 1);
    bool ok = key < k_end;
    if constexpr (PAGED) {
      ok = ok && page_ok(a, id);
      const int row = kc - static_cast<int>(div_by(kc, a.page)) * static_cast<int>(a.page.d);
      kr = reinterpret_cast<const char*>(a.kp.at(static_cast<int>(id.lo), kvh, row));
      vr = reinterpret_cast<const char*>(a.vp.at(static_cast<int>(id.lo), kvh, row));
    } else {
      kr = reinterpret_cast<const char*>(a.k.at(w.s.first + kc, kvh));
      vr = reinterpret_cast<const char*>(a.v.at(w.s.first + kc, kvh));
    }
    if (!ok) kr = vr = zeros;
    there = __ballot(ok);
  };
  auto row_of = [&](const char* p, int r) {
    const uint64_t v = reinterpret_cast<uint64_t>(p);
    const uint32_t lo = static_cast<uint32_t>(__builtin_amdgcn_ds_bpermute(4 * r, static_cast<int>(v)));
    const uint32_t hi = static_cast<uint32_t>(__builtin_amdgcn_ds_bpermute(4 * r, static_cast<int>(v >> 32)));
    return reinterpret_cast<const char*>((static_cast<uint64_t>(hi) << 32) | lo);
  };
  auto load_tile = [&](char* kt, char* vt) {
#pragma unroll
    for (int i = 0; i < P::KI; ++i) {
      const char* p = row_of(kr, krow[i]) + 2 * kdim[i];
      load_lds16(kdim[i] < a.dqk ? p : zeros, kt + wave * 1024 + i * kWaves * 1024);
    }
#pragma unroll
    for (int i = 0; i < P::VI; ++i) {
      const char* p = row_of(vr, vrow[i]) + 2 * vdim[i];
      load_lds16(vdim[i] < a.dv ? p : zeros, vt + wave * 1024 + i * kWaves * 1024);
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
  // this lane's places in a tile: key row 32 u + lr, chunk 2 ks + lh; value rows 16 st + 4 lh + (lane % 16) / 4 (+ 8), dims
  // 32 dt + 16 ((lane / 16) % 2) + 4 (lane % 4) .. + 3
  const int vfr = 4 * lh + (lane & 15) / 4;
  const int vplace = vfr * P::VC * 16 + v_chunk_of<P::VC>(vfr, 2 * ((lane >> 4) & 1) + (lane & 3) / 2) * 16 + (lane & 1) * 8;
  floatx16 o[ND];
  float m = -INFINITY, l = 0.f;
#pragma unroll
  for (int dt = 0; dt < ND; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[dt][i] = 0.f;
  const float sc = a.scale * 1.4426950408889634f;

  if (tid < 2) s_flag[tid] = 0;
  PageId next{0, 0};
  auto tile = [&](int it, char* kt, char* vt, char* kt_next, char* vt_next, int* flag, int* flag_next) {
    const int j0 = k_begin + it * kKeys;
    const uint64_t mine = there;
    wait_vmcnt<0>();  // this wave's part of the tile
    __syncthreads();  // every wave's part; and the other buffer has been read
    if (it + 1 < tiles) {
      find_rows(it + 1, next);
      if constexpr (PAGED) next = page_id(a, w.b, key_of(it + 2));
      load_tile(kt_next, vt_next);
    }
    const bool mixed = j0 + kKeys > lim_block;  // some row does not see some key: 0 * inf must not reach it
    if (mixed) {
      if (tid == 0) *flag_next = 0;
      bool bad = false;
#pragma unroll
      for (int i = 0; i < P::VI; ++i) {
        const uint4 x = *reinterpret_cast<const uint4*>(vt + wave * 1024 + i * kWaves * 1024 + lane * 16);
        bad = bad || not_finite<T>(x.x) || not_finite<T>(x.y) || not_finite<T>(x.z) || not_finite<T>(x.w);
      }
      if (bad) *flag = 1;
      __syncthreads();
    }
    if (j0 < lim_max) {
      floatx16 s[2];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[u][i] = 0.f;
#pragma unroll
      for (int ks = 0; ks < NK; ++ks)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const uint4 x = *reinterpret_cast<const uint4*>(kt + (32 * u + lr) * P::KC * 16 + k_chunk_at<P::KC>(lr, 2 * ks + lh) * 16);
          s[u] = Mfma<T>::m32(x, qf[ks], s[u]);
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
      float tmax = fmaxf(s[0][0], s[1][0]);
#pragma unroll
      for (int i = 1; i < 16; ++i) tmax = fmaxf(tmax, fmaxf(s[0][i], s[1][i]));
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
      if (mixed && __builtin_amdgcn_readfirstlane(*flag) != 0) {
        // key by key; lane: row lr, dims 32 dt + 8 (i / 4) + 4 lh + i % 4
#pragma unroll
        for (int st = 0; st < 4; ++st) {
          const uint32_t w0 = pf[st].x, w1 = pf[st].y, w2 = pf[st].z, w3 = pf[st].w;
#pragma unroll 1
          for (int k = 0; k < 16; ++k) {
            const int e = k % 4 + 4 * (k / 8), key = 16 * st + k;
            const uint32_t pw = e < 2 ? w0 : e < 4 ? w1 : e < 6 ? w2 : w3;
            const uint32_t pk = static_cast<uint32_t>(__builtin_amdgcn_ds_bpermute(4 * (lr + 32 * (k % 8 / 4)), static_cast<int>(pw)));
            const uint32_t see = (sees >> key) & 1u ? ~0u : 0u;
            const float p = value_of<T>((e & 1 ? pk >> 16 : pk) & see);
#pragma unroll
            for (int dt = 0; dt < ND; ++dt)
#pragma unroll
              for (int i = 0; i < 16; i += 4) {
                const uint2 x = *reinterpret_cast<const uint2*>(vt + key * P::VC * 16 + v_chunk_of<P::VC>(key, 4 * dt + i / 4) * 16 + 8 * lh);
                o[dt][i] = fmaf(p, value_of<T>(x.x & see), o[dt][i]);
                o[dt][i + 1] = fmaf(p, value_of<T>((x.x & see) >> 16), o[dt][i + 1]);
                o[dt][i + 2] = fmaf(p, value_of<T>(x.y & see), o[dt][i + 2]);
                o[dt][i + 3] = fmaf(p, value_of<T>((x.y & see) >> 16), o[dt][i + 3]);
              }
          }
        }
      } else {
#pragma unroll
        for (int st = 0; st < 4; ++st)
#pragma unroll
          for (int dt = 0; dt < ND; ++dt)
            o[dt] = Mfma<T>::m32(v_frag(vt + (vplace ^ (64 * dt)) + 16 * st * P::VC * 16, 8 * P::VC * 16), pf[st], o[dt]);
      }
    }
  };
  if (tiles > 0) {
    if constexpr (PAGED) next = page_id(a, w.b, key_of(0));
    find_rows(0, next);
    if constexpr (PAGED) next = page_id(a, w.b, key_of(1));
    load_tile(s_k0, s_v0);
  }
  for (int it = 0; it < tiles; it += 2) {
    tile(it, s_k0, s_v0, s_k1, s_v1, s_flag, s_flag + 1);
    if (it + 1 < tiles) tile(it + 1, s_k1, s_v1, s_k0, s_v0, s_flag + 1, s_flag);
  }
  if (lr >= wrows) return;
  l += __shfl_xor(l, 32, kWave);
  const int r = kRows * wave + lr;  // of the workgroup
  if (pieces > 1) {
    float* state = state_at<BR>(a, w.slot + w.piece, kvh);
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

template <class T, int NK, int ND, bool PAGED>
int launch_shape(const AttnArgs& a, const AttnPlan& p, hipStream_t st, const char* what) {
  hipLaunchKernelGGL((many_kernel<T, NK, ND, PAGED>), dim3(static_cast<unsigned>((p.blocks + p.target) * a.nkv)),
                     dim3(kWaves * kWave), 0, st, a);
  return mm::check_launch(what);
}

template <class T, bool PAGED>
int launch_type(const AttnArgs& a, const AttnPlan& p, hipStream_t st, const char* what) {
  if (a.dqk <= 64 && a.dv <= 64) return launch_shape<T, 4, 2, PAGED>(a, p, st, what);
  if (a.dqk <= 128 && a.dv <= 128) return launch_shape<T, 8, 4, PAGED>(a, p, st, what);
  if (a.dqk <= 192 && a.dv <= 128) return launch_shape<T, 12, 4, PAGED>(a, p, st, what);
  return launch_shape<T, 16, 8, PAGED>(a, p, st, what);
}

}  // namespace

int launch_many(const AttnArgs& a, const AttnPlan& p, int dtype, bool paged, hipStream_t st, const char* what) {
  int rc = dtype == MM_BF16 ? (paged ? launch_type<BF16, true>(a, p, st, what) : launch_type<BF16, false>(a, p, st, what))
                            : (paged ? launch_type<FP16, true>(a, p, st, what) : launch_type<FP16, false>(a, p, st, what));
  if (rc || p.target == 0) return rc;
  return launch_join_many(a, p, dtype, st, what);
}

}  // namespace mmp
