// Attention of few rows over many keys (decode steps, short pieces): 16 rows to a workgroup, the keys shared out among its
// waves, and among workgroups where the keys are many (paged_common.h: find_work).
#include "paged_common.h"

namespace mmp {

namespace {

constexpr int kKeys = 32;  // keys per tile

// The shape of few_kernel: NW waves, head dims up to 32 NKQ (q, k) and 16 NT (v).
template <int NW, int NKQ, int NT>
struct Few {
  static constexpr int BR = 16;
  static constexpr int GR = NW * kKeys;                  // a granule: a tile for every wave
  static constexpr int DVM = 16 * NT;
  static constexpr int KC = 4 * NKQ, VC = 2 * NT;        // 16-byte chunks of a key, value row in LDS
  static constexpr int KI = kKeys * KC / kWave, VI = kKeys * VC / kWave;  // loads per key, value tile
  static constexpr int K_BYTES = kKeys * KC * 16, V_BYTES = kKeys * VC * 16;
  static constexpr int OROW = DVM + 4;
  static constexpr int ML = BR * OROW;                   // the wave's maxima and sums, after its outputs
  static constexpr int MET = ML + 2 * BR;                // and whether it met a value that is not finite
  static constexpr int O_BYTES = (MET + 4) * 4;
  static constexpr int WAVE_BYTES = K_BYTES + V_BYTES > O_BYTES ? K_BYTES + V_BYTES : O_BYTES;
  static constexpr size_t LDS = static_cast<size_t>(NW) * WAVE_BYTES;
  static_assert(LDS <= 160 * 1024 && KI % 2 == 0 && NT % 4 == 0, "tile shape");
};

// Softmax attention of up to 16 rows over a piece of their keys, one pass with a running maximum and sum. 16 rows, the
// matrix instruction's side: a decode step has G of them a stream, and more would only add to a block's states. Eight waves
// to a block (four past 192 / 128 dims, where their tiles fill the LDS): at one stream of 700 positions 8.2 us, 9.7 with
// four. Grid (work x key / value heads) x NW waves. Wave w takes tiles w, w + NW, ... of 32 keys of the piece; the waves'
// states meet in LDS.
// Per tile, on the 16x16x32 MFMA (bf16 or fp16, fp32 sums):
//   S^T [32 keys, 16 rows] = K Q^T: the key rows as A fragments from LDS, the rows' queries held as B fragments;
//   the softmax update per row is lane-local (a lane of S^T holds 8 keys of row lane % 16), the maximum over 4 lanes;
//   O^T [dv, 16 rows] += V^T P^T: P^T straight from the S^T registers (weights rounded to the cache's type: the matrix
//     units' operand, 2^-9 of a weight), V^T by transposing LDS reads.
// Bound by the cache rows' way from memory, 184 us for the 1.04 GB of 16 streams behind 4000 to 40000 positions (8 heads of
// 128, 5.7 TB/s), or where the keys are few by the chain of reads length, page number, key, value (64 streams of up to 1000
// positions 9.8 us). The rows come by loads straight into the wave's own LDS, the next tile's keys requested as soon as this
// one's are in registers, its values as soon as this one's are; the page numbers of the tile after that are read one tile
// ahead, lane l for key l % 32, and handed to the loading lanes by ds_bpermute. Keys that no row sees (past the piece, in a
// missing page) read a row of zeros. A value that some rows must not see could still be an infinity or NaN (0 * inf): the
// waves look for it in the tiles that can hold one (row_by_keys).
template <class T, int NW, int NKQ, int NT, bool PAGED>
__global__ __launch_bounds__(NW * kWave) void few_kernel(AttnArgs a) {
  using P = Few<NW, NKQ, NT>;
  constexpr int BR = P::BR;
  extern __shared__ __align__(16) char s_few[];
  const int tid = threadIdx.x, lane = lane_id();
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int lr = lane & 15, lq = lane >> 4, G = static_cast<int>(a.group.d);
  const int unit = static_cast<int>(blockIdx.x) / a.nkv, kvh = static_cast<int>(blockIdx.x) - unit * a.nkv;
  const Work w = scalars(find_work<BR, P::GR, false>(a, unit));
  if (w.b < 0) return;
  const int r0 = w.blk * BR, rows = min(BR, w.s.n * G - r0), n4 = a.dv / 4;
  auto out_at = [&](int r) {  // row r0 + r of the stream
    const int i = static_cast<int>(div_by(r0 + r, a.group));
    return a.out.at(w.s.first + i, kvh * G + (r0 + r - i * G));
  };
  if (w.s.kv < 0) {
    for (int i = tid; i < rows * a.dv; i += NW * kWave) T::st(out_at(i / a.dv), i % a.dv, NAN);
    return;
  }
  const int keys = keys_of<BR>(w.s, w.blk, a.group), pieces = pieces_of<P::GR>(keys, w.cut);
  if (w.piece >= pieces) return;
  const Range part = keys_of_piece<P::GR>(keys, pieces, w.piece);
  const int k_begin = part.begin, k_end = part.end;
  const int tiles = (k_end - k_begin + kKeys - 1) / kKeys;
  char* kt = s_few + wave * P::WAVE_BYTES;
  char* vt = kt + P::K_BYTES;
  // load i of a key tile fills LDS chunks 64 i + lane: row krow[i % KH] (+ 16 for the second half), dims kdim[i % KH] ..;
  // of a value tile row vrow + VPI i, dims vdim[i % VP] ..
  constexpr int KH = P::KI / 2, VPI = kWave / P::VC, VP = P::VC == 32 ? 4 : 2;
  int krow[KH], kdim[KH], vdim[VP];
#pragma unroll
  for (int i = 0; i < KH; ++i) {
    krow[i] = (kWave * i + lane) / P::KC;
    kdim[i] = 8 * k_chunk_at<P::KC>(krow[i], (kWave * i + lane) % P::KC);
  }
  const int vrow = lane / P::VC;
#pragma unroll
  for (int i = 0; i < VP; ++i) vdim[i] = 8 * v_chunk_at<P::VC>(vrow + VPI * i, lane % P::VC);

  const char* zeros = reinterpret_cast<const char*>(kZeroRow);
  // lane l's key of a tile, clamped into the piece
  auto key_of = [&](int it) { return min(k_begin + it * kKeys + (lane & (kKeys - 1)), k_end - 1); };
  // the rows of a tile's keys: lane l's key and value row, and which of the 32 exist
  const char *kr, *vr;
  uint32_t there = 0;
  auto find_rows = [&](int it, Index id) {
    const int key = k_begin + it * kKeys + (lane & (kKeys - 1));
    bool ok = key < k_end;
    const int kc = min(key, k_end - 1);
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
    there = static_cast<uint32_t>(__ballot(ok));
  };
  auto row_of = [&](const char* p, int r) {  // row r's address, from the lane that found it
    const uint64_t v = reinterpret_cast<uint64_t>(p);
    const uint32_t lo = static_cast<uint32_t>(__builtin_amdgcn_ds_bpermute(4 * r, static_cast<int>(v)));
    const uint32_t hi = static_cast<uint32_t>(__builtin_amdgcn_ds_bpermute(4 * r, static_cast<int>(v >> 32)));
    return reinterpret_cast<const char*>((static_cast<uint64_t>(hi) << 32) | lo);
  };
  auto load_k = [&] {
#pragma unroll
    for (int i = 0; i < P::KI; ++i) {
      const char* p = row_of(kr, krow[i % KH] + (i / KH) * 16) + 2 * kdim[i % KH];
      load_lds16(kdim[i % KH] < a.dqk ? p : zeros, kt + i * 1024);
    }
  };
  auto load_v = [&] {
#pragma unroll
    for (int i = 0; i < P::VI; ++i) {
      const char* p = row_of(vr, vrow + VPI * i) + 2 * vdim[i % VP];
      load_lds16(vdim[i % VP] < a.dv ? p : zeros, vt + i * 1024);
    }
  };
  // LDS places of this lane's fragment pieces: key row 16 f + lr, chunk 4 kk + lq; value rows 4 lq + lr / 4 (+ 16), dims
  // 16 nt + 4 (lr % 4) .. + 3
  const char* kfrag = kt + lr * P::KC * 16;
  const int vfr = 4 * lq + lr / 4;
  const int vplace = vfr * P::VC * 16 + v_chunk_at<P::VC>(vfr, (lr % 4) / 2) * 16 + (lr & 1) * 8;

  uint4 qf[NKQ];
  const int my_row = r0 + min(lr, rows - 1), my_i = static_cast<int>(div_by(my_row, a.group));
  const int lim = w.s.kv - w.s.n + my_i + 1;  // keys that this lane's row sees
  {
    const uint16_t* qrow = a.q.at(w.s.first + my_i, kvh * G + (my_row - my_i * G));
    const uint32_t sign = a.negative ? 0x80008000u : 0u;
#pragma unroll
    for (int kk = 0; kk < NKQ; ++kk) {
      const int d = 32 * kk + 8 * lq;
      const bool ok = d < a.dqk;
      const uint4 x = and_mask16(ld16(qrow + (ok ? d : 0)), ok);
      qf[kk] = make_uint4(x.x ^ sign, x.y ^ sign, x.z ^ sign, x.w ^ sign);
    }
  }
  const int lim_all = w.s.kv - w.s.n + static_cast<int>(div_by(r0, a.group)) + 1;  // keys that every row sees
  floatx4 o[NT];
  float m = -INFINITY, l = 0.f;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) o[nt] = floatx4{0.f, 0.f, 0.f, 0.f};
  const float sc = a.scale * 1.4426950408889634f;  // scores in units of log2: exp2 gives the weights
  uint32_t seen = 0;  // exponents of values that some row must not meet
  if (wave < tiles) {
    Index next{0, 0};
    if constexpr (PAGED) next = page_id(a, w.b, key_of(wave));
    find_rows(wave, next);
    if constexpr (PAGED) next = page_id(a, w.b, key_of(wave + NW));
    wait_vmcnt<0>();  // the queries and pages: from here on only tiles and page numbers are in flight
    load_k();
    load_v();
    for (int it = wave; it < tiles; it += NW) {
      const int j0 = k_begin + it * kKeys;
      const uint32_t mine = there;  // the tile's keys that exist
      wait_vmcnt<P::VI>();  // the tile's keys (its values still in flight)
      wave_lds_fence();
      uint4 kx[2][NKQ];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int kk = 0; kk < NKQ; ++kk)
          kx[u][kk] = *reinterpret_cast<const uint4*>(kfrag + u * 16 * P::KC * 16 + k_chunk_at<P::KC>(lr, 4 * kk + lq) * 16);
      wait_lgkm0();  // read before the next tile overwrites them
      const bool more = it + NW < tiles;
      if (more) {
        find_rows(it + NW, next);
        if constexpr (PAGED) next = page_id(a, w.b, key_of(it + 2 * NW));
        load_k();
      }
      floatx4 s[2] = {floatx4{0.f, 0.f, 0.f, 0.f}, floatx4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int kk = 0; kk < NKQ; ++kk)
#pragma unroll
        for (int u = 0; u < 2; ++u) s[u] = Mfma<T>::m16(kx[u][kk], qf[kk], s[u]);
      const bool mixed = j0 + kKeys > lim_all;  // some row does not see some key: its value must be finite, or 0 * inf reaches the row
      const int n = lim - j0;
      const uint32_t sees = n >= kKeys ? mine : n <= 0 ? 0u : mine & ((1u << n) - 1u);
      const uint32_t lo4 = sees >> (4 * lq), hi4 = sees >> (16 + 4 * lq);
      float sv[8];
      float tmax = -INFINITY;
#pragma unroll
      for (int e = 0; e < 8; ++e) {  // slot e < 4 is key 4 lq + e of the tile, slot e >= 4 key 16 + 4 lq + e - 4
        const bool see = e < 4 ? (lo4 >> e) & 1u : (hi4 >> (e - 4)) & 1u;
        sv[e] = see ? (e < 4 ? s[0][e] : s[1][e - 4]) * sc : -INFINITY;
        tmax = larger(tmax, sv[e]);
      }
      const float mn = fmaxf(m, quarter_max(tmax));
      const float mu = mn == -INFINITY ? 0.f : mn;  // a row that has seen no key yet
      const float alpha = exp2_fast(m - mu);
      m = mn;
      float ps = 0.f;
      uint32_t pw[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p0 = exp2_fast(sv[2 * e] - mu), p1 = exp2_fast(sv[2 * e + 1] - mu);
        ps += p0 + p1;
        pw[e] = pack2<T>(p0, p1);
      }
      l = fmaf(l, alpha, ps);
      const uint4 pf = make_uint4(pw[0], pw[1], pw[2], pw[3]);
      if (__any(alpha != 1.f)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) o[nt] *= alpha;
      }
      if (more) wait_vmcnt<P::KI>();  // the tile's values (the next tile's keys still in flight)
      else wait_vmcnt<0>();
      wave_lds_fence();
#pragma unroll
      for (int n0 = 0; n0 < NT; n0 += 4) {
        uint32_t place[4];
        uint64_t lo[4], hi[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) place[b] = lds_place(vt) + (vplace ^ (32 * (n0 + b)));
        lds_tr4x2<16 * P::VC * 16>(place, lo, hi);
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const uint4 vf = make_uint4(static_cast<uint32_t>(lo[b]), static_cast<uint32_t>(lo[b] >> 32),
                                      static_cast<uint32_t>(hi[b]), static_cast<uint32_t>(hi[b] >> 32));
          if (mixed) seen = add_exponents<T>(seen, vf);
          o[n0 + b] = Mfma<T>::m16(vf, pf, o[n0 + b]);
        }
      }
      wait_lgkm0();  // read before the next tile overwrites them
      if (more) load_v();
    }
  }
  // the wave's state into its own LDS region, then the merge
  float* so = reinterpret_cast<float*>(s_few + wave * P::WAVE_BYTES);
  wave_lds_fence();
  l += __shfl_xor(l, 16, kWave);
  l += __shfl_xor(l, 32, kWave);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) *reinterpret_cast<floatx4*>(so + lr * P::OROW + 16 * nt + 4 * lq) = o[nt];
  if (lq == 0) {
    so[P::ML + lr] = m;
    so[P::ML + BR + lr] = l;
  }
  const bool mine_met = __any((seen & kNotFinite) != 0);
  if (lane == 0) so[P::MET] = mine_met ? 1.f : 0.f;
  __syncthreads();
  float* state = pieces > 1 ? state_at<BR>(a, w.slot + w.piece, kvh) : nullptr;
  float met = 0.f;
#pragma unroll
  for (int x = 0; x < NW; ++x) met += reinterpret_cast<const float*>(s_few + x * P::WAVE_BYTES)[P::MET];
  if (__builtin_amdgcn_readfirstlane(met != 0.f)) {
    rows_by_keys<T, BR>(a, w, kvh, rows, wave, NW, k_begin, k_end, state);
    return;
  }
  for (int i = tid; i < rows * n4; i += NW * kWave) {
    const int r = i / n4, d = 4 * (i - r * n4);
    auto of = [&](int x) { return reinterpret_cast<const float*>(s_few + x * P::WAVE_BYTES); };
    float mx = of(0)[P::ML + r];
#pragma unroll
    for (int x = 1; x < NW; ++x) mx = fmaxf(mx, of(x)[P::ML + r]);
    const float mu = mx == -INFINITY ? 0.f : mx;
    float lt = 0.f;
    floatx4 acc = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < NW; ++x) {
      const float wt = exp2_fast(of(x)[P::ML + r] - mu);
      lt = fmaf(of(x)[P::ML + BR + r], wt, lt);
      acc += wt * *reinterpret_cast<const floatx4*>(of(x) + r * P::OROW + d);
    }
    if (state) {
      *reinterpret_cast<floatx4*>(state + r * a.dv + d) = acc;
      if (d == 0) {
        state[BR * a.dv + r] = mx;
        state[BR * a.dv + BR + r] = lt;
      }
    } else {
      const float inv = mx == -INFINITY ? 0.f : 1.f / lt;
      *reinterpret_cast<uint2*>(out_at(r) + d) = make_uint2(pack2<T>(acc[0] * inv, acc[1] * inv), pack2<T>(acc[2] * inv, acc[3] * inv));
    }
  }
}

// Joins the pieces of a row block that was cut: out = sum_p exp2(m_p - M) acc_p / sum_p exp2(m_p - M) l_p. Grid (cut
// blocks, key / value heads, BR / ROWS) x 256: RW rows at a time, 256 / RW lanes to a row, of which dv / 4 read a piece's
// sums side by side and the rest other pieces'. Bound by latency: finding the block, one round of 8 pieces a lane, the
// exchange in LDS; 6.3 us after the 184 us above.
template <class T, int BR, int GR, int ROWS, int RW>
__global__ __launch_bounds__(256) void join_kernel(AttnArgs a) {
  constexpr int LANES = 256 / RW;
  __shared__ float s_m[256], s_l[256];
  __shared__ __align__(16) floatx4 s_acc[256];
  const int tid = threadIdx.x, kvh = blockIdx.y, G = static_cast<int>(a.group.d);
  const Work w = scalars(find_work<BR, GR, true>(a, blockIdx.x));
  if (w.b < 0) return;
  const int keys = keys_of<BR>(w.s, w.blk, a.group), pieces = pieces_of<GR>(keys, w.cut);
  if (pieces == 1) return;  // a block of few keys in a stream that is cut: written by the piece itself
  const int n4 = a.dv / 4, rows = min(BR, w.s.n * G - w.blk * BR);
  const int t = tid % LANES, side = LANES / n4, p0 = t / n4, d = 4 * (t - p0 * n4);
  const float* first = state_at<BR>(a, w.slot, kvh);
  const int64_t step = static_cast<int64_t>(a.nkv) * BR * (a.dv + 2);
  const int end = min(rows, static_cast<int>(blockIdx.z) * ROWS + ROWS);
  for (int r0 = static_cast<int>(blockIdx.z) * ROWS; r0 < end; r0 += RW) {
    const int r = r0 + tid / LANES;
    float m = -INFINITY, l = 0.f;
    floatx4 acc = floatx4{0.f, 0.f, 0.f, 0.f};
    if (r < end && p0 < side) {
      constexpr int kAtOnce = 8;
      for (int p = p0; p < pieces; p += side * kAtOnce) {
        float pm[kAtOnce], pl[kAtOnce];
        floatx4 pa[kAtOnce];
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
          const float* s = first + min(p + u * side, pieces - 1) * step;
          pm[u] = s[BR * a.dv + r];
          pl[u] = s[BR * a.dv + BR + r];
          pa[u] = *reinterpret_cast<const floatx4*>(s + r * a.dv + d);
        }
        float mn = m;
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) mn = fmaxf(mn, p + u * side < pieces ? pm[u] : -INFINITY);
        const float mu = mn == -INFINITY ? 0.f : mn, alpha = exp2_fast(m - mu);
        m = mn;
        l *= alpha;
        acc *= alpha;
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u)
          if (p + u * side < pieces) {
            const float wt = exp2_fast(pm[u] - mu);
            l = fmaf(pl[u], wt, l);
            acc += wt * pa[u];
          }
      }
    }
    __syncthreads();  // the last rows' values have been read
    s_m[tid] = m;
    s_l[tid] = l;
    s_acc[tid] = acc;
    __syncthreads();
    if (r >= end || p0 != 0) continue;
    float mx = m;
    for (int x = 1; x < side; ++x) mx = fmaxf(mx, s_m[tid + x * n4]);
    const float mu = mx == -INFINITY ? 0.f : mx;
    float lt = 0.f;
    floatx4 sum = floatx4{0.f, 0.f, 0.f, 0.f};
    for (int x = 0; x < side; ++x) {
      const float wt = exp2_fast(s_m[tid + x * n4] - mu);
      lt = fmaf(s_l[tid + x * n4], wt, lt);
      sum += wt * s_acc[tid + x * n4];
    }
    const int row = w.blk * BR + r, i = static_cast<int>(div_by(row, a.group));
    const float inv = mx == -INFINITY ? 0.f : 1.f / lt;
    *reinterpret_cast<uint2*>(a.out.at(w.s.first + i, kvh * G + (row - i * G)) + d) =
        make_uint2(pack2<T>(sum[0] * inv, sum[1] * inv), pack2<T>(sum[2] * inv, sum[3] * inv));
  }
}

// The same for blocks of many rows, which are cut into few pieces: dv / 4 lanes to a row, each through all pieces. Grid (cut
// blocks, key / value heads, BR / ROWS) x 256. Bound by latency too: 8 us after pieces of 100 to 500 tokens of 32/8 heads
// behind 611 to 5000 positions (75 us).
template <class T, int BR, int GR, int ROWS>
__global__ __launch_bounds__(256) void join_rows_kernel(AttnArgs a) {
  const int tid = threadIdx.x, kvh = blockIdx.y, G = static_cast<int>(a.group.d);
  const Work w = scalars(find_work<BR, GR, true>(a, blockIdx.x));
  if (w.b < 0) return;
  const int keys = keys_of<BR>(w.s, w.blk, a.group), pieces = pieces_of<GR>(keys, w.cut);
  if (pieces == 1) return;
  const int n4 = a.dv / 4, at_once = 256 / n4, rows = min(BR, w.s.n * G - w.blk * BR);
  const int my = tid / n4, d = 4 * (tid - my * n4);
  const float* first = state_at<BR>(a, w.slot, kvh);
  const int64_t step = static_cast<int64_t>(a.nkv) * BR * (a.dv + 2);
  const int end = min(rows, static_cast<int>(blockIdx.z) * ROWS + ROWS);
  if (my >= at_once) return;
  for (int r = static_cast<int>(blockIdx.z) * ROWS + my; r < end; r += at_once) {
    float m = -INFINITY, l = 0.f;
    floatx4 acc = floatx4{0.f, 0.f, 0.f, 0.f};
    constexpr int kAtOnce = 4;
    for (int p = 0; p < pieces; p += kAtOnce) {
      float pm[kAtOnce], pl[kAtOnce];
      floatx4 pa[kAtOnce];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        const float* s = first + min(p + u, pieces - 1) * step;
        pm[u] = s[BR * a.dv + r];
        pl[u] = s[BR * a.dv + BR + r];
        pa[u] = *reinterpret_cast<const floatx4*>(s + r * a.dv + d);
      }
      float mn = m;
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) mn = fmaxf(mn, p + u < pieces ? pm[u] : -INFINITY);
      const float mu = mn == -INFINITY ? 0.f : mn, alpha = exp2_fast(m - mu);
      m = mn;
      l *= alpha;
      acc *= alpha;
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u)
        if (p + u < pieces) {
          const float wt = exp2_fast(pm[u] - mu);
          l = fmaf(pl[u], wt, l);
          acc += wt * pa[u];
        }
    }
    const int row = w.blk * BR + r, i = static_cast<int>(div_by(row, a.group));
    const float inv = m == -INFINITY ? 0.f : 1.f / l;
    *reinterpret_cast<uint2*>(a.out.at(w.s.first + i, kvh * G + (row - i * G)) + d) =
        make_uint2(pack2<T>(acc[0] * inv, acc[1] * inv), pack2<T>(acc[2] * inv, acc[3] * inv));
  }
}

template <class T, int BR, int GR, int ROWS, int RW>
int launch_join(const AttnArgs& a, const AttnPlan& p, hipStream_t st, const char* what) {
  hipLaunchKernelGGL((join_kernel<T, BR, GR, ROWS, RW>),
                     dim3(static_cast<unsigned>(p.blocks < p.target ? p.blocks : p.target), static_cast<unsigned>(a.nkv), BR / ROWS),
                     dim3(256), 0, st, a);
  return mm::check_launch(what);
}

template <class T, int NW, int NKQ, int NT, bool PAGED>
int launch_shape(const AttnArgs& a, const AttnPlan& p, hipStream_t st, const char* what) {
  using P = Few<NW, NKQ, NT>;
  auto kern = few_kernel<T, NW, NKQ, NT, PAGED>;
  int rc = mm::allow_lds(kern, P::LDS, what);
  if (rc || (rc = launch_index<P::BR, P::GR>(a, st, what))) return rc;
  hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>((p.blocks + p.target) * a.nkv)), dim3(NW * kWave), P::LDS, st, a);
  rc = mm::check_launch(what);
  if (rc || p.target == 0) return rc;
  // Rows of the join: a workgroup takes four, each with 4 x 8 pieces a round (dv = 64), or where a block can have more than 32
  // pieces one, with four times as many. us a call, four | one: one Talker stream behind 5000 positions 10.7 | 11.2, behind
  // 20000 13.8 | 12.2, 120000 37 | 26; 16 / 2 heads of 256 behind 60000 109 | 66; 32 streams of 4 tokens of 32/8 heads of 128
  // behind 8000 205 | 217.
  const int64_t most = (PAGED ? a.batch.max_keys : a.batch.tokens) / P::GR;
  return p.target > 32 * p.blocks && most > 32 ? launch_join<T, P::BR, P::GR, 1, 1>(a, p, st, what)
                                               : launch_join<T, P::BR, P::GR, 4, 4>(a, p, st, what);
}

template <class T, bool PAGED>
int launch_type(const AttnArgs& a, const AttnPlan& p, hipStream_t st, const char* what) {
  if (a.dqk <= 64 && a.dv <= 64) return launch_shape<T, 8, 2, 4, PAGED>(a, p, st, what);
  if (a.dqk <= 128 && a.dv <= 128) return launch_shape<T, 8, 4, 8, PAGED>(a, p, st, what);
  if (a.dqk <= 192 && a.dv <= 128) return launch_shape<T, 8, 6, 8, PAGED>(a, p, st, what);
  return launch_shape<T, 4, 8, 16, PAGED>(a, p, st, what);
}

}  // namespace

namespace {

int64_t most_blocks(int64_t rows, int64_t seqs, int64_t br) { return rows / br + seqs < rows ? rows / br + seqs : rows; }

// Bytes of keys and values that blocks of 16 rows would read, each all the keys that its stream can have.
int64_t reads_of_few(int64_t rows, int64_t seqs, int64_t max_keys, int nkv, int dqk, int dv) {
  return most_blocks(rows, seqs, 16) * nkv * (dqk + dv) * 2 * max_keys;
}
constexpr int64_t kFewReads = 64 << 20;

// Streams up to which every wave finds its work by itself, 64 of them at a time; of more, index_kernel writes down where each
// stream's begins. us a call without | with it: one token of 192 Talker streams behind 1500 positions 54 | 46, behind 200 10.0 |
// 12.3; 8 tokens each behind 300 38 | 29; of 128 streams 35 | 34, 8.0 | 10.6, 25 | 25; of 1024 311 | 155, 65 | 39; of 4096 behind
// 200 601 | 134; 2048 prompts of 20 tokens 173 | 100, 192 of them 22.3 | 22.6.
constexpr int64_t kIndexed = 128;

int64_t few_granule(int dqk, int dv) { return (dqk <= 192 && dv <= 128 ? 8 : 4) * kKeys; }
// pieces aimed at for one key / value head
int64_t few_target(int nkv) { return (4 * mm::cu_count() + nkv - 1) / nkv; }
// of many rows, as many as the device holds workgroups at once: three a CU by registers at 64 dims, two, or one by shared
// memory
int64_t many_target(int nkv, int dqk, int dv) {
  const int64_t at_once = dqk <= 64 && dv <= 64 ? 3 : dqk <= 192 && dv <= 128 ? 2 : 1;
  return (at_once * mm::cu_count() + nkv - 1) / nkv;
}
int64_t index_bytes(int64_t seqs) { return seqs > kIndexed ? 16 * (seqs + 1) : 0; }
int64_t state_bytes(int64_t target, int nkv, int br, int dv) { return 2 * target * nkv * br * (dv + 2) * 4; }

}  // namespace

// Few rows or many: 16-row blocks where the streams have no more rows than that on average (a decode step), and where the
// keys that such blocks read are so few that the caches bring them quicker than 128 rows get through them. us a call, 16 |
// 128 rows (reads at 16): a prompt of 37 Talker tokens 5.0 | 6.2, of 200 5.6 | 9.2 (9 MB), of 500 8.0 | 13.2 (56 MB); 100
// Talker tokens behind 1000 13.6 | 15.6 (25 MB); 20 heads of one key / value head behind 6000 10.7 | 16.6 (3 MB); 30 thinker
// tokens behind 3000 23.9 | 23.2 (62 MB); 300 tokens of 32/8 heads of 128 16.9 | 13.7 (92 MB); 64 tokens of those behind 8000
// 66 | 39 (528 MB).
// Cutting: few rows above 4 granules of keys (one stream at 700 positions: 10.0 us cut, 8.4 not), then 4 pieces a CU (decode of
// 16 streams behind 4000 to 40000 positions: 397 us uncut, 239 at 1 piece a CU, 217 at 2, 197 at 4, 202 at 8). Many rows over
// a cache, above 4 granules: the workgroups that the device holds at once (64 dims, 2000 tokens behind 20000: 280 us at 1.5 a
// CU, 250 at 3, 242 at 4; 8000 tokens of 2 heads 65 at 1, 50 at 2, 42 at 3, 51 at 4; 128 dims, pieces of 100 to 500 tokens
// behind 611 to 5000: 149 uncut, 98 at 1, 83 at 2, 97 at 4; 256 dims, 300 tokens behind 5000: 69 at 1, 83 at 2, 600 behind 4000
// 95 and 106, four times 200 behind 4000 105 and 87). Prompts, whose keys are their own tokens, only where their row blocks
// leave half of the CUs idle and can be long (2 heads of 64, 2000 tokens: 24.8 us uncut, 15.6 cut; 2000 Talker tokens, 220
// blocks: 26.6 and 31; 300 tokens of 32/8 heads of 128: 14.0 and 16.5).
// Two groups of waves to a block where a prompt's blocks are fewer than 4 a CU: they halve the time of the last block (12
// ragged Talker prompts 42.8 -> 38.5 us, 2000 Talker tokens 37.4 -> 29.6, 4000 72 -> 59), but in a long run two workgroups
// of one group mix matrix and vector work better (8192 tokens of 32/8 heads of 128: 590 | 643), and over a cache the cut
// does as much (91 | 95).
AttnPlan plan_attn(bool paged, int64_t tokens, int64_t seqs, int64_t max_keys, int nh, int nkv, int dqk, int dv) {
  AttnPlan p{};
  const int64_t rows = tokens * (nh / nkv), cus = mm::cu_count();
  p.many = rows > 16 * seqs && reads_of_few(rows, seqs, max_keys, nkv, dqk, dv) > kFewReads;
  p.blocks = most_blocks(rows, seqs, p.many ? 128 : 16);
  if (p.many) {
    if (paged ? max_keys > 64 * kMinCut : 2 * p.blocks * nkv < cus && max_keys > 1024) p.target = many_target(nkv, dqk, dv);
    p.groups = !paged && p.target == 0 && p.blocks * nkv < 4 * cus && dqk <= 192 && dv <= 128 ? 2 : 1;
    p.workspace = state_bytes(p.target, nkv, 128, dv);
  } else {
    if (max_keys > 4 * few_granule(dqk, dv)) p.target = few_target(nkv);
    p.workspace = state_bytes(p.target, nkv, 16, dv);
  }
  p.indexed = seqs > kIndexed;
  p.workspace += index_bytes(seqs);
  return p;
}

int64_t workspace_of(bool paged, int64_t tokens, int64_t seqs, int64_t max_keys, int nh, int nkv, int dqk, int dv, bool at_most) {
  if (!at_most) return plan_attn(paged, tokens, seqs, max_keys, nh, nkv, dqk, dv).workspace;
  const int64_t few = max_keys > 4 * few_granule(dqk, dv) ? state_bytes(few_target(nkv), nkv, 16, dv) : 0;
  const bool many = max_keys > 64 * kMinCut && reads_of_few(tokens * (nh / nkv), seqs, max_keys, nkv, dqk, dv) > kFewReads;
  const int64_t of_many = many ? state_bytes(many_target(nkv, dqk, dv), nkv, 128, dv) : 0;
  return (few > of_many ? few : of_many) + index_bytes(seqs);
}

int launch_few(const AttnArgs& a, const AttnPlan& p, int dtype, bool paged, hipStream_t st, const char* what) {
  if (dtype == MM_BF16)
    return paged ? launch_type<BF16, true>(a, p, st, what) : launch_type<BF16, false>(a, p, st, what);
  return paged ? launch_type<FP16, true>(a, p, st, what) : launch_type<FP16, false>(a, p, st, what);
}

int launch_join_many(const AttnArgs& a, const AttnPlan& p, int dtype, hipStream_t st, const char* what) {
  constexpr int ROWS = 16;
  const dim3 grid(static_cast<unsigned>(p.blocks < p.target ? p.blocks : p.target), static_cast<unsigned>(a.nkv), 128 / ROWS);
  if (dtype == MM_BF16) hipLaunchKernelGGL((join_rows_kernel<BF16, 128, 64, ROWS>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((join_rows_kernel<FP16, 128, 64, ROWS>), grid, dim3(256), 0, st, a);
  return mm::check_launch(what);
}

}  // namespace mmp
