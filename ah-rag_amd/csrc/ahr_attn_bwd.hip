// Attention over packed sequences, backward (include/ahr.h ahr_attn_backward).
//
// With p = 2^(c s - lse), delta = sum_d do o and ds = p (do . v - delta):
//   dv_j = sum_i p_ij do_i,   dk_j = scale sum_i ds_ij q_i,   dq_i = scale sum_j ds_ij k_j.
// Two kernels recompute p, one for each direction of the sum: dk and dv stay in the registers of the
// wave that owns 32 keys while the query rows of every head of the group pass through LDS; dq stays
// with the wave that owns 32 rows while the keys pass. That is seven matrix products where one kernel
// needs five, but nothing is added through memory: no atomics, no fp32 copy of dq, the same bits
// every time.
#include "ahr_attn_common.h"

namespace ahr {
namespace attn {

constexpr int kRowsB = 64;  // query rows of one staged tile

// f16 holds ds only within 2^-24 .. 2^16, and ds of a long row with small gradients lies below it:
// its accumulators hold ds times a power of two, chosen from the first values so that their largest
// becomes 2^12 .. 2^13 and lowered (with the accumulators) when later ones pass 2^15. bf16 has fp32's
// range and skips all of it.
constexpr float kWide = 32768.f;
__device__ __forceinline__ float pick_scale(float largest) {
  const int ex = (int)((__float_as_uint(largest) >> 23) & 255) - 127;
  return ldexpf(1.f, min(12 - ex, 100));
}
// (p <= 1 is held times 2^14 for dv.)

// delta[t][head] = sum_d do o: 8 elements a lane, 16 lanes a row
template <typename T>
__global__ __launch_bounds__(256) void attn_delta_kernel(Params p, int64_t rows) {
  typedef typename Elem<T>::v8 v8;
  const int64_t r = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
  const int d = (threadIdx.x & 15) * 8;
  float x = 0.f;
  if (r < rows && d < p.dim) {
    const int64_t t = r / p.heads;
    const int hd = (int)(r - t * p.heads);
    const v8 a = *reinterpret_cast<const v8*>(p.o + (t * p.o_ts + hd * p.o_hs + d) * 2);
    const v8 b = *reinterpret_cast<const v8*>(p.d_o + (t * p.do_ts + hd * p.do_hs + d) * 2);
#pragma unroll
    for (int i = 0; i < 8; ++i) x = fmaf((float)a[i], (float)b[i], x);
  }
#pragma unroll
  for (int i = 1; i < 16; i *= 2) x += __shfl_xor(x, i, 64);
  if (r < rows && d == 0) p.delta[r] = x;
}

// dk, dv of NW * 32 keys of one key head
template <typename T, int DP, int NW>
__global__ __launch_bounds__(NW * 64, DP > 64 ? 1 : 2) void attn_dkv_kernel(Params p) {
  typedef typename Elem<T>::v8 v8;
  constexpr int NC = DP / 8, KS = DP / 16, DB = DP / 32;
  constexpr int kTile = kRowsB * DP * 2;
  constexpr int kBuf = 2 * kTile + 2 * kRowsB * 4;  // q tile, do tile, lse, delta
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x & 63, h = lane >> 5, n = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int hk = blockIdx.x % p.kv_heads;
  const KeyItem it = p.keys[blockIdx.x / p.kv_heads];
  const int dim = p.dim;

  if (DP != dim) {
    for (int b = 0; b < 2; ++b)
      for (int i = threadIdx.x; i < 2 * kTile / 16; i += NW * 64)
        reinterpret_cast<f32x4*>(smem + b * kBuf)[i] = f32x4{0, 0, 0, 0};
    __syncthreads();
  }

  const int key = wave * 32 + n;
  const bool live = key < it.nk;
  v8 kf[KS], vf[KS];
  {
    const int64_t at = it.k0 + (live ? key : 0);
    const char* kp = p.k + (at * p.k_ts + (int64_t)hk * p.k_hs) * 2;
    const char* vp = p.v + (at * p.v_ts + (int64_t)hk * p.v_hs) * 2;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int d = (2 * ks + h) * 8;
      const v8 z = {};
      const bool in = live && (DP == dim || d < dim);
      kf[ks] = in ? *reinterpret_cast<const v8*>(kp + d * 2) : z;
      vf[ks] = in ? *reinterpret_cast<const v8*>(vp + d * 2) : z;
    }
  }
  f32x16 gk[DB], gv[DB];
#pragma unroll
  for (int b = 0; b < DB; ++b)
#pragma unroll
    for (int r = 0; r < 16; ++r) gk[b][r] = gv[b][r] = 0.f;

  const Stager<NC, NW, kRowsB> stager(wave, lane);
  const int G = p.group;
  const int coff = it.klen - it.qlen;
  const int n_tok = it.qlen - it.t0;              // query tokens that matter
  const int64_t n_rows = (int64_t)n_tok * G;      // and their rows
  const int nt = (int)((n_rows + kRowsB - 1) / kRowsB);
  float st_l = 0.f, st_d = 0.f;  // lse and delta of the next tile's row, on their way to LDS
  auto stage = [&](int t, int buf) {
    const int64_t r0 = (int64_t)t * kRowsB;
    const int tok0 = (int)(r0 / G), g0 = (int)(r0 - (int64_t)tok0 * G);
    const int have = (int)min((int64_t)kRowsB, n_rows - r0);
    const int64_t at = it.q0 + it.t0 + tok0;
    const int qts = (int)p.q_ts * 2, qhs = (int)p.q_hs * 2, ots = (int)p.do_ts * 2, ohs = (int)p.do_hs * 2;
    const uint32_t span = (uint32_t)((g0 + have - 1) / G);  // tokens past the first
    const __amdgpu_buffer_rsrc_t qr = dense::tile_rsrc_u(p.q + (at * p.q_ts + (int64_t)hk * G * p.q_hs) * 2,
                                                         span * qts + (G - 1) * qhs + dim * 2);
    const __amdgpu_buffer_rsrc_t dr = dense::tile_rsrc_u(p.d_o + (at * p.do_ts + (int64_t)hk * G * p.do_hs) * 2,
                                                         span * ots + (G - 1) * ohs + dim * 2);
    char* tile = smem + buf * kBuf;
    auto off = [&](int r, int ts, int hs) {
      const int x = g0 + min(r, have - 1);
      const int tk = (x * p.group_inv) >> 16;
      return tk * ts + (x - tk * G) * hs;
    };
    stager.load(qr, tile, dim, [&](int r) { return off(r, qts, qhs); });
    stager.load(dr, tile + kTile, dim, [&](int r) { return off(r, ots, ohs); });
    if (threadIdx.x < kRowsB) {
      const int r = threadIdx.x, x = g0 + min(r, have - 1), tk = (x * p.group_inv) >> 16;
      const int64_t i = (at + tk) * p.heads + hk * G + (x - tk * G);
      st_l = p.lse[i];
      st_d = p.delta[i];
    }
  };
  auto land = [&](int buf) {
    float* f = reinterpret_cast<float*>(smem + buf * kBuf + 2 * kTile);
    if (threadIdx.x < kRowsB) {
      f[threadIdx.x] = st_l;
      f[kRowsB + threadIdx.x] = st_d;
    }
  };

  const bool wave_live = wave * 32 < it.nk;
  const int j = it.kpos + key;                               // this lane's key in its sequence
  const int j_hi = it.kpos + min(wave * 32 + 31, it.nk - 1);  // the wave's last
  const float c = p.scale_log2;
  float sc = Elem<T>::kNarrow ? 0.f : 1.f;  // factor of ds in gk (0: none chosen yet)
  if (nt > 0) {
    stage(0, 0);
    land(0);
  }
  for (int t = 0; t < nt; ++t) {
    __syncthreads();
    if (t + 1 < nt) stage(t + 1, (t + 1) & 1);
    const int64_t r0 = (int64_t)t * kRowsB;
    const int tok0 = (int)(r0 / G), g0 = (int)(r0 - (int64_t)tok0 * G);
    const int have = (int)min((int64_t)kRowsB, n_rows - r0);
    const char* q_lds = smem + (t & 1) * kBuf;
    const char* o_lds = q_lds + kTile;
    const float* f = reinterpret_cast<const float*>(o_lds + kTile);
    if (wave_live) {
#pragma unroll
      for (int u = 0; u < kRowsB / 32; ++u) {
        if (u * 32 >= have) break;
        f32x16 s, g;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = g[r] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) s = Elem<T>::mma(row_frag<T, NC>(q_lds, u * 32 + n, ks, h), kf[ks], s);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) g = Elem<T>::mma(row_frag<T, NC>(o_lds, u * 32 + n, ks, h), vf[ks], g);
        // a row reads keys j <= coff + its token; the rows' tokens rise
        const int tok_lo = it.t0 + tok0 + (((g0 + u * 32) * p.group_inv) >> 16);
        const bool cut = u * 32 + 32 > have || (p.causal && j_hi > coff + tok_lo);
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          const f32x4 ls = *reinterpret_cast<const f32x4*>(f + u * 32 + r4 * 8 + h * 4);
          const f32x4 de = *reinterpret_cast<const f32x4*>(f + kRowsB + u * 32 + r4 * 8 + h * 4);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = r4 * 4 + i;
            float pr = ex2(fmaf(s[r], c, -ls[i]));
            float ds = pr * (g[r] - de[i]);
            if (cut) {
              const int x = u * 32 + r4 * 8 + h * 4 + i;
              const int tok = it.t0 + tok0 + (((g0 + x) * p.group_inv) >> 16);
              const bool reads = x < have && (!p.causal || j <= coff + tok);
              pr = reads ? pr : 0.f;
              ds = reads ? ds : 0.f;
            }
            s[r] = Elem<T>::kNarrow ? pr * 0x1p14f : pr;
            g[r] = ds;
          }
        }
        if constexpr (Elem<T>::kNarrow) {  // one factor for the wave: dk sums over its rows
          float most = 0.f;
#pragma unroll
          for (int r = 0; r < 16; ++r) most = fmaxf(most, fabsf(g[r]));
          if (__any((most * sc > kWide || (sc == 0.f && most > 0.f)) && most < INFINITY)) {
            most = most < INFINITY ? most : 0.f;
#pragma unroll
            for (int x = 1; x < 64; x *= 2) most = fmaxf(most, __shfl_xor(most, x, 64));
            const float to = pick_scale(most), f2 = sc == 0.f ? 1.f : to / sc;
#pragma unroll
            for (int b = 0; b < DB; ++b)
#pragma unroll
              for (int r = 0; r < 16; ++r) gk[b][r] *= f2;
            sc = to;
          }
          const float mul = sc == 0.f ? 1.f : sc;
#pragma unroll
          for (int r = 0; r < 16; ++r) g[r] *= mul;
        }
#pragma unroll
        for (int k2 = 0; k2 < 2; ++k2) {
          const v8 pf = acc_frag<T>(s, k2 * 8), df = acc_frag<T>(g, k2 * 8);
#pragma unroll
          for (int b = 0; b < DB; ++b) {
            gv[b] = Elem<T>::mma(col_frag<T, NC>(o_lds, u * 32 + k2 * 16, b, lane), pf, gv[b]);
            gk[b] = Elem<T>::mma(col_frag<T, NC>(q_lds, u * 32 + k2 * 16, b, lane), df, gk[b]);
          }
        }
      }
    }
    if (t + 1 < nt) land((t + 1) & 1);
  }
  if (!live) return;
  const float k_out = p.scale / (sc == 0.f ? 1.f : sc), v_out = Elem<T>::kNarrow ? 0x1p-14f : 1.f;
  char* kp = p.dk + ((int64_t)(it.k0 + key) * p.dk_ts + (int64_t)hk * p.dk_hs) * 2;
  char* vp = p.dv + ((int64_t)(it.k0 + key) * p.dv_ts + (int64_t)hk * p.dv_hs) * 2;
#pragma unroll
  for (int b = 0; b < DB; ++b)
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int d = b * 32 + x * 8 + h * 4;
      if (DP == dim || d < dim) {
        store4<T>(kp + d * 2, gk[b][4 * x] * k_out, gk[b][4 * x + 1] * k_out, gk[b][4 * x + 2] * k_out, gk[b][4 * x + 3] * k_out);
        store4<T>(vp + d * 2, gv[b][4 * x] * v_out, gv[b][4 * x + 1] * v_out, gv[b][4 * x + 2] * v_out, gv[b][4 * x + 3] * v_out);
      }
    }
}

// dq of the rows of one item (32 rows a wave), transposed as in the forward pass
template <typename T, int DP, int NW>
__global__ __launch_bounds__(NW * 64, 2) void attn_dq_kernel(Params p) {
  typedef typename Elem<T>::v8 v8;
  constexpr int NC = DP / 8, KS = DP / 16, DB = DP / 32;
  constexpr int kTile = kKeys * DP * 2;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x & 63, h = lane >> 5, n = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int hk = blockIdx.x % p.kv_heads;
  const RowItem it = p.rows[blockIdx.x / p.kv_heads];
  const int dim = p.dim;
  if (DP != dim) {
    for (int i = threadIdx.x; i < 4 * kTile / 16; i += NW * 64) reinterpret_cast<f32x4*>(smem)[i] = f32x4{0, 0, 0, 0};
    __syncthreads();
  }
  const int n_rows = it.nq * p.group;
  const int row = wave * 32 + n;
  const bool live = row < n_rows;
  const int tok = live ? (row * p.group_inv) >> 16 : 0;
  const int head = hk * p.group + (live ? row - tok * p.group : 0);
  const int lim = live ? (p.causal ? min(it.klen, it.koff + tok + 1) : it.klen) : 0;
  const bool wave_live = wave * 32 < n_rows;
  v8 qf[KS], of[KS];
  {
    const char* qp = p.q + ((int64_t)(it.q0 + tok) * p.q_ts + (int64_t)head * p.q_hs) * 2;
    const char* op = p.d_o + ((int64_t)(it.q0 + tok) * p.do_ts + (int64_t)head * p.do_hs) * 2;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int d = (2 * ks + h) * 8;
      const v8 z = {};
      const bool in = live && (DP == dim || d < dim);
      qf[ks] = in ? *reinterpret_cast<const v8*>(qp + d * 2) : z;
      of[ks] = in ? *reinterpret_cast<const v8*>(op + d * 2) : z;
    }
  }
  const int64_t li = (int64_t)(it.q0 + tok) * p.heads + head;
  const float lse = live ? p.lse[li] : 0.f, delta = live ? p.delta[li] : 0.f;
  int lim_lo, lim_hi;
  {
    const int first = (wave * 32 * p.group_inv) >> 16, last = ((min(wave * 32 + 32, n_rows) - 1) * p.group_inv) >> 16;
    lim_lo = p.causal ? min(it.klen, it.koff + first + 1) : it.klen;
    lim_hi = p.causal ? min(it.klen, it.koff + last + 1) : it.klen;
  }
  f32x16 acc[DB];
#pragma unroll
  for (int b = 0; b < DB; ++b)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[b][r] = 0.f;
  const float c = p.scale_log2;
  float sc = Elem<T>::kNarrow ? 0.f : 1.f;  // factor of ds in acc, one for each row (0: none chosen yet)

  const Stager<NC, NW, kKeys> stager(wave, lane);
  const int nt = (it.ke + kKeys - 1) / kKeys;
  auto stage = [&](int t, int buf) {
    const int kt = t * kKeys, have = min(kKeys, it.ke - kt);
    const int kst = (int)p.k_ts * 2, vst = (int)p.v_ts * 2;
    const __amdgpu_buffer_rsrc_t kr = dense::tile_rsrc_u(p.k + ((int64_t)(it.k0 + kt) * p.k_ts + (int64_t)hk * p.k_hs) * 2,
                                                         (uint32_t)((have - 1) * kst + dim * 2));
    const __amdgpu_buffer_rsrc_t vr = dense::tile_rsrc_u(p.v + ((int64_t)(it.k0 + kt) * p.v_ts + (int64_t)hk * p.v_hs) * 2,
                                                         (uint32_t)((have - 1) * vst + dim * 2));
    char* tile = smem + buf * 2 * kTile;
    stager.load(kr, tile, dim, [&](int r) { return min(r, have - 1) * kst; });
    stager.load(vr, tile + kTile, dim, [&](int r) { return min(r, have - 1) * vst; });
  };
  if (nt > 0) stage(0, 0);
  for (int t = 0; t < nt; ++t) {
    __syncthreads();
    if (t + 1 < nt) stage(t + 1, (t + 1) & 1);
    const int kt = t * kKeys;
    if (!wave_live || kt >= min(it.ke, lim_hi)) continue;
    const char* kt_lds = smem + (t & 1) * 2 * kTile;
    const char* vt_lds = kt_lds + kTile;
    const bool cut = kt + kKeys > it.ke || kt + kKeys > lim_lo;
    const int mine = min(lim, it.ke) - kt;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      f32x16 s, g;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = g[r] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) s = Elem<T>::mma(row_frag<T, NC>(kt_lds, u * 32 + n, ks, h), qf[ks], s);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) g = Elem<T>::mma(row_frag<T, NC>(vt_lds, u * 32 + n, ks, h), of[ks], g);
#pragma unroll
      for (int r = 0; r < 16; ++r) g[r] = ex2(fmaf(s[r], c, -lse)) * (g[r] - delta);
      if (cut) {
#pragma unroll
        for (int r = 0; r < 16; ++r) g[r] = u * 32 + acc_row(r, h) < mine ? g[r] : 0.f;
      }
      if constexpr (Elem<T>::kNarrow) {
        float most = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) most = fmaxf(most, fabsf(g[r]));
        most = fmaxf(most, other_half(most));
        const bool grow = (most * sc > kWide || (sc == 0.f && most > 0.f)) && most < INFINITY;
        if (__any(grow)) {
          const float to = grow ? pick_scale(most) : sc, f2 = grow && sc != 0.f ? to / sc : 1.f;
#pragma unroll
          for (int b = 0; b < DB; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[b][r] *= f2;
          sc = to;
        }
        const float mul = sc == 0.f ? 1.f : sc;
#pragma unroll
        for (int r = 0; r < 16; ++r) g[r] *= mul;
      }
#pragma unroll
      for (int k2 = 0; k2 < 2; ++k2) {
        const v8 df = acc_frag<T>(g, k2 * 8);
#pragma unroll
        for (int b = 0; b < DB; ++b)
          acc[b] = Elem<T>::mma(col_frag<T, NC>(kt_lds, u * 32 + k2 * 16, b, lane), df, acc[b]);
      }
    }
  }
  if (!live) return;
  const float q_out = p.scale / (sc == 0.f ? 1.f : sc);
  char* qp = p.dq + ((int64_t)(it.q0 + tok) * p.dq_ts + (int64_t)head * p.dq_hs) * 2;
#pragma unroll
  for (int b = 0; b < DB; ++b)
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int d = b * 32 + x * 8 + h * 4;
      if (DP == dim || d < dim)
        store4<T>(qp + d * 2, acc[b][4 * x] * q_out, acc[b][4 * x + 1] * q_out, acc[b][4 * x + 2] * q_out, acc[b][4 * x + 3] * q_out);
    }
}

template <typename T, int DP, int NW>
static int launch_dkv(const Params& p, hipStream_t s) {
  constexpr int lds = 2 * (2 * kRowsB * DP * 2 + 2 * kRowsB * 4);
  static std::atomic<uint64_t> done{0};
  ensure_lds_attr(done, reinterpret_cast<const void*>(attn_dkv_kernel<T, DP, NW>), lds);
  attn_dkv_kernel<T, DP, NW><<<dim3((unsigned)(p.n_keys * p.kv_heads)), NW * 64, lds, s>>>(p);
  AHR_HIP(hipGetLastError());
  return AHR_OK;
}

template <typename T, int DP, int NW>
static int launch_dq(const Params& p, hipStream_t s) {
  constexpr int lds = 4 * kKeys * DP * 2;
  static std::atomic<uint64_t> done{0};
  ensure_lds_attr(done, reinterpret_cast<const void*>(attn_dq_kernel<T, DP, NW>), lds);
  attn_dq_kernel<T, DP, NW><<<dim3((unsigned)(p.n_rows * p.kv_heads)), NW * 64, lds, s>>>(p);
  AHR_HIP(hipGetLastError());
  return AHR_OK;
}

template <typename T, int DP>
static int launch_bwd_d(const ahr_attn_plan& pl, const Params& p, hipStream_t s) {
  int st = AHR_OK;
  if (p.n_keys) {
    if (pl.key_waves == 1) st = launch_dkv<T, DP, 1>(p, s);
    else if (pl.key_waves == 2) st = launch_dkv<T, DP, 2>(p, s);
    else st = launch_dkv<T, DP, 4>(p, s);
    if (st != AHR_OK) return st;
  }
  if (p.n_rows) {
    if (pl.waves == 1) st = launch_dq<T, DP, 1>(p, s);
    else if (pl.waves == 2) st = launch_dq<T, DP, 2>(p, s);
    else st = launch_dq<T, DP, 4>(p, s);
  }
  return st;
}

template <typename T>
static int launch_bwd(const ahr_attn_plan& pl, const Params& p, hipStream_t s) {
  const int64_t rows = pl.tokens * p.heads;
  if (rows > 0) {
    attn_delta_kernel<T><<<dim3((unsigned)((rows + 15) / 16)), 256, 0, s>>>(p, rows);
    AHR_HIP(hipGetLastError());
  }
  if (p.dim <= 32) return launch_bwd_d<T, 32>(pl, p, s);
  if (p.dim <= 64) return launch_bwd_d<T, 64>(pl, p, s);
  if (p.dim <= 96) return launch_bwd_d<T, 96>(pl, p, s);
  return launch_bwd_d<T, 128>(pl, p, s);
}

int launch_backward(const ahr_attn_args* a, const Params& p, hipStream_t s) {
  if (a->plan->shape.dtype == AHR_BF16) return launch_bwd<__bf16>(*a->plan, p, s);
  return launch_bwd<_Float16>(*a->plan, p, s);
}

}  // namespace attn
}  // namespace ahr
