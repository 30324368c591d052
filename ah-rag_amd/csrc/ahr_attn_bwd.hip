// Attention over packed sequences, backward (include/ahr.h ahr_attn_backward).
//
// With p = 2^(c s - lse), delta = sum_d do o (= sum_j p (do . v)) and ds = p (do . v - delta):
//   dv_j = sum_i p_ij do_i,   dk_j = scale sum_i ds_ij q_i,   dq_i = scale sum_j ds_ij k_j.
// Two kernels recompute p, one for each direction of the sum: dk and dv stay in the registers of the
// wave that owns 32 keys while the query rows of every head of the group pass through LDS; dq stays
// with the wave that owns 32 rows while the keys pass. That is seven matrix products where one kernel
// needs five, but nothing is added through memory: no atomics, no fp32 copy of dq, the same bits
// every time.
//
// What bounds it (kernel times in calls one after the other): 3 causal sequences of 0.7k-4.1k tokens, 16/4 heads of 128,
// bf16: dq 143 us (three products, 0.79 PFLOP/s), dk and dv 200 us (four, 0.75), the sums of cut key tiles 11. The dk/dv
// kernel holds 128 accumulators and 64 registers of keys and values a lane, so one wave a SIMD, which issues products (38 %
// of its time) and the vector instructions between them in turn; its pieces fill 256 slots to 0.8. 64 texts of up to 384
// tokens, 12 heads of 64: dq 30 us, dk and dv 41. Measured and not kept (of dk and dv, then at 235 us): the exponentials of
// one half of a tile issued between the products of the other (228 us; 43 for the texts), accumulators in ordinary
// registers (about 290), eight waves with the products' roles split between them.
#include "ahr_attn_common.h"

namespace ahr {
namespace attn {

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

// f16: ds of the tile times the state's factor, which is chosen and lowered here (ROW: one factor for each
// row, held by its lane; else one for the wave). acc: the accumulators that hold ds already.
template <int DB, bool ROW>
__device__ __forceinline__ void scale_ds(f32x16& g, f32x16 (&acc)[DB], float& sc) {
  float most = 0.f;
#pragma unroll
  for (int r = 0; r < 16; ++r) most = fmaxf(most, fabsf(g[r]));
  if (ROW) most = fmaxf(most, other_half(most));
  bool grow = (most * sc > kWide || (sc == 0.f && most > 0.f)) && most < INFINITY;
  if (__any(grow)) {
    if (!ROW) {
      most = most < INFINITY ? most : 0.f;
#pragma unroll
      for (int x = 1; x < 64; x *= 2) most = fmaxf(most, __shfl_xor(most, x, 64));
      grow = true;
    }
    const float to = grow ? pick_scale(most) : sc, f = grow && sc != 0.f ? to / sc : 1.f;
#pragma unroll
    for (int b = 0; b < DB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[b][r] *= f;
    sc = to;
  }
  const float mul = sc == 0.f ? 1.f : sc;
#pragma unroll
  for (int r = 0; r < 16; ++r) g[r] *= mul;
}

// ---- dk, dv ------------------------------------------------------------------------------------

constexpr int kStageRows = 64;  // query rows of a staged tile

template <int DP>
struct KeyCfg {
  static constexpr int kTile = kStageRows * DP * 2;
  static constexpr int kRowVals = 2 * kTile;               // lse and delta of the rows (and two spare copies)
  static constexpr int kBuf = kRowVals + 4 * kStageRows * 4;
  // Three tiles: with wide heads a SIMD holds one wave, and the loads of one tile take about as long as its
  // products, so they are issued two tiles ahead.
  static constexpr int kBufs = 3;
  static constexpr int kLoads = 2 * Stager<DP / 8, kWaves, kStageRows>::kPer + 1;  // of a tile, for each wave
};

// A wave's 32 keys: their rows of k and v, and the transposed sums.
template <typename T, int DP>
struct KeyState {
  typename Elem<T>::v8 kf[DP / 16], vf[DP / 16];
  f32x16 gk[DP / 32], gv[DP / 32];
  float sc;  // factor of ds in gk (0: none chosen yet)
};

// 32 query rows (from row u0 of the staged tiles) against the wave's keys; `cut`: only rows [from, have) of
// the tile read this lane's key.
template <typename T, int DP>
__device__ __forceinline__ void key_tile(const char* __restrict__ q_lds, const char* __restrict__ o_lds, const float* __restrict__ f,
                                         KeyState<T, DP>& st, int u0, bool cut, int from, int have, float c, int lane) {
  typedef typename Elem<T>::v8 v8;
  constexpr int NC = DP / 8, KS = DP / 16, DB = DP / 32;
  const int h = lane >> 5, n = lane & 31;
  f32x16 s, g;
#pragma unroll
  for (int r = 0; r < 16; ++r) s[r] = g[r] = 0.f;
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    s = Elem<T>::mma(row_frag<T, NC>(q_lds, u0 + n, ks, h), st.kf[ks], s);
    g = Elem<T>::mma(row_frag<T, NC>(o_lds, u0 + n, ks, h), st.vf[ks], g);
  }
  reads_ahead<2 * KS, 1>();
#pragma unroll
  for (int r4 = 0; r4 < 4; ++r4) {
    const f32x4 ls = *reinterpret_cast<const f32x4*>(f + u0 + r4 * 8 + h * 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) s[r4 * 4 + i] = ex2(fmaf(s[r4 * 4 + i], c, -ls[i]));
    const f32x4 de = *reinterpret_cast<const f32x4*>(f + kStageRows + u0 + r4 * 8 + h * 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) g[r4 * 4 + i] = s[r4 * 4 + i] * (g[r4 * 4 + i] - de[i]);
  }
  if (cut) {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int x = u0 + acc_row(r, h);
      const bool in = x >= from && x < have;
      s[r] = in ? s[r] : 0.f;
      g[r] = in ? g[r] : 0.f;
    }
  }
  if constexpr (Elem<T>::kNarrow) {
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] *= 0x1p14f;
    scale_ds<DB, false>(g, st.gk, st.sc);
  }
#pragma unroll
  for (int k2 = 0; k2 < 2; ++k2) {
    const v8 pf = acc_frag<T>(s, k2 * 8), df = acc_frag<T>(g, k2 * 8);
#pragma unroll
    for (int b = 0; b < DB; ++b) {
      st.gv[b] = Elem<T>::mma(col_frag<T, NC>(o_lds, u0 + k2 * 16, b, lane), pf, st.gv[b]);
      st.gk[b] = Elem<T>::mma(col_frag<T, NC>(q_lds, u0 + k2 * 16, b, lane), df, st.gk[b]);
    }
  }
  reads_ahead<4 * DB, 2>();
}

// The query rows (token, head of the group) of an item from token t0 on, tile by tile: where a tile starts.
struct KeyWalk {
  int G, ginv, coff;
  int64_t n_rows;
  int tok0, g0;  // first token (past t0) and head
  __device__ __forceinline__ void next(int rows_tok, int rows_g) {  // rows of a tile = rows_tok * G + rows_g
    tok0 += rows_tok;
    g0 += rows_g;
    if (g0 >= G) {
      g0 -= G;
      ++tok0;
    }
  }
};

// Loads of the tile that starts at w, `have` rows.
template <int DP>
__device__ __forceinline__ void key_stage(char* __restrict__ nxt, const Stager<DP / 8, kWaves, kStageRows>& stager, const Params& p,
                                          const KeyItem& it, const KeyWalk& w, int hk, int have) {
  typedef KeyCfg<DP> Cfg;
  const int G = w.G, g0 = w.g0;
  const int64_t at = (int64_t)it.q0 + it.t0 + w.tok0;
  const int qts = (int)p.q_ts * 2, qhs = (int)p.q_hs * 2, ots = (int)p.do_ts * 2, ohs = (int)p.do_hs * 2;
  const uint32_t span = (uint32_t)((g0 + have - 1) * w.ginv) >> 16;  // tokens past the first
  const __amdgpu_buffer_rsrc_t qr =
      dense::tile_rsrc_u(p.q + (at * p.q_ts + (int64_t)hk * G * p.q_hs) * 2, span * qts + (G - 1) * qhs + p.dim * 2);
  const __amdgpu_buffer_rsrc_t dr =
      dense::tile_rsrc_u(p.d_o + (at * p.do_ts + (int64_t)hk * G * p.do_hs) * 2, span * ots + (G - 1) * ohs + p.dim * 2);
  constexpr int step = Stager<DP / 8, kWaves, kStageRows>::kStep;
  if (DP != 96 && have == kStageRows && step % G == 0) {  // whole tokens a step, so g0 = 0
    const int tk = (stager.row0 * w.ginv) >> 16, g = stager.row0 - tk * G;
    if (p.dim == DP || stager.c0 * 8 < p.dim) {
      stager.load_full(qr, nxt, __mul24(tk, qts) + g * qhs, step / G * qts);
      stager.load_full(dr, nxt + Cfg::kTile, __mul24(tk, ots) + g * ohs, step / G * ots);
    }
  } else {
    auto off = [&](int r, int ts, int hs) {
      const int x = g0 + min(r, have - 1);
      const int tk = __mul24(x, w.ginv) >> 16;
      return __mul24(tk, ts) + (x - __mul24(tk, G)) * hs;
    };
    stager.load(qr, nxt, p.dim, [&](int r) { return off(r, qts, qhs); });
    stager.load(dr, nxt + Cfg::kTile, p.dim, [&](int r) { return off(r, ots, ohs); });
  }
  // one value a lane: lse by wave 0, delta by wave 1 (2 and 3 repeat them, so that all waves count the same loads)
  const float* vals = (stager.wave & 1 ? p.delta : p.lse) + at * p.heads + (int64_t)hk * G;
  const __amdgpu_buffer_rsrc_t vr = dense::tile_rsrc_u(vals, (span * p.heads + G) * 4);
  const int x = g0 + min(stager.lane, have - 1), tk = __mul24(x, w.ginv) >> 16;
  __builtin_amdgcn_raw_ptr_buffer_load_lds(vr, (__attribute__((address_space(3))) void*)(nxt + Cfg::kRowVals + stager.wave * kStageRows * 4), 4,
                                           (tk * p.heads + x - __mul24(tk, G)) * 4, 0, 0, 0);
}

template <typename T, int DP>
__device__ __forceinline__ void key_step(const char* __restrict__ cur, char* __restrict__ nxt, KeyState<T, DP>& st,
                                         const Stager<DP / 8, kWaves, kStageRows>& stager, const Params& p, const KeyItem& it,
                                         const KeyWalk& w, const KeyWalk& wn, int hk, int t, int nt, bool wave_live, int j, int j_hi, int lane) {
  typedef KeyCfg<DP> Cfg;
  constexpr int ahead = Cfg::kBufs - 1;
  if (t + ahead < nt) key_stage<DP>(nxt, stager, p, it, wn, hk, (int)min((int64_t)kStageRows, w.n_rows - (int64_t)(t + ahead) * kStageRows));
  if (!wave_live) return;
  const int G = w.G, tok0 = w.tok0, g0 = w.g0;
  const int have = (int)min((int64_t)kStageRows, w.n_rows - (int64_t)t * kStageRows);
  const float* f = reinterpret_cast<const float*>(cur + Cfg::kRowVals);
  // A row reads keys j <= coff + its token, which is (g0 + x) / G past tok0: row x reads key j from
  // x = G (j - coff - t0 - tok0) - g0 on.
  const int from = p.causal ? min(max(j - w.coff - it.t0 - tok0, -1), 1 << 20) * G - g0 : 0;
#pragma unroll
  for (int u0 = 0; u0 < kStageRows; u0 += 32) {
    if (u0 >= have) break;
    const int tok_lo = it.t0 + tok0 + (((g0 + u0) * w.ginv) >> 16);
    const bool cut = u0 + 32 > have || (p.causal && j_hi > w.coff + tok_lo);
    key_tile<T, DP>(cur, cur + Cfg::kTile, f, st, u0, cut, from, have, p.scale_log2, lane);
  }
}

// Wide heads: the sums stay in accumulation registers, at both ends of the loop (held in others there, all
// 128 are moved over and back each tile).
template <int DP>
__device__ __forceinline__ void pin(f32x16 (&a)[DP / 32], f32x16 (&b)[DP / 32]) {
  if constexpr (DP > 64) {
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) asm volatile("" : "+a"(a[i]), "+a"(b[i]));
  }
}

template <typename T, int DP>
__device__ __forceinline__ void key_loop(const Params& p, const KeyItem& it, int hk, char* smem, int wave, int lane) {
  typedef KeyCfg<DP> Cfg;
  constexpr int KS = DP / 16, DB = DP / 32;
  const int h = lane >> 5, n = lane & 31, dim = p.dim;
  const int key = wave * 32 + n;
  const bool live = key < it.nk;
  KeyState<T, DP> st;
  {
    const int64_t at = it.k0 + (live ? key : 0);
    load_row<T, DP>(st.kf, p.k + (at * p.k_ts + (int64_t)hk * p.k_hs) * 2, dim, h);
    load_row<T, DP>(st.vf, p.v + (at * p.v_ts + (int64_t)hk * p.v_hs) * 2, dim, h);
  }
#pragma unroll
  for (int b = 0; b < DB; ++b)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      st.gk[b][r] = 0.f;
      st.gv[b][r] = 0.f;
    }
  st.sc = Elem<T>::kNarrow ? 0.f : 1.f;

  const Stager<DP / 8, kWaves, kStageRows> stager(wave, lane);
  KeyWalk w;
  w.G = p.group;
  w.ginv = p.group_inv;
  w.coff = it.klen - it.qlen;
  w.n_rows = (int64_t)(it.t1 - it.t0) * p.group;
  w.tok0 = w.g0 = 0;
  const int nt = (int)((w.n_rows + kStageRows - 1) / kStageRows);
  const bool wave_live = wave * 32 < it.nk;
  const int j = it.kpos + key;                               // this lane's key in its sequence
  const int j_hi = it.kpos + min(wave * 32 + 31, it.nk - 1);  // the wave's last
  const int rows_tok = kStageRows / p.group, rows_g = kStageRows - rows_tok * p.group;
  KeyWalk wn = w;
#pragma unroll
  for (int t = 0; t < Cfg::kBufs - 1; ++t) {
    if (t < nt) key_stage<DP>(smem + t * Cfg::kBuf, stager, p, it, wn, hk, (int)min((int64_t)kStageRows, w.n_rows - (int64_t)t * kStageRows));
    wn.next(rows_tok, rows_g);
  }
  int cur = 0, nxt = (Cfg::kBufs - 1) * Cfg::kBuf;
  pin<DP>(st.gk, st.gv);
  for (int t = 0; t < nt; ++t) {
    // the next tile's loads may stay in flight (all are waited for where lanes without a chunk may skip some)
    if (dim == DP && t + 1 < nt) tile_barrier<Cfg::kLoads>();
    else tile_barrier();
    pin<DP>(st.gk, st.gv);
    key_step<T, DP>(smem + cur, smem + nxt, st, stager, p, it, w, wn, hk, t, nt, wave_live, j, j_hi, lane);
    w.next(rows_tok, rows_g);
    wn.next(rows_tok, rows_g);
    cur = cur + Cfg::kBuf == Cfg::kBufs * Cfg::kBuf ? 0 : cur + Cfg::kBuf;
    nxt = nxt + Cfg::kBuf == Cfg::kBufs * Cfg::kBuf ? 0 : nxt + Cfg::kBuf;
    pin<DP>(st.gk, st.gv);
  }
  if (!live) return;
  const float k_out = p.scale / (st.sc == 0.f ? 1.f : st.sc), v_out = Elem<T>::kNarrow ? 0x1p-14f : 1.f;
  if (it.plane >= 0) {  // [plane][row][key head][dk, dv][dim]
    float* out = p.part_o + ((((int64_t)it.plane * p.prows + it.prow + key) * p.kv_heads + hk) * 2) * dim;
#pragma unroll
    for (int b = 0; b < DB; ++b)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int d = b * 32 + x * 8 + h * 4;
        if (DP != dim && d >= dim) continue;
        const f32x16 &a = st.gk[b], &e = st.gv[b];
        *reinterpret_cast<f32x4*>(out + d) = f32x4{a[4 * x], a[4 * x + 1], a[4 * x + 2], a[4 * x + 3]} * k_out;
        *reinterpret_cast<f32x4*>(out + dim + d) = f32x4{e[4 * x], e[4 * x + 1], e[4 * x + 2], e[4 * x + 3]} * v_out;
      }
    return;
  }
  char* kp = p.dk + ((int64_t)(it.k0 + key) * p.dk_ts + (int64_t)hk * p.dk_hs) * 2;
  char* vp = p.dv + ((int64_t)(it.k0 + key) * p.dv_ts + (int64_t)hk * p.dv_hs) * 2;
#pragma unroll
  for (int b = 0; b < DB; ++b)
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int d = b * 32 + x * 8 + h * 4;
      if (DP != dim && d >= dim) continue;
      const f32x16 &a = st.gk[b], &e = st.gv[b];
      store4<T>(kp + d * 2, a[4 * x] * k_out, a[4 * x + 1] * k_out, a[4 * x + 2] * k_out, a[4 * x + 3] * k_out);
      store4<T>(vp + d * 2, e[4 * x] * v_out, e[4 * x + 1] * v_out, e[4 * x + 2] * v_out, e[4 * x + 3] * v_out);
    }
}

// dk, dv of one item for one key head
template <typename T, int DP>
__global__ __launch_bounds__(kWaves * 64, DP > 64 ? 1 : 2) void attn_dkv_kernel(Params p) {
  typedef KeyCfg<DP> Cfg;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int hk = blockIdx.x % p.kv_heads;
  const KeyItem it = p.keys[blockIdx.x / p.kv_heads];
  if (DP != p.dim) {
    for (int b = 0; b < Cfg::kBufs; ++b)
      for (int i = threadIdx.x; i < 2 * Cfg::kTile / 16; i += kWaves * 64)
        reinterpret_cast<f32x4*>(smem + b * Cfg::kBuf)[i] = f32x4{0, 0, 0, 0};
    __syncthreads();
  }
  key_loop<T, DP>(p, it, hk, smem, wave, lane);
}

// Adds the partial sums of dk and dv, plane after plane: 4 values a thread.
template <typename T>
__global__ __launch_bounds__(256) void attn_sum_kernel(Params p) {
  const JoinItem it = p.join[blockIdx.x];
  const int per = p.kv_heads * 2 * p.dim;  // values of a key
  const int64_t i = ((int64_t)blockIdx.y * 256 + threadIdx.x) * 4;
  if (i >= (int64_t)it.nq * per) return;
  const float* x = p.part_o + (int64_t)it.prow * per + i;
  const int64_t plane = p.prows * per;
  f32x4 s = {0, 0, 0, 0};
#pragma unroll 4
  for (int j = 0; j < it.np; ++j) s += *reinterpret_cast<const f32x4*>(x + j * plane);
  const int key = (int)(i / per), rest = (int)(i - (int64_t)key * per);
  const int hk = rest / (2 * p.dim), at = rest - hk * 2 * p.dim;
  const bool v = at >= p.dim;
  char* o = v ? p.dv + ((int64_t)(it.q0 + key) * p.dv_ts + (int64_t)hk * p.dv_hs + at - p.dim) * 2
              : p.dk + ((int64_t)(it.q0 + key) * p.dk_ts + (int64_t)hk * p.dk_hs + at) * 2;
  store4<T>(o, s[0], s[1], s[2], s[3]);
}

// ---- dq ----------------------------------------------------------------------------------------

template <typename T, int DP>
struct RowState {
  typename Elem<T>::v8 qf[DP / 16], of[DP / 16];
  f32x16 acc[DP / 32];
  float lse, delta, sc;
};

// One staged tile of keys and values for one wave's rows, transposed as in the forward pass.
template <typename T, int DP>
__device__ __forceinline__ void row_tile(const char* __restrict__ cur, RowState<T, DP>& st, bool cut, int mine, float c, int lane) {
  typedef typename Elem<T>::v8 v8;
  constexpr int NC = DP / 8, KS = DP / 16, DB = DP / 32;
  constexpr int kTile = kKeys * DP * 2;
  const int h = lane >> 5, n = lane & 31;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    f32x16 s, g;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = g[r] = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      s = Elem<T>::mma(row_frag<T, NC>(cur, u * 32 + n, ks, h), st.qf[ks], s);
      g = Elem<T>::mma(row_frag<T, NC>(cur + kTile, u * 32 + n, ks, h), st.of[ks], g);
    }
    reads_ahead<2 * KS, 1>();
#pragma unroll
    for (int r = 0; r < 16; ++r) g[r] = ex2(fmaf(s[r], c, -st.lse)) * (g[r] - st.delta);
    if (cut) {
#pragma unroll
      for (int r = 0; r < 16; ++r) g[r] = u * 32 + acc_row(r, h) < mine ? g[r] : 0.f;
    }
    if constexpr (Elem<T>::kNarrow) scale_ds<DB, true>(g, st.acc, st.sc);
#pragma unroll
    for (int k2 = 0; k2 < 2; ++k2) {
      const v8 df = acc_frag<T>(g, k2 * 8);
#pragma unroll
      for (int b = 0; b < DB; ++b) st.acc[b] = Elem<T>::mma(col_frag<T, NC>(cur, u * 32 + k2 * 16, b, lane), df, st.acc[b]);
    }
    reads_ahead<2 * DB, 2>();
  }
}

// delta = sum_j p_j (do . v_j) of this lane's row, whose keys all lie in the first staged tile. Equal to sum_d do o but
// for o's rounding to 16 bits, which with few keys is as large as that of ds (in units of dq, bf16, against
// 0.0024 with an exact delta: 0.0030 for 4 keys a row, 0.0025 for 16, 0.0024 from 64 on, where it hardly counts). So too
// the early rows of a causal sequence whose row tile reads on (31 texts of up to 1154 tokens, 12 heads of 32: dq 0.00255
// off with o's delta for them, 0.00241 so).
template <typename T, int DP>
__device__ __forceinline__ float row_delta(const char* __restrict__ cur, const RowState<T, DP>& st, int mine, float c, int lane) {
  constexpr int NC = DP / 8, KS = DP / 16;
  constexpr int kTile = kKeys * DP * 2;
  const int h = lane >> 5, n = lane & 31;
  float sum = 0.f;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    f32x16 s, g;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = g[r] = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      s = Elem<T>::mma(row_frag<T, NC>(cur, u * 32 + n, ks, h), st.qf[ks], s);
      g = Elem<T>::mma(row_frag<T, NC>(cur + kTile, u * 32 + n, ks, h), st.of[ks], g);
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) sum += u * 32 + acc_row(r, h) < mine ? ex2(fmaf(s[r], c, -st.lse)) * g[r] : 0.f;
  }
  return sum + other_half(sum);
}

template <typename T, int DP>
__device__ __forceinline__ void row_step(const char* __restrict__ cur, char* __restrict__ nxt, RowState<T, DP>& st,
                                         const Stager<DP / 8, kWaves, kKeys>& stager, const Params& p, const RowItem& it, int hk, int t, int nt,
                                         bool wave_live, int lim, int lim_lo, int lim_hi, int lane) {
  if (t + 1 < nt) {
    const int kt = (t + 1) * kKeys;
    const int64_t at = (int64_t)it.k0 + kt;
    stage_kv<DP>(nxt, stager, p.k + (at * p.k_ts + (int64_t)hk * p.k_hs) * 2, p.v + (at * p.v_ts + (int64_t)hk * p.v_hs) * 2, p.k_ts, p.v_ts,
                     min(kKeys, it.ke - kt), p.dim);
  }
  if (t < 0) return;
  const int kt = t * kKeys;
  if (!wave_live || kt >= lim_hi) return;
  row_tile<T, DP>(cur, st, kt + kKeys > it.ke || kt + kKeys > lim_lo, min(lim, it.ke) - kt, p.scale_log2, lane);
}

// dq of the rows of one item, 32 a wave
template <typename T, int DP>
__global__ __launch_bounds__(kWaves * 64, 2) void attn_dq_kernel(Params p) {
  constexpr int KS = DP / 16, DB = DP / 32;
  constexpr int kTile = kKeys * DP * 2;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x & 63, h = lane >> 5, n = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int hk = blockIdx.x % p.kv_heads;
  const RowItem it = p.rows[blockIdx.x / p.kv_heads];
  const int dim = p.dim;
  if (DP != dim) {
    for (int i = threadIdx.x; i < 4 * kTile / 16; i += kWaves * 64) reinterpret_cast<f32x4*>(smem)[i] = f32x4{0, 0, 0, 0};
    __syncthreads();
  }
  const int n_rows = it.nq * p.group;
  const int row = wave * 32 + n;
  const bool live = row < n_rows;
  const int tok = live ? (row * p.group_inv) >> 16 : 0;
  const int head = hk * p.group + (live ? row - tok * p.group : 0);
  const int lim = live ? (p.causal ? min(it.klen, it.koff + tok + 1) : it.klen) : 0;
  const bool wave_live = wave * 32 < n_rows;
  const int first = (wave * 32 * p.group_inv) >> 16, last = ((min(wave * 32 + 32, n_rows) - 1) * p.group_inv) >> 16;
  const int lim_lo = p.causal ? min(it.klen, it.koff + first + 1) : it.klen;
  const int lim_hi = p.causal ? min(it.klen, it.koff + last + 1) : it.klen;
  RowState<T, DP> st;
  const int64_t qt = it.q0 + tok;
  typename Elem<T>::v8 ov[KS];
  load_row<T, DP>(st.qf, p.q + (qt * p.q_ts + (int64_t)head * p.q_hs) * 2, dim, h);
  load_row<T, DP>(st.of, p.d_o + (qt * p.do_ts + (int64_t)head * p.do_hs) * 2, dim, h);
  load_row<T, DP>(ov, p.o + (qt * p.o_ts + (int64_t)head * p.o_hs) * 2, dim, h);
  const int64_t li = qt * p.heads + head;
  st.lse = live ? p.lse[li] : 0.f;
  st.sc = Elem<T>::kNarrow ? 0.f : 1.f;
#pragma unroll
  for (int b = 0; b < DB; ++b)
#pragma unroll
    for (int r = 0; r < 16; ++r) st.acc[b][r] = 0.f;

  const Stager<DP / 8, kWaves, kKeys> stager(wave, lane);
  const int nt = (it.ke + kKeys - 1) / kKeys;
  if (nt > 0) row_step<T, DP>(smem, smem, st, stager, p, it, hk, -1, nt, false, 0, 0, 0, lane);
  {  // delta of this lane's row, written for the dk/dv kernel that follows
    float x = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int i = 0; i < 8; ++i) x = fmaf((float)ov[ks][i], (float)st.of[ks][i], x);
    st.delta = x + other_half(x);
    // where the rows of the workgroup's first wave, which read the fewest keys, have them in the first tile
    const int few = p.causal ? min(it.klen, it.koff + (((min(32, n_rows) - 1) * p.group_inv) >> 16) + 1) : it.klen;
    if (nt > 0 && few <= kKeys) {
      tile_barrier();
      if (wave_live && lim_hi <= kKeys) st.delta = row_delta<T, DP>(smem, st, min(lim, it.ke), p.scale_log2, lane);
    }
    if (live && h == 0) p.delta[li] = st.delta;
  }
  if (nt > 0) {
    for (int t = 0; t < nt; ++t) {
      tile_barrier();
      row_step<T, DP>(smem + (t & 1) * 2 * kTile, smem + ((t + 1) & 1) * 2 * kTile, st, stager, p, it, hk, t, nt, wave_live, lim, lim_lo,
                          lim_hi, lane);
    }
  }
  if (!live) return;
  const float q_out = p.scale / (st.sc == 0.f ? 1.f : st.sc);
  char* qp = p.dq + ((int64_t)(it.q0 + tok) * p.dq_ts + (int64_t)head * p.dq_hs) * 2;
#pragma unroll
  for (int b = 0; b < DB; ++b)
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int d = b * 32 + x * 8 + h * 4;
      if (DP == dim || d < dim) {
        const f32x16& a = st.acc[b];
        store4<T>(qp + d * 2, a[4 * x] * q_out, a[4 * x + 1] * q_out, a[4 * x + 2] * q_out, a[4 * x + 3] * q_out);
      }
    }
}

template <typename T, int DP>
static int launch_dkv(const ahr_attn_plan& pl, const Params& p, hipStream_t s) {
  constexpr int lds = KeyCfg<DP>::kBufs * KeyCfg<DP>::kBuf;
  static std::atomic<uint64_t> done{0};
  ensure_lds_attr(done, reinterpret_cast<const void*>(attn_dkv_kernel<T, DP>), lds);
  attn_dkv_kernel<T, DP><<<dim3((unsigned)(p.n_keys * p.kv_heads)), kWaves * 64, lds, s>>>(p);
  AHR_HIP(hipGetLastError());
  if (p.n_join) {
    const int64_t vals = (int64_t)pl.join_tokens * p.kv_heads * 2 * p.dim;
    attn_sum_kernel<T><<<dim3((unsigned)p.n_join, (unsigned)((vals + 1023) / 1024)), 256, 0, s>>>(p);
    AHR_HIP(hipGetLastError());
  }
  return AHR_OK;
}

template <typename T, int DP>
static int launch_dq(const Params& p, hipStream_t s) {
  constexpr int lds = 4 * kKeys * DP * 2;
  static std::atomic<uint64_t> done{0};
  ensure_lds_attr(done, reinterpret_cast<const void*>(attn_dq_kernel<T, DP>), lds);
  attn_dq_kernel<T, DP><<<dim3((unsigned)(p.n_rows * p.kv_heads)), kWaves * 64, lds, s>>>(p);
  AHR_HIP(hipGetLastError());
  return AHR_OK;
}

template <typename T, int DP>
static int launch_bwd_d(const ahr_attn_plan& pl, const Params& p, hipStream_t s) {
  if (p.n_rows) {
    const int st = launch_dq<T, DP>(p, s);  // writes delta, so it comes first
    if (st != AHR_OK) return st;
  }
  return p.n_keys ? launch_dkv<T, DP>(pl, p, s) : AHR_OK;
}

template <typename T>
static int launch_bwd(const ahr_attn_plan& pl, const Params& p, hipStream_t s) {
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
