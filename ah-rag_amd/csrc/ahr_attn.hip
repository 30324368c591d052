// Attention over packed sequences, forward (include/ahr.h ahr_attn_forward), and the host planner of
// both directions.
//
// For a row (query token t, head h) with keys j: o = sum_j p_j v_j / sum_j p_j, p_j = 2^(c s_j - m),
// s_j = q . k_j, c = scale log2(e). One pass over the keys with a running reference m: p and the
// accumulators are relative to m, which is raised (and they are rescaled) only when a tile's maximum
// exceeds it by more than 8, so p <= 2^8 and almost every tile skips the rescale.
//
// Layout. A workgroup takes 32 rows per wave; the rows of a tile are (token, head of the group), so
// the query heads that share a key head read its keys once. Scores are computed transposed,
// S^T = K Q^T (32x32x16 MFMA): a lane then holds one row's scores of 16 keys, the maximum and sum
// stay within the lane and its other half, and S^T's registers are, converted to 16 bits, exactly the
// second operand of O^T = V^T P^T when V^T is read with its keys in accumulator order (col_frag). Keys
// and values go through LDS by DMA, double buffered, one barrier per 64 keys.
//
// What bounds it (kernel times in calls one after the other on the same inputs). Many rows: the matrix units, whose
// products and the exponentials between them overlap only across the two waves of a SIMD (4 causal sequences of
// 1.5k-8.2k tokens, 32/8 heads of 128, bf16: 1.09-1.12 ms, 1.0 PFLOP/s where a library product of 8192^3 reaches 1.18; up to
// 1.30 ms where each call follows a pause). Single tokens: memory (24 over 1k-33k keys each, 8 key heads of 128, f16: 236
// us and 7 for the join, 5.5 TB/s). Short texts lie between (256 of up to 384 tokens, 12 heads of 64: 73 to 87 us from
// one card to the next, 2.8 to 3.3 TB/s). Few workgroups (64 queries of 4-40 tokens behind a prefix of 900, 16/8 heads of
// 64: 19 us and 5 for the join) wait out each tile's chain of barrier, products, exponentials, products, at most five in
// a row; that chain, the start and the partial rows' way through memory were not told apart. Measured and not kept, each
// against the form of its time: three tile buffers instead of two (a third slower for the long sequences, no change for
// the prefix), two waves that share a tile's keys where an item has few rows (6 % less for the prefix, but 2 % more for
// the long ones) and an order of the workgroups that spreads key heads over the XCDs (10 % more).
#include "ahr_attn_common.h"

#include <algorithm>
#include <cmath>
#include <cstring>
#include <vector>

namespace ahr {
namespace attn {

constexpr float kRaise = 8.f;  // how far (log2) a score may exceed the reference before it is raised
// The exponent c s - m is one rounding of the exact value, while m itself is rounded: past 2^24 the largest weight is off
// by a power of two, which l shares, but which passes f16's range from 2^27 on and fp32's from 2^31.
constexpr float kFar = 0x1p26f;
constexpr float kNone = -3.4028234663852886e38f;  // log-sum of a piece whose keys' scores are all minus infinity

// What a wave carries from tile to tile: its 32 rows' queries, and one row for each lane (the other
// half-lane the same row, other keys).
template <typename T, int DP>
struct FwdState {
  typename Elem<T>::v8 qf[DP / 16];
  f32x16 acc[DP / 32];  // o, transposed
  float m, l;           // reference (of c s), this half-lane's part of the sum
};

// One staged tile of keys and values (cur) for one wave: the first `mine` keys count for this lane's
// row; `cut`: not the same 64 for all rows of the wave.
// (cur is restrict: the reads must not wait for the DMA that fills the other buffer meanwhile.)
template <typename T, int DP>
__device__ __forceinline__ void fwd_tile(const char* __restrict__ cur, FwdState<T, DP>& st, bool cut, int mine, float c, int lane) {
  typedef typename Elem<T>::v8 v8;
  constexpr int NC = DP / 8, KS = DP / 16, DB = DP / 32;
  constexpr int kTile = kKeys * DP * 2;
  const int h = lane >> 5, n = lane & 31;
  f32x16 s[2];
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int r = 0; r < 16; ++r) s[u][r] = 0.f;
#pragma unroll
  for (int ks = 0; ks < KS; ++ks)
#pragma unroll
    for (int u = 0; u < 2; ++u) s[u] = Elem<T>::mma(row_frag<T, NC>(cur, u * 32 + n, ks, h), st.qf[ks], s[u]);
  reads_ahead<2 * KS, 1>();

  if (cut) {  // keys that a row does not read: selected away, whatever their scores are
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[u][r] = u * 32 + acc_row(r, h) < mine ? s[u][r] : -INFINITY;
  }

  float top = s[0][0];
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int r = 0; r < 16; ++r) top = fmaxf(top, s[u][r]);
  top = fmaxf(top, other_half(top)) * c;
  if (__any(top > st.m + kRaise)) {  // (m = -inf before the first key)
    const float to = fmaxf(st.m, top);
    const float f = to == -INFINITY ? 1.f : ex2(st.m - to);
    st.l *= f;
#pragma unroll
    for (int b = 0; b < DB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) st.acc[b][r] *= f;
    st.m = to;
  }
  const float ref = st.m == -INFINITY ? 0.f : st.m;
  float add = 0.f;
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      s[u][r] = ex2(fmaf(s[u][r], c, -ref));
      add += s[u][r];
    }
  st.l += add;

#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const v8 pf = acc_frag<T>(s[g >> 1], (g & 1) * 8);
#pragma unroll
    for (int b = 0; b < DB; ++b) st.acc[b] = Elem<T>::mma(col_frag<T, NC>(cur + kTile, g * 16, b, lane), pf, st.acc[b]);
  }
  reads_ahead<4 * DB, 2>();
}

// The row of this lane again, in plain steps: where a product of zero weights with a value that is not finite
// reached an accumulator (a tile's matrix product multiplies every row's weight, also the zero of a key that
// the row does not read, with every value), where inputs that the row does read are not finite, or where its scores
// are too large for weights relative to a rounded reference (the largest score is subtracted before the scale).
template <typename T, int DP>
__device__ __forceinline__ void strict_row(FwdState<T, DP>& st, const Params& p, const RowItem& it, int hk, int head, int tok, int lim, int h) {
  typedef typename Elem<T>::v8 v8;
  typedef typename Elem<T>::v4 v4;
  const char* qp = p.q + ((int64_t)(it.q0 + tok) * p.q_ts + (int64_t)head * p.q_hs) * 2;
  auto score = [&](const char* k) {
    float x = 0.f;
    for (int d = 0; d < p.dim; d += 8) {
      const v8 a = *reinterpret_cast<const v8*>(qp + d * 2), b = *reinterpret_cast<const v8*>(k + d * 2);
#pragma unroll
      for (int i = 0; i < 8; ++i) x = fmaf((float)a[i], (float)b[i], x);
    }
    return x;
  };
  auto each = [&](auto f) {
    for (int j = it.pb; j < it.pe; ++j) f(p.pk + ((int64_t)j * p.pk_ts + hk * p.pk_hs) * 2, p.pv + ((int64_t)j * p.pv_ts + hk * p.pv_hs) * 2);
    for (int j = it.kb; j < min(it.ke, lim); ++j)
      f(p.k + ((int64_t)(it.k0 + j) * p.k_ts + hk * p.k_hs) * 2, p.v + ((int64_t)(it.k0 + j) * p.v_ts + hk * p.v_hs) * 2);
  };
  float m = -INFINITY;
  each([&](const char* k, const char*) { m = fmaxf(m, score(k)); });
  const float ref = m == -INFINITY ? 0.f : m;
  st.m = m == -INFINITY ? m : fminf(fmaxf(m * p.scale_log2, 0.5f * kNone), -0.5f * kNone);
  st.l = 0.f;
#pragma unroll
  for (int b = 0; b < DP / 32; ++b)
#pragma unroll
    for (int r = 0; r < 16; ++r) st.acc[b][r] = 0.f;
  each([&](const char* k, const char* v) {
    const float w = ex2((score(k) - ref) * p.scale_log2);
    if (h == 0) st.l += w;
#pragma unroll
    for (int b = 0; b < DP / 32; ++b)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d = b * 32 + g * 8 + h * 4;
        if (DP != p.dim && d >= p.dim) continue;
        const v4 x = *reinterpret_cast<const v4*>(v + d * 2);
#pragma unroll
        for (int i = 0; i < 4; ++i) st.acc[b][4 * g + i] = fmaf(w, (float)x[i], st.acc[b][4 * g + i]);
      }
  });
}

// Where a partial row lies: planes of the first prows rows one behind the other from the start, those of the far_rows
// others from the end.
__device__ __forceinline__ int64_t part_row(const Params& p, int plane, int row) {
  return row < p.prows ? plane * p.prows + row : p.parts - (plane + 1) * p.far_rows + row - p.prows;
}

template <typename T, int DP>
__device__ __forceinline__ void fwd_step(const char* __restrict__ cur, char* __restrict__ nxt, FwdState<T, DP>& st,
                                         const Stager<DP / 8, kWaves, kKeys>& stager, const Params& p, const RowItem& it, int hk, int t, int np,
                                         int nt, bool wave_live, int lim, int lim_lo, int lim_hi, int lane) {
  auto stage = [&](int t) {
    const bool pre = t < np;
    const int kt = pre ? it.pb + t * kKeys : it.kb + (t - np) * kKeys;
    const int have = min(kKeys, (pre ? it.pe : it.ke) - kt);
    const int64_t at = pre ? kt : (int64_t)it.k0 + kt;
    const int64_t kts = pre ? p.pk_ts : p.k_ts, vts = pre ? p.pv_ts : p.v_ts;
    stage_kv<DP>(nxt, stager, (pre ? p.pk : p.k) + (at * kts + hk * (pre ? p.pk_hs : p.k_hs)) * 2,
                     (pre ? p.pv : p.v) + (at * vts + hk * (pre ? p.pv_hs : p.v_hs)) * 2, kts, vts, have, p.dim);
  };
  if (t + 1 < nt) stage(t + 1);
  if (t < 0) return;
  const bool pre = t < np;
  const int kt = pre ? it.pb + t * kKeys : it.kb + (t - np) * kKeys;
  const int stop = pre ? it.pe : it.ke;
  if (!wave_live || (!pre && kt >= lim_hi)) return;  // no row of the wave reads from here on
  fwd_tile<T, DP>(cur, st, kt + kKeys > stop || (!pre && kt + kKeys > lim_lo), (pre ? stop : min(lim, stop)) - kt, p.scale_log2, lane);
}

// (Up to 64 wide: 128 registers, four waves a SIMD. 256 texts of up to 384 tokens, 12 heads of 64: 73 us, 79
// with the 162 registers that the compiler takes when left alone. 20 bytes a lane are put aside for it, before the loop
// over the tiles, and read back after it.)
template <typename T, int DP>
__global__ __launch_bounds__(kWaves * 64, DP <= 64 ? 4 : 2) void attn_fwd_kernel(Params p) {
  constexpr int DB = DP / 32;
  constexpr int kTile = kKeys * DP * 2;
  extern __shared__ __attribute__((aligned(16))) char smem[];  // [2][K tile, V tile]
  const int lane = threadIdx.x & 63, h = lane >> 5, n = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int hk = blockIdx.x % p.kv_heads;
  const RowItem it = p.rows[blockIdx.x / p.kv_heads];
  const int dim = p.dim;

  if (DP != dim) {  // the chunks past dim are never loaded
    for (int i = threadIdx.x; i < 4 * kTile / 16; i += kWaves * 64) reinterpret_cast<f32x4*>(smem)[i] = f32x4{0, 0, 0, 0};
    __syncthreads();
  }

  // this lane's row
  const int n_rows = it.nq * p.group;
  const int row = wave * 32 + n;
  const bool live = row < n_rows;
  const int tok = live ? (row * p.group_inv) >> 16 : 0;
  const int head = hk * p.group + (live ? row - tok * p.group : 0);
  const int lim = live ? (p.causal ? min(it.klen, it.koff + tok + 1) : it.klen) : 0;  // own keys it reads
  const bool wave_live = wave * 32 < n_rows;
  // smallest and largest number of own keys that a row of this wave reads
  const int first = (wave * 32 * p.group_inv) >> 16, last = ((min(wave * 32 + 32, n_rows) - 1) * p.group_inv) >> 16;
  const int lim_lo = p.causal ? min(it.klen, it.koff + first + 1) : it.klen;
  const int lim_hi = p.causal ? min(it.klen, it.koff + last + 1) : it.klen;

  FwdState<T, DP> st;
  load_row<T, DP>(st.qf, p.q + ((int64_t)(it.q0 + tok) * p.q_ts + (int64_t)head * p.q_hs) * 2, dim, h);
#pragma unroll
  for (int b = 0; b < DB; ++b)
#pragma unroll
    for (int r = 0; r < 16; ++r) st.acc[b][r] = 0.f;
  st.m = -INFINITY;
  st.l = 0.f;

  const Stager<DP / 8, kWaves, kKeys> stager(wave, lane);
  const int np = (it.pe - it.pb + kKeys - 1) / kKeys;
  const int nt = np + (it.ke - it.kb + kKeys - 1) / kKeys;
  if (nt > 0) {
    fwd_step<T, DP>(smem, smem, st, stager, p, it, hk, -1, np, nt, false, 0, 0, 0, lane);  // the first tile's loads
    for (int t = 0; t < nt; ++t) {
      tile_barrier();  // tile t has landed, tile t - 1 is no longer read
      fwd_step<T, DP>(smem + (t & 1) * 2 * kTile, smem + ((t + 1) & 1) * 2 * kTile, st, stager, p, it, hk, t, np, nt, wave_live, lim,
                          lim_lo, lim_hi, lane);
    }
  }

  {
    float x[4] = {st.l, 0.f, 0.f, 0.f};
#pragma unroll
    for (int b = 0; b < DB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r & 3] = fmaf(st.acc[b][r], 0.f, x[r & 3]);
    const bool far = st.m > -INFINITY && !(fabsf(st.m) < kFar);
    const bool odd = live && (far || !(fabsf((x[0] + x[1]) + (x[2] + x[3])) < INFINITY));
    if (__any(odd)) {
      // Both halves of a row take the strict path where either has to: they share its weights and its sum. (The
      // exchange runs in every lane: a lane that a branch has switched off hands over nothing.)
      const bool other = __shfl_xor((int)odd, 32, 64) != 0;
      if (odd || other) strict_row<T, DP>(st, p, it, hk, head, tok, lim, h);
    }
  }
  if (!live) return;
  const float l = st.l + other_half(st.l);
  // Without a weight: a row that reads no key here, or keys whose scores are all minus infinity. The first gives zeros, the
  // second has no softmax; in a piece it only adds nothing.
  const bool none = l == 0.f && (it.pe > it.pb || min(it.ke, lim) > it.kb);
  const float inv = l == 0.f ? (none && it.plane < 0 ? NAN : 0.f) : 1.f / l;
  const float lse = l == 0.f ? (none && it.plane >= 0 ? kNone : -INFINITY) : st.m + __log2f(l);
  if (it.plane >= 0) {
    const int64_t at = part_row(p, it.plane, it.prow + tok) * p.heads + head;
    if (h == 0) p.part_l[at] = lse;
    float* op = p.part_o + at * dim;
#pragma unroll
    for (int b = 0; b < DB; ++b)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d = b * 32 + g * 8 + h * 4;
        if (DP == dim || d < dim)
          *reinterpret_cast<f32x4*>(op + d) = f32x4{st.acc[b][4 * g] * inv, st.acc[b][4 * g + 1] * inv,
                                                    st.acc[b][4 * g + 2] * inv, st.acc[b][4 * g + 3] * inv};
      }
    return;
  }
  if (p.lse && h == 0) p.lse[(int64_t)(it.q0 + tok) * p.heads + head] = lse;
  char* op = p.o + ((int64_t)(it.q0 + tok) * p.o_ts + (int64_t)head * p.o_hs) * 2;
#pragma unroll
  for (int b = 0; b < DB; ++b)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = b * 32 + g * 8 + h * 4;
      if (DP == dim || d < dim)
        store4<T>(op + d * 2, st.acc[b][4 * g] * inv, st.acc[b][4 * g + 1] * inv, st.acc[b][4 * g + 2] * inv,
                  st.acc[b][4 * g + 3] * inv);
    }
}

// Joins partial results: o = sum_i 2^(lse_i - max) o_i / sum_i 2^(lse_i - max). dim / 4 lanes (a power of
// two or, with idle lanes, the next) take a row, 4 elements each; every partial value is read once.
template <typename T>
__global__ __launch_bounds__(256) void attn_join_kernel(Params p, int lanes) {
  const JoinItem it = p.join[blockIdx.x];
  const int per = 256 / lanes;  // rows of a workgroup
  const int r = blockIdx.y * per + threadIdx.x / lanes, d = (threadIdx.x % lanes) * 4;
  if (r >= it.nq * p.heads || d >= p.dim) return;
  const int i = r / p.heads, head = r - i * p.heads;
  const int64_t plane = (it.prow < p.prows ? p.prows : -p.far_rows) * p.heads, at = part_row(p, 0, it.prow + i) * p.heads + head;
  const float* pl = p.part_l + at;
  const float* po = p.part_o + at * p.dim + d;
  float m = -INFINITY, sum = 0.f;
  f32x4 a = {0, 0, 0, 0};
  for (int j0 = 0; j0 < it.np; j0 += 8) {  // the loads of 8 planes are in flight together
    float l[8];
    f32x4 x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int64_t o = min(j0 + j, it.np - 1) * plane;
      l[j] = j0 + j < it.np ? pl[o] : -INFINITY;
      x[j] = *reinterpret_cast<const f32x4*>(po + o * p.dim);
    }
    float to = m;
#pragma unroll
    for (int j = 0; j < 8; ++j) to = fmaxf(to, l[j]);
    const float ref = to == -INFINITY ? 0.f : to, f = ex2(m - ref);
    sum *= f;
    a *= f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float w = ex2(l[j] - ref);
      if (j0 + j >= it.np) break;
      sum += w;
      a += w * x[j];
    }
    m = to;
  }
  const float inv = sum == 0.f ? 0.f : m == kNone ? NAN : 1.f / sum;
  if (p.lse && d == 0) p.lse[(int64_t)(it.q0 + i) * p.heads + head] = sum == 0.f || m == kNone ? -INFINITY : m + __log2f(sum);
  store4<T>(p.o + ((int64_t)(it.q0 + i) * p.o_ts + (int64_t)head * p.o_hs + d) * 2, a[0] * inv, a[1] * inv, a[2] * inv, a[3] * inv);
}

// ---- host: plans ---------------------------------------------------------------------------

static int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b; }

struct Lists {
  std::vector<RowItem> rows;
  std::vector<KeyItem> keys;
  std::vector<JoinItem> join;
  int planes = 0, join_tokens = 0;
  int64_t prows = 0, far_rows = 0;  // partial rows of a plane, those behind the grid of the others among them
  int64_t parts = 0;                // forward: partial rows of all planes
};

struct Seq {
  int64_t q0, k0;
  int qlen, klen;
};

// own keys that tokens [t, t + n) of a sequence may read
static int keys_of(const Seq& s, bool causal, int t, int n) {
  if (!causal) return s.klen;
  return (int)std::max<int64_t>(0, std::min<int64_t>(s.klen, (int64_t)s.klen - s.qlen + t + n));
}

// Row lists: a tile takes the rows of as many tokens of one sequence as fit. Where there are fewer
// workgroups than fill the chip, or some far longer than the others, key ranges are cut into pieces and joined; a shared
// prefix is read
// within each sequence's tiles or, where those are mostly empty, by tiles over all tokens, and joined.
static void plan_rows(const std::vector<Seq>& seqs, const ahr_attn_shape& sh, int64_t prefix, bool may_split, Lists& L) {
  const int G = sh.heads / sh.kv_heads;
  const int per = kRows / G;  // tokens of a tile
  int64_t total = 0, tiles = 0, waves = 0;
  for (const Seq& s : seqs) {
    total += s.qlen;
    tiles += up(s.qlen, per);
    waves += up((int64_t)s.qlen * G, 32);
  }
  const int64_t ptiles = up(prefix, kKeys), across = up(total, per);
  // Apart takes fewer tiles, each a little dearer for its fuller waves, and a join: its launch, a start of each
  // tile's own keys (both in units of a key tile, 2.6 ns of the whole card; less where workgroups are few and join
  // anyway) and the partial rows through memory. 64 sequences, 16/8 heads of 64: 22 tokens, prefix 900 / 2000 / 6000:
  // within 29 / 53 / 136 us, apart 30 / 39 / 75; 14 tokens: 25 / 45 / 114 and 24 / 30 / 52; 32/8 heads of 128,
  // 22 tokens: 39 / 70 / 182 and 56 / 80 / 177; 40 sequences of 20 tokens, 12 heads of 64, prefix 300 / 900: 13 / 27
  // and 16 / 22; 30 of 8 tokens, 4/1 heads of 128, prefix 2000 / 8000: 15 / 30 and 17 / 23.
  const double saved = ((double)tiles - 1.25 * across) * ptiles * sh.kv_heads;
  const double join = 1000 + 2600 * std::min(1.0, (double)tiles * sh.kv_heads / 512) + (double)total * sh.heads * sh.head_dim / 1300;
  const bool apart = prefix > 0 && may_split && saved > join;
  std::vector<RowItem> base;
  std::vector<int> load, seq_of;
  for (size_t i = 0; i < seqs.size(); ++i)
    for (int t = 0; t < seqs[i].qlen; t += per) {
      const Seq& s = seqs[i];
      RowItem r;
      memset(&r, 0, sizeof r);
      r.q0 = (int32_t)(s.q0 + t);
      r.nq = std::min(per, s.qlen - t);
      r.k0 = (int32_t)s.k0;
      r.klen = s.klen;
      r.koff = s.klen - s.qlen + t;
      r.ke = keys_of(s, sh.causal, t, r.nq);
      r.pe = apart ? 0 : (int32_t)prefix;
      r.plane = -1;
      base.push_back(r);
      seq_of.push_back((int)i);
      load.push_back((int)(up(r.ke, kKeys) + (apart ? 0 : ptiles)));
    }
  int64_t work = 0;
  for (int x : load) work += x;
  const int64_t ptl = apart ? across : 0;  // prefix row tiles
  work += ptl * ptiles;
  const int64_t blocks = ((int64_t)base.size() + ptl) * sh.kv_heads;
  // Pieces of about `chunk` key tiles, at least four (256 keys); an item of up to one and a half stays whole. Tiles of
  // one wave's rows stream their keys from memory and gain from many workgroups (24 sequences of one token over 1k-33k
  // keys, 8 key heads of 128: 512 / 1024 / 2048 / 4096 pieces 295 / 279 / 258 / 278 us); fuller ones compute, and take
  // one round of resident workgroups (200 tokens, 32/8 heads, prefix 16000: 256 / 512 / 1024 / 2048 110 / 93 / 100 / 120
  // us). Where there are 512 workgroups without it, only items far above their share are cut, so that none is left
  // running alone (single tokens, 32/8 heads of 128: 64 sequences, one over 32768 keys and the others over 1000, 84 us,
  // uncut 656; 1000, one over 100000 and the others over 300, 301 and 2016); even batches take no join (64 over 1000
  // keys each 44 us, in 2048 pieces 49; 128 over 4000 355 and 367).
  const int64_t want = !apart && blocks < 512 && waves <= tiles ? 2048 : 512;
  int64_t chunk = INT32_MAX;
  if (may_split) chunk = std::max<int64_t>(4, up(work * sh.kv_heads, want));

  auto pieces_of = [&](int64_t tiles) { return tiles > chunk + chunk / 2 ? (int)up(tiles, chunk) : 1; };

  // Apart, the partial rows are a grid: planes (the prefix's pieces, then own keys) by tokens. Few sequences whose own
  // keys are cut would add their planes to every token (16000 single tokens, 8 heads of 128, prefix 2000, own keys 2 but
  // for one sequence with 131072: 22 planes, 1.45 GB, 302 us), so from 256 MB on those read the prefix in their own
  // tiles instead, and have a grid of their own behind the others' (132 MB, 306 us).
  int prefix_pieces = 0;
  int64_t step = 0;  // keys of a piece of the prefix
  if (apart) {
    step = up(ptiles, std::max<int64_t>(1, up(ptiles, chunk))) * kKeys;
    prefix_pieces = (int)up(prefix, step);
  }
  std::vector<char> alone(seqs.size(), 0);
  if (apart) {
    int most = 1;
    for (int x : load) most = std::max(most, pieces_of(x));
    if (most > 1 && (prefix_pieces + most) * total * sh.heads * (sh.head_dim + 1) * 4 > (int64_t)256 << 20)
      for (size_t b = 0; b < base.size(); ++b) alone[seq_of[b]] |= pieces_of(load[b]) > 1;
  }
  std::vector<int64_t> row0(seqs.size(), 0);  // apart: the first partial row of a sequence
  int64_t near_rows = 0;
  if (apart)
    for (size_t i = 0; i < seqs.size();) {
      if (alone[i]) {
        ++i;
        continue;
      }
      const int64_t t0 = seqs[i].q0, at = near_rows;
      for (; i < seqs.size() && !alone[i]; ++i) {
        row0[i] = near_rows;
        near_rows += seqs[i].qlen;
      }
      const int64_t t1 = t0 + near_rows - at;
      for (int64_t t = t0; t < t1; t += per)
        for (int j = 0; j < prefix_pieces; ++j) {
          RowItem r;
          memset(&r, 0, sizeof r);
          r.q0 = (int32_t)t;
          r.nq = (int32_t)std::min<int64_t>(per, t1 - t);
          r.pb = (int32_t)(j * step);
          r.pe = (int32_t)std::min<int64_t>(prefix, (j + 1) * step);
          r.plane = j;
          r.prow = (int32_t)(at + t - t0);
          L.rows.push_back(r);
        }
    }
  L.prows = near_rows;
  int near_planes = near_rows ? prefix_pieces : 0, far_planes = 0;
  for (size_t b = 0; b < base.size(); ++b) {
    RowItem r = base[b];
    const bool near = apart && !alone[seq_of[b]];
    if (apart && !near) {
      r.pe = (int32_t)prefix;
      load[b] += (int)ptiles;
    }
    const int pieces = pieces_of(load[b]);
    if (pieces == 1 && !near) {
      L.rows.push_back(r);
      continue;
    }
    // the key tiles of the item, prefix first, dealt to its pieces
    const int64_t own0 = near ? 0 : ptiles;
    const int64_t len = up(load[b], pieces);
    const int64_t prow = near ? row0[seq_of[b]] + r.q0 - seqs[seq_of[b]].q0 : L.prows;
    int made = near ? prefix_pieces : 0;
    if (load[b] > 0)
      for (int64_t t = 0; t < load[b]; t += len) {
        RowItem x = r;
        const int64_t e = std::min<int64_t>(load[b], t + len);
        x.pb = (int32_t)std::min<int64_t>(r.pe, t * kKeys);
        x.pe = (int32_t)std::min<int64_t>(r.pe, e * kKeys);
        x.kb = (int32_t)std::min<int64_t>(r.ke, std::max<int64_t>(0, t - own0) * kKeys);
        x.ke = (int32_t)std::min<int64_t>(r.ke, std::max<int64_t>(0, e - own0) * kKeys);
        x.plane = made++;
        x.prow = (int32_t)prow;
        L.rows.push_back(x);
      }
    int& planes = near || !apart ? near_planes : far_planes;
    planes = std::max(planes, made);
    if (!near) L.prows += r.nq;
    L.join.push_back(JoinItem{r.q0, r.nq, (int32_t)prow, made});
    L.join_tokens = std::max(L.join_tokens, r.nq);
  }
  if (!apart) near_rows = L.prows;
  L.far_rows = L.prows - near_rows;
  L.parts = near_planes * near_rows + far_planes * L.far_rows;
  L.planes = std::max(near_planes, far_planes);
  std::stable_sort(L.rows.begin(), L.rows.end(), [](const RowItem& a, const RowItem& b) {
    return (a.pe - a.pb) + (a.ke - a.kb) > (b.pe - b.pb) + (b.ke - b.kb);  // longest first
  });
}

// Key lists: a tile takes 128 keys of a sequence. Where few tiles have very unequal numbers of query rows
// (long causal sequences), their rows are cut into pieces whose sums are added.
static void plan_keys(const std::vector<Seq>& seqs, const ahr_attn_shape& sh, Lists& L) {
  const int G = sh.heads / sh.kv_heads;
  std::vector<KeyItem> base;
  int64_t work = 0;
  auto tiles_of = [&](int tokens) { return up((int64_t)tokens * G, 64); };
  for (const Seq& s : seqs)
    for (int j = 0; j < s.klen; j += kRows) {
      KeyItem k;
      memset(&k, 0, sizeof k);
      k.k0 = (int32_t)(s.k0 + j);
      k.nk = std::min(kRows, s.klen - j);
      k.kpos = j;
      k.klen = s.klen;
      k.q0 = (int32_t)s.q0;
      k.qlen = k.t1 = s.qlen;
      k.t0 = sh.causal ? (int32_t)std::min<int64_t>(s.qlen, std::max<int64_t>(0, (int64_t)j - (s.klen - s.qlen))) : 0;
      k.plane = -1;
      base.push_back(k);
      work += tiles_of(k.t1 - k.t0);
    }
  const int64_t slots = sh.head_dim > 64 ? 256 : 512;  // resident workgroups
  // (5.8k causal tokens in 3 sequences, 16/4 heads of 128: two thirds of a slot's share 457 us for the whole
  // step, a whole share 493, half 493, two shares 612, in one run)
  const int64_t piece = std::max<int64_t>(16, up(work * sh.kv_heads * 2, slots * 3));
  for (const KeyItem& k : base) {
    const int64_t tiles = tiles_of(k.t1 - k.t0);
    const int pieces = tiles * 4 > piece * 5 ? (int)up(tiles, piece) : 1;
    if (pieces == 1) {
      L.keys.push_back(k);
      continue;
    }
    const int step = (int)up(k.t1 - k.t0, pieces);
    int made = 0;
    for (int t = k.t0; t < k.t1; t += step) {
      KeyItem x = k;
      x.t0 = t;
      x.t1 = std::min(k.t1, t + step);
      x.plane = made++;
      x.prow = (int32_t)L.prows;
      L.keys.push_back(x);
    }
    L.planes = std::max(L.planes, made);
    L.join.push_back(JoinItem{k.k0, k.nk, (int32_t)L.prows, made});
    L.join_tokens = std::max(L.join_tokens, k.nk);
    L.prows += k.nk;
  }
  std::stable_sort(L.keys.begin(), L.keys.end(), [](const KeyItem& a, const KeyItem& b) { return a.t1 - a.t0 > b.t1 - b.t0; });
}

static int check_shape(const ahr_attn_shape& sh) {
  if (sh.dtype != AHR_F16 && sh.dtype != AHR_BF16) return fail(AHR_EUNSUP, "attention takes f16 and bf16");
  if (sh.heads < 1 || sh.kv_heads < 1 || sh.heads % sh.kv_heads) return fail(AHR_EINVAL, "heads must be a positive multiple of kv_heads");
  if (sh.heads / sh.kv_heads > kMaxGroup) return fail(AHR_EUNSUP, "more than 128 query heads share a key head");
  if (sh.head_dim < 8 || sh.head_dim % 8 || sh.head_dim > kMaxDim) return fail(AHR_EUNSUP, "head_dim must be a multiple of 8, at most 128");
  if (sh.prefix < 0 || sh.prefix > INT32_MAX - kKeys) return fail(AHR_EINVAL, "prefix out of range");
  if (sh.backward && sh.prefix) return fail(AHR_EUNSUP, "a shared prefix has no backward pass");
  if ((sh.causal | sh.backward) & ~1) return fail(AHR_EINVAL, "causal and backward are 0 or 1");
  return AHR_OK;
}

static int build(const int32_t* q_len, const int32_t* k_len, int n, const ahr_attn_shape& sh, ahr_attn_plan* plan,
                 int32_t* buf, int64_t cap) {
  std::vector<Seq> seqs((size_t)n);
  int64_t t = 0, tk = 0;
  for (int i = 0; i < n; ++i) {
    const int a = q_len[i], b = k_len ? k_len[i] : a;
    if (a < 0 || b < 0) return fail(AHR_EINVAL, "negative length");
    seqs[i] = Seq{t, tk, a, b};
    t += a;
    tk += b;
  }
  if (t > INT32_MAX / 2 || tk > INT32_MAX / 2) return fail(AHR_EINVAL, "more than 2^30 packed tokens");
  Lists L;
  plan_rows(seqs, sh, sh.backward ? 0 : sh.prefix, !sh.backward, L);
  if (sh.backward) plan_keys(seqs, sh, L);
  // a launch takes fewer than 2^32 threads in x and 2^16 workgroups in y (of the kernels that join or add partial results)
  const int64_t blocks = std::max<int64_t>(std::max(L.rows.size(), L.keys.size()) * (size_t)sh.kv_heads, L.join.size());
  const int64_t join_values = (int64_t)L.join_tokens * (sh.backward ? 2 * sh.kv_heads : sh.heads) * sh.head_dim;
  if (blocks >= 1 << 24 || join_values >= 1 << 24) return fail(AHR_EUNSUP, "too many sequences or heads for one call");
  memset(plan, 0, sizeof *plan);
  plan->shape = sh;
  plan->tokens = t;
  plan->key_tokens = tk;
  plan->n_rows = (int32_t)L.rows.size();
  plan->n_keys = (int32_t)L.keys.size();
  plan->n_join = (int32_t)L.join.size();
  plan->join_tokens = L.join_tokens;
  plan->planes = L.planes;
  plan->part_rows = L.prows;
  plan->far_rows = (int32_t)L.far_rows;
  plan->ints = (int64_t)(L.rows.size() * sizeof(RowItem) + L.keys.size() * sizeof(KeyItem) + L.join.size() * sizeof(JoinItem)) / 4;
  // forward: partial rows and their lse; backward: delta, partial dk and dv
  plan->ws_bytes = sh.backward ? up(t * sh.heads, 4) * 16 + (int64_t)L.planes * L.prows * sh.kv_heads * 2 * sh.head_dim * 4
                               : L.parts * sh.heads * (sh.head_dim + 1) * 4;
  if (!buf) return AHR_OK;
  if (cap < plan->ints) return fail(AHR_EINVAL, "buffer smaller than the plan's lists");
  char* b = reinterpret_cast<char*>(buf);
  memcpy(b, L.rows.data(), L.rows.size() * sizeof(RowItem));
  b += L.rows.size() * sizeof(RowItem);
  memcpy(b, L.keys.data(), L.keys.size() * sizeof(KeyItem));
  b += L.keys.size() * sizeof(KeyItem);
  memcpy(b, L.join.data(), L.join.size() * sizeof(JoinItem));
  return AHR_OK;
}

// ---- host: argument checks and launches ------------------------------------------------------

static int check_tensor(const ahr_tensor3& t, int64_t rows, int heads, const char* name) {
  if (rows == 0) return AHR_OK;
  if (!t.p) return fail(AHR_EINVAL, std::string(name) + ": null tensor");
  if (reinterpret_cast<uintptr_t>(t.p) % 16 || t.ts % 8 || t.hs % 8) return fail(AHR_EINVAL, std::string(name) + ": rows must start at multiples of 16 bytes");
  // offsets within a staged tile: 24-bit token strides in bytes, 32 bits for its tokens and all heads
  if (t.ts < 0 || t.hs < 0 || t.ts >= (1 << 22) || t.hs > ((int64_t)1 << 29) / heads) return fail(AHR_EUNSUP, std::string(name) + ": stride too large");
  return AHR_OK;
}

static int fill(const ahr_attn_args* a, bool backward, Params* out) {
  if (!a || !a->plan) return fail(AHR_EINVAL, "null arguments");
  const ahr_attn_plan& pl = *a->plan;
  const ahr_attn_shape& sh = pl.shape;
  int st = check_shape(sh);
  if (st != AHR_OK) return st;
  if ((sh.backward != 0) != backward) return fail(AHR_EINVAL, backward ? "not a backward plan" : "not a forward plan");
  if (!(a->scale > 0.f) || !std::isfinite((float)((double)a->scale * 1.4426950408889634))) return fail(AHR_EINVAL, "scale must be positive and finite");
  if (pl.ints > 0 && !a->lists) return fail(AHR_EINVAL, "null plan lists");
  if (pl.ws_bytes > 0 && (!a->ws || a->ws_bytes < pl.ws_bytes || reinterpret_cast<uintptr_t>(a->ws) % 16)) return fail(AHR_EINVAL, "workspace smaller than the plan's ws_bytes, or not aligned");
  const struct { const ahr_tensor3* t; int64_t rows; int heads; const char* name; bool on; } all[] = {
      {&a->q, pl.tokens, sh.heads, "q", true},           {&a->k, pl.key_tokens, sh.kv_heads, "k", true},
      {&a->v, pl.key_tokens, sh.kv_heads, "v", true},    {&a->prefix_k, sh.prefix, sh.kv_heads, "prefix_k", !backward},
      {&a->prefix_v, sh.prefix, sh.kv_heads, "prefix_v", !backward}, {&a->o, pl.tokens, sh.heads, "o", true},
      {&a->d_o, pl.tokens, sh.heads, "d_o", backward},   {&a->dq, pl.tokens, sh.heads, "dq", backward},
      {&a->dk, pl.key_tokens, sh.kv_heads, "dk", backward}, {&a->dv, pl.key_tokens, sh.kv_heads, "dv", backward}};
  for (const auto& x : all)
    if (x.on && (st = check_tensor(*x.t, x.rows, x.heads, x.name)) != AHR_OK) return st;
  if (backward && pl.tokens > 0 && !a->lse) return fail(AHR_EINVAL, "null lse");
  Params p;
  memset(&p, 0, sizeof p);
  p.q = (const char*)a->q.p, p.q_ts = a->q.ts, p.q_hs = a->q.hs;
  p.k = (const char*)a->k.p, p.k_ts = a->k.ts, p.k_hs = a->k.hs;
  p.v = (const char*)a->v.p, p.v_ts = a->v.ts, p.v_hs = a->v.hs;
  p.pk = (const char*)a->prefix_k.p, p.pk_ts = a->prefix_k.ts, p.pk_hs = a->prefix_k.hs;
  p.pv = (const char*)a->prefix_v.p, p.pv_ts = a->prefix_v.ts, p.pv_hs = a->prefix_v.hs;
  p.o = (char*)a->o.p, p.o_ts = a->o.ts, p.o_hs = a->o.hs;
  p.d_o = (const char*)a->d_o.p, p.do_ts = a->d_o.ts, p.do_hs = a->d_o.hs;
  p.dq = (char*)a->dq.p, p.dq_ts = a->dq.ts, p.dq_hs = a->dq.hs;
  p.dk = (char*)a->dk.p, p.dk_ts = a->dk.ts, p.dk_hs = a->dk.hs;
  p.dv = (char*)a->dv.p, p.dv_ts = a->dv.ts, p.dv_hs = a->dv.hs;
  p.lse = a->lse;
  if (backward) {
    p.delta = (float*)a->ws;
    p.part_o = (float*)a->ws + up(pl.tokens * sh.heads, 4) * 4;
  } else {
    p.part_o = (float*)a->ws;  // [parts][heads][dim], then the lse of each
    p.parts = pl.ws_bytes / ((int64_t)sh.heads * (sh.head_dim + 1) * 4);
    p.part_l = (float*)a->ws + p.parts * sh.heads * sh.head_dim;
  }
  p.prows = pl.part_rows - pl.far_rows;
  p.far_rows = pl.far_rows;
  p.n_rows = pl.n_rows, p.n_keys = pl.n_keys, p.n_join = pl.n_join;
  p.rows = reinterpret_cast<const RowItem*>(a->lists);
  p.keys = reinterpret_cast<const KeyItem*>(p.rows + pl.n_rows);
  p.join = reinterpret_cast<const JoinItem*>(p.keys + pl.n_keys);
  p.heads = sh.heads, p.kv_heads = sh.kv_heads, p.group = sh.heads / sh.kv_heads;
  p.group_inv = (65536 + p.group - 1) / p.group;  // x / group = x * group_inv >> 16 for x < 512
  p.dim = sh.head_dim, p.causal = sh.causal;
  p.scale = a->scale;
  p.scale_log2 = (float)((double)a->scale * 1.4426950408889634);
  *out = p;
  return AHR_OK;
}

template <typename T, int DP>
static int launch_fwd(const Params& p, int join_tokens, hipStream_t s) {
  constexpr int lds = 4 * kKeys * DP * 2;
  static std::atomic<uint64_t> done{0};
  ensure_lds_attr(done, reinterpret_cast<const void*>(attn_fwd_kernel<T, DP>), lds);
  attn_fwd_kernel<T, DP><<<dim3((unsigned)(p.n_rows * p.kv_heads)), kWaves * 64, lds, s>>>(p);
  AHR_HIP(hipGetLastError());
  if (p.n_join) {
    const int lanes = p.dim <= 32 ? 8 : (p.dim <= 64 ? 16 : 32), per = 256 / lanes;
    attn_join_kernel<T><<<dim3((unsigned)p.n_join, (unsigned)((join_tokens * p.heads + per - 1) / per)), 256, 0, s>>>(p, lanes);
    AHR_HIP(hipGetLastError());
  }
  return AHR_OK;
}

template <typename T>
static int launch_fwd_d(const Params& p, int join_tokens, hipStream_t s) {
  if (p.dim <= 32) return launch_fwd<T, 32>(p, join_tokens, s);
  if (p.dim <= 64) return launch_fwd<T, 64>(p, join_tokens, s);
  if (p.dim <= 96) return launch_fwd<T, 96>(p, join_tokens, s);
  return launch_fwd<T, 128>(p, join_tokens, s);
}

}  // namespace attn
}  // namespace ahr

extern "C" {

int ahr_attn_plan_build(const int32_t* q_len, const int32_t* k_len, int n, const ahr_attn_shape* shape,
                        ahr_attn_plan* plan, int32_t* buf, int64_t cap) {
  using namespace ahr;
  if (!shape || !plan || n < 0 || (n > 0 && !q_len)) return fail(AHR_EINVAL, "null lengths, shape or plan");
  int st = attn::check_shape(*shape);
  if (st != AHR_OK) return st;
  try {
    return attn::build(q_len, k_len, n, *shape, plan, buf, cap);
  } catch (...) {
    return fail(AHR_ENOMEM, "out of host memory for the work lists");
  }
}

int ahr_attn_forward(const ahr_attn_args* a, void* stream) {
  using namespace ahr;
  attn::Params p;
  int st = attn::fill(a, false, &p);
  if (st != AHR_OK) return st;
  if (p.n_rows == 0) return AHR_OK;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (a->plan->shape.dtype == AHR_BF16) return attn::launch_fwd_d<__bf16>(p, a->plan->join_tokens, s);
  return attn::launch_fwd_d<_Float16>(p, a->plan->join_tokens, s);
}

int ahr_attn_backward(const ahr_attn_args* a, void* stream) {
  using namespace ahr;
  attn::Params p;
  int st = attn::fill(a, true, &p);
  if (st != AHR_OK) return st;
  return attn::launch_backward(a, p, reinterpret_cast<hipStream_t>(stream));
}

}  // extern "C"
