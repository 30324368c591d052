// Row operators of packed sequences: q/k norm with rotation, and mean pooling (include/ahr.h).
//
// Both are bound by memory: every value is read once and written once, the reductions stay in
// registers, and sums that cross workgroups go through fp32 partial rows added in a fixed order.
#include "ahr_common.h"
#include "ahr.h"

#include <algorithm>
#include <cmath>
#include <cstring>
#include <type_traits>

namespace ahr {
namespace packed {

typedef float f32x4 __attribute__((ext_vector_type(4)));

template <typename T, int N>
__device__ __forceinline__ void load_f32(float* to, const T* from) {  // N consecutive, aligned to N * sizeof(T) or 16 B
  constexpr int W = (int)sizeof(T) * N >= 16 ? 16 / (int)sizeof(T) : N;
#pragma unroll
  for (int i = 0; i < N; i += W) {
    typedef T vec __attribute__((ext_vector_type(W)));
    const vec v = *reinterpret_cast<const vec*>(from + i);
#pragma unroll
    for (int j = 0; j < W; ++j) to[i + j] = (float)v[j];
  }
}
template <typename T, int N>
__device__ __forceinline__ void store_f32(T* to, const float* from) {
  constexpr int W = (int)sizeof(T) * N >= 16 ? 16 / (int)sizeof(T) : N;
#pragma unroll
  for (int i = 0; i < N; i += W) {
    typedef T vec __attribute__((ext_vector_type(W)));
    vec v;
#pragma unroll
    for (int j = 0; j < W; ++j) v[j] = (T)from[i + j];
    *reinterpret_cast<vec*>(to + i) = v;
  }
}

struct Rope {
  const void *q, *k, *yq, *yk;
  void *oq, *ok;  // forward: outputs; backward: gradients
  int64_t q_ts, q_hs, k_ts, k_hs, yq_ts, yq_hs, yk_ts, yk_hs, oq_ts, oq_hs, ok_ts, ok_hs;
  const float *wq, *wk, *cos, *sin;
  const int32_t* pos;
  float* part;  // backward: [part_q + part_k][dim], the weights' gradients of q's and k's workgroups
  int64_t tokens, n_pos;
  int heads, kv_heads, dim, rot;
  int q_blocks;  // vector form: workgroups (x) of q, the others take k
  float eps;
};

// Vector form (rot == head_dim, a multiple of 8, aligned rows). LPR lanes share a head's row; a lane
// owns P pairs of the rotation (8; 4 where head_dim is no multiple of 16): elements a = e0 .. e0+P-1 and
// b = e0 + dim/2 .. (interleaved: 2 P consecutive elements, pair i = (2i, 2i+1)), so the rotation needs
// no exchange between lanes. D is head_dim, or 0: read at run time, with LPR of any size. A
// workgroup takes q or k, so that a lane keeps one side's weights (and one side's part of their
// gradients: both sides' took 138 registers, three waves a SIMD, and a select for each use; 170 us
// backward where this takes 150); a wave keeps the lane's cos and sin for all heads of its token. BWD:
// dx and the weights' gradients; each lane adds its part of dw over its tokens in registers, the
// workgroup joins them into one partial row.
// Bound by memory: 22.8k tokens of 32 + 8 heads of 128 in bf16 take 95 us forward (467 MB, 4.9 TB/s,
// which is what a copy reaches) and 150 us backward (700 MB, 4.7 TB/s).
template <typename T, int D, int P, bool IL, bool BWD>
__global__ __launch_bounds__(256, 4) void rope_vec_kernel(Rope p) {
  const int dim = D ? D : p.dim;
  const int LPR = dim / (2 * P), RPW = 64 / LPR;  // lanes of a row, rows of a wave (lanes past them idle)
  const float mean = 1.f / dim;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int sub = lane / LPR, li = lane % LPR;
  const int e0 = IL ? li * 2 * P : li * P;
  const bool normed = p.wq != nullptr, is_k = (int)blockIdx.x >= p.q_blocks;
  const int heads = is_k ? p.kv_heads : p.heads;
  const int block = is_k ? blockIdx.x - p.q_blocks : blockIdx.x, blocks = is_k ? gridDim.x - p.q_blocks : p.q_blocks;
  const T* xs = (const T*)(is_k ? p.k : p.q);
  const T* ys = (const T*)(is_k ? p.yk : p.yq);
  T* os = (T*)(is_k ? p.ok : p.oq);
  const int64_t x_ts = is_k ? p.k_ts : p.q_ts, x_hs = is_k ? p.k_hs : p.q_hs, y_ts = is_k ? p.yk_ts : p.yq_ts, y_hs = is_k ? p.yk_hs : p.yq_hs,
                o_ts = is_k ? p.ok_ts : p.oq_ts, o_hs = is_k ? p.ok_hs : p.oq_hs;
  float w[2 * P], dw[2 * P];
#pragma unroll
  for (int i = 0; i < 2 * P; ++i) {
    const int e = IL || i < P ? e0 + i : dim / 2 + e0 + i - P;
    w[i] = normed ? (is_k ? p.wk : p.wq)[e] : 1.f;
    dw[i] = 0.f;
  }
  auto load = [&](float* to, const T* row) {
    if (IL) {
      load_f32<T, 2 * P>(to, row + e0);
    } else {
      load_f32<T, P>(to, row + e0);
      load_f32<T, P>(to + P, row + dim / 2 + e0);
    }
  };
  auto row_sum = [&](float x) {  // over the row's lanes, the same in all of them
    if (D) {
#pragma unroll
      for (int m = 1; m < 64; m *= 2)
        if (m < LPR) x += __shfl_xor(x, m, 64);
      return x;
    }
    float all = 0.f;
    for (int j = 0; j < LPR; ++j) all += __shfl(x, sub * LPR + j, 64);
    return all;
  };
  // Heads of a token are dealt to gridDim.y slices; with fewer heads than rows a wave takes several tokens
  // (23.5k tokens of 12 + 1 heads of 128, forward and backward: 92 us, one token a wave 206).
  const int per = heads < RPW ? RPW / heads : 1;
  const int token = per > 1 ? sub / heads : 0, head = sub - token * heads;
  const bool on = sub < (per > 1 ? per * heads : RPW);
  for (int64_t t0 = ((int64_t)block * 4 + wave) * per; t0 < p.tokens; t0 += (int64_t)blocks * 4 * per) {
    const int64_t t = t0 + token;
    const int64_t at = p.pos[t < p.tokens ? t : t0];
    const bool known = at >= 0 && at < p.n_pos;
    float c[P], s[P];
    {
      const int64_t o = (known ? at : 0) * (dim / 2) + li * P;
      load_f32<float, P>(c, p.cos + o);
      load_f32<float, P>(s, p.sin + o);
      if (!known) {
#pragma unroll
        for (int i = 0; i < P; ++i) c[i] = s[i] = NAN;
      }
    }
    for (int h0 = blockIdx.y * RPW; h0 < heads; h0 += gridDim.y * RPW) {
      const int hd = h0 + head;
      const bool have = on && t < p.tokens && hd < heads;
      float x[2 * P], y[2 * P];
      if (have) {
        load(x, xs + t * x_ts + hd * x_hs);
        if (BWD) load(y, ys + t * y_ts + hd * y_hs);
      } else {
#pragma unroll
        for (int i = 0; i < 2 * P; ++i) x[i] = y[i] = 0.f;
      }
      float r = 1.f;
      if (normed) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 2 * P; ++i) sum = fmaf(x[i], x[i], sum);
        r = 1.f / sqrtf(row_sum(sum) * mean + p.eps);
      }
      float o[2 * P];
      if (!BWD) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
          const int a = IL ? 2 * i : i, b = IL ? 2 * i + 1 : i + P;
          const float na = x[a] * r * w[a], nb = x[b] * r * w[b];
          o[a] = na * c[i] - nb * s[i];
          o[b] = nb * c[i] + na * s[i];
        }
      } else {
        // dn = R^T dy; dw += dn x r; dx = r (dn w - x r^2 mean(dn w x))
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < P; ++i) {
          const int a = IL ? 2 * i : i, b = IL ? 2 * i + 1 : i + P;
          float da = y[a] * c[i] + y[b] * s[i], db = y[b] * c[i] - y[a] * s[i];
          // (idle rows hold zeros; an unknown position's NaN belongs to rows that exist)
          if (have) {
            dw[a] = fmaf(da, x[a] * r, dw[a]);
            dw[b] = fmaf(db, x[b] * r, dw[b]);
          }
          da *= w[a];
          db *= w[b];
          dot = fmaf(da, x[a], fmaf(db, x[b], dot));
          o[a] = da;
          o[b] = db;
        }
        if (normed) {
          const float f = row_sum(dot) * mean * r * r;
#pragma unroll
          for (int i = 0; i < 2 * P; ++i) o[i] = r * (o[i] - x[i] * f);
        }
      }
      if (have) {
        T* op = os + t * o_ts + hd * o_hs;
        if (IL) {
          store_f32<T, 2 * P>(op + e0, o);
        } else {
          store_f32<T, P>(op + e0, o);
          store_f32<T, P>(op + dim / 2 + e0, o + P);
        }
      }
    }
  }
  if (BWD && normed) {
    // the rows of a wave, then the four waves, in a fixed order
    __shared__ float acc[4][64 * 2 * P];
    if (sub < RPW) {
#pragma unroll
      for (int i = 0; i < 2 * P; ++i) acc[wave][sub * dim + (IL || i < P ? e0 + i : dim / 2 + e0 + i - P)] = dw[i];
    }
    __syncthreads();
    for (int e = threadIdx.x; e < dim; e += 256) {
      float sum = 0.f;
      for (int a = 0; a < 4; ++a)
        for (int b = 0; b < RPW; ++b) sum += acc[a][b * dim + e];
      const int row = (is_k ? p.q_blocks * gridDim.y : 0) + blockIdx.y * blocks + block;
      p.part[(int64_t)row * dim + e] = sum;
    }
  }
}

// General form: any even head_dim up to 512, any even rot <= head_dim, any alignment; one wave per
// head row at a time, element e of a row in lane e % 64. Rotation partners are read from memory again.
// (23.5k tokens of 20 + 4 heads of 80 in bf16, forward and backward: 887 us, 119 in the vector form.)
template <typename T, bool BWD>
__global__ __launch_bounds__(256) void rope_any_kernel(Rope p, int il) {
  constexpr int E = 8;  // 512 / 64
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const bool normed = p.wq != nullptr;
  const int all = p.heads + p.kv_heads, half = p.rot / 2;
  float dw[2][E];
#pragma unroll
  for (int i = 0; i < E; ++i) dw[0][i] = dw[1][i] = 0.f;
  for (int64_t row = (int64_t)blockIdx.x * 4 + wave; row < p.tokens * all; row += (int64_t)gridDim.x * 4) {
    const int64_t t = row / all;
    const int hd = (int)(row - t * all);
    const bool is_k = hd >= p.heads;
    const int hh = is_k ? hd - p.heads : hd;
    const T* xp = (const T*)(is_k ? p.k : p.q) + (is_k ? t * p.k_ts + hh * p.k_hs : t * p.q_ts + hh * p.q_hs);
    const T* yp = (const T*)(is_k ? p.yk : p.yq) + (is_k ? t * p.yk_ts + hh * p.yk_hs : t * p.yq_ts + hh * p.yq_hs);
    T* op = (T*)(is_k ? p.ok : p.oq) + (is_k ? t * p.ok_ts + hh * p.ok_hs : t * p.oq_ts + hh * p.oq_hs);
    const float* w = is_k ? p.wk : p.wq;
    const int64_t at = p.pos[t];
    const bool known = at >= 0 && at < p.n_pos;
    const float* cp = p.cos + (known ? at : 0) * half;
    const float* sp = p.sin + (known ? at : 0) * half;
    float sum = 0.f;
    if (normed)
      for (int e = lane; e < p.dim; e += 64) sum = fmaf((float)xp[e], (float)xp[e], sum);
#pragma unroll
    for (int m = 1; m < 64; m *= 2) sum += __shfl_xor(sum, m, 64);
    const float r = normed ? 1.f / sqrtf(sum / p.dim + p.eps) : 1.f;
    float dot = 0.f, g[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int e = lane + 64 * i;
      g[i] = 0.f;
      if (e >= p.dim) continue;
      // the other element of e's pair, its table entry, and the sign of its sine term
      const bool turned = e < p.rot;
      const int mate = !turned ? e : (il ? e ^ 1 : (e < half ? e + half : e - half));
      const int ti = !turned ? 0 : (il ? e >> 1 : (e < half ? e : e - half));
      const float sg = (il ? (e & 1) : e >= half) ? 1.f : -1.f;
      const float c = turned ? (known ? cp[ti] : NAN) : (known ? 1.f : NAN);
      const float s = turned ? (known ? sp[ti] : NAN) : 0.f;
      if (!BWD) {
        const float a = (float)xp[e] * r * (normed ? w[e] : 1.f), b = (float)xp[mate] * r * (normed ? w[mate] : 1.f);
        g[i] = a * c + sg * b * s;
      } else {
        float d = (float)yp[e] * c - sg * (float)yp[mate] * s;
        const float x = (float)xp[e];
        if (is_k) dw[1][i] += d * x * r; else dw[0][i] += d * x * r;
        if (normed) d *= w[e];
        dot = fmaf(d, x, dot);
        g[i] = d;
      }
    }
    if (BWD && normed) {
#pragma unroll
      for (int m = 1; m < 64; m *= 2) dot += __shfl_xor(dot, m, 64);
      const float f = dot / p.dim * r * r;
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (lane + 64 * i < p.dim) g[i] = r * (g[i] - (float)xp[lane + 64 * i] * f);
    }
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (lane + 64 * i < p.dim) op[lane + 64 * i] = (T)g[i];
  }
  if (BWD && normed) {
    __shared__ float acc[4][2][512];
#pragma unroll
    for (int i = 0; i < E; ++i) {
      acc[wave][0][lane + 64 * i] = dw[0][i];
      acc[wave][1][lane + 64 * i] = dw[1][i];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * p.dim; i += 256) {
      const int s = i / p.dim, e = i % p.dim;
      p.part[((int64_t)s * gridDim.x + blockIdx.x) * p.dim + e] = acc[0][s][e] + acc[1][s][e] + acc[2][s][e] + acc[3][s][e];
    }
  }
}

// dw = the sum of the workgroups' partial rows: a workgroup per 16 columns, 64 threads a column, so that few
// loads of a thread follow each other (1024 rows of 128, 16 threads a column: 17 us, 64: 6)
__global__ __launch_bounds__(1024) void rope_dw_kernel(const float* part, int part_q, int part_k, int dim, float* dwq, float* dwk) {
  __shared__ float acc[16][16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = blockIdx.x * 16 + (lane & 15);
  const bool is_k = col >= dim;
  const int rows = col < 2 * dim ? (is_k ? part_k : part_q) : 0;
  const float* from = part + (is_k ? (int64_t)part_q * dim + col - dim : col);
  float s = 0.f;
#pragma unroll 8
  for (int b = threadIdx.x >> 4; b < rows; b += 64) s += from[(int64_t)b * dim];
  s += __shfl_xor(s, 16, 64);
  s += __shfl_xor(s, 32, 64);
  if (lane < 16) acc[wave][lane] = s;
  __syncthreads();
  if (threadIdx.x < 16 && col < 2 * dim) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) t += acc[i][threadIdx.x];
    (is_k ? dwk : dwq)[is_k ? col - dim : col] = t;
  }
}

constexpr int kRopeBlocks = 1024;

static int64_t rope_ws(int dim) { return (int64_t)kRopeBlocks * 2 * dim * 4; }

static int rope_check(const ahr_rope_args* a, bool bwd) {
  if (!a) return fail(AHR_EINVAL, "null arguments");
  if (a->dtype != AHR_F32 && a->dtype != AHR_F16 && a->dtype != AHR_BF16) return fail(AHR_EINVAL, "unknown dtype");
  if (a->heads < 0 || a->kv_heads < 0 || a->heads + a->kv_heads < 1 || a->heads > 65536 || a->kv_heads > 65536) return fail(AHR_EINVAL, "heads out of range");
  if (a->head_dim < 2 || a->head_dim % 2 || a->head_dim > 512) return fail(AHR_EUNSUP, "head_dim must be even, at most 512");
  if (a->rot < 2 || a->rot % 2 || a->rot > a->head_dim) return fail(AHR_EINVAL, "rot must be even, between 2 and head_dim");
  if (a->tokens < 0 || a->n_pos < 0) return fail(AHR_EINVAL, "negative size");
  if ((a->wq == nullptr) != (a->wk == nullptr)) return fail(AHR_EINVAL, "one norm weight without the other");
  if (!(a->eps >= 0.f) || !std::isfinite(a->eps)) return fail(AHR_EINVAL, "eps must be finite and not negative");
  if (a->tokens == 0) return AHR_OK;
  if (a->n_pos < 1 || !a->cos || !a->sin || !a->positions) return fail(AHR_EINVAL, "null positions or table");
  const ahr_tensor3 *t[6] = {&a->q, &a->yq, &a->dq, &a->k, &a->yk, &a->dk};
  for (int i = 0; i < 6; ++i) {
    if ((i < 3 ? a->heads : a->kv_heads) == 0 || (i % 3 == 2 && !bwd)) continue;
    if (!t[i]->p || t[i]->ts < 0 || t[i]->hs < 0) return fail(AHR_EINVAL, "null tensor or negative stride");
  }
  if (bwd && a->wq) {
    if (!a->dwq || !a->dwk) return fail(AHR_EINVAL, "null weight gradients");
    if (!a->ws || a->ws_bytes < rope_ws(a->head_dim)) return fail(AHR_EINVAL, "workspace smaller than ahr_rope_ws_bytes");
  }
  return AHR_OK;
}

template <typename T, bool BWD>
static int rope_launch(const ahr_rope_args* a, Rope p, hipStream_t s) {
  const ahr_tensor3* t[6] = {&a->q, &a->yq, &a->dq, &a->k, &a->yk, &a->dk};
  const int al = 16 / (int)sizeof(T);
  bool vec = a->rot == a->head_dim && a->head_dim % 8 == 0;
  for (int i = 0; i < 6; ++i) {
    if ((i < 3 ? a->heads : a->kv_heads) == 0 || (i % 3 == 2 && !BWD)) continue;
    vec = vec && reinterpret_cast<uintptr_t>(t[i]->p) % 16 == 0 && t[i]->ts % al == 0 && t[i]->hs % al == 0;
  }
  vec = vec && reinterpret_cast<uintptr_t>(p.cos) % 16 == 0 && reinterpret_cast<uintptr_t>(p.sin) % 16 == 0;
  const int all = a->heads + a->kv_heads;
  int part_q = 0, part_k = 0;
  const int il = a->interleaved;
#define AHR_ROPE(D, P)                                                                                  \
  {                                                                                                     \
    const int rpw = 64 / (a->head_dim / (2 * P)), rounds = (std::max(a->heads, a->kv_heads) + rpw - 1) / rpw; \
    auto want = [&](int heads) {                                                                        \
      const int64_t per = 4 * (heads > 0 && heads < rpw ? rpw / heads : 1);                             \
      return (a->tokens + per - 1) / per;                                                               \
    };                                                                                                  \
    /* few tokens: a token's heads are spread over more waves, for latency */                           \
    int gy = 1;                                                                                         \
    while (gy < rounds && (a->tokens + 3) / 4 * gy < 512) gy *= 2;                                                   \
    /* backward: one round of resident workgroups, dealt to q and k as the heads are */                 \
    const int most = BWD ? kRopeBlocks / gy : 65536;                                                    \
    const int k_most = BWD ? std::max(1, (int)((int64_t)most * a->kv_heads / all)) : most;              \
    const int bq = a->heads ? (int)std::min<int64_t>(want(a->heads), BWD ? std::max(1, most - k_most) : most) : 0; \
    const int bk = a->kv_heads ? (int)std::min<int64_t>(want(a->kv_heads), k_most) : 0;                 \
    p.q_blocks = bq;                                                                                    \
    part_q = bq * gy, part_k = bk * gy;                                                                 \
    if (il) rope_vec_kernel<T, D, P, true, BWD><<<dim3(bq + bk, gy), 256, 0, s>>>(p);                      \
    else rope_vec_kernel<T, D, P, false, BWD><<<dim3(bq + bk, gy), 256, 0, s>>>(p);                        \
  }
  if (vec && a->head_dim == 32) AHR_ROPE(32, 8)
  else if (vec && a->head_dim == 64) AHR_ROPE(64, 8)
  else if (vec && a->head_dim == 128) AHR_ROPE(128, 8)
  else if (vec && a->head_dim == 256) AHR_ROPE(256, 8)
  else if (vec && a->head_dim % 16 == 0) AHR_ROPE(0, 8)
  else if (vec) AHR_ROPE(0, 4)
  else {
    const int blocks = (int)std::min<int64_t>((a->tokens * all + 3) / 4, BWD ? kRopeBlocks : 65536);
    part_q = part_k = blocks;
    rope_any_kernel<T, BWD><<<dim3(blocks), 256, 0, s>>>(p, il);
  }
#undef AHR_ROPE
  AHR_HIP(hipGetLastError());
  if (BWD && a->wq) {
    rope_dw_kernel<<<dim3((2 * a->head_dim + 15) / 16), 1024, 0, s>>>(p.part, part_q, part_k, a->head_dim, a->dwq, a->dwk);
    AHR_HIP(hipGetLastError());
  }
  return AHR_OK;
}

template <bool BWD>
static int rope(const ahr_rope_args* a, void* stream) {
  const int st = rope_check(a, BWD);
  if (st != AHR_OK) return st;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  Rope p;
  memset(&p, 0, sizeof p);
  p.q = a->q.p, p.q_ts = a->q.ts, p.q_hs = a->q.hs;
  p.k = a->k.p, p.k_ts = a->k.ts, p.k_hs = a->k.hs;
  const ahr_tensor3 &oq = BWD ? a->dq : a->yq, &ok = BWD ? a->dk : a->yk;
  p.yq = a->yq.p, p.yq_ts = a->yq.ts, p.yq_hs = a->yq.hs;
  p.yk = a->yk.p, p.yk_ts = a->yk.ts, p.yk_hs = a->yk.hs;
  p.oq = oq.p, p.oq_ts = oq.ts, p.oq_hs = oq.hs;
  p.ok = ok.p, p.ok_ts = ok.ts, p.ok_hs = ok.hs;
  p.wq = a->wq, p.wk = a->wk, p.cos = a->cos, p.sin = a->sin, p.pos = a->positions;
  p.part = (float*)a->ws;
  p.tokens = a->tokens, p.n_pos = a->n_pos;
  p.heads = a->heads, p.kv_heads = a->kv_heads, p.dim = a->head_dim, p.rot = a->rot;
  p.eps = a->eps;
  if (a->tokens == 0) {
    if (BWD && a->wq) {  // no rows: zero weight gradients
      rope_dw_kernel<<<dim3((2 * a->head_dim + 15) / 16), 1024, 0, s>>>(p.part, 0, 0, a->head_dim, a->dwq, a->dwk);
      AHR_HIP(hipGetLastError());
    }
    return AHR_OK;
  }
  if (a->dtype == AHR_F32) return rope_launch<float, BWD>(a, p, s);
  if (a->dtype == AHR_F16) return rope_launch<_Float16, BWD>(a, p, s);
  return rope_launch<__bf16, BWD>(a, p, s);
}

// ---- mean pooling ----------------------------------------------------------------------------

constexpr float kPoolEps = 1e-12f;

// Sum of a chunk's rows: a workgroup per chunk and 64 * V columns, its four waves take every fourth row.
// Bound by memory: 40k rows of 768 in bf16 (256 texts) 12 us, 5.1 TB/s.
template <typename T, int V>
__global__ __launch_bounds__(256) void pool_sum_kernel(const T* rows, int64_t rs, int width, const int4* chunks, float* ws, int ld) {
  __shared__ float acc[4][64 * V];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int4 ch = chunks[blockIdx.x];
  const int col = (blockIdx.y * 64 + lane) * V;
  float s[V];
#pragma unroll
  for (int i = 0; i < V; ++i) s[i] = 0.f;
  if (col < width) {
    const T* p = rows + (int64_t)ch.x * rs + col;
#pragma unroll 4
    for (int r = wave; r < ch.y; r += 4) {
      float x[V];
      load_f32<T, V>(x, p + (int64_t)r * rs);
#pragma unroll
      for (int i = 0; i < V; ++i) s[i] += x[i];
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) acc[wave][i * 64 + lane] = s[i];
  __syncthreads();
  float* o = ws + (int64_t)blockIdx.x * ld + (int64_t)blockIdx.y * 64 * V;
  for (int i = threadIdx.x; i < 64 * V; i += 256) {  // column i = lane' * V + part
    const int j = (i % V) * 64 + i / V;
    if (blockIdx.y * 64 * V + i < ld) o[i] = acc[0][j] + acc[1][j] + acc[2][j] + acc[3][j];  // (zeros past width)
  }
}

template <int WAVES>
__device__ __forceinline__ float block_sum(float x, float* red) {
#pragma unroll
  for (int m = 1; m < 64; m *= 2) x += __shfl_xor(x, m, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
  __syncthreads();
  x = 0.f;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) x += red[i];
  __syncthreads();
  return x;
}

// Mean and norm of a sequence: the sums of its chunks in a fixed order, four chunks at a time and 4
// columns a thread (a long document's partial rows are all that one workgroup has to read: wide loads,
// several in flight, 63 partial rows of 1024 in 7 us, 118 with one column a thread).
__global__ __launch_bounds__(1024) void pool_mean_kernel(const float* ws, int ld, int width, const int4* seqs, int normalize, float* out,
                                                         float* norm) {
  __shared__ f32x4 part[4][256];
  __shared__ float red[16];
  const int4 sq = seqs[blockIdx.x];  // rows, first chunk, chunks
  const int x = threadIdx.x & 255, y = threadIdx.x >> 8;
  float* o = out + (int64_t)blockIdx.x * width;
  float ss = 0.f;
  for (int g0 = 0; g0 < ld / 4; g0 += 256) {
    const int g = g0 + x;
    f32x4 s = {0, 0, 0, 0};
    if (g < ld / 4) {
      const f32x4* p = reinterpret_cast<const f32x4*>(ws + (int64_t)sq.y * ld) + g;
#pragma unroll 8
      for (int i = y; i < sq.z; i += 4) s += p[(int64_t)i * (ld / 4)];
    }
    part[y][x] = s;
    __syncthreads();
    if (y == 0 && g < ld / 4) {
      s = part[0][x] + part[1][x] + part[2][x] + part[3][x];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float v = sq.x > 0 ? s[i] / (float)sq.x : 0.f;
        if (g * 4 + i < width) o[g * 4 + i] = v;
        ss = fmaf(v, v, ss);  // (zeros past width)
      }
    }
    __syncthreads();
  }
  const float nm = sqrtf(block_sum<16>(ss, red));
  if (threadIdx.x == 0 && norm) norm[blockIdx.x] = nm;
  if (!normalize || y != 0) return;
  const float d = fmaxf(nm, kPoolEps);
  for (int g = x; g < ld / 4; g += 256)
    for (int c = g * 4; c < min(width, g * 4 + 4); ++c) o[c] /= d;  // (each thread its own values)
}

// Gradient of the rows: the same for every row of a sequence, (d_out - out (out . d_out)) / (norm rows),
// written to the rows of one chunk. Bound by the writes: 40k rows of 1024 in f16 (12 documents) 17 us, 4.8 TB/s.
template <typename T, int V>
__global__ __launch_bounds__(256) void pool_grad_kernel(T* d_rows, int width, const int4* chunks, const int4* seqs, int normalize,
                                                        const float* d_out, const float* out, const float* norm) {
  __shared__ float red[4];
  const int4 ch = chunks[blockIdx.x];
  const float* dy = d_out + (int64_t)ch.z * width;
  const float* y = out + (int64_t)ch.z * width;
  float dot = 0.f, d = 1.f;
  if (normalize) {
    const float nm = norm[ch.z];
    if (nm >= kPoolEps) {  // below it the division is by a constant
      for (int c = threadIdx.x; c < width; c += 256) dot = fmaf(dy[c], y[c], dot);
    }
    dot = block_sum<4>(dot, red);
    d = fmaxf(nm, kPoolEps);
  }
  const float f = 1.f / (d * (float)seqs[ch.z].x);
  T* p = d_rows + (int64_t)ch.x * width;
  for (int c = threadIdx.x * V; c < width; c += 256 * V) {
    float g[V];
#pragma unroll
    for (int i = 0; i < V; ++i) g[i] = (dy[c + i] - (normalize ? y[c + i] * dot : 0.f)) * f;
    for (int r = 0; r < ch.y; ++r) store_f32<T, V>(p + (int64_t)r * width + c, g);
  }
}

template <typename T>
static int pool_sum(const void* rows, int64_t rs, int width, const int4* chunks, int n_chunks, float* ws, int ld, hipStream_t s) {
  constexpr int V = 16 / (int)sizeof(T);
  if (width % V == 0 && rs % V == 0 && reinterpret_cast<uintptr_t>(rows) % 16 == 0)
    pool_sum_kernel<T, V><<<dim3(n_chunks, (width + 64 * V - 1) / (64 * V)), 256, 0, s>>>((const T*)rows, rs, width, chunks, ws, ld);
  else
    pool_sum_kernel<T, 1><<<dim3(n_chunks, (width + 63) / 64), 256, 0, s>>>((const T*)rows, rs, width, chunks, ws, ld);
  AHR_HIP(hipGetLastError());
  return AHR_OK;
}

template <typename T>
static int pool_grad(void* d_rows, int width, const int4* chunks, int n_chunks, const int4* seqs, int normalize,
                     const float* d_out, const float* out, const float* norm, hipStream_t s) {
  constexpr int V = 16 / (int)sizeof(T);
  if (width % V == 0 && reinterpret_cast<uintptr_t>(d_rows) % 16 == 0)
    pool_grad_kernel<T, V><<<n_chunks, 256, 0, s>>>((T*)d_rows, width, chunks, seqs, normalize, d_out, out, norm);
  else
    pool_grad_kernel<T, 1><<<n_chunks, 256, 0, s>>>((T*)d_rows, width, chunks, seqs, normalize, d_out, out, norm);
  AHR_HIP(hipGetLastError());
  return AHR_OK;
}

}  // namespace packed
}  // namespace ahr

extern "C" {

int ahr_rope_ws_bytes(int64_t tokens, int head_dim, int64_t* bytes) {
  if (!bytes || tokens < 0 || head_dim < 2 || head_dim > 512) return ahr::fail(AHR_EINVAL, "null output or bad size");
  *bytes = ahr::packed::rope_ws(head_dim);
  return AHR_OK;
}

int ahr_qk_norm_rope(const ahr_rope_args* a, void* stream) { return ahr::packed::rope<false>(a, stream); }

int ahr_qk_norm_rope_backward(const ahr_rope_args* a, void* stream) { return ahr::packed::rope<true>(a, stream); }

int ahr_pool_plan_build(const int32_t* lengths, int n, int32_t* buf, int64_t cap, int* n_chunks) {
  using namespace ahr;
  if (n < 0 || (n > 0 && !lengths) || !n_chunks) return fail(AHR_EINVAL, "null lengths or output");
  int64_t tokens = 0, count = 0;
  for (int i = 0; i < n; ++i) {
    if (lengths[i] < 0) return fail(AHR_EINVAL, "negative length");
    tokens += lengths[i];
  }
  if (tokens > INT32_MAX / 2) return fail(AHR_EINVAL, "more than 2^30 packed tokens");
  // rows of a chunk: as few as keep about 512 chunks (each of which leaves a partial row to be added)
  int64_t rows = 64;
  while (rows < 1024 && rows * 512 < tokens) rows *= 2;
  for (int i = 0; i < n; ++i) count += (lengths[i] + rows - 1) / rows;
  *n_chunks = (int)count;
  if (!buf) return AHR_OK;
  if (cap < (count + n) * 4) return fail(AHR_EINVAL, "buffer smaller than the lists");
  int32_t *c = buf, *s = buf + count * 4;
  int64_t row = 0;
  int32_t made = 0;
  for (int i = 0; i < n; ++i, s += 4) {
    s[0] = lengths[i];
    s[1] = made;
    for (int64_t t = 0; t < lengths[i]; t += rows, ++made, c += 4) {
      c[0] = (int32_t)(row + t);
      c[1] = (int32_t)std::min<int64_t>(rows, lengths[i] - t);
      c[2] = i;
      c[3] = 0;
    }
    s[2] = made - s[1];
    s[3] = 0;
    row += lengths[i];
  }
  return AHR_OK;
}

static int pool_check(int dtype, int width, const int32_t* lists, int n_chunks, int n) {
  using namespace ahr;
  if (dtype != AHR_F32 && dtype != AHR_F16 && dtype != AHR_BF16) return fail(AHR_EINVAL, "unknown dtype");
  if (width < 1 || width > (1 << 20)) return fail(AHR_EINVAL, "width out of range");
  if (n < 0 || n_chunks < 0 || (n > 0 && !lists) || reinterpret_cast<uintptr_t>(lists) % 16) return fail(AHR_EINVAL, "null or unaligned lists");
  // a launch takes fewer than 2^32 threads: 1024 for a sequence, 256 for a chunk
  if (n >= 1 << 22 || n_chunks >= 1 << 24) return fail(AHR_EUNSUP, "too many sequences for one call");
  return AHR_OK;
}

int ahr_pool_mean(int dtype, const void* rows, int64_t rs, int width, const int32_t* lists, int n_chunks, int n,
                  int normalize, float* out, float* norm, float* ws, int64_t ws_bytes, void* stream) {
  using namespace ahr;
  int st = pool_check(dtype, width, lists, n_chunks, n);
  if (st != AHR_OK) return st;
  if (n == 0) return AHR_OK;
  if (!out || rs < 0 || (n_chunks > 0 && (!rows || !ws))) return fail(AHR_EINVAL, "null tensor or negative stride");
  const int ld = (width + 3) / 4 * 4;
  if (ws_bytes < (int64_t)n_chunks * ld * 4 || reinterpret_cast<uintptr_t>(ws) % 16) return fail(AHR_EINVAL, "workspace too small, or not aligned");
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const int4* ch = reinterpret_cast<const int4*>(lists);
  const int4* sq = reinterpret_cast<const int4*>(lists + (int64_t)n_chunks * 4);
  if (n_chunks > 0) {
    if (dtype == AHR_F32) st = packed::pool_sum<float>(rows, rs, width, ch, n_chunks, ws, ld, s);
    else if (dtype == AHR_F16) st = packed::pool_sum<_Float16>(rows, rs, width, ch, n_chunks, ws, ld, s);
    else st = packed::pool_sum<__bf16>(rows, rs, width, ch, n_chunks, ws, ld, s);
    if (st != AHR_OK) return st;
  }
  packed::pool_mean_kernel<<<n, 1024, 0, s>>>(ws, ld, width, sq, normalize, out, norm);
  AHR_HIP(hipGetLastError());
  return AHR_OK;
}

int ahr_pool_mean_backward(int dtype, void* d_rows, int width, const int32_t* lists, int n_chunks, int n, int normalize,
                           const float* d_out, const float* out, const float* norm, void* stream) {
  using namespace ahr;
  int st = pool_check(dtype, width, lists, n_chunks, n);
  if (st != AHR_OK) return st;
  if (n_chunks == 0) return AHR_OK;
  if (!d_rows || !d_out || (normalize && (!out || !norm))) return fail(AHR_EINVAL, "null tensor");
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const int4* ch = reinterpret_cast<const int4*>(lists);
  const int4* sq = reinterpret_cast<const int4*>(lists + (int64_t)n_chunks * 4);
  if (dtype == AHR_F32) return packed::pool_grad<float>(d_rows, width, ch, n_chunks, sq, normalize, d_out, out, norm, s);
  if (dtype == AHR_F16) return packed::pool_grad<_Float16>(d_rows, width, ch, n_chunks, sq, normalize, d_out, out, norm, s);
  return packed::pool_grad<__bf16>(d_rows, width, ch, n_chunks, sq, normalize, d_out, out, norm, s);
}

}  // extern "C"
