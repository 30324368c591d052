// Device helpers of the packed-attention kernels (gfx950): element types, the LDS swizzle of a
// staged tile, fragment reads and the LDS-DMA that fills it.
#pragma once

#include "ahr_attn.h"
#include "ahr_dense_common.h"

namespace ahr {
namespace attn {

using dense::bf16x8;
using dense::f16x8;
using dense::f32x16;
using dense::f32x4;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

template <typename T>
struct Elem;
template <>
struct Elem<__bf16> {
  typedef bf16x8 v8;
  typedef bf16x4 v4;
  static constexpr bool kNarrow = false;
  static __device__ __forceinline__ f32x16 mma(v8 a, v8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Elem<_Float16> {
  typedef f16x8 v8;
  typedef f16x4 v4;
  static constexpr bool kNarrow = true;  // a 5-bit exponent
  static __device__ __forceinline__ f32x16 mma(v8 a, v8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};

// A staged tile holds rows of NC = DP / 8 chunks of 16 B without padding; chunk c of row r sits in
// slot c ^ swz<NC>(r). It serves both ways a tile is read: 16-B row fragments (32 rows, the same
// chunk) reach all sixteen 16-B slots of the 256-B bank row within a lane group, and transposed
// 8-B reads (4 rows x 64 B) reach its four 64-B parts.
template <int NC>
__device__ __forceinline__ int swz(int r) {
  if constexpr (NC == 16) return ((r & 3) << 2) | ((r >> 2) & 3);
  if constexpr (NC == 8) return ((r & 2) << 1) | ((r >> 2) & 3);
  return (r >> 2) & 3;
}

// 8 consecutive elements of row r at chunk 2 * ks + h: an A operand of 32x32x16 whose rows are the
// tile's rows (lane l: row l & 31, k = 8 * (l >> 5) + 0..7).
template <typename T, int NC>
__device__ __forceinline__ typename Elem<T>::v8 row_frag(const char* tile, int r, int ks, int h) {
  return *reinterpret_cast<const typename Elem<T>::v8*>(tile + r * (NC * 16) + (((2 * ks + h) ^ swz<NC>(r)) << 4));
}

// The transposed operand: rows of the result are 32 columns (block db) of the tile, k runs over 16
// of its rows from r0 in the order in which a 32x32 accumulator holds them (lane half h: rows
// 4h..4h+3, 8+4h..8+4h+3), so that accumulator values become the other operand without moving
// between lanes. Each 16-lane group of the read transposes 4 rows x 16 columns.
template <typename T, int NC>
__device__ __forceinline__ typename Elem<T>::v8 col_frag(const char* tile, int r0, int db, int lane) {
  typedef __attribute__((address_space(3))) s16x4* lds4;
  const int h = lane >> 5, lr = (lane & 15) >> 2;
  const int c = db * 4 + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
  const int ra = r0 + 4 * h + lr, rb = ra + 8;
  const char* pa = tile + ra * (NC * 16) + ((c ^ swz<NC>(ra)) << 4) + (lane & 1) * 8;
  const char* pb = tile + rb * (NC * 16) + ((c ^ swz<NC>(rb)) << 4) + (lane & 1) * 8;
  const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)pa);
  const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)pb);
  const s16x8 ab = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  return __builtin_bit_cast(typename Elem<T>::v8, ab);
}

// values x[o .. o+7] of an accumulator as the other operand
template <typename T>
__device__ __forceinline__ typename Elem<T>::v8 acc_frag(const f32x16& x, int o) {
  typename Elem<T>::v8 f;
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = (T)x[o + j];
  return f;
}

// Before a tile that LDS-DMA fills is read: this wave's loads have landed, then every wave's (the
// compiler's own barrier does not wait for LDS-DMA). All waves of the workgroup pass here once per tile,
// whether or not they have work in it. The wait is the builtin, which the compiler counts: after one in
// inline asm it waits again, at the first use of registers loaded before the loop, for whatever the tile
// has in flight by then.
// N: loads of this wave that may still be in flight (of tiles further ahead).
template <int N = 0>
__device__ __forceinline__ void tile_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((N & 15) | 0x0070 | (N >> 4) << 14);  // vmcnt(N) lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Asks the scheduler, for N matrix products of the block before it whose operands take R LDS reads each,
// to keep the reads AHEAD products ahead (left alone it reads each fragment right before its product,
// which then waits out the LDS latency).
template <int N, int R, int AHEAD = 4>
__device__ __forceinline__ void reads_ahead() {
  constexpr int A = N < AHEAD ? N : AHEAD;
  __builtin_amdgcn_sched_group_barrier(0x100, A * R, 0);  // 0x100: LDS reads, 8: matrix products
#pragma unroll
  for (int i = 0; i < N - A; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, R, 0);
  }
  __builtin_amdgcn_sched_group_barrier(0x008, A, 0);
}

// A row's fragments from memory (lane half h: elements 16 ks + 8 h ..), zeros past dim. The loads are
// unconditional, so that all are in flight together and nothing waits for them before the first tile's
// loads are issued: lanes without a row of their own read a valid one (their results go nowhere), chunks
// past dim the last.
template <typename T, int DP>
__device__ __forceinline__ void load_row(typename Elem<T>::v8 (&f)[DP / 16], const char* row, int dim, int h) {
#pragma unroll
  for (int ks = 0; ks < DP / 16; ++ks) f[ks] = *reinterpret_cast<const typename Elem<T>::v8*>(row + min((2 * ks + h) * 8, dim - 8) * 2);
  if (dim != DP) {
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) {
      const typename Elem<T>::v8 z = {};
      if ((2 * ks + h) * 8 >= dim) f[ks] = z;
    }
  }
}

// row of a 32x32 accumulator register r in lane half h
__device__ __forceinline__ int acc_row(int r, int h) { return (r & 3) + 8 * (r >> 2) + 4 * h; }

__device__ __forceinline__ float other_half(float x) { return __shfl_xor(x, 32, 64); }

__device__ __forceinline__ float ex2(float x) { return __builtin_amdgcn_exp2f(x); }

template <typename T>
__device__ __forceinline__ void store4(char* p, float a, float b, float c, float d) {
  typename Elem<T>::v4 x;
  x[0] = (T)a;
  x[1] = (T)b;
  x[2] = (T)c;
  x[3] = (T)d;
  *reinterpret_cast<typename Elem<T>::v4*>(p) = x;
}

// LDS-DMA of a tile of ROWS rows: its NC * ROWS / 64 loads of 16 B a lane are dealt to the NW waves. A
// wave's loads are kStep rows apart; where the swizzle repeats after that many rows (all but NC = 12),
// its lanes keep one row and chunk, and the step goes into the scalar offset.
template <int NC, int NW, int ROWS>
struct Stager {
  static constexpr int kLoads = NC * ROWS / 64, kPer = (kLoads + NW - 1) / NW;
  static_assert(NC == 12 || kLoads % NW == 0, "every wave has the same loads");
  static constexpr int kStep = NC == 12 ? 0 : NW * 64 / NC;
  int wave, lane, row0, c0;
  __device__ __forceinline__ Stager(int w, int l) : wave(w), lane(l) {
    row0 = (w * 64 + l) / NC;
    c0 = ((w * 64 + l) % NC) ^ swz<NC>(row0);
  }
  // a whole tile of rows (of lanes whose chunk lies within dim): row r lies at row_off (of row0) + (r - row0) / kStep * step
  __device__ __forceinline__ void load_full(__amdgpu_buffer_rsrc_t r, char* tile, int row_off, int step) const {
    const uint32_t v = (uint32_t)(row_off + c0 * 16);
#pragma unroll
    for (int i = 0; i < kPer; ++i) dense::blds16_soff(r, v, (uint32_t)(i * step), tile + (i * NW + wave) * 1024);
  }
  // any: off(row) -> byte offset of the row from the descriptor's base (rows past the range repeat a valid
  // one: every load stays inside the tensors). Chunks past dim are left alone (zeroed once).
  template <typename F>
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t r, char* tile, int dim, F off) const {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (kLoads % NW != 0 && i * NW + wave >= kLoads) break;
      const int ci = (i * NW + wave) * 64 + lane, row = ci / NC, c = (ci % NC) ^ swz<NC>(row);
      if (c * 8 < dim) dense::blds16(r, (uint32_t)(off(row) + c * 16), tile + (i * NW + wave) * 1024);
    }
  }
};

// Keys and values [kt, kt + have) of one key head into a buffer.
template <int DP>
__device__ __forceinline__ void stage_kv(char* __restrict__ nxt, const Stager<DP / 8, kWaves, kKeys>& stager, const char* k, const char* v,
                                         int64_t kts, int64_t vts, int have, int dim) {
  const int kst = (int)kts * 2, vst = (int)vts * 2;
  const __amdgpu_buffer_rsrc_t kr = dense::tile_rsrc_u(k, (uint32_t)((have - 1) * kst + dim * 2));
  const __amdgpu_buffer_rsrc_t vr = dense::tile_rsrc_u(v, (uint32_t)((have - 1) * vst + dim * 2));
  if (DP != 96 && have == kKeys) {
    constexpr int step = Stager<DP / 8, kWaves, kKeys>::kStep;
    if (dim == DP || stager.c0 * 8 < dim) {  // (chunks past dim: left alone)
      stager.load_full(kr, nxt, __mul24(stager.row0, kst), step * kst);
      stager.load_full(vr, nxt + kKeys * DP * 2, __mul24(stager.row0, vst), step * vst);
    }
  } else {
    stager.load(kr, nxt, dim, [&](int r) { return __mul24(min(r, have - 1), kst); });
    stager.load(vr, nxt + kKeys * DP * 2, dim, [&](int r) { return __mul24(min(r, have - 1), vst); });
  }
}

}  // namespace attn
}  // namespace ahr
