// Attention over packed sequences: work lists and kernel parameters shared by the host planner and
// the kernels (ahr_attn.hip, ahr_attn_bwd.hip).
#pragma once

#include "ahr.h"
#include "ahr_common.h"

namespace ahr {
namespace attn {

constexpr int kKeys = 64;     // keys of one staged tile
constexpr int kWaves = 4;     // waves of a workgroup
constexpr int kRows = 128;    // rows of a row tile, keys of a key tile: 32 a wave
constexpr int kMaxDim = 128;  // head dimensions: multiples of 8 up to this
constexpr int kMaxGroup = 128;  // query heads that share a key head

// One workgroup's share of the forward pass or of dq, for each key head: the rows (token, head of
// the group) of nq tokens against a range of the shared prefix and a range of their own keys.
struct RowItem {
  int32_t q0, nq;      // packed query tokens [q0, q0 + nq)
  int32_t k0, klen;    // packed position and number of the sequence's keys
  int32_t koff;        // causal: token i of the item reads keys < min(klen, koff + i + 1)
  int32_t kb, ke;      // own keys [kb, ke) of this item, relative to k0
  int32_t pb, pe;      // prefix keys [pb, pe)
  int32_t plane, prow; // partial results: plane and row of the first token; plane < 0: final
  int32_t pad;
};

// One workgroup's share of dk and dv, for each key head: nk keys against query rows of their sequence.
struct KeyItem {
  int32_t k0, nk;      // packed keys [k0, k0 + nk)
  int32_t kpos, klen;  // position of the first within the sequence, keys of the sequence
  int32_t q0, qlen;    // the sequence's packed query tokens
  int32_t t0, t1;      // query tokens [t0, t1) of the sequence (those before read none of the keys)
  int32_t plane, prow; // partial sums: plane and row of the first key; plane < 0: final
  int32_t pad[2];
};

// Tokens (backward: keys) whose np partial results (planes 0..np-1) are joined.
struct JoinItem {
  int32_t q0, nq, prow, np;
};

struct Params {
  const char *q, *k, *v, *pk, *pv, *d_o;
  char *o, *dq, *dk, *dv;
  float *lse, *delta;
  float *part_o, *part_l;
  // strides in elements
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, pk_ts, pk_hs, pv_ts, pv_hs, o_ts, o_hs, do_ts, do_hs;
  int64_t dq_ts, dq_hs, dk_ts, dk_hs, dv_ts, dv_hs;
  int64_t prows, far_rows, parts;  // partial rows of a plane, of the planes behind, of all planes
  const RowItem* rows;
  const KeyItem* keys;
  const JoinItem* join;
  int n_rows, n_keys, n_join;
  int heads, kv_heads, group, group_inv, dim, causal;
  float scale, scale_log2;
};

int launch_backward(const ahr_attn_args* a, const Params& p, hipStream_t s);

}  // namespace attn
}  // namespace ahr
