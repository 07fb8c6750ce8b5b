// Attention over tokens: s_ij = scale q_i . k_j + table[bucket_of[clip(j - i)], h],  p_i = softmax of s_i over the keys that count,
// o_i = sum_j p_ij v_j, for the tokens of one sequence; heads of the queries share those of the keys and values in groups.
// Backward, with D_i = dO_i . o_i:  ds_ij = p_ij (dO_i . v_j - D_i),  dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,
// dv_j = sum_i p_ij dO_i,  dtable[b, h] = sum of ds over the pairs of the bucket.
//
// Which keys count: those of the query's sequence that the mask leaves, with `causal` none behind the query. A query that the mask
// leaves out has none. Rows without a key, and rows of no sequence, are zero and have zero gradients.
#pragma once

#include "../../include/b200_tokens.h"
#include "ptx.cuh"

namespace trimul {

struct AttentionTensor {
  const void* base;
  long long row, head;  // strides in elements
};

struct AttentionParams {
  AttentionTensor q, k, v, dout;  // [rows, heads, d]
  const int* offsets;             // sequence s: rows offsets[s] .. offsets[s + 1]; null: `length` rows each
  const uint8_t* mask;            // [rows]
  const void* table;              // [buckets, heads]
  const int* bucket_of;           // [2 reach + 1]
  void *o, *rest, *dq, *dk, *dv;  // [rows, heads, d]; rest: what rounding o took away
  float* lse;                     // [heads][rows]: log2 of the softmax's denominator, +inf where a row has no key
  float* delta;                   // [heads][rows]
  float* most;                    // [kv_heads][delta_blocks][2]: greatest |dO|^2 and |v|^2 (fp16)
  float* partial;                 // [heads][places][2 reach + 1]: sums of ds by distance; null: not asked for
  void* dtable;
  long long rows, places;
  int sequences, length, heads, kv_heads, d, buckets, reach, delta_blocks;
  bool causal, wide_table;  // fp32 table
  float scale;
};

__device__ __forceinline__ long long attention_offset(const AttentionParams& p, int s) {
  if (p.offsets == nullptr) return static_cast<long long>(s) * p.length;
  return s == 0 ? 0 : min(max(static_cast<long long>(__ldcg(p.offsets + s)), 0ll), p.rows);
}
constexpr float kLog2e = 1.4426950408889634f;

// In units of log2. Finite biases beyond fp16's range count as its ends: next to greater ones fp32 would lose the scores, the powers of two
// that fp16 probabilities are held times and the logarithm of a row's sum, and at the type's lowest value the unit's factor makes them infinite.
// (Where a row has greater ones too, the probability of a pair that far below is zero either way.)
__device__ __forceinline__ float attention_bias(const AttentionParams& p, int distance, int head, bool f16) {
  if (p.table == nullptr) return 0.f;
  const int b = min(max(__ldcg(p.bucket_of + min(max(distance, -p.reach), p.reach) + p.reach), 0), p.buckets - 1);
  const long long at = static_cast<long long>(b) * p.heads + head;
  const float v = p.wide_table ? __ldcg(static_cast<const float*>(p.table) + at)
                  : f16        ? __half2float(__ldcg(static_cast<const __half*>(p.table) + at))
                               : __bfloat162float(__ldcg(static_cast<const __nv_bfloat16*>(p.table) + at));
  return (fabsf(v) > B200_ATTENTION_MAX_BIAS && fabsf(v) < INFINITY ? copysignf(B200_ATTENTION_MAX_BIAS, v) : v) * kLog2e;
}

template <typename T>
__device__ __forceinline__ const T* attention_at(const AttentionTensor& t, long long row, int head) {
  return static_cast<const T*>(t.base) + row * t.row + head * t.head;
}
__device__ __forceinline__ float warp_sum(float v) {
  for (int i = 16; i > 0; i /= 2) v += __shfl_xor_sync(0xFFFFFFFFu, v, i);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
  for (int i = 16; i > 0; i /= 2) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, i));
  return v;
}

}  // namespace trimul
