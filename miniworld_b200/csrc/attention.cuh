// Attention over tokens: s_ij = scale q_i . k_j + table[bucket_of[clip(j - i)], h],  p_i = softmax of s_i over the keys that count,
// o_i = sum_j p_ij v_j, for the tokens of one sequence; heads of the queries share those of the keys and values in groups.
// Backward, with D_i = dO_i . o_i:  ds_ij = p_ij (dO_i . v_j - D_i),  dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,
// dv_j = sum_i p_ij dO_i,  dtable[b, h] = sum of ds over the pairs of the bucket.
//
// Which keys count: those of the query's sequence that the mask leaves, with `causal` none behind the query. A query that the mask
// leaves out has none. Rows without a key, and rows of no sequence, are zero and have zero gradients.
#pragma once

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
  float* partial;                 // [heads][blocks][2 reach + 1]: sums of ds by distance
  void* dtable;
  long long rows;
  int sequences, length, heads, kv_heads, d, buckets, reach, blocks;
  bool causal, wide_table;  // fp32 table
  float scale;
};

struct AttentionRow {
  long long first, last;  // its sequence
  bool there;             // the row takes part
};
__device__ __forceinline__ long long attention_offset(const AttentionParams& p, int s) {
  if (p.offsets == nullptr) return static_cast<long long>(s) * p.length;
  return s == 0 ? 0 : min(max(static_cast<long long>(__ldcg(p.offsets + s)), 0ll), p.rows);
}
__device__ __forceinline__ AttentionRow attention_row(const AttentionParams& p, long long row) {
  int lo = 0, hi = p.sequences;  // the last sequence that begins at or before the row
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    (attention_offset(p, mid) <= row ? lo : hi) = mid;
  }
  AttentionRow r = {attention_offset(p, lo), attention_offset(p, lo + 1), true};
  r.there = row >= r.first && row < r.last && (p.mask == nullptr || __ldcg(p.mask + row) != 0);
  return r;
}
__device__ __forceinline__ float attention_bias(const AttentionParams& p, int distance, int head, bool f16) {
  if (p.table == nullptr) return 0.f;
  const int b = min(max(__ldcg(p.bucket_of + min(max(distance, -p.reach), p.reach) + p.reach), 0), p.buckets - 1);
  const long long at = static_cast<long long>(b) * p.heads + head;
  if (p.wide_table) return __ldcg(static_cast<const float*>(p.table) + at);
  return f16 ? __half2float(__ldcg(static_cast<const __half*>(p.table) + at)) : __bfloat162float(__ldcg(static_cast<const __nv_bfloat16*>(p.table) + at));
}

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kAttentionWarps = 4;
constexpr int kAttentionMostWidth = 128;

template <typename T>
__device__ __forceinline__ const T* attention_at(const AttentionTensor& t, long long row, int head) {
  return static_cast<const T*>(t.base) + row * t.row + head * t.head;
}
template <typename T>
__device__ __forceinline__ float attention_dot(const float* a, const T* b, int d) {
  float s = 0.f;
  for (int c = 0; c < d; ++c) s = fmaf(a[c], static_cast<float>(__ldcg(b + c)), s);
  return s;
}
__device__ __forceinline__ float warp_sum(float v) {
  for (int i = 16; i > 0; i /= 2) v += __shfl_xor_sync(0xFFFFFFFFu, v, i);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
  for (int i = 16; i > 0; i /= 2) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, i));
  return v;
}

// delta, dq and the sums of ds by distance: a warp a query row
template <typename T>
__global__ void __launch_bounds__(kAttentionWarps * 32) attention_dq_kernel(const AttentionParams p) {
  extern __shared__ float by_distance[];  // [warps][2 reach + 1]
  __shared__ float row_q[kAttentionWarps][kAttentionMostWidth], row_g[kAttentionWarps][kAttentionMostWidth];
  constexpr bool f16 = __is_same(T, __half);
  grid_dependency_wait();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, head = blockIdx.y, kv_head = head / (p.heads / p.kv_heads);
  float *q = row_q[warp], *g = row_g[warp];
  const int distances = p.table != nullptr ? 2 * p.reach + 1 : 0;
  for (int i = threadIdx.x; i < distances * kAttentionWarps; i += blockDim.x) by_distance[i] = 0.f;
  __syncthreads();
  float* sums = by_distance + warp * distances;
  for (long long row = static_cast<long long>(blockIdx.x) * kAttentionWarps + warp; row < p.rows; row += static_cast<long long>(gridDim.x) * kAttentionWarps) {
    const AttentionRow r = attention_row(p, row);
    T* out = static_cast<T*>(p.dq) + (row * p.heads + head) * p.d;
    float acc[4] = {0.f, 0.f, 0.f, 0.f}, delta = 0.f;
    const float lse = __ldcg(p.lse + head * p.rows + row);
    if (r.there && lse != INFINITY) {
      __syncwarp();
      const T* o = static_cast<const T*>(p.o) + (row * p.heads + head) * p.d;
      const T* rest = static_cast<const T*>(p.rest) + (row * p.heads + head) * p.d;
      for (int c = lane; c < p.d; c += 32) {
        q[c] = static_cast<float>(__ldcg(attention_at<T>(p.q, row, head) + c));
        g[c] = static_cast<float>(__ldcg(attention_at<T>(p.dout, row, head) + c));
        delta = fmaf(g[c], static_cast<float>(__ldcg(o + c)) + static_cast<float>(__ldcg(rest + c)) * (f16 ? 1.f / 2048.f : 1.f), delta);
      }
      delta = warp_sum(delta);
      __syncwarp();
      const long long last = p.causal ? row + 1 : r.last;
      for (long long j0 = r.first; j0 < last; j0 += 32) {
        const long long j = j0 + lane;
        const bool counts = j < last && (p.mask == nullptr || __ldcg(p.mask + j) != 0);
        float ds = 0.f;
        if (counts) {
          const float s = (attention_dot(q, attention_at<T>(p.k, j, kv_head), p.d) * p.scale + attention_bias(p, static_cast<int>(j - row), head, f16)) * kLog2e;
          ds = exp2f(s - lse) * (attention_dot(g, attention_at<T>(p.v, j, kv_head), p.d) - delta);
        }
        if (distances != 0) {
          const long long d = j - row;
          const bool low = d <= -p.reach, high = !low && d >= p.reach;  // (a reach of 0 is one bucket)
          const float lows = warp_sum(low ? ds : 0.f), highs = warp_sum(high ? ds : 0.f);
          if (!low && !high) sums[d + p.reach] += ds;
          if (lane == 0) {
            sums[0] += lows;
            sums[2 * p.reach] += highs;
          }
          __syncwarp();
        }
        uint32_t left = __ballot_sync(0xFFFFFFFFu, counts);
        while (left != 0) {
          const int i = __ffs(left) - 1;
          left &= left - 1;
          const float w = __shfl_sync(0xFFFFFFFFu, ds, i);
          const T* k = attention_at<T>(p.k, j0 + i, kv_head);
          for (int a = 0; a < 4; ++a)
            if (lane + 32 * a < p.d) acc[a] = fmaf(w, static_cast<float>(__ldcg(k + lane + 32 * a)), acc[a]);
        }
      }
    }
    for (int a = 0; a < 4; ++a)
      if (lane + 32 * a < p.d) out[lane + 32 * a] = static_cast<T>(acc[a] * p.scale);
    if (lane == 0) p.delta[head * p.rows + row] = delta;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < distances; i += blockDim.x) {
    float s = 0.f;
    for (int w = 0; w < kAttentionWarps; ++w) s += by_distance[w * distances + i];
    p.partial[(static_cast<long long>(head) * gridDim.x + blockIdx.x) * distances + i] = s;
  }
}

// dk and dv: a warp a key row, over the query heads of its group
template <typename T>
__global__ void __launch_bounds__(kAttentionWarps * 32) attention_dkv_kernel(const AttentionParams p) {
  __shared__ float row_k[kAttentionWarps][kAttentionMostWidth], row_v[kAttentionWarps][kAttentionMostWidth];
  constexpr bool f16 = __is_same(T, __half);
  grid_dependency_wait();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, kv_head = blockIdx.y, group = p.heads / p.kv_heads;
  float *k = row_k[warp], *v = row_v[warp];
  for (long long row = static_cast<long long>(blockIdx.x) * kAttentionWarps + warp; row < p.rows; row += static_cast<long long>(gridDim.x) * kAttentionWarps) {
    const AttentionRow r = attention_row(p, row);
    float dk[4] = {0.f, 0.f, 0.f, 0.f}, dv[4] = {0.f, 0.f, 0.f, 0.f};
    if (r.there) {
      __syncwarp();
      for (int c = lane; c < p.d; c += 32) {
        k[c] = static_cast<float>(__ldcg(attention_at<T>(p.k, row, kv_head) + c));
        v[c] = static_cast<float>(__ldcg(attention_at<T>(p.v, row, kv_head) + c));
      }
      __syncwarp();
      for (int head = kv_head * group; head < (kv_head + 1) * group; ++head)
        for (long long i0 = p.causal ? row : r.first; i0 < r.last; i0 += 32) {
          const long long i = i0 + lane;
          const bool counts = i < r.last && (p.mask == nullptr || __ldcg(p.mask + i) != 0);
          float e = 0.f, ds = 0.f;
          if (counts) {
            const float s = (attention_dot(k, attention_at<T>(p.q, i, head), p.d) * p.scale + attention_bias(p, static_cast<int>(row - i), head, f16)) * kLog2e;
            e = exp2f(s - __ldcg(p.lse + head * p.rows + i));
            ds = e * (attention_dot(v, attention_at<T>(p.dout, i, head), p.d) - __ldcg(p.delta + head * p.rows + i));
          }
          uint32_t left = __ballot_sync(0xFFFFFFFFu, counts);
          while (left != 0) {
            const int at = __ffs(left) - 1;
            left &= left - 1;
            const float wv = __shfl_sync(0xFFFFFFFFu, e, at), wk = __shfl_sync(0xFFFFFFFFu, ds, at);
            const T *q = attention_at<T>(p.q, i0 + at, head), *g = attention_at<T>(p.dout, i0 + at, head);
            for (int a = 0; a < 4; ++a)
              if (lane + 32 * a < p.d) {
                dk[a] = fmaf(wk, static_cast<float>(__ldcg(q + lane + 32 * a)), dk[a]);
                dv[a] = fmaf(wv, static_cast<float>(__ldcg(g + lane + 32 * a)), dv[a]);
              }
          }
        }
    }
    const long long at = (row * p.kv_heads + kv_head) * p.d;
    for (int a = 0; a < 4; ++a)
      if (lane + 32 * a < p.d) {
        static_cast<T*>(p.dk)[at + lane + 32 * a] = static_cast<T>(dk[a] * p.scale);
        static_cast<T*>(p.dv)[at + lane + 32 * a] = static_cast<T>(dv[a]);
      }
  }
}

// The table's gradient: a block a head; a thread a distance adds the blocks' sums up, then a thread a bucket its distances.
template <typename T>
__global__ void __launch_bounds__(256) attention_table_kernel(const AttentionParams p) {
  extern __shared__ float distance[];  // [2 reach + 1]
  grid_dependency_wait();
  const int distances = 2 * p.reach + 1, head = blockIdx.x;
  const float* in = p.partial + static_cast<long long>(head) * p.blocks * distances;
  for (int i = threadIdx.x; i < distances; i += blockDim.x) {
    float s = 0.f;
    for (int b = 0; b < p.blocks; ++b) s += __ldcg(in + static_cast<long long>(b) * distances + i);
    distance[i] = s;
  }
  __syncthreads();
  for (int b = threadIdx.x; b < p.buckets; b += blockDim.x) {
    float s = 0.f;
    for (int i = 0; i < distances; ++i)
      if (min(max(__ldcg(p.bucket_of + i), 0), p.buckets - 1) == b) s += distance[i];
    static_cast<T*>(p.dtable)[static_cast<long long>(b) * p.heads + head] = static_cast<T>(s);
  }
}

}  // namespace trimul
