// Relative position added to the pair tensor: y[b, i, j] = z[b, i, j] + table[bucket(b, i, j)], where the bucket is that of the distance
// index[b, j] - index[b, i] (those beyond the reach count as the outermost), or the table's last row for tokens of different chains.
// Gradient of the table: the sum of dy over the pairs of each bucket; dz is dy.
#pragma once

#include "ptx.cuh"

namespace trimul {

struct PositionParams {
  const void *z, *dy;
  const float* table;   // [buckets, c]
  const void* index;    // [b, n], 32 or 64 bits
  const void* chain;    // likewise; null: one chain
  const int* bucket_of; // [2 reach + 1]
  void* y;
  float* partial;       // backward: [chunks][blocks of a chunk][buckets][kPositionChunk]
  float* dtable;
  int b, n, c, buckets, reach;
  bool wide;            // index and chain are 64-bit
  int chunks, blocks;   // backward: pieces of kPositionChunk channels, blocks of each
};

// index and chain of token j of sample b
__device__ __forceinline__ longlong2 position_token(const PositionParams& p, long long at) {
  longlong2 t;
  if (p.wide) {
    t.x = __ldcg(static_cast<const long long*>(p.index) + at);
    t.y = p.chain != nullptr ? __ldcg(static_cast<const long long*>(p.chain) + at) : 0;
  } else {
    t.x = __ldcg(static_cast<const int*>(p.index) + at);
    t.y = p.chain != nullptr ? __ldcg(static_cast<const int*>(p.chain) + at) : 0;
  }
  return t;
}
__device__ __forceinline__ int position_bucket(const PositionParams& p, longlong2 i, longlong2 j) {
  if (i.y != j.y) return p.buckets - 1;
  // (the difference of any two 64-bit indices: compared before it could wrap)
  const long long reach = p.reach;
  long long d;
  if (j.x >= i.x)
    d = static_cast<unsigned long long>(j.x) - static_cast<unsigned long long>(i.x) > static_cast<unsigned long long>(reach) ? reach : j.x - i.x;
  else
    d = static_cast<unsigned long long>(i.x) - static_cast<unsigned long long>(j.x) > static_cast<unsigned long long>(reach) ? -reach : j.x - i.x;
  return min(max(__ldcg(p.bucket_of + d + reach), 0), p.buckets - 1);
}

template <typename T, int V>
struct alignas(sizeof(T) * V) Piece {
  T v[V];
};
// past L1, which may hold what the launch before this one has read and its predecessor written
template <typename T, int V>
__device__ __forceinline__ Piece<T, V> load_piece(const T* p) {
  Piece<T, V> r;
  if constexpr (sizeof(r) == 16)
    *reinterpret_cast<uint4*>(&r) = __ldcg(reinterpret_cast<const uint4*>(p));
  else if constexpr (sizeof(r) == 8)
    *reinterpret_cast<uint2*>(&r) = __ldcg(reinterpret_cast<const uint2*>(p));
  else if constexpr (sizeof(r) == 4)
    *reinterpret_cast<uint32_t*>(&r) = __ldcg(reinterpret_cast<const uint32_t*>(p));
  else
    *reinterpret_cast<unsigned short*>(&r) = __ldcg(reinterpret_cast<const unsigned short*>(p));
  return r;
}

constexpr int kPositionThreads = 256;

// HBM bound. A block walks rows (b, i); threads take pieces of V channels of neighbouring cells.
template <typename T, int V>
__global__ void __launch_bounds__(kPositionThreads) position_forward_kernel(const PositionParams p) {
  grid_dependency_wait();
  grid_dependents_launch();
  const T* z = static_cast<const T*>(p.z);
  T* y = static_cast<T*>(p.y);
  const int pieces = p.c / V;
  const long long rows = static_cast<long long>(p.b) * p.n, row_pieces = static_cast<long long>(p.n) * pieces;
  for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
    const longlong2 ti = position_token(p, row);
    const long long sample = row / p.n * p.n;
    for (long long q = static_cast<long long>(blockIdx.y) * blockDim.x + threadIdx.x; q < row_pieces; q += static_cast<long long>(gridDim.y) * blockDim.x) {
      const int j = static_cast<int>(q / pieces), c = static_cast<int>(q - static_cast<long long>(j) * pieces) * V;
      Piece<T, V> v = load_piece<T, V>(z + (row * p.n + j) * p.c + c);
      const float* t = p.table + static_cast<long long>(position_bucket(p, ti, position_token(p, sample + j))) * p.c + c;
#pragma unroll
      for (int e = 0; e < V; ++e) v.v[e] = static_cast<T>(static_cast<float>(v.v[e]) + __ldcg(t + e));
      *reinterpret_cast<Piece<T, V>*>(y + (row * p.n + j) * p.c + c) = v;
    }
  }
}

constexpr int kPositionChunk = 64;  // channels of a warp: two a lane
constexpr int kPositionRun = 32;    // positions that a warp looks at together

// Sums over the buckets, in fixed orders: a warp owns 64 channels of a run of positions and a table of sums in shared memory; it adds
// up neighbouring positions of one bucket in registers (most pairs are far apart and share the outer two). The block adds its warps'
// tables up, and position_sums_kernel the blocks'.
template <typename T, int V>
__global__ void position_backward_kernel(const PositionParams p) {
  extern __shared__ float sums[];  // [warps][buckets][kPositionChunk]
  grid_dependency_wait();
  grid_dependents_launch();
  const T* dy = static_cast<const T*>(p.dy);
  const int warps = blockDim.x / 32, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int table = p.buckets * kPositionChunk;
  for (int i = threadIdx.x; i < warps * table; i += blockDim.x) sums[i] = 0.f;
  __syncthreads();
  const int chunk = blockIdx.x % p.chunks, block = blockIdx.x / p.chunks;
  float* own = sums + warp * table + lane * 2;
  const int c = chunk * kPositionChunk + lane * 2;
  const int runs = (p.n + kPositionRun - 1) / kPositionRun;  // of a row
  const long long units = static_cast<long long>(p.b) * p.n * runs, teams = static_cast<long long>(p.blocks) * warps;
  const long long team = static_cast<long long>(block) * warps + warp;
  float2 sum = make_float2(0.f, 0.f);
  int run = -1;
  auto flush = [&]() {
    if (run >= 0) {
      float2* t = reinterpret_cast<float2*>(own + run * kPositionChunk);
      const float2 have = *t;
      *t = make_float2(have.x + sum.x, have.y + sum.y);
    }
    sum = make_float2(0.f, 0.f);
  };
  auto value = [&](const T* at) {  // two channels of a position
    float2 v = make_float2(0.f, 0.f);
    if constexpr (V == 2) {
      if (c < p.c) {
        const Piece<T, 2> w = load_piece<T, 2>(at + c);
        v = make_float2(static_cast<float>(w.v[0]), static_cast<float>(w.v[1]));
      }
    } else {
      if (c < p.c) v.x = static_cast<float>(load_piece<T, 1>(at + c).v[0]);
      if (c + 1 < p.c) v.y = static_cast<float>(load_piece<T, 1>(at + c + 1).v[0]);
    }
    return v;
  };
  const long long last = units * (team + 1) / teams;
  for (long long unit = units * team / teams; unit < last; ++unit) {
    const long long row = unit / runs;
    const int j0 = static_cast<int>(unit - row * runs) * kPositionRun, count = min(kPositionRun, p.n - j0);
    int bucket = -1;
    if (lane < count) bucket = position_bucket(p, position_token(p, row), position_token(p, row / p.n * p.n + j0 + lane));
    const T* at = dy + (row * p.n + j0) * p.c;
    float2 v[kPositionRun];
#pragma unroll
    for (int i = 0; i < kPositionRun; ++i)
      if (i < count) v[i] = value(at + static_cast<long long>(i) * p.c);
#pragma unroll
    for (int i = 0; i < kPositionRun; ++i) {
      if (i >= count) break;
      const int b = __shfl_sync(0xFFFFFFFFu, bucket, i);
      if (b != run) {
        flush();
        run = b;
      }
      sum.x += v[i].x;
      sum.y += v[i].y;
    }
  }
  flush();
  __syncthreads();
  float* out = p.partial + (static_cast<long long>(chunk) * p.blocks + block) * table;
  for (int i = threadIdx.x; i < table; i += blockDim.x) {
    float s = sums[i];
    for (int w = 1; w < warps; ++w) s += sums[w * table + i];
    out[i] = s;
  }
}

__global__ void __launch_bounds__(256) position_sums_kernel(const PositionParams p) {
  __shared__ float part[4][kPositionChunk];
  grid_dependency_wait();
  grid_dependents_launch();
  const int bucket = blockIdx.x, chunk = blockIdx.y, c = threadIdx.x % kPositionChunk, part_of = threadIdx.x / kPositionChunk;
  const long long table = static_cast<long long>(p.buckets) * kPositionChunk;
  const float* in = p.partial + static_cast<long long>(chunk) * p.blocks * table + static_cast<long long>(bucket) * kPositionChunk + c;
  float s = 0.f;
#pragma unroll 8
  for (int i = part_of; i < p.blocks; i += 4) s += __ldcg(in + i * table);
  part[part_of][c] = s;
  __syncthreads();
  const int channel = chunk * kPositionChunk + c;
  if (part_of == 0 && channel < p.c) p.dtable[static_cast<long long>(bucket) * p.c + channel] = (part[0][c] + part[1][c]) + (part[2][c] + part[3][c]);
}

}  // namespace trimul
