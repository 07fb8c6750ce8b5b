// Relative position added to the pair tensor: y[b, i, j] = z[b, i, j] + table[bucket(b, i, j)], where the bucket is that of the distance
// index[b, j] - index[b, i] (those beyond the reach count as the outermost), or the table's last row for tokens of different chains.
// Gradient of the table: the sum of dy over the pairs of each bucket; dz is dy.
#pragma once

#include <type_traits>

#include "../../include/b200_tokens.h"
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
  int cells;            // forward: cells of a tile
  uint32_t magic;       // ceil(2^32 / pieces of a cell)
  bool table_in_smem;
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
__device__ __forceinline__ int position_bucket(const PositionParams& p, const int* bucket_of, longlong2 i, longlong2 j) {
  if (i.y != j.y) return p.buckets - 1;
  // (the difference of any two 64-bit indices: compared before it could wrap)
  const long long reach = p.reach;
  long long d;
  if (j.x >= i.x)
    d = static_cast<unsigned long long>(j.x) - static_cast<unsigned long long>(i.x) > static_cast<unsigned long long>(reach) ? reach : j.x - i.x;
  else
    d = static_cast<unsigned long long>(i.x) - static_cast<unsigned long long>(j.x) > static_cast<unsigned long long>(reach) ? -reach : j.x - i.x;
  return bucket_of[d + reach];
}
// the buckets of all distances, brought into the table's range
__device__ __forceinline__ void position_buckets(const PositionParams& p, int* bucket_of) {
  for (int i = threadIdx.x; i < 2 * p.reach + 1; i += blockDim.x) bucket_of[i] = min(max(__ldcg(p.bucket_of + i), 0), p.buckets - 1);
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

// v += t, rounded once
template <typename T, int Q>
__device__ __forceinline__ void add_piece(T* v, const Piece<float, Q>& t) {
  if constexpr (sizeof(T) == 2 && Q >= 2) {
    uint32_t* w = reinterpret_cast<uint32_t*>(v);
#pragma unroll
    for (int e = 0; e < Q; e += 2) {
      constexpr bool f16 = std::is_same_v<T, __half>;
      const float2 s = __fadd2_rn(f16 ? f16x2_to_float2(w[e / 2]) : bf16x2_to_float2(w[e / 2]), make_float2(t.v[e], t.v[e + 1]));
      w[e / 2] = f16 ? pack_f16x2(s) : pack_bf16x2(s);
    }
  } else {
#pragma unroll
    for (int e = 0; e < Q; ++e) v[e] = static_cast<T>(static_cast<float>(v[e]) + t.v[e]);
  }
}

constexpr int kPositionThreads = 256;
constexpr int kPositionMostCells = 512;
constexpr int kPositionFlight = 4;  // pieces of V channels that a thread loads at once

// HBM bound: 768 x 768 x 128 bf16 50 to 54 us (302 MB, 0.86 to 0.92 of the measured rate); with buckets looked up and table entries loaded
// by every piece 569. A block takes tiles of consecutive cells (b, i, j), whatever rows they are of: the buckets of a tile first (a thread a cell,
// loads for the next tile while this one streams), then its pieces of V channels. The table lies in shared memory, the floats of a piece
// a quarter-warp's stride apart, so that neighbouring lanes read neighbouring words.
template <typename T, int V>
__global__ void __launch_bounds__(kPositionThreads) position_forward_kernel(const PositionParams p) {
  extern __shared__ float4 table_smem[];
  __shared__ int bucket_of[2 * B200_POSITION_MAX_REACH + 1];
  __shared__ int buckets[2][kPositionMostCells];
  grid_dependency_wait();
  grid_dependents_launch();
  const T* z = static_cast<const T*>(p.z);
  T* y = static_cast<T*>(p.y);
  float* const table = reinterpret_cast<float*>(table_smem);
  constexpr int Q = V < 4 ? V : 4, QUADS = V / Q;  // floats read at once, and how often for a piece
  const int pieces = p.c / V;
  position_buckets(p, bucket_of);
  if (p.table_in_smem) {
    const int row_quads = pieces * QUADS;
#pragma unroll 8
    for (int i = threadIdx.x; i < p.buckets * row_quads; i += kPositionThreads) {
      const int row = i / row_quads, at = i - row * row_quads, d = at / pieces, piece = at - d * pieces;
      *reinterpret_cast<Piece<float, Q>*>(table + static_cast<long long>(i) * Q) = load_piece<float, Q>(p.table + row * p.c + piece * V + d * Q);
    }
  }
  __syncthreads();
  const long long cells = static_cast<long long>(p.b) * p.n * p.n, tiles = (cells + p.cells - 1) / p.cells;
  auto bucket_at = [&](long long cell) {
    const long long row = cell / p.n;  // (b, i)
    const long long j = cell - row * p.n, sample = row / p.n;
    return position_bucket(p, bucket_of, position_token(p, row), position_token(p, sample * p.n + j));
  };
  int next[2];
  auto look = [&](long long tile) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int i = threadIdx.x + k * kPositionThreads;
      const long long cell = tile * p.cells + i;
      next[k] = i < p.cells && cell < cells ? bucket_at(cell) : 0;
    }
  };
  look(blockIdx.x);
  int turn = 0;
  for (long long tile = blockIdx.x; tile < tiles; tile += gridDim.x, turn ^= 1) {
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (threadIdx.x + k * kPositionThreads < p.cells) buckets[turn][threadIdx.x + k * kPositionThreads] = next[k];
    __syncthreads();  // (the other buffer was read before the barrier of the tile before)
    const int count = static_cast<int>(min(static_cast<long long>(p.cells), cells - tile * p.cells)) * pieces;
    const T* from = z + tile * p.cells * p.c;
    T* to = y + tile * p.cells * p.c;
    bool looked = false;
    for (int q0 = threadIdx.x; q0 < count || !looked; q0 += kPositionFlight * kPositionThreads) {
      Piece<T, V> v[kPositionFlight];
#pragma unroll
      for (int k = 0; k < kPositionFlight; ++k)
        if (q0 + k * kPositionThreads < count) v[k] = load_piece<T, V>(from + static_cast<long long>(q0 + k * kPositionThreads) * V);
      if (!looked) {
        if (tile + gridDim.x < tiles) look(tile + gridDim.x);
        looked = true;
      }
#pragma unroll
      for (int k = 0; k < kPositionFlight; ++k) {
        const int q = q0 + k * kPositionThreads;
        if (q >= count) break;
        const int cell = p.magic == 0 ? q : static_cast<int>(__umulhi(static_cast<uint32_t>(q), p.magic)), piece = q - cell * pieces;
        const int row = buckets[turn][cell];
#pragma unroll
        for (int d = 0; d < QUADS; ++d) {
          const Piece<float, Q> t = p.table_in_smem ? *reinterpret_cast<const Piece<float, Q>*>(table + row * p.c + (d * pieces + piece) * Q)
                                                    : load_piece<float, Q>(p.table + row * p.c + piece * V + d * Q);
          add_piece<T, Q>(v[k].v + d * Q, t);
        }
        *reinterpret_cast<Piece<T, V>*>(to + static_cast<long long>(q) * V) = v[k];
      }
    }
  }
}

constexpr int kPositionChunk = 64;  // channels of a warp: two a lane
constexpr int kPositionWarps = 13;  // tables of sums of 66 buckets that fit into shared memory

// Sums over the buckets, in fixed orders: a warp owns 64 channels and a run of positions, of which it has 32 (fp32: 16) on their way while
// it adds up as many before them. Neighbouring positions of one bucket are added up in registers (most pairs are far apart and share the
// outer two), others in the warp's table in shared memory. The block adds its warps' tables up, and position_sums_kernel the blocks'.
// 768 x 768 x 128 bf16: 53 us for 151 MB, with 13 warps and 53 KB on their way an SM. What bounds it is the work between the loads, of
// 4 bytes a lane each, and in mixed runs a shuffle, a branch and a read and write of shared memory for a position (issue 49 % busy): two
// units on their way in 12 warps were slower (step 111 -> 120 us). More rows leave fewer warps: 130, 258 and 512 take 152, 349 and 804 us for
// a step's forward and backward where 66 take 104. (Buckets found after the values they are for had been asked for: 75; values
// converted as they came: 398.)
template <typename T, int V>
__global__ void __launch_bounds__(kPositionWarps * 32, 1) position_backward_kernel(const PositionParams p) {
  constexpr int R = sizeof(T) == 2 ? 32 : 16;  // positions that a warp looks at together
  extern __shared__ float4 sums_smem[];
  __shared__ int bucket_of[2 * B200_POSITION_MAX_REACH + 1];
  float* const sums = reinterpret_cast<float*>(sums_smem);  // [warps][buckets][kPositionChunk]
  grid_dependency_wait();
  grid_dependents_launch();
  const T* dy = static_cast<const T*>(p.dy);
  const int warps = blockDim.x / 32, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int table = p.buckets * kPositionChunk;
  for (int i = threadIdx.x; i < warps * table / 4; i += blockDim.x) sums_smem[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  position_buckets(p, bucket_of);
  __syncthreads();
  const int chunk = blockIdx.x % p.chunks, block = blockIdx.x / p.chunks;
  float* const own = sums + warp * table + lane * 2;
  // a lane without a channel of its own (or with one) reads the last ones again and writes them to columns that nobody reads
  const int c = min(chunk * kPositionChunk + lane * 2, p.c - V);
  const bool second = V == 1 && c + 1 < p.c;
  const int runs = (p.n + R - 1) / R;  // of a row
  const long long units = static_cast<long long>(p.b) * p.n * runs, teams = static_cast<long long>(p.blocks) * warps;
  const long long team = static_cast<long long>(block) * warps + warp, last = units * (team + 1) / teams;
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
  using Word = std::conditional_t<sizeof(T) == 2, uint32_t, uint2>;  // two channels of a position
  struct Unit {
    Word v[R];
    int bucket;
  };
  auto values = [](Word w) {
    if constexpr (sizeof(T) == 4)
      return make_float2(__uint_as_float(w.x), __uint_as_float(w.y));
    else if constexpr (std::is_same_v<T, __half>)
      return f16x2_to_float2(w);
    else
      return bf16x2_to_float2(w);
  };
  auto fetch = [&](long long unit, Unit& u) {
    const long long row = unit / runs;
    const int j0 = static_cast<int>(unit - row * runs) * R, most = p.n - 1 - j0;
    const T* at = dy + (row * p.n + j0) * p.c + c;
    auto read = [&](const T* from) -> Word {
      if constexpr (V == 2) {
        return __ldcg(reinterpret_cast<const Word*>(from));
      } else if constexpr (sizeof(T) == 4) {
        return make_uint2(__ldcg(reinterpret_cast<const uint32_t*>(from)), second ? __ldcg(reinterpret_cast<const uint32_t*>(from) + 1) : 0u);
      } else {
        const unsigned short* at16 = reinterpret_cast<const unsigned short*>(from);
        return __ldcg(at16) | (second ? static_cast<uint32_t>(__ldcg(at16 + 1)) << 16 : 0u);
      }
    };
    if (most >= R - 1) {
#pragma unroll
      for (int i = 0; i < R; ++i) u.v[i] = read(at + i * p.c);
    } else {  // (positions past the row's end: its last, not added)
#pragma unroll
      for (int i = 0; i < R; ++i) u.v[i] = read(at + min(i, most) * p.c);
    }
  };
  // its tokens, a lane a position, are asked for a unit before that, and their buckets found after the work on the unit between
  longlong2 mine, other;
  auto ask = [&](long long unit) {
    const long long row = unit / runs;
    const int j0 = static_cast<int>(unit - row * runs) * R;
    mine = position_token(p, row);
    other = position_token(p, row / p.n * p.n + min(j0 + lane, p.n - 1));
  };
  auto find = [&](long long unit) {
    const int j = static_cast<int>(unit % runs) * R + lane;
    return lane < R && j < p.n ? position_bucket(p, bucket_of, mine, other) : -1;
  };
  auto add = [&](const Unit& u) {
    const int bucket = __shfl_sync(0xFFFFFFFFu, u.bucket, 0);
    if (__all_sync(0xFFFFFFFFu, u.bucket == bucket || lane >= R)) {
      if (bucket != run) {
        flush();
        run = bucket;
      }
#pragma unroll
      for (int i = 0; i < R; ++i) {
        sum = __fadd2_rn(sum, values(u.v[i]));
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int b = __shfl_sync(0xFFFFFFFFu, u.bucket, i);
      if (b != run) {
        flush();
        run = b;
      }
      // (run -1: past the row's end; the sum is dropped)
      sum = __fadd2_rn(sum, values(u.v[i]));
    }
  };
  const long long begin = units * team / teams;
  Unit a, b;
  if (begin < last) {
    fetch(begin, a);
    ask(begin);
    a.bucket = find(begin);
    if (begin + 1 < last) ask(begin + 1), b.bucket = find(begin + 1);
  }
  auto step = [&](long long unit, Unit& now, Unit& next) {
    const bool more = unit + 2 < last;
    if (more) ask(unit + 2);  // (in front of the values: they come in the order they were asked for)
    if (unit + 1 < last) fetch(unit + 1, next);
    add(now);
    if (more) now.bucket = find(unit + 2);
  };
  for (long long unit = begin; unit < last; unit += 2) {
    step(unit, a, b);
    if (unit + 1 < last) step(unit + 1, b, a);
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
