// The join of two blocks on tiles of consecutive rows (see join.cuh for the formulas): what almost every call runs on.
//
// HBM bounds the join, and what a thread can keep in flight with loads of its own is bounded by its registers: the backward's five
// tensors a row, its sums over the rows and its parameters leave none for the next row (the kernels in join.cuh reach 0.5 to 1 TB/s).
// Here a warp of its own moves tiles of R consecutive rows, contiguous in memory, between HBM and a ring of stages in shared memory
// with bulk copies, in flight while 15 warps work on the stages before. A tile's start and size are multiples of 16 bytes whatever
// the width (R is chosen so; the last tile's odd bytes are copied by lanes), so rows of odd widths, which start anywhere, cost HBM
// what aligned ones cost. A thread reads its elements of a row from the stage, writes its results over its own inputs (y over x, h
// over u, dx over x or dy, du over u, dgate over gate) and the copying warp stores them from there.
// Parameters lie in shared memory as fp32 with the residual scale folded in (w_s = w scale, b_s = b scale): with z = e valid
// sigmoid(g), t scale = n w_s + b_s and the sums over the rows are four,  S1 = sum z n, S2 = sum z, S3 = sum dh n_y, S4 = sum dh:
//   d scale = w S1 + b S2 (or S1),  d w_post = scale S1,  d b_post = scale S2,  d w_pre = S3,  d b_pre = S4.
// What bounds it now is the issue of its arithmetic (about 500 instructions for a warp's 256 elements forward, 650 backward): bf16, every
// part, forward of 147456 x 128 38 us (5.0 TB/s), backward of 131072 x 128 72 us (3.7 TB/s), of 8192 x 1024 41 us (2.5 TB/s: four warps
// a row, whose sums meet at barriers); norm of 196608 x 64 16 and 25 us (3.1, 3.0 TB/s).
#pragma once

#include "blocks_status.cuh"
#include "join.cuh"

namespace trimul {

// Warps that compute; one more copies: four to a scheduler with 128 registers a thread, or two such blocks an SM with 64 (the
// backward of a norm alone, and the forward with eight elements of a row a thread, which rows of up to eight elements have).
constexpr int kTileWarps = 15;
constexpr int kTileThreads = kTileWarps * 32 + 32;
constexpr int kTileTeams = 7;                          // most teams of several warps
constexpr int kTileMaxStages = 8;
constexpr int kTileSmem = 224 * 1024;                  // of the 227 KB a block may have (the 228 KB of an SM)
constexpr int kTileSmemHalf = 112 * 1024;              // two blocks an SM: see above

struct JoinTileParams {
  JoinParams j;
  int tile_rows;       // R
  int tiles;           // ceil(rows / R)
  int stages;
  int slot;            // bytes of one tensor's place in a stage
  int slots;           // tensors in a stage
  int slot_of[5];      // x, u, gate, dy, dh: place in a stage, -1: not there
  int out_slot[3];     // forward: y, h; backward: dx, du, dgate; -1: not asked for
  int params;          // floats of one parameter vector in shared memory (the width of all threads of a row)
  int workers;         // threads that compute
  int block_tiles;     // backward with a shared gate: consecutive tiles of a block (0: every grid-th tile)
  int group_slots;     // ... and the gate rows that they can touch
};

// Shared memory by its 32-bit address: the compiler keeps no 64-bit pointers for it
__device__ __forceinline__ uint4 lds4(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void sts4(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
// Single words under a predicate: a branch for each would cost more than the access (82646 rows of 203, forward on tiles of one round: 129
// against 121 us)
__device__ __forceinline__ uint32_t lds_if(uint32_t a, bool on) {
  uint32_t v;
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %2, 0;\n\tmov.b32 %0, 0;\n\t@p ld.shared.b32 %0, [%1];\n\t}" : "=r"(v) : "r"(a), "r"(static_cast<uint32_t>(on)) : "memory");
  return v;
}
__device__ __forceinline__ void sts_if(uint32_t a, uint32_t v, bool on) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %2, 0;\n\t@p st.shared.b32 [%0], %1;\n\t}" ::"r"(a), "r"(v), "r"(static_cast<uint32_t>(on)) : "memory");
}
__device__ __forceinline__ void sts16_if(uint32_t a, uint32_t v, bool on) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %2, 0;\n\t@p st.shared.u16 [%0], %1;\n\t}" ::"r"(a), "h"(static_cast<unsigned short>(v)), "r"(static_cast<uint32_t>(on)) : "memory");
}
__device__ __forceinline__ float2 as_f2(uint32_t x, uint32_t y) { return make_float2(__uint_as_float(x), __uint_as_float(y)); }
__device__ __forceinline__ uint32_t bits(float v) { return __float_as_uint(v); }

// offset of parameter c in shared memory: pieces of four of eight neighbours apart, so that a warp's 16-byte reads are conflict-free
template <int VEC>
__device__ __forceinline__ int tile_param(int c, int params) {
  return VEC == 8 ? ((c >> 2) & 1) * (params >> 1) + (c >> 3) * 4 + (c & 3) : c;
}
// Column of element i of thread t. VEC neighbours are read at once: 8 (widths that are a multiple of eight), 2 (even ones), 3: two of a
// 16-bit type in rows of an odd width, of which every other one starts in the middle of a 32-bit word; 1 (fp32 rows of an odd width).
template <int VEC>
__device__ __forceinline__ int tile_col(int i, int t, int team) {
  constexpr int N = VEC == 3 ? 2 : VEC;
  return ((i / N) * team + t) * N + i % N;
}
template <int VEC, int NV>
__device__ __forceinline__ void tile_params(uint32_t w, int params, int t, int team, float2 (&v)[4 * NV]) {
  if constexpr (VEC == 8) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const uint32_t at = w + (j * team + t) * 16;
      const uint4 a = lds4(at), b = lds4(at + params * 2);
      v[4 * j] = as_f2(a.x, a.y);
      v[4 * j + 1] = as_f2(a.z, a.w);
      v[4 * j + 2] = as_f2(b.x, b.y);
      v[4 * j + 3] = as_f2(b.z, b.w);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4 * NV; ++i) {
      if constexpr (VEC == 2 || VEC == 3) {
        asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v[i].x), "=f"(v[i].y) : "r"(w + (i * team + t) * 8) : "memory");
      } else {
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v[i].x) : "r"(w + (2 * i * team + t) * 4) : "memory");
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v[i].y) : "r"(w + ((2 * i + 1) * team + t) * 4) : "memory");
      }
    }
  }
}

// A row's elements of this thread from a stage; zero past the width (EXACT: there is nothing past it, 8 NV elements of every thread are there)
template <typename T, int VEC, int NV, bool EXACT>
__device__ __forceinline__ void tile_load(uint32_t p, int d, int t, int team, float2 (&v)[4 * NV]) {
  if constexpr (VEC == 8) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * team + t) * 8;
      if (EXACT || c < d) {
        if constexpr (sizeof(T) == 2) {
          const uint4 w = lds4(p + c * 2);
          v[4 * j] = Io<T>::two(w.x);
          v[4 * j + 1] = Io<T>::two(w.y);
          v[4 * j + 2] = Io<T>::two(w.z);
          v[4 * j + 3] = Io<T>::two(w.w);
        } else {
          const uint4 a = lds4(p + c * 4), b = lds4(p + c * 4 + 16);
          v[4 * j] = as_f2(a.x, a.y);
          v[4 * j + 1] = as_f2(a.z, a.w);
          v[4 * j + 2] = as_f2(b.x, b.y);
          v[4 * j + 3] = as_f2(b.z, b.w);
        }
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) v[4 * j + k] = make_float2(0.f, 0.f);
      }
    }
  } else if constexpr (VEC == 2) {
#pragma unroll
    for (int i = 0; i < 4 * NV; ++i) {
      const int c = (i * team + t) * 2;
      if constexpr (sizeof(T) == 2)
        v[i] = Io<T>::two(lds_if(p + c * 2, c < d));
      else
        v[i] = as_f2(lds_if(p + c * 4, c < d), lds_if(p + c * 4 + 4, c < d));
    }
  } else if constexpr (VEC == 3) {
    // the two words that the pair may lie in, and the halves of them that it does
    const uint32_t word = p & ~3u, pick = (p & 2u) != 0 ? 0x5432u : 0x3210u;
#pragma unroll
    for (int i = 0; i < 4 * NV; ++i) {
      const int c = (i * team + t) * 2;
      const uint32_t w = __byte_perm(lds_if(word + c * 2, c < d), lds_if(word + c * 2 + 4, c < d), pick);
      v[i] = Io<T>::two(c + 1 == d ? w & 0xFFFFu : w);  // (past the end the other half is the next row's)
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4 * NV; ++i) {
      const int a = 2 * i * team + t, b = a + team;
      v[i] = as_f2(lds_if(p + a * 4, a < d), lds_if(p + b * 4, b < d));
    }
  }
}
template <typename T, int VEC, int NV, bool EXACT>
__device__ __forceinline__ void tile_store(uint32_t p, int d, int t, int team, const float2 (&v)[4 * NV]) {
  if constexpr (VEC == 8) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * team + t) * 8;
      if (!EXACT && c >= d) continue;
      if constexpr (sizeof(T) == 2) {
        sts4(p + c * 2, Io<T>::pack(v[4 * j].x, v[4 * j].y), Io<T>::pack(v[4 * j + 1].x, v[4 * j + 1].y), Io<T>::pack(v[4 * j + 2].x, v[4 * j + 2].y),
             Io<T>::pack(v[4 * j + 3].x, v[4 * j + 3].y));
      } else {
        sts4(p + c * 4, bits(v[4 * j].x), bits(v[4 * j].y), bits(v[4 * j + 1].x), bits(v[4 * j + 1].y));
        sts4(p + c * 4 + 16, bits(v[4 * j + 2].x), bits(v[4 * j + 2].y), bits(v[4 * j + 3].x), bits(v[4 * j + 3].y));
      }
    }
  } else if constexpr (VEC == 2) {
#pragma unroll
    for (int i = 0; i < 4 * NV; ++i) {
      const int c = (i * team + t) * 2;
      if constexpr (sizeof(T) == 2) {
        sts_if(p + c * 2, Io<T>::pack(v[i].x, v[i].y), c < d);
      } else {
        sts_if(p + c * 4, bits(v[i].x), c < d);
        sts_if(p + c * 4 + 4, bits(v[i].y), c < d);
      }
    }
  } else if constexpr (VEC == 3) {
    const bool odd = (p & 2u) != 0;
#pragma unroll
    for (int i = 0; i < 4 * NV; ++i) {
      const int c = (i * team + t) * 2;
      const uint32_t w = Io<T>::pack(v[i].x, v[i].y);
      const bool whole = !odd && c + 1 < d;
      sts_if(p + c * 2, w, whole);
      sts16_if(p + c * 2, w, !whole && c < d);
      sts16_if(p + c * 2 + 2, w >> 16, odd && c + 1 < d);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4 * NV; ++i) {
      const int a = 2 * i * team + t, b = a + team;
      sts_if(p + a * 4, bits(v[i].x), a < d);
      sts_if(p + b * 4, bits(v[i].y), b < d);
    }
  }
}
// A gate row that many rows share, from L2
template <typename T, int VEC, int NV>
__device__ __forceinline__ void tile_gate(const void* gate, long long row, int d, int t, int team, float2 (&v)[4 * NV]) {
  const T* p = static_cast<const T*>(gate) + row * d;
  if constexpr (VEC == 8) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * team + t) * 8;
      uint4 w = make_uint4(0u, 0u, 0u, 0u), u = w;
      if (c < d) {
        w = __ldcg(reinterpret_cast<const uint4*>(p + c));
        if (sizeof(T) == 4) u = __ldcg(reinterpret_cast<const uint4*>(p + c) + 1);
      }
      if constexpr (sizeof(T) == 2) {
        v[4 * j] = Io<T>::two(w.x);
        v[4 * j + 1] = Io<T>::two(w.y);
        v[4 * j + 2] = Io<T>::two(w.z);
        v[4 * j + 3] = Io<T>::two(w.w);
      } else {
        v[4 * j] = as_f2(w.x, w.y);
        v[4 * j + 1] = as_f2(w.z, w.w);
        v[4 * j + 2] = as_f2(u.x, u.y);
        v[4 * j + 3] = as_f2(u.z, u.w);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4 * NV; ++i) {
      const int a = tile_col<VEC>(2 * i, t, team), b = tile_col<VEC>(2 * i + 1, t, team);
      v[i] = make_float2(a < d ? Io<T>::get(p + a) : 0.f, b < d ? Io<T>::get(p + b) : 0.f);
    }
  }
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}
__device__ __forceinline__ void bulk_store(void* dst, uint32_t src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(src), "r"(bytes) : "memory");
}

__device__ __forceinline__ float exp2f_fast(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float reciprocal_fast(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float2 f2(float v) { return make_float2(v, v); }
// 1 / (1 + 2^(-g log2 e)), two at a time
__device__ __forceinline__ float2 sigmoid2(float2 g) {
  const float2 n = __fmul2_rn(g, f2(-1.44269504f));
  const float2 e = __fadd2_rn(make_float2(exp2f_fast(n.x), exp2f_fast(n.y)), f2(1.f));
  return make_float2(reciprocal_fast(e.x), reciprocal_fast(e.y));
}

// What both directions share: barriers, the ring, the copying warp
template <typename T>
struct TileRing {
  const JoinTileParams& p;
  uint8_t* stage0;     // shared memory
  uint32_t bars;       // full[stages], done[stages]
  volatile int* abort_flag;
  __device__ __forceinline__ uint32_t full(int s) const { return bars + 8u * s; }
  __device__ __forceinline__ uint32_t done(int s) const { return bars + 8u * (kTileMaxStages + s); }
  __device__ __forceinline__ uint8_t* stage(int s) const { return stage0 + s * p.slots * p.slot; }
  __device__ __forceinline__ int first() const { return p.block_tiles != 0 ? blockIdx.x * p.block_tiles : blockIdx.x; }
  __device__ __forceinline__ int step() const { return p.block_tiles != 0 ? 1 : gridDim.x; }
  __device__ __forceinline__ int count() const {
    if (p.block_tiles != 0) return max(0, min(p.block_tiles, p.tiles - first()));
    return first() < p.tiles ? (p.tiles - first() + gridDim.x - 1) / gridDim.x : 0;
  }
  // The copying warp. `in`: tensors by place (slot_of), `out`: by out_slot.
  template <int IN, int OUT>
  __device__ __forceinline__ void copy(const void* const (&in)[IN], void* const (&out)[OUT], int lane) const {
    const int n = count(), S = p.stages;
    const size_t row_bytes = static_cast<size_t>(p.j.d) * sizeof(T);
    auto bytes_of = [&](int tile) {
      const long long r0 = static_cast<long long>(tile) * p.tile_rows;
      const long long left = p.j.rows - r0;
      return static_cast<uint32_t>((left < p.tile_rows ? left : p.tile_rows) * row_bytes);
    };
    auto store = [&](int k) -> bool {
      const int tile = first() + k * step(), s = k % S;
      const bool got = mbar_wait_thread(done(s), (k / S) & 1, abort_flag, &blocks_status, kDevTimeoutProducer);
      if (!__all_sync(0xFFFFFFFFu, got && *abort_flag == 0)) return false;
      const size_t at = static_cast<size_t>(tile) * p.tile_rows * row_bytes;
      const uint32_t bytes = bytes_of(tile), whole = bytes & ~15u;
#pragma unroll
      for (int o = 0; o < OUT; ++o) {
        if (p.out_slot[o] < 0) continue;
        uint8_t* src = stage(s) + p.out_slot[o] * p.slot;
        uint8_t* dst = static_cast<uint8_t*>(out[o]) + at;
        if (lane == 0 && whole != 0) bulk_store(dst, smem_u32(src), whole);
        const uint32_t i = whole + lane * static_cast<uint32_t>(sizeof(T));
        if (i < bytes) *reinterpret_cast<T*>(dst + i) = *reinterpret_cast<const T*>(src + i);
      }
      if (lane == 0) bulk_commit();
      return true;
    };
    int stored = 0;
    bool ok = true;
    for (int k = 0; k < n && ok; ++k) {
      const int tile = first() + k * step(), s = k % S;
      while (ok && stored <= k - S) ok = store(stored++);
      if (!ok) break;
      if (k >= S) {
        if (lane == 0) bulk_wait_read<0>();
        __syncwarp();
      }
      const size_t at = static_cast<size_t>(tile) * p.tile_rows * row_bytes;
      const uint32_t bytes = bytes_of(tile), whole = bytes & ~15u;
      uint32_t expect = 0;
#pragma unroll
      for (int i = 0; i < IN; ++i) {
        if (p.slot_of[i] < 0 || in[i] == nullptr) continue;
        expect += whole;
        const uint32_t b = whole + lane * static_cast<uint32_t>(sizeof(T));
        if (b < bytes) {
          const T* src = reinterpret_cast<const T*>(static_cast<const uint8_t*>(in[i]) + at + b);
          Io<T>::put(reinterpret_cast<T*>(stage(s) + p.slot_of[i] * p.slot + b), Io<T>::get(src));
        }
      }
      __syncwarp();
      if (lane == 0) {
        mbar_arrive_expect_tx(full(s), expect);
        if (whole != 0) {
#pragma unroll
          for (int i = 0; i < IN; ++i)
            if (p.slot_of[i] >= 0 && in[i] != nullptr)
              bulk_load(smem_u32(stage(s) + p.slot_of[i] * p.slot), static_cast<const uint8_t*>(in[i]) + at, whole, full(s));
        }
      }
    }
    while (ok && stored < n) ok = store(stored++);
    if (lane == 0) bulk_wait<0>();
    if (!ok) {  // loads that no warp has waited for have landed before the block may exit
      for (int s = 0; s < S; ++s) {
        const long long t0 = clock64();
        while (stored + s < n && !mbar_try_wait(full((stored + s) % S), ((stored + s) / S) & 1) && clock64() - t0 < kWaitLimitCycles) {
        }
      }
    }
  }
};

// Sums over a team, the same bits in every thread (as TeamSum, the steps unrolled)
struct TileSum {
  float2* scratch;
  int team, warps, id, half, warp_in_team;
  template <typename F>
  __device__ __forceinline__ void steps(F f) const {
    if (team >= 32) {
      f(16), f(8), f(4), f(2), f(1);
    } else if (team == 16) {
      f(8), f(4), f(2), f(1);
    } else {
      if (team >= 8) f(4);
      if (team >= 4) f(2);
      if (team >= 2) f(1);
    }
  }
  // every warp's value in shared memory, ready to be read
  __device__ __forceinline__ const float2* exchange(float2 v) {
    float2* s = scratch + half * 16;
    half ^= 1;
    if ((threadIdx.x & 31) == 0) s[warp_in_team] = v;
    named_bar_sync(1 + id, team);
    return s;
  }
  __device__ __forceinline__ float one(float v) {
    steps([&](int o) { v += __shfl_xor_sync(0xFFFFFFFFu, v, o); });
    if (warps > 1) {
      const float2* s = exchange(make_float2(v, 0.f));
      v = 0.f;
      for (int i = 0; i < warps; ++i) v += s[i].x;
    }
    return v;
  }
  __device__ __forceinline__ float2 two(float2 v) {
    steps([&](int o) {
      const float a = __shfl_xor_sync(0xFFFFFFFFu, v.x, o), b = __shfl_xor_sync(0xFFFFFFFFu, v.y, o);
      v = __fadd2_rn(v, make_float2(a, b));
    });
    if (warps > 1) {
      const float2* s = exchange(v);
      v = f2(0.f);
      for (int i = 0; i < warps; ++i) v = __fadd2_rn(v, s[i]);
    }
    return v;
  }
  // Mean and sum of squared deviations of a row from those of each thread's `n` values, merged pairwise (the deviations of two
  // equal parts add (difference of the means)^2 n / 2): one exchange instead of one for the mean and one for the deviations
  __device__ __forceinline__ float2 merge(float mean, float dev, float n) {
    steps([&](int o) {
      const float m = __shfl_xor_sync(0xFFFFFFFFu, mean, o), q = __shfl_xor_sync(0xFFFFFFFFu, dev, o);
      const float delta = m - mean;
      mean = 0.5f * (mean + m);
      dev = fmaf(delta * delta, 0.5f * n, dev + q);
      n += n;
    });
    if (warps > 1) {
      const float2* s = exchange(make_float2(mean, dev));
      mean = dev = 0.f;
      for (int i = 0; i < warps; ++i) mean += s[i].x;
      mean = __fdividef(mean, static_cast<float>(warps));
      for (int i = 0; i < warps; ++i) {
        const float delta = s[i].x - mean;
        dev += fmaf(delta * delta, n, s[i].y);
      }
    }
    return make_float2(mean, dev);
  }
};

// mean and 1 / sigma of a row. (With eight elements a thread, rows of eight, where two blocks share an SM, the merged form's
// instructions cost more than the second exchange's latency.)
template <int VEC, int NV, bool EXACT>
__device__ __forceinline__ float2 tile_stats(const float2 (&v)[4 * NV], int kind, float eps, int d, float inv, int t, int team, TileSum& sum) {
  float mean = 0.f, dev;
  if (EXACT && NV > 1 && kind == kNormLayer) {
    float2 a = v[0], q = f2(0.f);
#pragma unroll
    for (int i = 1; i < 4 * NV; ++i) a = __fadd2_rn(a, v[i]);
    mean = (a.x + a.y) * (1.0f / (8 * NV));
#pragma unroll
    for (int i = 0; i < 4 * NV; ++i) {
      const float2 c = __fadd2_rn(v[i], f2(-mean));
      q = __ffma2_rn(c, c, q);
    }
    const float2 all = sum.merge(mean, q.x + q.y, 8 * NV);
    mean = all.x;
    dev = all.y;
  } else {
    if (kind == kNormLayer) {
      float2 a = f2(0.f);
#pragma unroll
      for (int i = 0; i < 4 * NV; ++i) a = __fadd2_rn(a, v[i]);
      mean = sum.one(a.x + a.y) * inv;
    }
    float2 q = f2(0.f);
#pragma unroll
    for (int i = 0; i < 4 * NV; ++i) {
      float2 c = __fadd2_rn(v[i], f2(-mean));
      if (!EXACT && tile_col<VEC>(2 * i, t, team) >= d) c.x = 0.f;
      if (!EXACT && tile_col<VEC>(2 * i + 1, t, team) >= d) c.y = 0.f;
      q = __ffma2_rn(c, c, q);
    }
    dev = sum.one(q.x + q.y);
  }
  return make_float2(mean, rsqrtf(fmaf(dev, inv, eps)));
}

// Shared memory: parameters | scratch of the sums | barriers | stages | what the last row's words reach past its end (odd widths)
constexpr int kTileScratch = kTileTeams * 32 * 8 + 2 * kTileMaxStages * 8 + 16;
constexpr int kTileTail = 16;

template <typename T, int VEC, int NV, bool EXACT>
__global__ void __launch_bounds__(kTileThreads, NV == 1 ? 2 : 1) join_tile_forward_kernel(const JoinTileParams p) {
  extern __shared__ __align__(128) uint8_t smem[];
  float* par = reinterpret_cast<float*>(smem);  // w_s, b_s, w_pre, b_pre
  const uint32_t par_at = smem_u32(smem);
  uint8_t* at = smem + 4 * p.params * 4;
  float2* scratch = reinterpret_cast<float2*>(at);
  const uint32_t bars = smem_u32(at + kTileTeams * 32 * 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(at + kTileTeams * 32 * 8 + 2 * kTileMaxStages * 8);
  const TileRing<T> ring{p, at + kTileScratch, bars, abort_flag};
  const JoinParams& j = p.j;
  const int lane = threadIdx.x & 31;
  const int workers = blockDim.x - 32;
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(ring.full(s), 1);
      mbar_init(ring.done(s), workers / 32);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  grid_dependency_wait();
  grid_dependents_launch();
  for (int c = threadIdx.x; c < p.params; c += blockDim.x) {
    const bool in = c < j.d;
    const float s = in ? (j.scale != nullptr ? __ldcg(j.scale + c) : 1.f) : 0.f;
    const int o = tile_param<VEC>(c, p.params);
    par[o] = in && j.post_w != nullptr ? __ldcg(j.post_w + c) * s : s;
    par[p.params + o] = in && j.post_b != nullptr ? __ldcg(j.post_b + c) * s : 0.f;
    par[2 * p.params + o] = in ? (j.pre_w != nullptr ? __ldcg(j.pre_w + c) : 1.f) : 0.f;
    par[3 * p.params + o] = in && j.pre_b != nullptr ? __ldcg(j.pre_b + c) : 0.f;
  }
  __syncthreads();
  if (static_cast<int>(threadIdx.x) >= workers) {
    const void* const in[3] = {j.x, j.u, j.gate};
    void* const out[2] = {j.y, j.h};
    ring.copy(in, out, lane);
    return;
  }
  const int d = j.d, team = j.team, t = threadIdx.x % team, id = threadIdx.x / team, teams = workers / team;
  TileSum sum{scratch + (team > 32 ? id : 0) * 32, team, (team + 31) / 32, id, 0, t >> 5};
  const float inv = 1.0f / static_cast<float>(d);
  const int row_bytes = d * static_cast<int>(sizeof(T));
  const int n = ring.count();
  const uint32_t stage_bytes = p.slots * p.slot, ring_at = smem_u32(ring.stage0);
  const long long tile_step = static_cast<long long>(ring.step()) * p.tile_rows;
  long long r0 = static_cast<long long>(ring.first()) * p.tile_rows;
  int s = 0;
  uint32_t ph = 0, stage = ring_at;
  for (int k = 0; k < n; ++k) {
    // (a wait that gave up: the warps go on over what there is, every later wait returns at once, and none is missing at a barrier)
    mbar_wait_warp(ring.full(s), ph, abort_flag, &blocks_status, kDevTimeoutStats);
    const int rows = j.rows - r0 < p.tile_rows ? static_cast<int>(j.rows - r0) : p.tile_rows;
    for (int r = id; r - id < p.tile_rows; r += teams) {
      const long long row = r0 + r;
      const bool on = r < rows;
      const int off = on ? r * row_bytes : 0;
      float2 x[4 * NV], w[4 * NV];
      tile_load<T, VEC, NV, EXACT>(stage + p.slot_of[0] * p.slot + off, d, t, team, x);
      if (j.u != nullptr) {
        const bool valid = on && (j.mask == nullptr || __ldcg(j.mask + row) != 0);
        float2 u[4 * NV];
        tile_load<T, VEC, NV, EXACT>(stage + p.slot_of[1] * p.slot + off, d, t, team, u);
        if (j.post_kind != kNormNone) {
          const float2 st = tile_stats<VEC, NV, EXACT>(u, j.post_kind, j.post_eps, d, inv, t, team, sum);
          if (on && t == 0 && j.post_stats != nullptr) j.post_stats[row] = st;
#pragma unroll
          for (int i = 0; i < 4 * NV; ++i) u[i] = __fmul2_rn(__fadd2_rn(u[i], f2(-st.x)), f2(st.y));
        }
        // (without weight and scale too where a layer norm has left -mean / sigma past the width: the zeros that stand there keep it out of
        // the next norm's mean; selects in that mean would cost every call of such widths 3 %)
        if (j.post_w != nullptr || j.scale != nullptr || (!EXACT && j.post_kind == kNormLayer)) {
          tile_params<VEC, NV>(par_at, p.params, t, team, w);
#pragma unroll
          for (int i = 0; i < 4 * NV; ++i) u[i] = __fmul2_rn(u[i], w[i]);
        }
        if (j.post_b != nullptr) {
          tile_params<VEC, NV>(par_at + 4 * p.params, p.params, t, team, w);
#pragma unroll
          for (int i = 0; i < 4 * NV; ++i) u[i] = __fadd2_rn(u[i], w[i]);
        }
        if (j.gate != nullptr) {
          if (p.slot_of[2] >= 0) {
            tile_load<T, VEC, NV, EXACT>(stage + p.slot_of[2] * p.slot + off, d, t, team, w);
          } else {
            tile_gate<T, VEC, NV>(j.gate, on ? row / j.gate_rows : 0, d, t, team, w);
          }
#pragma unroll
          for (int i = 0; i < 4 * NV; ++i) u[i] = __fmul2_rn(u[i], sigmoid2(w[i]));
        }
        if (valid) {
#pragma unroll
          for (int i = 0; i < 4 * NV; ++i) x[i] = __fadd2_rn(x[i], u[i]);
        }
        if (on) tile_store<T, VEC, NV, EXACT>(stage + p.out_slot[0] * p.slot + off, d, t, team, x);
      }
      if (j.pre_kind != kNormNone) {
        const float2 st = tile_stats<VEC, NV, EXACT>(x, j.pre_kind, j.pre_eps, d, inv, t, team, sum);
        if (on && t == 0 && j.pre_stats != nullptr) j.pre_stats[row] = st;
        tile_params<VEC, NV>(par_at + 4 * 2 * p.params, p.params, t, team, w);
#pragma unroll
        for (int i = 0; i < 4 * NV; ++i) x[i] = __fmul2_rn(__fmul2_rn(__fadd2_rn(x[i], f2(-st.x)), f2(st.y)), w[i]);
        if (j.pre_b != nullptr) {
          tile_params<VEC, NV>(par_at + 4 * 3 * p.params, p.params, t, team, w);
#pragma unroll
          for (int i = 0; i < 4 * NV; ++i) x[i] = __fadd2_rn(x[i], w[i]);
        }
        if (on) tile_store<T, VEC, NV, EXACT>(stage + p.out_slot[1] * p.slot + off, d, t, team, x);
      }
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(ring.done(s));
    r0 += tile_step;
    stage += stage_bytes;
    if (++s == p.stages) {
      s = 0;
      ph ^= 1u;
      stage = ring_at;
    }
  }
}

// A shared gate's gradient: a team adds up its rows of the current gate row in registers and leaves them in fp32 when the gate row
// changes, in a place of its own for each gate row that the block's tiles touch ([blocks][group_slots][teams][8 team]);
// join_tile_gate_kernel adds them up in the order of the blocks and teams.
template <typename T, int VEC, bool EXACT, bool JOIN>
__global__ void __launch_bounds__(kTileThreads, JOIN ? 1 : 2) join_tile_backward_kernel(const JoinTileParams p) {
  extern __shared__ __align__(128) uint8_t smem[];
  float* par = reinterpret_cast<float*>(smem);  // w_s, b_s, w_pre
  const uint32_t par_at = smem_u32(smem);
  uint8_t* at = smem + 3 * p.params * 4;
  float2* scratch = reinterpret_cast<float2*>(at);
  const uint32_t bars = smem_u32(at + kTileTeams * 32 * 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(at + kTileTeams * 32 * 8 + 2 * kTileMaxStages * 8);
  const TileRing<T> ring{p, at + kTileScratch, bars, abort_flag};
  const JoinParams& j = p.j;
  const int lane = threadIdx.x & 31;
  const int workers = blockDim.x - 32;
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(ring.full(s), 1);
      mbar_init(ring.done(s), workers / 32);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  grid_dependency_wait();
  grid_dependents_launch();
  for (int c = threadIdx.x; c < p.params; c += blockDim.x) {
    const bool in = c < j.d;
    const float s = in ? (j.scale != nullptr ? __ldcg(j.scale + c) : 1.f) : 0.f;
    const int o = tile_param<VEC>(c, p.params);
    par[o] = in && j.post_w != nullptr ? __ldcg(j.post_w + c) * s : s;
    par[p.params + o] = in && j.post_b != nullptr ? __ldcg(j.post_b + c) * s : 0.f;
    par[2 * p.params + o] = in ? (j.pre_w != nullptr ? __ldcg(j.pre_w + c) : 1.f) : 0.f;
  }
  __syncthreads();
  const int d = j.d, team = j.team, t = threadIdx.x % team, id = threadIdx.x / team, teams = workers / team;
  const int n = ring.count();
  float2 s1[4], s2[4], s3[4], s4[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) s1[i] = s2[i] = s3[i] = s4[i] = f2(0.f);
  if (static_cast<int>(threadIdx.x) >= workers) {
    const void* const in[5] = {j.x, j.u, j.gate, j.dy, j.dh};
    void* const out[3] = {j.dx, j.du, j.dgate};
    ring.copy(in, out, lane);
  } else {
    TileSum sum{scratch + (team > 32 ? id : 0) * 32, team, (team + 31) / 32, id, 0, t >> 5};
    const float inv = 1.0f / static_cast<float>(d);
    const int row_bytes = d * static_cast<int>(sizeof(T));
    const bool shared_gate = JOIN && p.block_tiles != 0;
    float2 sg_sum[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) sg_sum[i] = f2(0.f);
    const long long first_row = static_cast<long long>(ring.first()) * p.tile_rows;
    const long long first_group = shared_gate ? first_row / j.gate_rows : 0;
    long long group = first_group;
    auto leave_gate = [&]() {
      float* o = j.gate_part + ((static_cast<long long>(blockIdx.x) * p.group_slots + (group - first_group)) * teams + id) * (8 * team);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        o[2 * i * team + t] = sg_sum[i].x;
        o[(2 * i + 1) * team + t] = sg_sum[i].y;
        sg_sum[i] = f2(0.f);
      }
    };
    const uint32_t stage_bytes = p.slots * p.slot, ring_at = smem_u32(ring.stage0);
    const long long tile_step = static_cast<long long>(ring.step()) * p.tile_rows;
    long long r0 = first_row;
    int s = 0;
    uint32_t ph = 0, stage = ring_at;
    // statistics and mask of the team's next row, asked for while this one is worked on
    float2 next_post = f2(0.f), next_pre = f2(0.f);
    int next_valid = 0;
    auto row_facts = [&](long long tile_row, int r) {
      const long long row = tile_row + r;
      next_valid = 0;
      if (r >= p.tile_rows || row >= j.rows) return;
      if (JOIN) next_valid = j.mask == nullptr ? 1 : __ldcg(j.mask + row);
      if (JOIN && j.post_kind != kNormNone) next_post = __ldcg(j.post_stats + row);
      if (j.pre_kind != kNormNone) next_pre = __ldcg(j.pre_stats + row);
    };
    if (n > 0) row_facts(r0, id);
    for (int k = 0; k < n; ++k) {
      const int rows = j.rows - r0 < p.tile_rows ? static_cast<int>(j.rows - r0) : p.tile_rows;
      mbar_wait_warp(ring.full(s), ph, abort_flag, &blocks_status, kDevTimeoutStats);  // (as in the forward)
      for (int r = id; r - id < p.tile_rows; r += teams) {
        const bool on = r < rows;
        const bool valid = next_valid != 0;
        const float2 post = next_post, pre = next_pre;
        if (r - id + teams < p.tile_rows)
          row_facts(r0, r + teams);
        else if (k + 1 < n)
          row_facts(r0 + tile_step, id);
        const long long row = r0 + r;
        const int off = on ? r * row_bytes : 0;
        float2 x[4], e[4], q[4], u[4], g[4], w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = e[i] = u[i] = f2(0.f), g[i] = f2(1.f);
        if (j.pre_kind != kNormNone && on) tile_load<T, VEC, 1, EXACT>(stage + p.slot_of[0] * p.slot + off, d, t, team, x);
        if (JOIN && j.dy != nullptr && on) tile_load<T, VEC, 1, EXACT>(stage + p.slot_of[3] * p.slot + off, d, t, team, e);
        if (JOIN && valid) {
          tile_load<T, VEC, 1, EXACT>(stage + p.slot_of[1] * p.slot + off, d, t, team, u);
          if (j.gate != nullptr) {
            if (!shared_gate) {
              tile_load<T, VEC, 1, EXACT>(stage + p.slot_of[2] * p.slot + off, d, t, team, g);
            } else {
              tile_gate<T, VEC, 1>(j.gate, row / j.gate_rows, d, t, team, g);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) g[i] = sigmoid2(g[i]);
          }
          if (j.post_kind != kNormNone) {
#pragma unroll
            for (int i = 0; i < 4; ++i) u[i] = __fmul2_rn(__fadd2_rn(u[i], f2(-post.x)), f2(post.y));
          }
        }
        if (j.pre_kind != kNormNone) {
          if (JOIN && valid) {
            tile_params<VEC, 1>(par_at, p.params, t, team, w);
            if (j.post_b != nullptr) {
              tile_params<VEC, 1>(par_at + 4 * p.params, p.params, t, team, q);
#pragma unroll
              for (int i = 0; i < 4; ++i) x[i] = __ffma2_rn(__ffma2_rn(u[i], w[i], q[i]), g[i], x[i]);
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i) x[i] = __ffma2_rn(__fmul2_rn(u[i], w[i]), g[i], x[i]);
            }
          }
          if (j.dh != nullptr && on) {
            tile_load<T, VEC, 1, EXACT>(stage + p.slot_of[4] * p.slot + off, d, t, team, q);
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) q[i] = f2(0.f);
          }
          tile_params<VEC, 1>(par_at + 4 * 2 * p.params, p.params, t, team, w);
          float2 c1 = f2(0.f), c2 = f2(0.f);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            x[i] = __fmul2_rn(__fadd2_rn(x[i], f2(-pre.x)), f2(pre.y));
            s3[i] = __ffma2_rn(q[i], x[i], s3[i]);
            s4[i] = __fadd2_rn(s4[i], q[i]);
            q[i] = __fmul2_rn(q[i], w[i]);
            c1 = __fadd2_rn(c1, q[i]);
            c2 = __ffma2_rn(q[i], x[i], c2);
          }
          const float2 c = sum.two(make_float2(c1.x + c1.y, c2.x + c2.y));
          const float m1 = j.pre_kind == kNormLayer ? -c.x * inv : 0.f, m2 = -c.y * inv;
#pragma unroll
          for (int i = 0; i < 4; ++i) e[i] = __ffma2_rn(f2(pre.y), __ffma2_rn(x[i], f2(m2), __fadd2_rn(q[i], f2(m1))), e[i]);
        }
        if (on && p.out_slot[0] >= 0) tile_store<T, VEC, 1, EXACT>(stage + p.out_slot[0] * p.slot + off, d, t, team, e);
        if constexpr (!JOIN) continue;
        float2 a1 = f2(0.f), a2 = f2(0.f);
        tile_params<VEC, 1>(par_at, p.params, t, team, w);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          e[i] = valid ? __fmul2_rn(e[i], g[i]) : f2(0.f);  // z
          s1[i] = __ffma2_rn(e[i], u[i], s1[i]);
          s2[i] = __fadd2_rn(s2[i], e[i]);
          q[i] = __fmul2_rn(e[i], w[i]);
          a1 = __fadd2_rn(a1, q[i]);
          a2 = __ffma2_rn(q[i], u[i], a2);
        }
        if (j.gate != nullptr && j.dgate != nullptr) {
          // gradient of the logits: z (n w_s + b_s) (1 - sigmoid)
          float2 b[4];
          if (j.post_b != nullptr) {
            tile_params<VEC, 1>(par_at + 4 * p.params, p.params, t, team, b);
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) b[i] = f2(0.f);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i)
            g[i] = __fmul2_rn(__fmul2_rn(e[i], __ffma2_rn(u[i], w[i], b[i])), __fadd2_rn(f2(1.f), make_float2(-g[i].x, -g[i].y)));
          if (!shared_gate) {
            if (on) tile_store<T, VEC, 1, EXACT>(stage + p.out_slot[2] * p.slot + off, d, t, team, g);
          } else if (on) {
            const long long now = row / j.gate_rows;
            if (now != group) {
              leave_gate();
              for (++group; group < now; ++group) leave_gate();  // (gate rows between, of which this team has no row)
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) sg_sum[i] = __fadd2_rn(sg_sum[i], g[i]);
          }
        }
        if (j.post_kind != kNormNone) {
          const float2 c = sum.two(make_float2(a1.x + a1.y, a2.x + a2.y));
          const float m1 = j.post_kind == kNormLayer ? -c.x * inv : 0.f, m2 = -c.y * inv;
#pragma unroll
          for (int i = 0; i < 4; ++i) q[i] = __fmul2_rn(f2(post.y), __ffma2_rn(u[i], f2(m2), __fadd2_rn(q[i], f2(m1))));
        }
        if (!valid) {
#pragma unroll
          for (int i = 0; i < 4; ++i) q[i] = f2(0.f);
        }
        if (on && p.out_slot[1] >= 0) tile_store<T, VEC, 1, EXACT>(stage + p.out_slot[1] * p.slot + off, d, t, team, q);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(ring.done(s));
      r0 += tile_step;
      stage += stage_bytes;
      if (++s == p.stages) {
        s = 0;
        ph ^= 1u;
        stage = ring_at;
      }
    }
    if (shared_gate && j.dgate != nullptr && n > 0) {
      long long last = first_row + static_cast<long long>(n) * p.tile_rows;
      last = (last < j.rows ? last : j.rows) - 1;
      const long long end = last / j.gate_rows;
      for (; group <= end; ++group) leave_gate();
    }
  }
  if (j.sums == nullptr) return;
  // The block's teams, one sum after the other, through the (idle) stages
  float* buf = reinterpret_cast<float*>(ring.stage0);
  const bool worker = static_cast<int>(threadIdx.x) < workers;
#pragma unroll
  for (int s = JOIN ? 0 : 2; s < 4; ++s) {
    const float2(&v)[4] = s == 0 ? s1 : s == 1 ? s2 : s == 2 ? s3 : s4;
    __syncthreads();
    if (worker) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        buf[id * 8 * team + 2 * i * team + t] = v[i].x;
        buf[id * 8 * team + (2 * i + 1) * team + t] = v[i].y;
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < 8 * team; c += blockDim.x) {
      float a = 0.f;
      for (int k = 0; k < teams; ++k) a += buf[k * 8 * team + c];
      const int col = tile_col<VEC>(c / team, c % team, team);
      if (col < d) j.sums[(static_cast<size_t>(blockIdx.x) * 4 + s) * d + col] = a;
    }
  }
}

// The blocks' four sums, 32 chains a column, and the five gradients from them
struct JoinTileSums {
  const float* sums;  // [blocks][4][d]
  const float *scale, *post_w, *post_b;
  float* out[5];      // d scale, d post_w, d post_b, d pre_w, d pre_b; null: not asked for
  int blocks, d, post_kind;
};
__global__ void __launch_bounds__(1024) join_tile_sums_kernel(const JoinTileSums p) {
  __shared__ float part[2][32][33];
  grid_dependency_wait();
  grid_dependents_launch();
  const int x = threadIdx.x & 31, chain = threadIdx.x >> 5, c = blockIdx.x * 32 + x;
  const int pair = blockIdx.y;  // S1 and S2, or S3 and S4
  float a = 0.f, b = 0.f;
  if (c < p.d)
    for (int k0 = chain; k0 < p.blocks; k0 += 5 * 32) {  // (ten loads in flight, all that one block an SM leaves: 6.5 -> 5 us)
      float va[5], vb[5];
#pragma unroll
      for (int i = 0; i < 5; ++i) {
        const int k = k0 + i * 32;
        const float* s = p.sums + (static_cast<size_t>(k) * 4 + pair * 2) * p.d + c;
        va[i] = k < p.blocks ? __ldcg(s) : 0.f;
        vb[i] = k < p.blocks ? __ldcg(s + p.d) : 0.f;
      }
#pragma unroll
      for (int i = 0; i < 5; ++i) a += va[i], b += vb[i];
    }
  part[0][chain][x] = a;
  part[1][chain][x] = b;
  __syncthreads();
  if (chain != 0 || c >= p.d) return;
  a = b = 0.f;
  for (int k = 0; k < 32; ++k) {
    a += part[0][k][x];
    b += part[1][k][x];
  }
  if (pair == 1) {
    if (p.out[3] != nullptr) p.out[3][c] = a;
    if (p.out[4] != nullptr) p.out[4][c] = b;
    return;
  }
  const float scale = p.scale != nullptr ? __ldcg(p.scale + c) : 1.f;
  const float w = p.post_kind != kNormNone && p.post_w != nullptr ? __ldcg(p.post_w + c) : 1.f;
  const float bias = p.post_kind != kNormNone && p.post_b != nullptr ? __ldcg(p.post_b + c) : 0.f;
  if (p.out[0] != nullptr) p.out[0][c] = fmaf(w, a, bias * b);
  if (p.out[1] != nullptr) p.out[1][c] = scale * a;
  if (p.out[2] != nullptr) p.out[2][c] = scale * b;
}

// Gradient of the shared gate rows: the teams of every block that has rows of one, 32 chains a column
template <typename T, int VEC>
__global__ void __launch_bounds__(1024) join_tile_gate_kernel(const JoinTileParams p) {
  __shared__ float part[32][33];
  grid_dependency_wait();
  grid_dependents_launch();
  const JoinParams& j = p.j;
  const int x = threadIdx.x & 31, chain = threadIdx.x >> 5;
  const int team = j.team, teams = p.workers / team;
  const long long block_rows = static_cast<long long>(p.block_tiles) * p.tile_rows;
  const long long group = blockIdx.x, begin = group * j.gate_rows, end = begin + j.gate_rows;
  const int b0 = static_cast<int>(begin / block_rows), b1 = static_cast<int>((end - 1) / block_rows);
  const int c = blockIdx.y * 32 + x;  // element of the teams' order
  float a = 0.f;
  if (c < 8 * team) {
    // (the first block's rows may begin in an earlier gate row; every later block begins in this one)
    const int slot = static_cast<int>(group - b0 * block_rows / j.gate_rows);
    const int places = (b1 - b0 + 1) * teams;
#pragma unroll 4
    for (int k = chain; k < places; k += 32) {
      const int block = k / teams;
      const long long place = (static_cast<long long>(b0 + block) * p.group_slots + (block == 0 ? slot : 0)) * teams + k - block * teams;
      a += __ldcg(j.gate_part + place * (8 * team) + c);
    }
  }
  part[chain][x] = a;
  __syncthreads();
  if (chain != 0) return;
  a = 0.f;
  for (int k = 0; k < 32; ++k) a += part[k][x];
  const int col = tile_col<VEC>(c / team, c % team, team);
  if (c < 8 * team && col < j.d) Io<T>::put(static_cast<T*>(j.dgate) + group * j.d + col, a);
}

}  // namespace trimul
