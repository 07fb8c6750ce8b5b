// Dropout on a block's output with the residual add: y = x + keep u / (1 - p), and its gradient du = keep dy / (1 - p) by the same
// kernels without x. The mask is never stored: which elements stay follows from their place and a key of two 64-bit words, by the
// counter-based generator Philox-4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", 2011). Counter:
// the place of eight elements (two words) and the key's second word; key: its first. The eight 16-bit halves of the result, low half
// of each word first, are compared with the threshold round(65536 p): an element stays with probability 1 - threshold / 65536, and the
// kept ones are scaled by the inverse of exactly that, so that the expectation is u whatever p rounds to.
#pragma once

#include "ptx.cuh"

namespace trimul {

struct DropoutParams {
  const void* x;  // null: none
  const void* u;
  void* y;
  const long long* key;
  unsigned long long call;  // added to the key's second word
  long long outer, inner;   // mask elements: outer * inner; u: [outer, shared, inner]
  long long shared, chunk;  // rows under one mask, and how many of them a thread takes
  uint32_t threshold;
  float scale;
};

__device__ __forceinline__ uint4 philox(uint4 c, uint2 k) {
#pragma unroll
  for (int turn = 0; turn < 10; ++turn) {
    const uint64_t a = static_cast<uint64_t>(c.x) * 0xD2511F53u, b = static_cast<uint64_t>(c.z) * 0xCD9E8D57u;
    c = make_uint4(static_cast<uint32_t>(b >> 32) ^ c.y ^ k.x, static_cast<uint32_t>(b), static_cast<uint32_t>(a >> 32) ^ c.w ^ k.y,
                   static_cast<uint32_t>(a));
    k.x += 0x9E3779B9u;
    k.y += 0xBB67AE85u;
  }
  return c;
}

struct DropoutKey {
  uint2 k;
  uint32_t hi0, hi1;
  __device__ __forceinline__ explicit DropoutKey(const DropoutParams& p) {
    const unsigned long long a = static_cast<unsigned long long>(__ldcg(p.key)), b = static_cast<unsigned long long>(__ldcg(p.key + 1)) + p.call;
    k = make_uint2(static_cast<uint32_t>(a), static_cast<uint32_t>(a >> 32));
    hi0 = static_cast<uint32_t>(b);
    hi1 = static_cast<uint32_t>(b >> 32);
  }
  __device__ __forceinline__ uint4 numbers(long long block) const {
    return philox(make_uint4(static_cast<uint32_t>(block), static_cast<uint32_t>(static_cast<unsigned long long>(block) >> 32), hi0, hi1), k);
  }
};
__device__ __forceinline__ uint32_t half_of(uint4 r, int i) {
  const uint32_t w = i < 2 ? r.x : i < 4 ? r.y : i < 6 ? r.z : r.w;
  return i & 1 ? w >> 16 : w & 0xFFFFu;
}

template <typename T>
__device__ __forceinline__ float to_float(T v) {
  return static_cast<float>(v);
}
template <typename T>
__device__ __forceinline__ T from_float(float v) {
  return static_cast<T>(v);
}
// eight elements, as the words that they lie in
template <typename T>
struct Eight {
  static constexpr int kWords = sizeof(T) / 2;
  uint4 w[kWords];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = __ldcg(reinterpret_cast<const uint4*>(p) + i);
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < kWords; ++i) reinterpret_cast<uint4*>(p)[i] = w[i];
  }
  __device__ __forceinline__ T& at(int i) { return reinterpret_cast<T*>(w)[i]; }
};

template <typename T>
__device__ __forceinline__ T dropped(T x, T u, bool keep, float scale, bool residual) {
  // (an element that is dropped is x itself whatever u holds)
  if (!keep) return residual ? x : from_float<T>(0.f);
  return from_float<T>(residual ? fmaf(to_float(u), scale, to_float(x)) : to_float(u) * scale);
}

constexpr int kDropoutThreads = 256;
constexpr int kDropoutFlight = 4;  // pieces of eight elements that a thread loads at once

// Eight elements under one mask group: y from x and u
template <typename T, bool RESIDUAL>
__device__ __forceinline__ void drop_eight(const DropoutParams& p, uint4 r, Eight<T>& x, Eight<T>& u, T* y) {
#pragma unroll
  for (int i = 0; i < 8; ++i) u.at(i) = dropped(x.at(i), u.at(i), half_of(r, i) >= p.threshold, p.scale, RESIDUAL);
  u.store(y);
}

// No rows share: a thread takes a few groups of eight elements and draws their numbers while the elements are on their way. 16384 x 1024
// fp16 23 us with the residual, 20 without, where 100 and 67 MB have to move (0.67 and 0.51 of the measured rate): between memory and
// instructions, about 26 an element (issue 53 and 61 % busy; halves, choices and conversions go one element at a time). With one group a
// thread whose numbers came first 55 and 36.
template <typename T, bool RESIDUAL>
__global__ void __launch_bounds__(kDropoutThreads) dropout_kernel(const DropoutParams p) {
  grid_dependency_wait();
  grid_dependents_launch();
  const T* x = static_cast<const T*>(p.x);
  const T* u = static_cast<const T*>(p.u);
  T* y = static_cast<T*>(p.y);
  const DropoutKey key(p);
  const long long n = p.outer * p.inner;
  const long long first = static_cast<long long>(blockIdx.x) * (kDropoutThreads * kDropoutFlight) + threadIdx.x;
  Eight<T> a[kDropoutFlight], b[kDropoutFlight];
#pragma unroll
  for (int q = 0; q < kDropoutFlight; ++q) {
    const long long at = (first + q * kDropoutThreads) * 8;
    if (at + 8 <= n) {
      b[q].load(u + at);
      if (RESIDUAL) a[q].load(x + at);
    }
  }
#pragma unroll
  for (int q = 0; q < kDropoutFlight; ++q) {
    const long long g = first + q * kDropoutThreads, at = g * 8;
    if (at >= n) break;
    const uint4 r = key.numbers(g);
    if (at + 8 <= n) {
      drop_eight<T, RESIDUAL>(p, r, a[q], b[q], y + at);
    } else {
      for (int i = 0; at + i < n; ++i)
        y[at + i] = dropped(RESIDUAL ? __ldcg(x + at + i) : T(0.f), __ldcg(u + at + i), half_of(r, i) >= p.threshold, p.scale, RESIDUAL);
    }
  }
}

// Rows share a mask and have whole groups of eight: a thread draws a group's numbers once for `chunk` rows. 384 x 384 x 128 bf16, a
// mask for 384 rows: 23 us with the residual (113 MB), 18 to 20 without (75 MB).
template <typename T, bool RESIDUAL>
__global__ void __launch_bounds__(kDropoutThreads) dropout_shared_kernel(const DropoutParams p) {
  grid_dependency_wait();
  grid_dependents_launch();
  const T* x = static_cast<const T*>(p.x);
  const T* u = static_cast<const T*>(p.u);
  T* y = static_cast<T*>(p.y);
  const DropoutKey key(p);
  const long long g = static_cast<long long>(blockIdx.x) * kDropoutThreads + threadIdx.x;
  if (g * 8 >= p.outer * p.inner) return;
  const long long base = g * 8 + g * 8 / p.inner * (p.shared - 1) * p.inner;
  long long s = static_cast<long long>(blockIdx.y) * p.chunk;
  const long long last = min(p.shared, s + p.chunk);
  Eight<T> a[kDropoutFlight], b[kDropoutFlight];
  auto fetch = [&]() {
#pragma unroll
    for (int q = 0; q < kDropoutFlight; ++q)
      if (s + q < last) {
        b[q].load(u + base + (s + q) * p.inner);
        if (RESIDUAL) a[q].load(x + base + (s + q) * p.inner);
      }
  };
  fetch();
  const uint4 r = key.numbers(g);
  while (true) {
#pragma unroll
    for (int q = 0; q < kDropoutFlight; ++q)
      if (s + q < last) drop_eight<T, RESIDUAL>(p, r, a[q], b[q], y + base + (s + q) * p.inner);
    s += kDropoutFlight;
    if (s >= last) break;
    fetch();
  }
}

constexpr int kDropoutSingles = 8;  // rows in flight

// The same where rows of an odd width share a mask or a tensor does not start on 16 bytes: one mask element a thread, one element a load.
// 384 x 384 x 101 bf16, a mask for 384 rows: 33 us for 89 MB; 16384 x 1024 bf16 without shared rows, where numbers for eight elements are drawn
// for each: 409 us.
template <typename T, bool RESIDUAL>
__global__ void __launch_bounds__(kDropoutThreads) dropout_single_kernel(const DropoutParams p) {
  grid_dependency_wait();
  grid_dependents_launch();
  const T* x = static_cast<const T*>(p.x);
  const T* u = static_cast<const T*>(p.u);
  T* y = static_cast<T*>(p.y);
  const DropoutKey key(p);
  const long long n = p.outer * p.inner;
  const long long first_row = static_cast<long long>(blockIdx.y) * p.chunk, last_row = min(p.shared, first_row + p.chunk);
  for (long long e = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; e < n; e += static_cast<long long>(gridDim.x) * blockDim.x) {
    const bool keep = half_of(key.numbers(e / 8), static_cast<int>(e & 7)) >= p.threshold;
    const long long base = e + e / p.inner * (p.shared - 1) * p.inner;
    for (long long s = first_row; s < last_row; s += kDropoutSingles) {
      T a[kDropoutSingles], b[kDropoutSingles];
#pragma unroll
      for (int q = 0; q < kDropoutSingles; ++q)
        if (s + q < last_row) {
          b[q] = __ldcg(u + base + (s + q) * p.inner);
          a[q] = RESIDUAL ? __ldcg(x + base + (s + q) * p.inner) : T(0.f);
        }
#pragma unroll
      for (int q = 0; q < kDropoutSingles; ++q)
        if (s + q < last_row) y[base + (s + q) * p.inner] = dropped(a[q], b[q], keep, p.scale, RESIDUAL);
    }
  }
}

}  // namespace trimul
