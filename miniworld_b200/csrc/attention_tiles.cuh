// What the attention's kernels on the tensor cores share: which rows a block works on, operands in shared and tensor memory, the bias.
//
// Tiles are 128 queries by 128 keys. Scores and their gradients are products into tensor memory, a row a lane; threads take them into
// registers, and what comes of them (probabilities, gradients of scores) goes back into tensor memory in 16 bits as the first operand
// of the next product: neither of the two ever passes through shared memory.
#pragma once

#include "attention.cuh"

namespace trimul {

constexpr int kAtTile = 128;
constexpr int kAtTileBytes = 128 * 128;  // 128 rows of 64 elements
// what a result's rounding error is multiplied by before it is rounded itself
template <bool F16>
constexpr float kAtRest = F16 ? 2048.f : 1.f;

struct AttentionMaps {
  CUtensorMap q, k, v, dout;  // [rows][heads][d], boxes of 128 rows of 64 elements
};

__device__ __forceinline__ void umma_ta(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {  // (NaN: the greatest of the others)
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
template <bool F16>
__device__ __forceinline__ uint32_t pack_pair(float2 v) {
  if constexpr (F16)
    return pack_f16x2(v);
  else
    return pack_bf16x2(v);
}
template <bool F16>
__device__ __forceinline__ float2 unpack_pair(uint32_t v) {
  if constexpr (F16)
    return f16x2_to_float2(v);
  else
    return bf16x2_to_float2(v);
}
// 32 lanes x 8 consecutive 32-bit columns, registers -> TMEM
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
               "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
template <int REGS>
__device__ __forceinline__ void registers_more() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS));
}
template <int REGS>
__device__ __forceinline__ void registers_fewer() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS));
}

// The rows of a block. Sequences of equal lengths are cut into tiles one after the other. Packed ones get, for sequence s, the places
// from floor(offsets[s] / rows of a tile) + s on: at least as many as it has tiles, and found by looking for the greatest s whose first
// place is not beyond the block's, without any table. What is left at most is one place a sequence. Place `sequences` stands for the
// rows behind the last one.
struct AttentionPlace {
  long long first, last;  // the sequence's rows
  int tile;               // of `tile_rows` rows of it; beyond its end: nothing to do
  int behind;             // rows of no sequence
};
__host__ __device__ inline long long attention_places(const int* offsets, long long rows, int sequences, int length, int tile_rows) {
  if (offsets == nullptr) return static_cast<long long>(sequences) * ((length + tile_rows - 1) / tile_rows);
  return rows / tile_rows + sequences + 1;
}
// The heads of a place one after the other: their rows lie side by side in memory, and the longest rows of all heads of a causal sequence come
// first (38009 packed tokens, causal, 16 heads of 128: 847 -> 797 us against all places of a head first).
__device__ __forceinline__ int attention_block_head(int heads) { return static_cast<int>(blockIdx.x % static_cast<unsigned>(heads)); }
__device__ __forceinline__ long long attention_block_place(const AttentionParams& p, int heads, bool last_first) {
  const long long at = blockIdx.x / static_cast<unsigned>(heads);
  return last_first ? p.places - 1 - at : at;
}
// by a whole warp
__device__ __forceinline__ AttentionPlace attention_place(const AttentionParams& p, long long place, int tile_rows) {
  AttentionPlace r;
  if (p.offsets == nullptr) {
    const int tiles = (p.length + tile_rows - 1) / tile_rows;
    const long long s = place / tiles;
    r.first = s * p.length;
    r.last = r.first + p.length;
    r.tile = static_cast<int>(place - s * tiles);
    r.behind = 0;
    return r;
  }
  const int lane = threadIdx.x & 31;
  int lo = 0, n = p.sequences + 1;  // the sequence is one of lo .. lo + n - 1
  while (n > 32) {
    const int step = (n + 31) / 32, at = lane * step;
    const bool before = at < n && attention_offset(p, lo + at) / tile_rows + lo + at <= place;
    const int at_most = max(__popc(__ballot_sync(0xFFFFFFFFu, before)) - 1, 0) * step;
    lo += at_most;
    n = min(step, n - at_most);
  }
  // (the offsets of the last candidates are those of the sequence found: no load follows another here)
  const long long offset = attention_offset(p, min(lo + lane, p.sequences));
  const bool before = lane < n && offset / tile_rows + lo + lane <= place;
  const int found = max(__popc(__ballot_sync(0xFFFFFFFFu, before)) - 1, 0), s = lo + found;
  r.first = __shfl_sync(0xFFFFFFFFu, offset, found);
  r.last = __shfl_sync(0xFFFFFFFFu, offset, min(found + 1, 31));
  if (s == p.sequences) r.last = p.rows;
  else if (found == 31) r.last = attention_offset(p, s + 1);
  // (offsets out of order may leave any number of places to a sequence: its rows are counted in 32 bits)
  r.tile = static_cast<int>(min(max(place - (r.first / tile_rows + s), 0ll), p.rows / tile_rows + 1));
  r.behind = s == p.sequences;
  return r;
}

// Biases of all distances that tiles near the diagonal meet, in units of log2: entry i is that of the distance i - (reach + 255).
__host__ __device__ constexpr int attention_bias_entries(int reach) { return 2 * (reach + 255) + 1; }
__device__ __forceinline__ void attention_bias_fill(const AttentionParams& p, float* bias, int head, bool f16, int thread, int threads) {
  const int entries = attention_bias_entries(p.reach);
  for (int i = thread; i < entries; i += threads) bias[i] = attention_bias(p, i - (p.reach + 255), head, f16);
}

// Whether tiles of 128 keys and 128 queries, whose first ones are `d0` apart, have pairs within the reach
__device__ __forceinline__ bool attention_near(const AttentionParams& p, int d0) { return d0 + 127 > -p.reach && d0 - 127 < p.reach; }

// Rows first .. first + 32 W - 1 that lie before `last` and that the mask leaves, a bit each (whole warp)
template <int W>
__device__ __forceinline__ void attention_mask_bits(const AttentionParams& p, long long first, long long last, uint32_t (&bits)[W]) {
  const int lane = threadIdx.x & 31;
  bool there[W];
#pragma unroll
  for (int i = 0; i < W; ++i) {
    const long long row = first + 32 * i + lane;
    there[i] = row < last && __ldcg(p.mask + row) != 0;
  }
#pragma unroll
  for (int i = 0; i < W; ++i) bits[i] = __ballot_sync(0xFFFFFFFFu, there[i]);
}
// The first `count` of 32 as bits
__device__ __forceinline__ uint32_t first_bits(int count) { return count >= 32 ? ~0u : count > 0 ? (1u << count) - 1u : 0u; }
// The same of the rows from row0 of a sequence on, with or without a mask
template <int W>
__device__ __forceinline__ void attention_rows_there(const AttentionParams& p, const AttentionPlace& place, int length, int row0, uint32_t (&bits)[W]) {
  if (p.mask != nullptr) {
    attention_mask_bits(p, place.first + row0, place.last, bits);
    return;
  }
#pragma unroll
  for (int w = 0; w < W; ++w) bits[w] = first_bits(length - row0 - 32 * w);
}

// What the copying thread remembers of its ring, a bit a stage: whether it was used, the parity of that use, whether the copy went to
// landed() and not to ready(), and the parity of landed(), which only such copies have.
struct AttentionRing {
  uint32_t used = 0, odd = 0, through = 0, landed = 0, landed_odd = 0;
  __device__ __forceinline__ void use(int s, bool other) {
    const uint32_t bit = 1u << s;
    odd ^= used & bit;
    used |= bit;
    through = other ? through | bit : through & ~bit;
    if (other) {
      landed_odd ^= landed & bit;
      landed |= bit;
    }
  }
  // Copies that nothing waits for any more (a wait may give up at any time, also after the last copy was started) land before the block may
  // exit. Where all went well they have, or their readers are waiting too.
  template <int ST, typename Landed, typename Ready>
  __device__ __forceinline__ void drain(uint32_t first, Landed landed_bar, Ready ready_bar) const {
    auto land = [](uint32_t b, uint32_t phase) {
      const long long t0 = clock64();
      while (!mbar_try_wait(b, phase) && clock64() - t0 < kWaitLimitCycles) {
      }
    };
    land(first, 0);
    for (int s = 0; s < ST; ++s)
      if (used >> s & 1u) land(through >> s & 1u ? landed_bar(s) : ready_bar(s), (through >> s & 1u ? landed_odd : odd) >> s & 1u);
  }
};

// Zeroes the rows of a tile in shared memory that are not among the `bits` (whole warp): an operand's rows that belong to other
// sequences or are masked must not meet the zeros that stand for them in the other operand as infinities or NaN.
template <int W>
__device__ __forceinline__ void attention_clean_rows(uint32_t tile, int halves, const uint32_t (&bits)[W]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    if (bits[w] == ~0u) continue;
#pragma unroll 1
    for (int h = 0; h < halves; ++h)
#pragma unroll 1
      for (int r = lane / 8; r < 32; r += 4)
        if (!(bits[w] >> r & 1u))
          asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(tile + h * (W * 4096) + (w * 32 + r) * 128 + (lane & 7) * 16), "r"(0) : "memory");
  }
  fence_proxy_async_smem();
  __syncwarp();
}

}  // namespace trimul
