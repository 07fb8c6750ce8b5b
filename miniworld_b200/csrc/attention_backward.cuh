// Backward of the attention (formulas: attention.cuh) in three kernels, each with fixed orders of summation and without atomics:
// delta; dq with the sums of ds by distance (a block a tile of 128 queries, over the keys); dk and dv (a block a tile of 128 keys, over
// the queries of all heads of the group). Scores and dO v^T are formed again in both of the latter: 7 products where 5 would do, against
// adding dq up over blocks in whatever order they end.
//
// Sixteen warps do the arithmetic: a thread has a row and 32 columns of the scores and of dO v^T. Both are in registers while the next
// tile's are formed; probabilities and ds go back into tensor memory as the first operand of the sums.
//
// One B200, 2 x 4096 tokens, 16 heads of 64, alone: delta 17 us, dq 318 to 340, dk and dv 343 (tensor pipe busy 31 and 41 % of the time,
// special function unit 42 %). A tile takes about 2000 clocks of an SM, 1024 of them exponentials: the products of the next tile, the arithmetic
// and the sums' products hand over to one another four times a tile, at about 200 clocks each, and all warps are on the same tile
// (there are no columns for scores of another). A step with heads of 128 takes 1362 us where one with heads of 64 takes 874. With eight warps of twice the columns, masks in every element and rows' values loaded by the warps that use
// them 436 and 507.
//
// fp16: probabilities are held times 2^15, and ds times the power of two that brings its bound 2 max |dO| max |v| to 2^14 .. 2^15, so that
// nothing overflows and little is subnormal; both come off the fp32 sums again.
#pragma once

#include "../../include/b200_tokens.h"
#include "attention_tiles.cuh"
#include "tokens_status.cuh"

namespace trimul {

constexpr int kAtDeltaThreads = 256;
constexpr int kAtDeltaBlocks = 256;  // at most, of a key head

// delta[h][row] = dO . o, from o before it was rounded: the rounded one's error, times the probabilities' mass, would stand in the
// biases' gradients, where the true sums nearly cancel (4096 tokens: 0.027 of their norm). In fp16 also the greatest |dO|^2 of the rows
// that have keys, and |v|^2 of those that are keys: the two differ where biases of -inf leave a row without a key that others attend to.
template <typename T>
__global__ void __launch_bounds__(kAtDeltaThreads) attention_delta_kernel(const AttentionParams p) {
  constexpr bool f16 = __is_same(T, __half);
  __shared__ float most[2][kAtDeltaThreads / 32];
  grid_dependency_wait();
  grid_dependents_launch();
  int team = 1;  // lanes of a row: 8 elements each
  while (team * 8 < p.d) team *= 2;
  const int lane = threadIdx.x % team, group = p.heads / p.kv_heads, kv_head = blockIdx.y;
  const long long step = static_cast<long long>(gridDim.x) * (kAtDeltaThreads / team);
  const bool own = lane * 8 < p.d;
  float most_g = 0.f, most_v = 0.f;
  auto row_square = [&](float s) {
    for (int i = 1; i < team; i *= 2) s += __shfl_xor_sync(0xFFFFFFFFu, s, i);
    return s;
  };
  auto values = [&](const T* at, float2 (&v)[4]) {
    const uint4 w = own ? __ldcg(reinterpret_cast<const uint4*>(at + lane * 8)) : make_uint4(0, 0, 0, 0);
    v[0] = unpack_pair<f16>(w.x), v[1] = unpack_pair<f16>(w.y), v[2] = unpack_pair<f16>(w.z), v[3] = unpack_pair<f16>(w.w);
  };
  const long long rounds = (p.rows + step - 1) / step, keys_end = f16 && p.offsets != nullptr ? attention_offset(p, p.sequences) : p.rows;
  for (long long k = 0; k < rounds; ++k) {
    const long long row = k * step + static_cast<long long>(blockIdx.x) * (kAtDeltaThreads / team) + threadIdx.x / team;
    const bool inside = row < p.rows;
    const long long r = inside ? row : 0;
    for (int h = kv_head * group; h < (kv_head + 1) * group; ++h) {
      const bool there = inside && __ldcg(p.lse + h * p.rows + r) != INFINITY;
      float2 g[4], o[4], e[4];
      values(attention_at<T>(p.dout, r, h), g);
      const long long at = (r * p.heads + h) * p.d;
      values(static_cast<const T*>(p.o) + at, o);
      values(static_cast<const T*>(p.rest) + at, e);
      float s = 0.f, square = 0.f;
      if (there) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s = fmaf(g[i].x, fmaf(e[i].x, 1.f / kAtRest<f16>, o[i].x), s);
          s = fmaf(g[i].y, fmaf(e[i].y, 1.f / kAtRest<f16>, o[i].y), s);
          square = fmaf(g[i].x, g[i].x, fmaf(g[i].y, g[i].y, square));
        }
      }
      s = row_square(s);
      if (f16) {
        square = row_square(square);
        if (square < INFINITY) most_g = fmaxf(most_g, square);
      }
      if (inside && lane == 0) p.delta[h * p.rows + row] = s;
    }
    if (f16) {
      float2 v[4];
      values(attention_at<T>(p.v, r, kv_head), v);
      float square = 0.f;
      if (inside && row < keys_end && (p.mask == nullptr || __ldcg(p.mask + r) != 0)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) square = fmaf(v[i].x, v[i].x, fmaf(v[i].y, v[i].y, square));
      }
      square = row_square(square);
      if (square < INFINITY) most_v = fmaxf(most_v, square);
    }
  }
  if (f16) {
    most_g = warp_max(most_g);
    most_v = warp_max(most_v);
    if (threadIdx.x % 32 == 0) {
      most[0][threadIdx.x / 32] = most_g;
      most[1][threadIdx.x / 32] = most_v;
    }
    __syncthreads();
    if (threadIdx.x < 2) {
      float m = 0.f;
      for (int i = 0; i < kAtDeltaThreads / 32; ++i) m = fmaxf(m, most[threadIdx.x][i]);
      p.most[(static_cast<long long>(kv_head) * gridDim.x + blockIdx.x) * 2 + threadIdx.x] = m;
    }
  }
}

// The power of two that ds is held times (whole warp)
__device__ __forceinline__ float attention_ds_scale(const AttentionParams& p, int kv_head) {
  float g = 0.f, v = 0.f;
  for (int i = threadIdx.x & 31; i < p.delta_blocks; i += 32) {
    const float2 m = __ldcg(reinterpret_cast<const float2*>(p.most) + static_cast<long long>(kv_head) * p.delta_blocks + i);
    g = fmaxf(g, m.x);
    v = fmaxf(v, m.y);
  }
  const float bound = 2.f * sqrtf(warp_max(g)) * sqrtf(warp_max(v));
  return bound > 0.f && bound < INFINITY ? exp2f(static_cast<float>(min(max(14 - ilogbf(bound), -60), 60))) : 1.f;
}

constexpr int kAtBackWarps = 16;  // of the arithmetic: a thread has a row and 32 columns
constexpr int kAtBackThreads = kAtBackWarps * 32 + 128;
constexpr int kAtBackMany = 104, kAtBackFew = 64;  // registers: the launch's are 96, and 4 x 104 + 64 = 5 x 96

// ---------------------------------------------------------------- dq
template <int HALVES>
struct AtDq {
  static constexpr int kKeys = HALVES == 1 ? 3 : 2, kValues = HALVES == 1 ? 2 : 1;  // stages: keys are held until dq has them
  static constexpr int kStages = kKeys + kValues;
  __host__ __device__ static constexpr int key_stage(int j) { return j % kKeys; }
  __host__ __device__ static constexpr int value_stage(int j) { return kKeys + j % kValues; }
  static constexpr int kStageBytes = HALVES * kAtTileBytes;
  static constexpr uint32_t kScores = 0, kGrad = 128, kDs = 256, kSum = 320;  // columns of tensor memory
  static constexpr int kBars = 2 * HALVES * kAtTileBytes + kStages * kStageBytes;
  static constexpr int kBias = kBars + 320;
  static int smem(bool table, int reach) {
    // biases; sums by distance of every warp; what the threads of a row tell each other
    return 1024 + kBias + (table ? (attention_bias_entries(reach) + kAtBackWarps * (2 * reach + 1) + 4 * kAtTile) * 4 : 0);
  }
};

template <bool F16, int HALVES>
__global__ void __launch_bounds__(kAtBackThreads, 1) attention_dq_kernel(const __grid_constant__ AttentionMaps maps, const AttentionParams p) {
  using C = AtDq<HALVES>;
  constexpr int ST = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* const smem = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t q_s = base, do_s = q_s + HALVES * kAtTileBytes, ring = do_s + HALVES * kAtTileBytes, bars = base + C::kBars;
  auto landed = [&](int s) { return bars + 8u * s; };
  auto ready = [&](int s) { return bars + 8u * (ST + s); };
  auto empty = [&](int s) { return bars + 8u * (2 * ST + s); };
  const uint32_t q_ready = bars + 8u * (3 * ST), formed = q_ready + 8, read = q_ready + 16, ds_ready = q_ready + 24, ds_done = q_ready + 32;
  static_assert(8 * (3 * ST + 5) <= 240, "barriers");
  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(smem + C::kBars + 240);
  volatile int* const abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* const ds_scale_s = reinterpret_cast<float*>(tmem_slot + 2);
  int* const status = &tokens_status;
  AttentionPlace* const place_s = reinterpret_cast<AttentionPlace*>(smem + C::kBars + 256);
  float* const bias = reinterpret_cast<float*>(smem + C::kBias);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int load_warp = kAtBackWarps, mma_warp = load_warp + 1, clean_warp = load_warp + 2;
  const int head = attention_block_head(p.heads), kv_head = head / (p.heads / p.kv_heads);
  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(landed(s), 1);
      mbar_init(ready(s), 1);
      mbar_init(empty(s), 1);
    }
    mbar_init(q_ready, 1);
    mbar_init(formed, 1);
    mbar_init(read, kAtBackWarps);
    mbar_init(ds_ready, kAtBackWarps);
    mbar_init(ds_done, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == mma_warp) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  grid_dependency_wait();
  grid_dependents_launch();
  const long long place_index = attention_block_place(p, p.heads, p.causal);
  if (warp == 0) {
    const AttentionPlace r = attention_place(p, place_index, kAtTile);
    if (lane == 0) *place_s = r;
  }
  if (F16 && warp == 1) {
    const float c = attention_ds_scale(p, kv_head);
    if (lane == 0) *ds_scale_s = c;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const AttentionPlace place = *place_s;
  const int length = static_cast<int>(place.last - place.first), q0 = place.tile * kAtTile;
  int n = 0;  // key tiles
  if (!place.behind && q0 < length) n = p.causal ? place.tile + 1 : (length + kAtTile - 1) / kAtTile;
  auto dirty = [&](int j) { return p.mask != nullptr || (j + 1) * kAtTile > length; };

  if (warp >= kAtBackWarps) {
    registers_fewer<kAtBackFew>();
    if (warp == load_warp && lane == 0 && n > 0) {
      mbar_arrive_expect_tx(q_ready, 2 * HALVES * kAtTileBytes);
      for (int h = 0; h < HALVES; ++h) {
        tma_load_3d(q_s + h * kAtTileBytes, &maps.q, q_ready, h * 64, head, static_cast<int>(place.first) + q0);
        tma_load_3d(do_s + h * kAtTileBytes, &maps.dout, q_ready, h * 64, head, static_cast<int>(place.first) + q0);
      }
      int i = 0;
      AttentionRing state;
      for (; i < 2 * n; ++i) {
        const bool value = i & 1;
        const int j = i >> 1, s = value ? C::value_stage(j) : C::key_stage(j), turn = value ? j / C::kValues : j / C::kKeys;
        if (turn > 0 && !mbar_wait(empty(s), static_cast<uint32_t>(turn & 1) ^ 1u, abort_flag, status, kDevTimeoutProducer)) break;
        const bool other = !value && dirty(j);
        state.use(s, other);
        const uint32_t bar = other ? landed(s) : ready(s);
        mbar_arrive_expect_tx(bar, C::kStageBytes);
        for (int h = 0; h < HALVES; ++h)
          tma_load_3d(ring + s * C::kStageBytes + h * kAtTileBytes, value ? &maps.v : &maps.k, bar, h * 64, kv_head, static_cast<int>(place.first) + j * kAtTile);
      }
      state.drain<ST>(q_ready, landed, ready);
    } else if (warp == mma_warp && elect_one()) {
      constexpr uint32_t fmt = F16 ? kFmtF16 : kFmtBF16;
      constexpr uint32_t idesc_s = umma_idesc(128, 128, false, false, fmt, fmt);
      const int steps = (p.d + 15) / 16;
      const uint32_t idesc_q = umma_idesc(128, steps * 16, false, true, fmt, fmt);
      bool ok = n > 0 && mbar_wait(q_ready, 0, abort_flag, status, kDevTimeoutMma);
      auto wait = [&](uint32_t bar, uint32_t parity) { ok = ok && mbar_wait(bar, parity & 1u, abort_flag, status, kDevTimeoutMma); };
      auto form = [&](int j) {
        const int sk = C::key_stage(j), sv = C::value_stage(j);
        wait(ready(sk), j / C::kKeys);
        if (j > 0) wait(read, j - 1);
        if (!ok) return;
        tc_fence_after();
        for (int ks = 0; ks < steps; ++ks)
          umma_bf16(tmem + C::kScores, umma_desc_kmajor(q_s + (ks >> 2) * kAtTileBytes) + static_cast<uint64_t>((ks & 3) * 2),
                    umma_desc_kmajor(ring + sk * C::kStageBytes + (ks >> 2) * kAtTileBytes) + static_cast<uint64_t>((ks & 3) * 2), idesc_s, ks != 0 ? 1u : 0u);
        wait(ready(sv), j / C::kValues);
        if (!ok) return;
        tc_fence_after();
        for (int ks = 0; ks < steps; ++ks)
          umma_bf16(tmem + C::kGrad, umma_desc_kmajor(do_s + (ks >> 2) * kAtTileBytes) + static_cast<uint64_t>((ks & 3) * 2),
                    umma_desc_kmajor(ring + sv * C::kStageBytes + (ks >> 2) * kAtTileBytes) + static_cast<uint64_t>((ks & 3) * 2), idesc_s, ks != 0 ? 1u : 0u);
        umma_commit(formed);
        umma_commit(empty(sv));
      };
      if (ok) form(0);
      for (int j = 0; j < n && ok; ++j) {
        if (j + 1 < n) form(j + 1);
        wait(ds_ready, j);
        if (!ok) break;
        tc_fence_after();
        const int sk = C::key_stage(j), key_steps = (min(kAtTile, length - j * kAtTile) + 15) / 16;
        for (int ks = 0; ks < key_steps; ++ks)
          umma_ta(tmem + C::kSum, tmem + C::kDs + ks * 8, umma_desc_mnmajor(ring + sk * C::kStageBytes + ks * 2048, kAtTileBytes), idesc_q, (j | ks) != 0 ? 1u : 0u);
        umma_commit(ds_done);
        umma_commit(empty(sk));
      }
    } else if (warp == clean_warp) {
      uint32_t odd = 0;
      for (int j = 0; j < n; ++j) {
        if (!dirty(j)) continue;
        const int s = C::key_stage(j);
        uint32_t bits[4];
        attention_rows_there(p, place, length, j * kAtTile, bits);
        if (!mbar_wait_warp(landed(s), odd >> s & 1u, abort_flag, status, kDevTimeoutStats)) break;
        odd ^= 1u << s;
        attention_clean_rows(ring + s * C::kStageBytes, HALVES, bits);
        if (lane == 0) mbar_arrive(ready(s));
      }
    }
  } else {
    registers_more<kAtBackMany>();
    const int quarter = warp >> 2, row0 = (warp & 3) * 32, row = row0 + lane, q_row = q0 + row;
    const uint32_t own = tmem + (static_cast<uint32_t>(warp & 3) << 21);
    const bool inside = q_row < length;
    const bool there = inside && !place.behind && (p.mask == nullptr || __ldcg(p.mask + place.first + q_row) != 0);
    const bool sums = p.partial != nullptr;
    const int distances = 2 * p.reach + 1;
    float* const all_distances = bias + attention_bias_entries(p.reach);  // [warps][distances], then [4][128]
    float* const by_distance = all_distances + warp * distances;
    float low = 0.f, high = 0.f;
    if (p.table != nullptr && n > 0) {
      attention_bias_fill(p, bias, head, F16, threadIdx.x, kAtBackWarps * 32);
      if (sums)
        for (int i = lane; i < distances; i += 32) by_distance[i] = 0.f;
      named_bar_sync(1, kAtBackWarps * 32);
      low = bias[0];
      high = bias[2 * (p.reach + 255)];
    }
    const float c = F16 ? *ds_scale_s : 1.f, scale = p.scale * kLog2e;
    const float lse = there ? __ldcg(p.lse + head * p.rows + place.first + q_row) : INFINITY;
    const float delta = there ? __ldcg(p.delta + head * p.rows + place.first + q_row) : 0.f;
    const float2 c2 = make_float2(c, c), minus_delta = make_float2(-delta * c, -delta * c);
    // of the row: ds in all, of the outer two buckets, and the probabilities' mass there
    float all = 0.f, sum_low = 0.f, sum_high = 0.f, mass_low = 0.f, mass_high = 0.f;
    bool ok = true;
    for (int j = 0; j < n; ++j) {
      const int key0 = j * kAtTile + quarter * 32, d0 = key0 - q0, keys = length - key0;
      const bool near = p.table != nullptr && d0 + 31 > -p.reach && d0 - 127 < p.reach;
      const float add = p.table == nullptr || near ? 0.f : d0 > 0 ? high : low;
      const int limit = !there ? 0 : p.causal ? min(keys, q_row - key0 + 1) : keys;
      uint32_t bits[1] = {~0u};
      if (p.mask != nullptr) attention_mask_bits(p, place.first + key0, place.last, bits);
      const uint32_t counts = bits[0] & first_bits(limit);
      ok = mbar_wait_warp(formed, j & 1, abort_flag, status, kDevTimeoutEpilogue);
      if (!ok) break;
      tc_fence_after();
      uint32_t v[32], g[32];
      tmem_ld32(own + C::kScores + quarter * 32, v);
      tmem_ld32(own + C::kGrad + quarter * 32, g);
      tmem_ld_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(read);
      float factor = scale;
      const float shift = add - lse;
      if (near) {
        const float* b = bias + (p.reach + 255) + d0 - row;
#pragma unroll
        for (int k = 0; k < 32; ++k) v[k] = __float_as_uint(fmaf(__uint_as_float(v[k]), scale, b[k]));
        factor = 1.f;
      }
      if (counts != ~0u) {
        // (what does not count may be anything: the products are taken out before they meet numbers)
#pragma unroll
        for (int k = 0; k < 32; ++k) {
          const bool there_k = counts >> k & 1u;
          v[k] = there_k ? __float_as_uint(__uint_as_float(v[k]) * factor) : 0xFF800000u;
          g[k] = there_k ? g[k] : 0u;
        }
        factor = 1.f;
      }
      const float2 factor2 = make_float2(factor, factor), shift2 = make_float2(shift, shift);
      uint32_t w[16];
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        float2 e = __ffma2_rn(make_float2(__uint_as_float(v[2 * k]), __uint_as_float(v[2 * k + 1])), factor2, shift2);
        e.x = exp2_approx(e.x);
        e.y = exp2_approx(e.y);
        const float2 ds = __fmul2_rn(e, __ffma2_rn(make_float2(__uint_as_float(g[2 * k]), __uint_as_float(g[2 * k + 1])), c2, minus_delta));
        w[k] = pack_pair<F16>(ds);
        v[2 * k] = __float_as_uint(e.x), v[2 * k + 1] = __float_as_uint(e.y);
        g[2 * k] = __float_as_uint(ds.x), g[2 * k + 1] = __float_as_uint(ds.y);
      }
      if (j > 0) {
        ok = mbar_wait_warp(ds_done, (j - 1) & 1, abort_flag, status, kDevTimeoutEpilogue);
        if (!ok) break;
        tc_fence_after();
      }
      tmem_st16(own + C::kDs + quarter * 16, w);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(ds_ready);
      if (sums) {
        float2 total = make_float2(0.f, 0.f), mass = make_float2(0.f, 0.f);
#pragma unroll
        for (int k = 0; k < 32; k += 2) {
          total = __fadd2_rn(total, make_float2(__uint_as_float(g[k]), __uint_as_float(g[k + 1])));
          mass = __fadd2_rn(mass, make_float2(__uint_as_float(v[k]), __uint_as_float(v[k + 1])));
        }
        const float t = total.x + total.y;
        all += t;
        const int e0 = d0 - row0;  // distance of this square's first column from its first row
        if (e0 + 31 <= -p.reach) {
          sum_low += t;
          mass_low += mass.x + mass.y;
        } else if (e0 - 31 >= p.reach) {
          sum_high += t;
          mass_high += mass.x + mass.y;
        } else {
          // columns up to / from which on this row is in an outer bucket (a reach of 0 is one bucket: the lower)
          const int last_low = -p.reach - e0 + lane, first_high = max(p.reach - e0 + lane, last_low + 1);
          // Lane x adds up the square's diagonals x (of the rows above 32 - x) and x - 32: column k of row r is in the one or the other.
          float upper = 0.f, lower = 0.f;
#pragma unroll
          for (int k = 0; k < 32; ++k) {
            const float ds = __uint_as_float(g[k]), e = __uint_as_float(v[k]);
            if (k <= last_low) sum_low += ds, mass_low += e;
            if (k >= first_high) sum_high += ds, mass_high += e;
            const float turned = __shfl_sync(0xFFFFFFFFu, ds, k - lane);  // (of row k - lane modulo 32)
            if (lane <= k) upper += turned;
            else lower += turned;
          }
          const int du = e0 + lane, dl = du - 32;
          if (du > -p.reach && du < p.reach) by_distance[du + p.reach] += upper;
          if (dl > -p.reach && dl < p.reach) by_distance[dl + p.reach] += lower;
          __syncwarp();
        }
      }
    }
    if (n > 0 && ok) ok = mbar_wait_warp(ds_done, (n - 1) & 1, abort_flag, status, kDevTimeoutEpilogue);
    if (ok) {
      tc_fence_after();
      const float back = p.scale / c;
      const long long at = ((place.first + q_row) * p.heads + head) * p.d;
      for (int c0 = quarter * 16; c0 < p.d; c0 += 64) {
        uint32_t o[16], w[8];
        if (n > 0) {
          tmem_ld16(own + C::kSum + c0, o);
          tmem_ld_wait();
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
          w[k] = there ? pack_pair<F16>(make_float2(__uint_as_float(o[2 * k]) * back, __uint_as_float(o[2 * k + 1]) * back)) : 0u;
        if (inside) {
          uint4* out = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.dq) + at + c0);
          out[0] = make_uint4(w[0], w[1], w[2], w[3]);
          if (c0 + 8 < p.d) out[1] = make_uint4(w[4], w[5], w[6], w[7]);
        }
      }
    }
    if (sums) {
      // ds of a row adds up to nothing but what delta is off by: its share, by the probabilities' mass, comes off the outer buckets, of
      // whose terms most are of one sign otherwise
      float* const rows = all_distances + kAtBackWarps * distances;
      float* const out = p.partial + (head * p.places + place_index) * distances;
      if (n > 0) {
        rows[quarter * 128 + row] = all;
        named_bar_sync(1, kAtBackWarps * 32);
        const float off = (rows[row] + rows[128 + row]) + (rows[256 + row] + rows[384 + row]);
        const float l = warp_sum(sum_low - off * mass_low), h = warp_sum(sum_high - off * mass_high);
        named_bar_sync(1, kAtBackWarps * 32);
        if (lane == 0) {
          rows[warp] = l;
          rows[kAtBackWarps + warp] = h;
        }
        named_bar_sync(1, kAtBackWarps * 32);
      }
      for (int i = threadIdx.x; i < distances; i += kAtBackWarps * 32) {
        float s = 0.f;
        if (n > 0) {
          for (int k = 0; k < kAtBackWarps; ++k) s += all_distances[k * distances + i];
          if (i == 0)
            for (int k = 0; k < kAtBackWarps; ++k) s += rows[k];
          if (i == distances - 1)
            for (int k = 0; k < kAtBackWarps; ++k) s += rows[kAtBackWarps + k];
        }
        out[i] = s / c;
      }
    }
  }
  __syncthreads();
  if (warp == mma_warp) tmem_dealloc(tmem, 512);
}

// ---------------------------------------------------------------- dk and dv
template <int HALVES>
struct AtDkv {
  static constexpr bool kOver = HALVES == 2;  // probabilities and ds over the scores and dO v^T
  static constexpr int kStages = HALVES == 1 ? 6 : 4;
  static constexpr int kStageBytes = HALVES * kAtTileBytes;
  static constexpr uint32_t kScores = 0, kGrad = 128, kProbs = kOver ? 0 : 256, kDs = kOver ? 128 : 320, kDv = kOver ? 256 : 384, kDk = kOver ? 384 : 448;
  static constexpr int kBars = 2 * HALVES * kAtTileBytes + kStages * kStageBytes;
  static constexpr int kRowBuffers = 4;
  static constexpr int kRows = kBars + 320;       // of what a tile's queries have: -lse, -delta
  static constexpr int kBias = kRows + kRowBuffers * 2 * 128 * 4;
  static int smem(bool table, int reach) { return 1024 + kBias + (table ? attention_bias_entries(reach) * 4 : 0); }
};

template <bool F16, int HALVES>
__global__ void __launch_bounds__(kAtBackThreads, 1) attention_dkv_kernel(const __grid_constant__ AttentionMaps maps, const AttentionParams p) {
  using C = AtDkv<HALVES>;
  constexpr int ST = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* const smem = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t k_s = base, v_s = k_s + HALVES * kAtTileBytes, ring = v_s + HALVES * kAtTileBytes, bars = base + C::kBars;
  auto landed = [&](int s) { return bars + 8u * s; };
  auto ready = [&](int s) { return bars + 8u * (ST + s); };
  auto empty = [&](int s) { return bars + 8u * (2 * ST + s); };
  const uint32_t k_ready = bars + 8u * (3 * ST), formed = k_ready + 8, read = k_ready + 16, ds_ready = k_ready + 24, ds_done = k_ready + 32;
  auto rows_ready = [&](int b) { return k_ready + 40 + 8u * b; };
  auto rows_free = [&](int b) { return k_ready + 40 + 8u * (C::kRowBuffers + b); };
  static_assert(8 * (3 * ST + 5 + 2 * C::kRowBuffers) <= 256 && sizeof(AttentionPlace) + 12 <= 64, "barriers");
  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(smem + C::kBars + 256 + sizeof(AttentionPlace));
  volatile int* const abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* const ds_scale_s = reinterpret_cast<float*>(tmem_slot + 2);
  int* const status = &tokens_status;
  AttentionPlace* const place_s = reinterpret_cast<AttentionPlace*>(smem + C::kBars + 256);
  float* const of_rows = reinterpret_cast<float*>(smem + C::kRows);
  float* const bias = reinterpret_cast<float*>(smem + C::kBias);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int load_warp = kAtBackWarps, mma_warp = load_warp + 1, clean_warp = load_warp + 2, rows_warp = load_warp + 3;
  const int kv_head = attention_block_head(p.kv_heads), group = p.heads / p.kv_heads;
  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(landed(s), 1);
      mbar_init(ready(s), 1);
      mbar_init(empty(s), 1);
    }
    mbar_init(k_ready, 1);
    mbar_init(formed, 1);
    mbar_init(read, kAtBackWarps);
    mbar_init(ds_ready, kAtBackWarps);
    mbar_init(ds_done, 1);
    for (int b = 0; b < C::kRowBuffers; ++b) {
      mbar_init(rows_ready(b), 1);
      mbar_init(rows_free(b), kAtBackWarps);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == mma_warp) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  grid_dependency_wait();
  grid_dependents_launch();
  if (warp == 0) {
    const AttentionPlace r = attention_place(p, attention_block_place(p, p.kv_heads, false), kAtTile);
    if (lane == 0) *place_s = r;
  }
  if (F16 && warp == 1) {
    const float c = attention_ds_scale(p, kv_head);
    if (lane == 0) *ds_scale_s = c;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const AttentionPlace place = *place_s;
  const int length = static_cast<int>(place.last - place.first), key0 = place.tile * kAtTile;
  const int first_tile = p.causal ? place.tile : 0;  // of the queries
  int tiles = 0;
  if (!place.behind && key0 < length) tiles = (length + kAtTile - 1) / kAtTile - first_tile;
  const int n = tiles * group;  // (head, query tile) one after the other
  auto dirty = [&](int i) { return p.mask != nullptr || (i + 1) * kAtTile > length; };

  if (warp >= kAtBackWarps) {
    registers_fewer<kAtBackFew>();
    if (warp == load_warp && lane == 0 && n > 0) {
      mbar_arrive_expect_tx(k_ready, 2 * HALVES * kAtTileBytes);
      for (int h = 0; h < HALVES; ++h) {
        tma_load_3d(k_s + h * kAtTileBytes, &maps.k, k_ready, h * 64, kv_head, static_cast<int>(place.first) + key0);
        tma_load_3d(v_s + h * kAtTileBytes, &maps.v, k_ready, h * 64, kv_head, static_cast<int>(place.first) + key0);
      }
      int i = 0, head = kv_head * group, tile = first_tile;
      AttentionRing state;
      for (; i < 2 * n; ++i) {
        const bool grad = i & 1;
        const int s = i % ST;
        if (i >= ST && !mbar_wait(empty(s), static_cast<uint32_t>((i / ST) & 1) ^ 1u, abort_flag, status, kDevTimeoutProducer)) break;
        const bool other = dirty(tile);
        state.use(s, other);
        const uint32_t bar = other ? landed(s) : ready(s);
        mbar_arrive_expect_tx(bar, C::kStageBytes);
        for (int h = 0; h < HALVES; ++h)
          tma_load_3d(ring + s * C::kStageBytes + h * kAtTileBytes, grad ? &maps.dout : &maps.q, bar, h * 64, head, static_cast<int>(place.first) + tile * kAtTile);
        if (grad && ++tile == first_tile + tiles) tile = first_tile, ++head;
      }
      state.drain<ST>(k_ready, landed, ready);
    } else if (warp == mma_warp && elect_one()) {
      constexpr uint32_t fmt = F16 ? kFmtF16 : kFmtBF16;
      constexpr uint32_t idesc_s = umma_idesc(128, 128, false, false, fmt, fmt);
      const int steps = (p.d + 15) / 16;
      const uint32_t idesc_o = umma_idesc(128, steps * 16, false, true, fmt, fmt);
      bool ok = n > 0 && mbar_wait(k_ready, 0, abort_flag, status, kDevTimeoutMma);
      auto wait = [&](uint32_t bar, uint32_t parity) { ok = ok && mbar_wait(bar, parity & 1u, abort_flag, status, kDevTimeoutMma); };
      auto form = [&](int u) {
        const int iq = 2 * u, ig = iq + 1, sq = iq % ST, sg = ig % ST;
        wait(ready(sq), iq / ST);
        if (!C::kOver && u > 0) wait(read, u - 1);
        if (!ok) return;
        tc_fence_after();
        for (int ks = 0; ks < steps; ++ks)
          umma_bf16(tmem + C::kScores, umma_desc_kmajor(k_s + (ks >> 2) * kAtTileBytes) + static_cast<uint64_t>((ks & 3) * 2),
                    umma_desc_kmajor(ring + sq * C::kStageBytes + (ks >> 2) * kAtTileBytes) + static_cast<uint64_t>((ks & 3) * 2), idesc_s, ks != 0 ? 1u : 0u);
        wait(ready(sg), ig / ST);
        if (!ok) return;
        tc_fence_after();
        for (int ks = 0; ks < steps; ++ks)
          umma_bf16(tmem + C::kGrad, umma_desc_kmajor(v_s + (ks >> 2) * kAtTileBytes) + static_cast<uint64_t>((ks & 3) * 2),
                    umma_desc_kmajor(ring + sg * C::kStageBytes + (ks >> 2) * kAtTileBytes) + static_cast<uint64_t>((ks & 3) * 2), idesc_s, ks != 0 ? 1u : 0u);
        umma_commit(formed);
      };
      if (ok) form(0);
      for (int u = 0; u < n && ok; ++u) {
        if (!C::kOver && u + 1 < n) form(u + 1);
        wait(ds_ready, u);
        if (!ok) break;
        tc_fence_after();
        const int sq = (2 * u) % ST, sg = (2 * u + 1) % ST;
        const int key_steps = (min(kAtTile, length - (first_tile + u % tiles) * kAtTile) + 15) / 16;
        for (int ks = 0; ks < key_steps; ++ks)
          umma_ta(tmem + C::kDv, tmem + C::kProbs + ks * 8, umma_desc_mnmajor(ring + sg * C::kStageBytes + ks * 2048, kAtTileBytes), idesc_o, (u | ks) != 0 ? 1u : 0u);
        for (int ks = 0; ks < key_steps; ++ks)
          umma_ta(tmem + C::kDk, tmem + C::kDs + ks * 8, umma_desc_mnmajor(ring + sq * C::kStageBytes + ks * 2048, kAtTileBytes), idesc_o, (u | ks) != 0 ? 1u : 0u);
        umma_commit(ds_done);
        umma_commit(empty(sq));
        umma_commit(empty(sg));
        if (C::kOver && u + 1 < n) form(u + 1);
      }
    } else if (warp == clean_warp) {
      uint32_t odd = 0;
      for (int u = 0; u < n; ++u) {
        const int tile = first_tile + u % tiles;
        if (!dirty(tile)) continue;
        uint32_t bits[4];
        attention_rows_there(p, place, length, tile * kAtTile, bits);
        bool ok = true;
        for (int i = 2 * u; i < 2 * u + 2 && ok; ++i) {
          const int s = i % ST;
          ok = mbar_wait_warp(landed(s), odd >> s & 1u, abort_flag, status, kDevTimeoutStats);
          if (!ok) break;
          odd ^= 1u << s;
          attention_clean_rows(ring + s * C::kStageBytes, HALVES, bits);
          if (lane == 0) mbar_arrive(ready(s));
        }
        if (!ok) break;
      }
    } else if (warp == rows_warp) {
      // what a tile's queries have: -lse (with the outer bucket's bias, where the whole tile is in one) and -delta; the next tile's are on
      // their way while this one's are written
      const float held = F16 ? *ds_scale_s * (1.f / 32768.f) : 1.f;
      int head = kv_head * group, tile = first_tile;
      float low = 0.f, high = 0.f, l[4], d[4];
      auto fetch = [&]() {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int query = tile * kAtTile + i * 32 + lane;
          const long long at = head * p.rows + place.first + query;
          l[i] = query < length ? __ldcg(p.lse + at) : INFINITY;
          d[i] = query < length ? __ldcg(p.delta + at) : 0.f;
        }
      };
      if (n > 0) fetch();
      for (int u = 0; u < n; ++u) {
        if (p.table != nullptr && tile == first_tile) {
          low = attention_bias(p, -p.reach, head, F16);
          high = attention_bias(p, p.reach, head, F16);
        }
        const int d0 = key0 - tile * kAtTile, buffer = u % C::kRowBuffers;
        const float add = (F16 ? 15.f : 0.f) + (p.table == nullptr || attention_near(p, d0) ? 0.f : d0 > 0 ? high : low);
        float* const rows = of_rows + buffer * 256;
        if (u >= C::kRowBuffers && !mbar_wait_warp(rows_free(buffer), ((u / C::kRowBuffers) & 1) ^ 1, abort_flag, status, kDevTimeoutStats)) break;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          rows[i * 32 + lane] = add - l[i];
          rows[128 + i * 32 + lane] = -d[i] * held;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(rows_ready(buffer));
        if (++tile == first_tile + tiles) tile = first_tile, ++head;
        if (u + 1 < n) fetch();
      }
    }
  } else {
    registers_more<kAtBackMany>();
    const int quarter = warp >> 2, row = (warp & 3) * 32 + lane, k_row = key0 + row;
    const uint32_t own = tmem + (static_cast<uint32_t>(warp & 3) << 21);
    const bool inside = k_row < length;
    const bool there = inside && !place.behind && (p.mask == nullptr || __ldcg(p.mask + place.first + k_row) != 0);
    const float c = F16 ? *ds_scale_s : 1.f, held = F16 ? c * (1.f / 32768.f) : 1.f, scale = p.scale * kLog2e;
    const float2 held2 = make_float2(held, held);
    int head = kv_head * group, tile = first_tile;
    bool ok = true;
    // (every thread comes to every barrier of its group: after a wait has given up the others return at once)
    for (int u = 0; u < n; ++u) {
      const int q0 = tile * kAtTile, d0 = key0 - q0;
      if (p.table != nullptr && tile == first_tile) {
        if (u > 0) named_bar_sync(1, kAtBackWarps * 32);  // no thread reads the last head's biases any more
        attention_bias_fill(p, bias, head, F16, threadIdx.x, kAtBackWarps * 32);
        named_bar_sync(1, kAtBackWarps * 32);
      }
      const bool near = p.table != nullptr && attention_near(p, d0);
      const int buffer = u % C::kRowBuffers;
      if (++tile == first_tile + tiles) tile = first_tile, ++head;
      ok = mbar_wait_warp(rows_ready(buffer), (u / C::kRowBuffers) & 1, abort_flag, status, kDevTimeoutEpilogue);
      ok = mbar_wait_warp(formed, u & 1, abort_flag, status, kDevTimeoutEpilogue) && ok;
      tc_fence_after();
      uint32_t v[32], g[32];
      tmem_ld32(own + C::kScores + quarter * 32, v);
      tmem_ld32(own + C::kGrad + quarter * 32, g);
      tmem_ld_wait();
      tc_fence_before();
      if (!C::kOver) {
        __syncwarp();
        if (lane == 0) mbar_arrive(read);
      } else {
        named_bar_sync(2 + (warp & 3), 128);  // all of a row's columns have been read before results go over them
      }
      float factor = scale;
      if (near) {
        const float* b = bias + (p.reach + 255) + d0 + row - quarter * 32;
#pragma unroll
        for (int k = 0; k < 32; ++k) v[k] = __float_as_uint(fmaf(__uint_as_float(v[k]), scale, b[-k]));
        factor = 1.f;
      }
      if (p.causal && d0 == 0) {  // queries before the key do not count
        const int first = row - quarter * 32;
#pragma unroll
        for (int k = 0; k < 32; ++k) {
          v[k] = k >= first ? __float_as_uint(__uint_as_float(v[k]) * factor) : 0xFF800000u;
          g[k] = k >= first ? g[k] : 0u;
        }
        factor = 1.f;
      }
      const float2 factor2 = make_float2(factor, factor);
      const float* const rows = of_rows + buffer * 256 + quarter * 32;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t w[8], x[8];
#pragma unroll
        for (int k = 0; k < 8; k += 2) {
          const int at = i * 16 + 2 * k;
          const float4 l = *reinterpret_cast<const float4*>(rows + at), d = *reinterpret_cast<const float4*>(rows + 128 + at);
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const int col = at + 2 * q;
            float2 e = __ffma2_rn(make_float2(__uint_as_float(v[col]), __uint_as_float(v[col + 1])), factor2, q == 0 ? make_float2(l.x, l.y) : make_float2(l.z, l.w));
            e.x = exp2_approx(e.x);
            e.y = exp2_approx(e.y);
            const float2 ds = __fmul2_rn(e, __ffma2_rn(make_float2(__uint_as_float(g[col]), __uint_as_float(g[col + 1])), held2, q == 0 ? make_float2(d.x, d.y) : make_float2(d.z, d.w)));
            w[k + q] = pack_pair<F16>(e);
            x[k + q] = pack_pair<F16>(ds);
          }
        }
        if (i == 0 && u > 0 && ok) {
          ok = mbar_wait_warp(ds_done, (u - 1) & 1, abort_flag, status, kDevTimeoutEpilogue);
          tc_fence_after();
        }
        tmem_st8(own + C::kProbs + quarter * 16 + i * 8, w);
        tmem_st8(own + C::kDs + quarter * 16 + i * 8, x);
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(rows_free(buffer));
        mbar_arrive(ds_ready);
      }
    }
    if (n > 0 && ok) ok = mbar_wait_warp(ds_done, (n - 1) & 1, abort_flag, status, kDevTimeoutEpilogue);
    if (ok) {
      tc_fence_after();
      const long long at = ((place.first + k_row) * p.kv_heads + kv_head) * p.d;
      // two of a row's threads write dk, two dv
      const uint32_t from = own + (quarter < 2 ? C::kDk : C::kDv);
      const float back = quarter < 2 ? p.scale / c : F16 ? 1.f / 32768.f : 1.f;
      uint16_t* const to = static_cast<uint16_t*>(quarter < 2 ? p.dk : p.dv);
      for (int c0 = (quarter & 1) * 16; c0 < p.d; c0 += 32) {
        uint32_t o[16], w[8];
        if (n > 0) {
          tmem_ld16(from + c0, o);
          tmem_ld_wait();
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
          w[k] = there ? pack_pair<F16>(make_float2(__uint_as_float(o[2 * k]) * back, __uint_as_float(o[2 * k + 1]) * back)) : 0u;
        if (inside) {
          uint4* out = reinterpret_cast<uint4*>(to + at + c0);
          out[0] = make_uint4(w[0], w[1], w[2], w[3]);
          if (c0 + 8 < p.d) out[1] = make_uint4(w[4], w[5], w[6], w[7]);
        }
      }
    }
  }
  __syncthreads();
  if (warp == mma_warp) tmem_dealloc(tmem, 512);
}

// The table's gradient: a block a head adds the places' sums up, each distance in as many threads as there are, then a thread a bucket
// its distances. With the farthest reach one or two threads add up all places of a distance, tens of thousands where sequences are short, and
// terms that nearly cancel: a thread adds up runs of places in fp32 and the runs in 64 bits, in the same time as all in fp32 (every
// place in 64 bits took 3 us more with 1584 places and 257 distances).
constexpr int kAtTableRun = 32;
template <typename T>
__global__ void __launch_bounds__(1024) attention_table_kernel(const AttentionParams p) {
  __shared__ double distance[1024];
  __shared__ float whole[2 * B200_POSITION_MAX_REACH + 1];
  __shared__ int bucket[2 * B200_POSITION_MAX_REACH + 1];
  grid_dependency_wait();
  grid_dependents_launch();
  const int distances = 2 * p.reach + 1, head = blockIdx.x, teams = 1024 / distances;
  const int team = threadIdx.x / distances, i = threadIdx.x % distances;
  const float* in = p.partial + (static_cast<long long>(head) * p.places + team) * distances + i;
  const long long step = static_cast<long long>(teams) * distances;
  const int places = static_cast<int>(p.places);  // (no more than a grid has blocks)
  const int count = team < teams && team < places ? (places - 1 - team) / teams + 1 : 0;
  double s = 0.;
  for (int left = count; left > 0; left -= kAtTableRun, in += kAtTableRun * step) {
    float run = 0.f;
    if (left >= kAtTableRun) {
#pragma unroll 8
      for (int k = 0; k < kAtTableRun; ++k) run += __ldcg(in + k * step);
    } else {
#pragma unroll 8
      for (int k = 0; k < left; ++k) run += __ldcg(in + k * step);
    }
    s += run;
  }
  distance[threadIdx.x] = s;
  if (threadIdx.x < distances) bucket[threadIdx.x] = min(max(__ldcg(p.bucket_of + threadIdx.x), 0), p.buckets - 1);
  __syncthreads();
  if (threadIdx.x < distances)
    for (int t = 1; t < teams; ++t) s += distance[t * distances + threadIdx.x];
  if (threadIdx.x < distances) whole[threadIdx.x] = static_cast<float>(s);
  __syncthreads();
  for (int b = threadIdx.x; b < p.buckets; b += 1024) {
    float total = 0.f;
    for (int k = 0; k < distances; ++k)
      if (bucket[k] == b) total += whole[k];
    static_cast<T*>(p.dtable)[static_cast<long long>(b) * p.heads + head] = static_cast<T>(total);
  }
}

}  // namespace trimul
