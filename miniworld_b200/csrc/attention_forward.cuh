// Forward of the attention (formulas: attention.cuh). One pass over the keys with the running maximum and sum of the softmax; a block
// takes one tile of 128 queries (widths up to 64; two blocks an SM) or two (up to 128; each key and value tile then serves 256 queries)
// of one head. A warp copies key and value tiles into a ring in shared memory, one issues the products, one zeroes rows of value tiles
// that do not count; eight warps a query tile hold half a row of scores a thread.
//
// What bounds it is the exponential: 16 a clock and SM, 1024 clocks for a tile, against 512 (d = 64) of products. So the next tile's
// scores are formed as soon as this tile's are in registers, with the probabilities in columns of their own (d <= 64), or the two
// query tiles take turns (d > 64, probabilities over the scores). The accumulator is brought to a new maximum only where one grew by
// more than 2^8: the probabilities stay below 2^8 then (2^15 in fp16, where they begin at 2^7, so that small ones keep their bits),
// which costs nothing in floating point; the two threads of a row compare their maxima only where one of a warp pair's grew by that much.
//
// One B200, 2 x 4096 tokens, 16 heads: 218 us at d = 64 (the special function unit busy 56 % of the time over the launch, 82 % between
// a block's first and last tile), 284 us at d = 128 (970 TFLOP/s, 0.62 of measured). With a thread a row 250 and 341: one warp a
// scheduler and block waits out its own latencies. Tiles of 64 keys with four blocks an SM (d <= 64) or two buffers of scores (d > 64) 238
// and 368: a product of 64 columns takes as long as one of 128, for the rows of q that it reads from shared memory. Short sequences pay 4500 of a block's 14000
// clocks before its first scores and 2000 after its last (512 x 384 tokens, 8 heads of 32: 354 us). Blocks that stay and have the next
// work's tiles on their way, or a copying warp that does not wait for the others' set-up, cost registers that the softmax needs: 415
// and 430 us there.
#pragma once

#include "attention_tiles.cuh"
#include "tokens_status.cuh"

namespace trimul {

template <int HALVES>
struct AtForward {
  static constexpr int kTiles = HALVES;                 // query tiles of a block
  static constexpr bool kOver = HALVES == 2;            // probabilities over the scores
  static constexpr int kStages = HALVES == 1 ? 5 : 4;   // of key and value tiles
  static constexpr int kSoftmaxWarps = 8 * kTiles;
  static constexpr int kThreads = kSoftmaxWarps * 32 + 128;
  static constexpr int kBlocks = HALVES == 1 ? 2 : 1;   // an SM
  // registers: the launch's are 80 or 96; the softmax's warps take from the others (2 x 104 + 32 = 3 x 80, 4 x 104 + 64 = 5 x 96)
  static constexpr int kMany = 104, kFew = HALVES == 1 ? 32 : 64;
  static constexpr uint32_t kColumns = HALVES == 1 ? 256 : 512;
  static constexpr int kStageBytes = HALVES * kAtTileBytes;
  static constexpr int kBars = kTiles * HALVES * kAtTileBytes + kStages * kStageBytes;
  static constexpr int kSwap = kBars + 320;             // what the two threads of a row tell each other
  static constexpr int kBias = kSwap + kTiles * 2 * kAtTile * 4;
  static int smem(bool table, int reach) { return 1024 + kBias + (table ? attention_bias_entries(reach) * 4 : 0); }
  __host__ __device__ static constexpr uint32_t scores(int t) { return static_cast<uint32_t>(t) * 128; }
  __host__ __device__ static constexpr uint32_t probabilities(int t) { return kOver ? static_cast<uint32_t>(t) * 128 : 128u; }
  __host__ __device__ static constexpr uint32_t out(int t) { return kOver ? 256u + static_cast<uint32_t>(t) * 128 : 192u; }
};

template <bool F16, int HALVES>
__global__ void __launch_bounds__(AtForward<HALVES>::kThreads, AtForward<HALVES>::kBlocks)
    attention_forward_kernel(const __grid_constant__ AttentionMaps maps, const AttentionParams p) {
  using C = AtForward<HALVES>;
  constexpr int T = C::kTiles, ST = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* const smem = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t q_s = base, ring = q_s + T * HALVES * kAtTileBytes, bars = base + C::kBars;
  auto landed = [&](int s) { return bars + 8u * s; };          // a copy has landed, rows of it are still to be zeroed
  auto ready = [&](int s) { return bars + 8u * (ST + s); };    // the tile can be used
  auto empty = [&](int s) { return bars + 8u * (2 * ST + s); };
  constexpr int B0 = 3 * ST;
  const uint32_t q_ready = bars + 8u * B0;
  auto scores_ready = [&](int t) { return bars + 8u * (B0 + 1 + t); };
  auto scores_read = [&](int t) { return bars + 8u * (B0 + 1 + T + t); };
  auto probs_ready = [&](int t) { return bars + 8u * (B0 + 1 + 2 * T + t); };
  auto out_done = [&](int t) { return bars + 8u * (B0 + 1 + 3 * T + t); };
  static_assert(8 * (B0 + 1 + 4 * T) <= 240, "barriers");
  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(smem + C::kBars + 240);
  volatile int* const abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* const status = &tokens_status;
  AttentionPlace* const place_s = reinterpret_cast<AttentionPlace*>(smem + C::kBars + 256);
  float* const swap = reinterpret_cast<float*>(smem + C::kSwap);  // [query tile][half][row]
  float* const bias = reinterpret_cast<float*>(smem + C::kBias);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int load_warp = C::kSoftmaxWarps, mma_warp = load_warp + 1, clean_warp = load_warp + 2;
  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(landed(s), 1);
      mbar_init(ready(s), 1);
      mbar_init(empty(s), 1);
    }
    mbar_init(q_ready, 1);
    for (int t = 0; t < T; ++t) {
      mbar_init(scores_ready(t), 1);
      mbar_init(scores_read(t), 8);
      mbar_init(probs_ready(t), 8);
      mbar_init(out_done(t), 1);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == mma_warp) {
    tmem_alloc(smem_u32(tmem_slot), C::kColumns);
    tmem_relinquish();
  }
  grid_dependency_wait();
  grid_dependents_launch();
  const long long place_index = attention_block_place(p, p.heads, p.causal);
  if (warp == 0) {
    const AttentionPlace r = attention_place(p, place_index, T * kAtTile);
    if (lane == 0) *place_s = r;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const AttentionPlace place = *place_s;
  const int head = attention_block_head(p.heads), kv_head = head / (p.heads / p.kv_heads);
  const int length = static_cast<int>(place.last - place.first);
  // key tiles of query tile t
  auto tiles_of = [&](int t) {
    const long long q0 = (static_cast<long long>(place.tile) * T + t) * kAtTile;
    if (place.behind || q0 >= length) return 0;
    const int keys = p.causal ? static_cast<int>(min(q0 + kAtTile, static_cast<long long>(length))) : length;
    return (keys + kAtTile - 1) / kAtTile;
  };
  const int n0 = tiles_of(0), n1 = T == 2 ? tiles_of(T - 1) : 0, n = max(n0, n1);
  // places in the order of use: scores of the next tile come before the sum of this one where they have columns of their own
  auto key_place = [&](int j) { return C::kOver ? 2 * j : j == 0 ? 0 : 2 * j - 1; };
  auto value_place = [&](int j) { return C::kOver ? 2 * j + 1 : j < n - 1 ? 2 * j + 2 : 2 * n - 1; };
  auto dirty = [&](int j) { return p.mask != nullptr || (j + 1) * kAtTile > length; };  // value tile j has rows that may not count

  if (warp >= C::kSoftmaxWarps) {
    registers_fewer<C::kFew>();
    if (warp == load_warp && lane == 0 && n > 0) {
      mbar_arrive_expect_tx(q_ready, ((n0 > 0) + (n1 > 0)) * HALVES * kAtTileBytes);
      for (int t = 0; t < T; ++t)
        if ((t == 0 ? n0 : n1) > 0)
          for (int h = 0; h < HALVES; ++h)
            tma_load_3d(q_s + (t * HALVES + h) * kAtTileBytes, &maps.q, q_ready, h * 64, head, static_cast<int>(place.first) + (place.tile * T + t) * kAtTile);
      AttentionRing state;
      for (int i = 0; i < 2 * n; ++i) {
        // which tile is next
        bool value;
        int j;
        if (C::kOver) {
          value = i & 1;
          j = i >> 1;
        } else {
          value = i == 2 * n - 1 || (i != 0 && !(i & 1));
          j = i == 2 * n - 1 ? n - 1 : i == 0 ? 0 : value ? (i - 2) / 2 : (i + 1) / 2;
        }
        const int s = i % ST;
        if (i >= ST && !mbar_wait(empty(s), static_cast<uint32_t>((i / ST) & 1) ^ 1u, abort_flag, status, kDevTimeoutProducer)) break;
        const bool other = value && dirty(j);
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
      const uint32_t idesc_o = umma_idesc(128, steps * 16, false, true, fmt, fmt);
      bool ok = n > 0 && mbar_wait(q_ready, 0, abort_flag, status, kDevTimeoutMma);
      auto wait = [&](uint32_t bar, uint32_t parity) { ok = ok && mbar_wait(bar, parity & 1u, abort_flag, status, kDevTimeoutMma); };
      // (products are carried out in the order of their issue: scores go over the last tile's probabilities after these have been used)
      auto form_scores = [&](int t, int j, bool first, bool last) {
        const int i = key_place(j), s = i % ST;
        if (first) wait(ready(s), i / ST);
        if (!C::kOver && j > 0) wait(scores_read(t), j - 1);
        if (!ok) return;
        tc_fence_after();
        for (int ks = 0; ks < steps; ++ks)
          umma_bf16(tmem + C::scores(t), umma_desc_kmajor(q_s + (t * HALVES + (ks >> 2)) * kAtTileBytes) + static_cast<uint64_t>((ks & 3) * 2),
                    umma_desc_kmajor(ring + s * C::kStageBytes + (ks >> 2) * kAtTileBytes) + static_cast<uint64_t>((ks & 3) * 2), idesc_s, ks != 0 ? 1u : 0u);
        umma_commit(scores_ready(t));
        if (last) umma_commit(empty(s));
      };
      auto add_values = [&](int t, int j, bool first, bool last) {
        const int i = value_place(j), s = i % ST;
        if (first) wait(ready(s), i / ST);
        wait(probs_ready(t), j);
        if (!ok) return;
        tc_fence_after();
        const int key_steps = 2 * ((min(kAtTile, length - j * kAtTile) + 31) / 32);  // (probabilities come in pieces of 32)
        for (int ks = 0; ks < key_steps; ++ks)
          umma_ta(tmem + C::out(t), tmem + C::probabilities(t) + ks * 8, umma_desc_mnmajor(ring + s * C::kStageBytes + ks * 2048, kAtTileBytes), idesc_o,
                  (j | ks) != 0 ? 1u : 0u);
        umma_commit(out_done(t));
        if (last) umma_commit(empty(s));
      };
      // (the second query tile has at least as many key tiles as the first, or none)
      for (int j = -1; j < n && ok; ++j) {
        const bool a = j >= 0 && j < n0, b = j >= 0 && j < n1, next_a = j + 1 < n0, next_b = j + 1 < n1;
        if (!C::kOver && next_a) form_scores(0, j + 1, true, true);
        if (a && ok) add_values(0, j, true, !b);
        if (C::kOver && next_a && ok) form_scores(0, j + 1, true, !next_b);
        if (b && ok) add_values(1, j, !a, true);
        if (next_b && ok) form_scores(1, j + 1, !next_a, true);
      }
    } else if (warp == clean_warp) {
      uint32_t odd = 0;  // a bit a stage: parity of landed()'s next phase
      for (int j = 0; j < n; ++j) {
        if (!dirty(j)) continue;
        const int s = value_place(j) % ST;
        uint32_t bits[4];
        attention_rows_there(p, place, length, j * kAtTile, bits);
        if (!mbar_wait_warp(landed(s), odd >> s & 1u, abort_flag, status, kDevTimeoutStats)) break;
        odd ^= 1u << s;
        attention_clean_rows(ring + s * C::kStageBytes, HALVES, bits);
        if (lane == 0) mbar_arrive(ready(s));
      }
    }
  } else {
    registers_more<C::kMany>();
    // two threads a row: columns 0 .. 63 and 64 .. 127 of the scores, every other 16 columns of the sums
    const int t = warp >> 3, half = warp >> 2 & 1, nt = t == 0 ? n0 : n1, row = (warp & 3) * 32 + lane, pair = 2 + t * 4 + (warp & 3);
    const uint32_t own = tmem + (static_cast<uint32_t>(warp & 3) << 21);  // this warp's lanes
    const int q0 = (place.tile * T + t) * kAtTile, q_row = q0 + row;
    const bool inside = q_row < length;
    const bool there = inside && !place.behind && (p.mask == nullptr || __ldcg(p.mask + place.first + q_row) != 0);
    float* const mine = swap + (t * 2 + half) * kAtTile + row;
    const float* const other = swap + (t * 2 + (half ^ 1)) * kAtTile + row;
    float low = 0.f, high = 0.f;  // the outer buckets
    if (p.table != nullptr && n > 0) {
      attention_bias_fill(p, bias, head, F16, threadIdx.x, C::kSoftmaxWarps * 32);
      named_bar_sync(1, C::kSoftmaxWarps * 32);
      low = bias[0];
      high = bias[2 * (p.reach + 255)];
    }
    constexpr float kOffset = F16 ? 7.f : 0.f;  // log2 of what a probability of one is held as
    constexpr float kGrowth = 8.f;
    const float scale = p.scale * kLog2e;
    float m = -INFINITY;
    float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
    bool ok = true;
    // (every thread comes to every barrier of its pair: after a wait has given up the others return at once)
    for (int j = 0; j < nt; ++j) {
      const int key0 = j * kAtTile + half * 64, d0 = key0 - q0;
      const bool near = p.table != nullptr && d0 + 63 > -p.reach && d0 - 127 < p.reach;
      const float add = p.table == nullptr || near ? 0.f : d0 > 0 ? high : low;
      const int keys = length - key0, limit = p.causal ? min(keys, q_row - key0 + 1) : keys;
      uint32_t bits[2] = {~0u, ~0u};
      if (p.mask != nullptr) attention_mask_bits(p, place.first + key0, place.last, bits);
      ok = mbar_wait_warp(scores_ready(t), j & 1, abort_flag, status, kDevTimeoutEpilogue);
      tc_fence_after();
      uint32_t v[2][32];
#pragma unroll
      for (int i = 0; i < 2; ++i) tmem_ld32(own + C::scores(t) + half * 64 + i * 32, v[i]);
      tmem_ld_wait();
      if (!C::kOver) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(scores_read(t));
      }
      float factor = scale;
      if (near) {
        const float* b = bias + (p.reach + 255) + d0 - row;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int c = 0; c < 32; ++c) v[i][c] = __float_as_uint(fmaf(__uint_as_float(v[i][c]), scale, b[i * 32 + c]));
        factor = 1.f;
      } else if (scale <= 0.f) {  // (the greatest score is not that of the greatest product)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int c = 0; c < 32; ++c) v[i][c] = __float_as_uint(__uint_as_float(v[i][c]) * scale);
        factor = 1.f;
      }
      float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};  // (a chain of dependent instructions costs more than they have)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t counts = bits[i] & first_bits(limit - 32 * i);
        if (counts != ~0u) {
#pragma unroll
          for (int c = 0; c < 32; ++c)
            if (!(counts >> c & 1u)) v[i][c] = 0xFF800000u;
        }
#pragma unroll
        for (int c = 0; c < 32; c += 2) top[c / 2 % 4] = max3(top[c / 2 % 4], __uint_as_float(v[i][c]), __uint_as_float(v[i][c + 1]));
      }
      const float most = fmaf(max3(fmaxf(top[0], top[1]), top[2], top[3]), factor, add);
      // A new maximum only where it grew by much, or where there was none; only then do the two threads of a row compare theirs. (Both
      // have read their scores when one writes probabilities over them.)
      if (named_bar_or(pair, 64, most > m + kGrowth || (m == -INFINITY && most > m))) {
        *mine = most;
        named_bar_sync(pair, 64);
        const float both = fmaxf(most, *other);
        float shrink = 1.f;
        if (both > m + kGrowth || (m == -INFINITY && both > m)) {
          shrink = exp2_approx(m - both);
          m = both;
          sum[0] = make_float2(sum[0].x * shrink, sum[0].y * shrink);
          sum[1] = make_float2(sum[1].x * shrink, sum[1].y * shrink);
        }
        if (j > 0) {
          // (no product is adding to the accumulator after that: the next one waits for these probabilities)
          ok = ok && mbar_wait_warp(out_done(t), (j - 1) & 1, abort_flag, status, kDevTimeoutEpilogue);
          tc_fence_after();
          const float2 shrink2 = make_float2(shrink, shrink);
          for (int c0 = half * 16; c0 < p.d; c0 += 32) {
            uint32_t o[16];
            tmem_ld16(own + C::out(t) + c0, o);
            tmem_ld_wait();
#pragma unroll
            for (int c = 0; c < 16; c += 2) {
              const float2 s = __fmul2_rn(make_float2(__uint_as_float(o[c]), __uint_as_float(o[c + 1])), shrink2);
              o[c] = __float_as_uint(s.x);
              o[c + 1] = __float_as_uint(s.y);
            }
            tmem_st16(own + C::out(t) + c0, o);
          }
        }
      }
      const float shift = add + kOffset - (m == -INFINITY ? 0.f : m);
      const float2 factor2 = make_float2(factor, factor), shift2 = make_float2(shift, shift);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t w[16];
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          float2 e = __ffma2_rn(make_float2(__uint_as_float(v[i][2 * c]), __uint_as_float(v[i][2 * c + 1])), factor2, shift2);
          e.x = exp2_approx(e.x);
          e.y = exp2_approx(e.y);
          sum[c & 1] = __fadd2_rn(sum[c & 1], e);
          w[c] = pack_pair<F16>(e);
        }
        if (!C::kOver && i == 0 && j > 0 && ok) {
          // The products with the last tile's probabilities are done: their columns can be written. (Every warp waits, whether or not it
          // has columns with keys: one that went on would arrive for this tile while the others have yet to arrive for the last.)
          ok = mbar_wait_warp(out_done(t), (j - 1) & 1, abort_flag, status, kDevTimeoutEpilogue);
          tc_fence_after();
        }
        if (i * 32 < keys) tmem_st16(own + C::probabilities(t) + half * 32 + i * 16, w);
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(probs_ready(t));
    }
    if (nt > 0) {
      ok = ok && mbar_wait_warp(out_done(t), (nt - 1) & 1, abort_flag, status, kDevTimeoutEpilogue);
      named_bar_sync(pair, 64);  // (the other has read this one's maximum)
      *mine = (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
      named_bar_sync(pair, 64);
    }
    if (ok) {
      tc_fence_after();
      const float total = nt > 0 ? swap[t * 2 * kAtTile + row] + swap[(t * 2 + 1) * kAtTile + row] : 0.f;
      const bool some = there && total != 0.f;  // (NaN: some)
      const float inverse = some ? 1.f / total : 0.f;
      const long long at = ((place.first + q_row) * p.heads + head) * p.d;
      for (int c0 = half * 16; c0 < p.d; c0 += 32) {
        uint32_t o[16], w[8], rest[8];
        if (nt > 0) {
          tmem_ld16(own + C::out(t) + c0, o);
          tmem_ld_wait();
        }
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const float2 s = some ? make_float2(__uint_as_float(o[2 * c]) * inverse, __uint_as_float(o[2 * c + 1]) * inverse) : make_float2(0.f, 0.f);
          w[c] = pack_pair<F16>(s);
          // what the rounding took away, for the backward (in fp16 2^11 times as much: it would be subnormal)
          const float2 r = unpack_pair<F16>(w[c]);
          rest[c] = pack_pair<F16>(make_float2((s.x - r.x) * kAtRest<F16>, (s.y - r.y) * kAtRest<F16>));
        }
        if (inside) {
#pragma unroll
          for (int q = 0; q < 2; ++q)
            if (c0 + q * 8 < p.d) {
              *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.o) + at + c0 + q * 8) = make_uint4(w[q * 4], w[q * 4 + 1], w[q * 4 + 2], w[q * 4 + 3]);
              if (p.rest != nullptr)
                *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.rest) + at + c0 + q * 8) = make_uint4(rest[q * 4], rest[q * 4 + 1], rest[q * 4 + 2], rest[q * 4 + 3]);
            }
        }
      }
      if (half == 0 && inside && p.lse != nullptr) p.lse[head * p.rows + place.first + q_row] = some ? m - kOffset + log2f(total) : INFINITY;
    }
  }
  __syncthreads();
  if (warp == mma_warp) tmem_dealloc(tmem, C::kColumns);
}

}  // namespace trimul
