// The gated feed-forward of narrow tensors (D <= 128) in one kernel: h never leaves the SM.
//
// With two kernels h is written and read once, 4 H bytes a row against 4 D of x and y: at D = 64, H = 256 four fifths of the traffic
// (196608 rows: 38.5 + 22 us). Here a CTA pair works on 256 rows and walks the hidden width in blocks of 64 units, as the pair
// Transition does (transition.cuh, whose buffers and hand-overs these are):
//
//   G1(block): D1[row, 0:64 | 64:128] = x[row, :] * [W_a(block) ; W_b(block)]^T        (M 256, N 128, K D)
//   gate     : h[row, u] = act(D1[row, u]) * D1[row, 64 + u]  -> 16 bits, into tensor memory
//   G2(block): D2[row, :] += h[row, 0:64] * W_s[:, block]^T                            (M 256, N 64 or 128, A operand from tensor memory)
//
// CTA 0 loads the block's rows of W_a, CTA 1 those of W_b, each its half of the rows of W_s. Tensor memory: D1[0..2] (128 columns each)
// and D2 (two of 64 for D <= 64, one of 128). Blocks go round three groups of eight warps by their running number gb; a group reads its
// D1 into registers and leaves h in the same columns, which are free again once G2 of the block is complete.
// What bounds it is the special-function unit: an exponential a unit and a reciprocal for four, 1.25 x 64 x 128 / 16 = 640 cycles a
// block and SM, so the groups are there to keep it busy while others wait for products, tensor memory and barriers: 196608 x 64 x 256
// with two groups (h in the idle D2, a reciprocal for two) 42 us; now 31.8 us in a graph of calls, of which that unit is busy half of
// the time.
// Warps: 0 weights, 1 G1, 2 input tiles, 3 G2, 4-27 the gate's groups, 28-31 output. All waits are bounded.
#pragma once

#include "feed_forward.cuh"

namespace trimul {

struct FfNarrowParams {
  void* y;
  long long rows;
  int d;          // columns of y
  int num_tiles;  // of 256 rows
  int blocks;     // of 64 hidden units
};

constexpr int kNwThreads = 1024;
constexpr int kNwGroups = 3;
constexpr int kNwWStages = 5;
constexpr int kNwXStages = 3;
constexpr int kNwWStageBytes = 24576;  // 64 rows of W_a or W_b, up to 64 of W_s
constexpr int kNwXBytes = 32768;
constexpr int kNwSmemBytes = kNwXStages * kNwXBytes + kNwWStages * kNwWStageBytes + 256 + 1024;
constexpr uint32_t kNwColD2 = 128 * kNwGroups;

// HALVES: 64-wide parts of D
template <bool F16, int ACT, int HALVES>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kNwThreads, 1)
ff_narrow_kernel(const __grid_constant__ FfMaps maps, const FfNarrowParams p) {
  constexpr int WS = kNwWStages, XS = kNwXStages, G = kNwGroups;
  constexpr int kN2 = 64 * HALVES;  // columns of D2
  constexpr uint32_t kWBytes = HALVES * 8192 + (kN2 / 2) * 128;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t x_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t w_base = x_base + XS * kNwXBytes;
  const uint32_t bar_base = w_base + WS * kNwWStageBytes;
  // ("leader": only CTA 0's is used; "both": the commit signals the one in each CTA)
  auto x_full = [&](int s) { return bar_base + 8u * s; };                // leader: bytes of both CTAs
  auto x_empty = [&](int s) { return bar_base + 8u * (XS + s); };        // both: every G1 of the tile is complete
  constexpr int B0 = 2 * XS;
  auto w_full = [&](int s) { return bar_base + 8u * (B0 + s); };         // leader: bytes of both CTAs
  auto blk_done = [&](int s) { return bar_base + 8u * (B0 + WS + s); };  // both: G2 of the block in weight stage s is complete
  auto d1_full = [&](int g) { return bar_base + 8u * (B0 + 2 * WS + g); };          // both
  auto d1_free = [&](int g) { return bar_base + 8u * (B0 + 2 * WS + G + g); };      // both: G2 has read h out of it
  auto h_full = [&](int g) { return bar_base + 8u * (B0 + 2 * WS + 2 * G + g); };   // leader: 8 warps of each CTA
  constexpr int B1 = B0 + 2 * WS + 3 * G;
  auto d2_full = [&](int b) { return bar_base + 8u * (B1 + b); };        // both
  auto d2_empty = [&](int b) { return bar_base + 8u * (B1 + 2 + b); };   // leader: 4 warps of each CTA
  // the D2 buffer of tile t and how often it has been used before
  auto d2_of = [&](int t) { return HALVES == 1 ? t & 1 : 0; };
  auto d2_use = [&](int t) { return HALVES == 1 ? t >> 1 : t; };
  auto d2_col = [&](int t) { return kNwColD2 + (HALVES == 1 ? (t & 1) * 64u : 0u); };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem_raw + (bar_base - smem_u32(smem_raw)) + 8 * (B1 + 4));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* const status = &blocks_status;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int pair = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;
  if (threadIdx.x == 0) {
    for (int s = 0; s < XS; ++s) {
      mbar_init(x_full(s), 1);
      mbar_init(x_empty(s), 1);
    }
    for (int s = 0; s < WS; ++s) {
      mbar_init(w_full(s), 1);
      mbar_init(blk_done(s), 1);
    }
    for (int g = 0; g < G; ++g) {
      mbar_init(d1_full(g), 1);
      mbar_init(d1_free(g), 1);
      mbar_init(h_full(g), 16);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(d2_full(b), 1);
      mbar_init(d2_empty(b), 8);
    }
    *abort_flag = 0;
    fence_mbar_init();
    prefetch_tmap(&maps.a[0]);
    prefetch_tmap(&maps.b[rank]);
    prefetch_tmap(&maps.b[2]);
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(tmem_slot), 512);
    tmem_relinquish_pair();
  }
  grid_dependency_wait();
  grid_dependents_launch();
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // barriers of both CTAs are initialised before any signal crosses
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int nb = p.blocks;
  const int my_tiles = pair < p.num_tiles ? (p.num_tiles - pair + num_pairs - 1) / num_pairs : 0;
  const int total = my_tiles * nb;
  // a producer's copies that nothing has waited for (after a wait has given up) land before the CTA may exit
  auto drain = [&](int issued, int stages, auto full) {
    for (int i = issued > stages ? issued - stages : 0; i < issued; ++i) {
      const long long t0 = clock64();
      while (!mbar_try_wait(full(i % stages), static_cast<uint32_t>((i / stages) & 1))) {
        if (*abort_flag != 0 || clock64() - t0 > kWaitLimitCycles) {
          atomicCAS(status, 0, kDevTimeoutDrain);
          break;
        }
      }
    }
  };

  if (warp == 0) {
    // ------------------------------------------------------------ weights, block after block (both CTAs)
    if (lane == 0) {
      int gb = 0;
      for (; gb < total; ++gb) {
        const int slot = gb % WS, hb = gb % nb;
        if (!mbar_wait(blk_done(slot), static_cast<uint32_t>((gb / WS) & 1) ^ 1u, abort_flag, status, kDevTimeoutProducer)) break;
        if (rank == 0) mbar_arrive_expect_tx(w_full(slot), 2 * kWBytes);
        const uint32_t bar = map_to_cta(w_full(slot), 0), ws = w_base + slot * kNwWStageBytes;
#pragma unroll
        for (int i = 0; i < HALVES; ++i) tma_load_2d_pair(ws + i * 8192, &maps.b[rank], bar, i * 64, hb * 64);
        tma_load_2d_pair(ws + 16384, &maps.b[2], bar, hb * 64, static_cast<int>(rank) * (kN2 / 2));
      }
      if (rank == 0) drain(gb, WS, w_full);
    }
  } else if (warp == 2) {
    // ------------------------------------------------------------ input tiles (both CTAs); rows past the end read as zero
    if (lane == 0) {
      int t = 0;
      for (; t < my_tiles; ++t) {
        const int s = t % XS;
        if (!mbar_wait(x_empty(s), static_cast<uint32_t>((t / XS) & 1) ^ 1u, abort_flag, status, kDevTimeoutProducer)) break;
        if (rank == 0) mbar_arrive_expect_tx(x_full(s), 2 * HALVES * 16384);
        const uint32_t bar = map_to_cta(x_full(s), 0);
        const int row0 = (pair + t * num_pairs) * 256 + static_cast<int>(rank) * 128;
#pragma unroll
        for (int i = 0; i < HALVES; ++i) tma_load_2d_pair(x_base + s * kNwXBytes + i * 16384, &maps.a[0], bar, i * 64, row0);
      }
      if (rank == 0) drain(t, XS, x_full);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ G1 (leader)
    if (rank == 0 && elect_one()) {
      constexpr uint32_t idesc = umma_idesc(256, 128, false, false, F16 ? kFmtF16 : kFmtBF16, F16 ? kFmtF16 : kFmtBF16);
      int t = 0, hb = 0;
      for (int gb = 0; gb < total; ++gb) {
        const int s = t % XS, slot = gb % WS, g = gb % G;
        if (hb == 0 && !mbar_wait(x_full(s), (t / XS) & 1, abort_flag, status, kDevTimeoutMma)) break;
        if (!mbar_wait(w_full(slot), static_cast<uint32_t>((gb / WS) & 1), abort_flag, status, kDevTimeoutMma)) break;
        if (!mbar_wait(d1_free(g), static_cast<uint32_t>(((gb / G) & 1) ^ 1), abort_flag, status, kDevTimeoutMma)) break;
        tc_fence_after();
        const uint32_t xs = x_base + s * kNwXBytes, ws = w_base + slot * kNwWStageBytes;
#pragma unroll
        for (int ks = 0; ks < 4 * HALVES; ++ks)
          umma_pair(tmem + g * 128, umma_desc_kmajor(xs + (ks >> 2) * 16384) + static_cast<uint64_t>((ks & 3) * 2),
                    umma_desc_kmajor(ws + (ks >> 2) * 8192) + static_cast<uint64_t>((ks & 3) * 2), idesc, ks != 0 ? 1u : 0u);
        umma_commit_pair(d1_full(g));
        if (++hb == nb) {
          umma_commit_pair(x_empty(s));
          hb = 0;
          ++t;
        }
      }
    }
  } else if (warp == 3) {
    // ------------------------------------------------------------ G2 (leader). G1 of the same block was complete before h could be
    // formed, so one commit says that the block's weight stage and its h are free.
    if (rank == 0 && elect_one()) {
      constexpr uint32_t idesc = umma_idesc(256, kN2, false, false, F16 ? kFmtF16 : kFmtBF16, F16 ? kFmtF16 : kFmtBF16);
      int t = 0, hb = 0;
      for (int gb = 0; gb < total; ++gb) {
        const int slot = gb % WS, g = gb % G;
        if (hb == 0 && !mbar_wait(d2_empty(d2_of(t)), (d2_use(t) & 1) ^ 1u, abort_flag, status, kDevTimeoutMma)) break;
        if (!mbar_wait(h_full(g), static_cast<uint32_t>((gb / G) & 1), abort_flag, status, kDevTimeoutMma)) break;
        tc_fence_after();
        const uint32_t ws = w_base + slot * kNwWStageBytes + 16384;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)  // (h of units 0-31 and of units 32-63: see the gate)
          umma_pair_ta(tmem + d2_col(t), tmem + g * 128 + (ks >> 1) * 32 + (ks & 1) * 8, umma_desc_kmajor(ws) + static_cast<uint64_t>(ks * 2), idesc,
                       (hb | ks) != 0 ? 1u : 0u);
        umma_commit_pair(blk_done(slot));
        umma_commit_pair(d1_free(g));
        if (++hb == nb) {
          umma_commit_pair(d2_full(d2_of(t)));
          hb = 0;
          ++t;
        }
      }
    }
  } else if (warp < 4 + 8 * G) {
    // ------------------------------------------------------------ gate: a row and 32 of the block's 64 units a thread, 16 at a time.
    // h (16 columns) replaces the thread's own values of a, which no other thread reads.
    const int grp = (warp - 4) >> 3, uh = ((warp - 4) >> 2) & 1;
    const uint32_t d1 = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + grp * 128 + uh * 32;
    uint32_t ph = 0;
    for (int gb = grp; gb < total; gb += G, ph ^= 1u) {
      if (!mbar_wait_warp(d1_full(grp), ph, abort_flag, status, kDevTimeoutEpilogue)) break;
      tc_fence_after();
      uint32_t o[16];
      float most = 0.f;  // of |h|, NaN where one of them is
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t va[16], vb[16];
        tmem_ld16(d1 + c * 16, va);
        tmem_ld16(d1 + 64 + c * 16, vb);
        tmem_ld_wait();
        float h[16];
        ff_gate16(va, vb, ACT, h);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float2 v = make_float2(h[2 * j], h[2 * j + 1]);
          if (F16) asm("max.NaN.abs.f32 %0, %0, %1, %2;" : "+f"(most) : "f"(v.x), "f"(v.y));
          o[8 * c + j] = F16 ? pack_f16x2_sat(v) : pack_bf16x2(v.x, v.y);
        }
      }
      // fp16: a finite h beyond the range becomes +-65504, and so would an infinite one. It makes the whole row of y infinite or NaN in any
      // case, so two NaN in the place of two of the row's values say the same (one instruction for two values; with each value's own
      // infinity 34.1 us, GELU 48, against 32.8 and 45)
      if (F16 && !(most < INFINITY)) o[0] = 0x7FFF7FFFu;
      tmem_st16(d1, o);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_leader(h_full(grp), rank);
    }
  } else {
    // ------------------------------------------------------------ output: a row a thread
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    for (int t = 0; t < my_tiles; ++t) {
      const long long row = static_cast<long long>(pair + t * num_pairs) * 256 + static_cast<int>(rank) * 128 + (warp & 3) * 32 + lane;
      if (!mbar_wait_warp(d2_full(d2_of(t)), d2_use(t) & 1, abort_flag, status, kDevTimeoutEpilogue)) break;
      tc_fence_after();
      uint16_t* out = static_cast<uint16_t*>(p.y) + row * p.d;
#pragma unroll
      for (int c = 0; c < kN2; c += 32) {
        uint32_t v[2][16];
        tmem_ld16(tmem + lanes + d2_col(t) + c, v[0]);
        tmem_ld16(tmem + lanes + d2_col(t) + c + 16, v[1]);
        tmem_ld_wait();
        if (c + 32 == kN2) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_leader(d2_empty(d2_of(t)), rank);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int col = c + i * 16;
          if (row >= p.rows || col >= p.d) continue;
          uint32_t w[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) w[j] = ff_pack<F16>(__uint_as_float(v[i][2 * j]), __uint_as_float(v[i][2 * j + 1]));
          if (col + 16 <= p.d)
            ff_store32(out + col, w);
          else
            *reinterpret_cast<uint4*>(out + col) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // neither CTA leaves while the other may still signal its barriers or read its operands
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

}  // namespace trimul
