// The gated feed-forward of any width (multiples of eight), x [M, D], W_a and W_b [H, D], W_s [D, H]:
//
//   a = x W_a^T,  b = x W_b^T,  h = act(a) b,  y = h W_s^T                        (act: SiLU, or GELU with the error function)
//   dh = dy W_s,  da = dh b act'(a),  db = dh act(a),  dx = da W_a + db W_b,  dW_a = da^T x,  dW_b = db^T x,  dW_s = dy^T h
//
// Nothing but x is kept for the backward: a and b are formed again (16 M D H multiply-adds in all instead of 12, against two
// tensors [M, H] written and read, and their rounding). Five products on the tensor cores (fp32 accumulators in tensor memory), by
// one kernel template; what is between two products of a row is done in the first one's epilogue, on the accumulators:
//
//   kFfUp       a | b side by side in one accumulator, h leaves              K = D
//   kFfDown     y = h W_s^T                                                   K = H
//   kFfHidden   dh, and a | b again: da, db and h leave                       K = D, D
//   kFfInput    dx = da W_a + db W_b, one accumulator over both               K = H, H
//   kFfWeights  dW_a, dW_b and dW_s^T = h^T dy: three products of one shape, the rows (K = M) split over the CTAs; fp32 partials
//
// Operands as they lie in memory: the weights' other orientation and the rows-as-K operands are read MN-major, so nothing is
// transposed. h, da and db are rounded to the type of x (saturating for fp16), each once, as operands of 16-bit products have to be.
// The structure is the contraction's: persistent CTAs (pairs for large products: 256-row tiles, each CTA supplies its rows of the
// first operand and half of the second), one warp loads through TMA, one issues the MMAs, the others are the epilogue of the tile
// before. All waits are bounded; one that gives up leaves a code in blocks_status.
#pragma once

#include "blocks_status.cuh"
#include "ptx.cuh"

namespace trimul {

enum FfOp : int { kFfUp = 0, kFfDown = 1, kFfHidden = 2, kFfInput = 3, kFfWeights = 4 };
enum FfAct : int { kFfSilu = 0, kFfGelu = 1 };

struct FfMaps {
  CUtensorMap a[3];
  CUtensorMap b[3];
};

struct FfParams {
  void* out[3];        // h | y | da, db, h | dx | dW_a, dW_b, dW_s (kFfWeights with one part; null: not asked for)
  float* partial;      // kFfWeights with several: [splits][3][rows][cols]
  long long ld;        // elements from one row of `out` to the next
  int rows, cols;      // of the output
  int m_tiles, n_tiles;
  int kb, kb_second;   // 64-deep k blocks of the first and of the second segment
  int bn;              // accumulator columns of an output tile (kFfUp and kFfHidden: of its a | b part)
  int splits, kb_split;  // kFfWeights: parts of the k range, k blocks of each
  int type;            // kFfWeights: of `out`, 0 bf16, 1 fp32, 2 fp16
};

constexpr int kFfStages = 6;
constexpr int kFfStageBytes = 32768;  // 128 rows of the first operand, up to 128 of the second, 64 deep
constexpr int kFfEpilogueWarps = 16;
constexpr int kFfThreads = 64 + 32 * kFfEpilogueWarps;
constexpr int kFfSmemBytes = kFfStages * kFfStageBytes + 256 + 1024;

template <bool F16>
__device__ __forceinline__ uint32_t ff_pack(float a, float b) {
  return F16 ? pack_f16x2_sat(make_float2(a, b)) : pack_bf16x2(a, b);
}

__device__ __forceinline__ float2 ff_f2(float v) { return make_float2(v, v); }
// 1 / (1 + 2^(-a log2 e)) of two values with one reciprocal, of the product of the two denominators (the special-function unit, four
// lanes a clock, is what an epilogue of few products waits for). The exponent is held below 64, so that the product stays finite:
// sigmoid(a) is 2^-63 for a < -43, off by less than 1e-19.
__device__ __forceinline__ float2 ff_sigmoid2(float2 a) {
  const float2 n = __fmul2_rn(a, ff_f2(-1.44269504f));
  float2 x;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(x.x) : "f"(fminf(n.x, 63.f)));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(x.y) : "f"(fminf(n.y, 63.f)));
  x = __fadd2_rn(x, ff_f2(1.f));
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x.x * x.y));
  return __fmul2_rn(ff_f2(r), make_float2(x.y, x.x));
}
// Values of 16 neighbouring units: act(a) b
__device__ __forceinline__ void ff_gate16(const uint32_t (&a)[16], const uint32_t (&b)[16], int act, float (&h)[16]) {
  if (act == kFfSilu) {
#pragma unroll
    for (int j = 0; j < 16; j += 2) {
      const float2 va = make_float2(__uint_as_float(a[j]), __uint_as_float(a[j + 1])), vb = make_float2(__uint_as_float(b[j]), __uint_as_float(b[j + 1]));
      const float2 r = __fmul2_rn(__fmul2_rn(va, ff_sigmoid2(va)), vb);
      h[j] = r.x;
      h[j + 1] = r.y;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float v = __uint_as_float(a[j]);
      h[j] = 0.5f * v * (1.0f + erff(v * 0.70710678f)) * __uint_as_float(b[j]);
    }
  }
}
// ... and of the backward: dh b act'(a), dh act(a), act(a) b
__device__ __forceinline__ void ff_gate_back16(const uint32_t (&a)[16], const uint32_t (&b)[16], const uint32_t (&d)[16], int act, float (&da)[16],
                                               float (&db)[16], float (&h)[16]) {
#pragma unroll
  for (int j = 0; j < 16; j += 2) {
    const float2 va = make_float2(__uint_as_float(a[j]), __uint_as_float(a[j + 1])), vb = make_float2(__uint_as_float(b[j]), __uint_as_float(b[j + 1]));
    const float2 vd = make_float2(__uint_as_float(d[j]), __uint_as_float(d[j + 1]));
    float2 f, slope;
    if (act == kFfSilu) {
      const float2 s = ff_sigmoid2(va);
      f = __fmul2_rn(va, s);
      slope = __ffma2_rn(f, __fadd2_rn(ff_f2(1.f), make_float2(-s.x, -s.y)), s);  // s (1 + a (1 - s))
    } else {
      const float2 cdf = make_float2(0.5f * (1.0f + erff(va.x * 0.70710678f)), 0.5f * (1.0f + erff(va.y * 0.70710678f)));
      f = __fmul2_rn(va, cdf);
      slope = make_float2(fmaf(va.x * 0.39894228f, __expf(-0.5f * va.x * va.x), cdf.x), fmaf(va.y * 0.39894228f, __expf(-0.5f * va.y * va.y), cdf.y));
    }
    const float2 x = __fmul2_rn(__fmul2_rn(vd, vb), slope), y = __fmul2_rn(vd, f), z = __fmul2_rn(f, vb);
    da[j] = x.x;
    da[j + 1] = x.y;
    db[j] = y.x;
    db[j + 1] = y.y;
    h[j] = z.x;
    h[j + 1] = z.y;
  }
}

// 32 bytes in one request where the address allows: whole sectors of L2 (in halves a tile's stores took twice as long)
__device__ __forceinline__ void ff_store32(void* p, const uint32_t (&w)[8]) {
  if ((reinterpret_cast<uintptr_t>(p) & 31u) == 0) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]),
                 "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
  } else {
    reinterpret_cast<uint4*>(p)[0] = make_uint4(w[0], w[1], w[2], w[3]);
    reinterpret_cast<uint4*>(p)[1] = make_uint4(w[4], w[5], w[6], w[7]);
  }
}
__device__ __forceinline__ void ff_put(void* out, size_t i, float v, int type) {
  if (type == 1)
    static_cast<float*>(out)[i] = v;
  else if (type == 0)
    static_cast<__nv_bfloat16*>(out)[i] = __float2bfloat16_rn(v);
  else
    static_cast<__half*>(out)[i] = __float2half_rn(v);
}
// 16 neighbours of a row, those before `left` (a multiple of 8)
__device__ __forceinline__ void ff_put16(void* out, size_t i, const float (&v)[16], int left, int type) {
#pragma unroll
  for (int j = 0; j < 16; j += 8) {
    if (j >= left) break;
    if (type == 1) {
      uint32_t w[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) w[k] = __float_as_uint(v[j + k]);
      ff_store32(static_cast<float*>(out) + i + j, w);
    } else {
      uint32_t w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = type == 0 ? pack_bf16x2(v[j + 2 * k], v[j + 2 * k + 1]) : pack_f16x2(make_float2(v[j + 2 * k], v[j + 2 * k + 1]));
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + i + j) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

template <int OP, bool PAIR, bool F16, int ACT>
__global__ void __launch_bounds__(kFfThreads, 1) ff_kernel(const __grid_constant__ FfMaps maps, const FfParams p) {
  constexpr int S = kFfStages;
  constexpr bool A_MN = OP == kFfWeights;
  constexpr bool SECOND = OP == kFfHidden || OP == kFfInput;  // two segments of k
  constexpr int G = PAIR ? 2 : 1;                              // CTAs of a tile
  constexpr int kUnits = PAIR ? 128 : 64;                      // hidden units of a tile (kFfUp, kFfHidden)
  constexpr uint32_t kAcc = OP == kFfHidden ? kUnits : (PAIR ? 256 : 128);  // columns from one of the two accumulators to the other
  constexpr uint32_t kAcc0 = OP == kFfHidden ? 2 * kUnits : 0;  // (kFfHidden: a | b first, then dh of even and odd tiles)
  constexpr uint32_t kTmemCols = PAIR ? 512 : 256;

  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t bar_base = base + S * kFfStageBytes;
  auto full = [&](int s) { return bar_base + 8u * s; };
  auto empty = [&](int s) { return bar_base + 8u * (S + s); };
  auto acc_full = [&](int a) { return bar_base + 8u * (2 * S + a); };
  auto acc_empty = [&](int a) { return bar_base + 8u * (2 * S + 2 + a); };
  const uint32_t ab_empty = bar_base + 8u * (2 * S + 4);  // kFfHidden: a | b are in registers
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem_raw + (bar_base - smem_u32(smem_raw)) + 8 * (2 * S + 5));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? cluster_ctarank() : 0;
  const int first = PAIR ? blockIdx.x >> 1 : blockIdx.x, step = PAIR ? gridDim.x >> 1 : gridDim.x;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(acc_full(a), 1);
      mbar_init(acc_empty(a), kFfEpilogueWarps * G);
    }
    mbar_init(ab_empty, kFfEpilogueWarps * G);
    *abort_flag = 0;
    fence_mbar_init();
    for (int i = 0; i < 3; ++i) {
      if (i == 0 || OP == kFfWeights || (i == 1 && SECOND)) prefetch_tmap(&maps.a[i]);
      if (i == 0 || OP == kFfHidden || (i == 1 && OP != kFfDown)) prefetch_tmap(&maps.b[i]);
    }
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      tmem_alloc_pair(smem_u32(tmem_slot), kTmemCols);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(smem_u32(tmem_slot), kTmemCols);
      tmem_relinquish();
    }
  }
  grid_dependency_wait();
  grid_dependents_launch();
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync_all();  // barriers of both CTAs are initialised before any signal crosses
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  const int per_split = p.m_tiles * p.n_tiles * (OP == kFfWeights ? 3 : 1);
  const int tiles = per_split * p.splits;
  struct Tile {
    int split, product, m, n, kb0, kb1;
  };
  // the second operand's tiles run fastest (they share the rows of the first), the parts of a split k range slowest (tiles in
  // flight read the same rows)
  auto tile_at = [&](int i) {
    Tile t;
    t.split = OP == kFfWeights ? i / per_split : 0;
    i -= t.split * per_split;
    t.n = i % p.n_tiles;
    i /= p.n_tiles;
    t.m = i % p.m_tiles;
    t.product = i / p.m_tiles;
    t.kb0 = OP == kFfWeights ? t.split * p.kb_split : 0;
    t.kb1 = OP == kFfWeights ? min(p.kb, t.kb0 + p.kb_split) : p.kb + (SECOND ? p.kb_second : 0);
    return t;
  };

  if (warp == 0) {
    // ------------------------------------------------------------ loads (both CTAs of a pair)
    if (lane == 0) {
      int s = 0, issued = 0;
      uint32_t ph = 0;
      bool ok = true;
      const int bn_cta = p.bn / G;
      for (int i = first; ok && i < tiles; i += step) {
        const Tile t = tile_at(i);
        const int m0 = (t.m * G + static_cast<int>(rank)) * 128;
        for (int kb = t.kb0; kb < t.kb1; ++kb) {
          if (!mbar_wait(empty(s), ph ^ 1u, abort_flag, &blocks_status, kDevTimeoutProducer)) {
            ok = false;
            break;
          }
          const bool second = SECOND && kb >= p.kb;
          const int k0 = (second ? kb - p.kb : kb) * 64;
          // kFfHidden: first dh (half as many columns), then a | b
          const int cols = OP == kFfHidden && !second ? bn_cta / 2 : bn_cta;
          if (rank == 0) mbar_arrive_expect_tx(full(s), G * (16384u + cols * 128u));
          const uint32_t sa = base + s * kFfStageBytes, sb = sa + 16384;
          auto load = [&](uint32_t dst, const CUtensorMap* m, int c0, int c1) {
            if constexpr (PAIR)
              tma_load_2d_pair(dst, m, map_to_cta(full(s), 0), c0, c1);
            else
              tma_load_2d(dst, m, full(s), c0, c1);
          };
          if constexpr (A_MN) {
            load(sa, &maps.a[t.product], m0, k0);
            load(sa + 8192, &maps.a[t.product], m0 + 64, k0);
          } else {
            load(sa, &maps.a[second ? 1 : 0], k0, m0);
          }
          if constexpr (OP == kFfUp) {
            if constexpr (PAIR) {
              load(sb, &maps.b[rank], k0, t.n * kUnits);
            } else {
              load(sb, &maps.b[0], k0, t.n * kUnits);
              load(sb + 8192, &maps.b[1], k0, t.n * kUnits);
            }
          } else if constexpr (OP == kFfDown) {
            load(sb, &maps.b[0], k0, t.n * p.bn + static_cast<int>(rank) * bn_cta);
          } else if constexpr (OP == kFfHidden) {
            if (!second) {
              load(sb, &maps.b[2], t.n * kUnits + static_cast<int>(rank) * 64, k0);
            } else if constexpr (PAIR) {
              load(sb, &maps.b[rank], k0, t.n * kUnits);
            } else {
              load(sb, &maps.b[0], k0, t.n * kUnits);
              load(sb + 8192, &maps.b[1], k0, t.n * kUnits);
            }
          } else {
            const CUtensorMap* m = OP == kFfInput ? &maps.b[second ? 1 : 0] : &maps.b[t.product == 2 ? 1 : 0];
            const int n0 = t.n * p.bn + static_cast<int>(rank) * bn_cta;
            for (int c = 0; c < bn_cta; c += 64) load(sb + c * 128, m, n0 + c, k0);
          }
          ++issued;
          if (++s == S) {
            s = 0;
            ph ^= 1u;
          }
        }
      }
      // every copy that was started lands before the CTA may exit (a pair's leader counts the bytes of both CTAs; the closing
      // cluster barrier keeps the other one)
      if (rank == 0) {
        const int pending = issued < S ? issued : S;
        for (int q = 0; q < pending; ++q) {
          if (s == 0) {
            s = S;
            ph ^= 1u;
          }
          --s;
          const long long t0 = clock64();
          while (!mbar_try_wait(full(s), ph)) {
            if (*abort_flag != 0 || clock64() - t0 > kWaitLimitCycles) {
              atomicCAS(&blocks_status, 0, kDevTimeoutDrain);
              break;
            }
          }
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMAs (the pair's leader)
    if (rank == 0 && elect_one()) {
      int s = 0, it = 0;
      uint32_t ph = 0;
      bool ok = true;
      const uint32_t fmt = F16 ? kFmtF16 : kFmtBF16;
      for (int i = first; ok && i < tiles; i += step, ++it) {
        const Tile t = tile_at(i);
        const int acc = it & 1;
        if (!mbar_wait(acc_empty(acc), ((it >> 1) & 1) ^ 1u, abort_flag, &blocks_status, kDevTimeoutMma)) break;
        tc_fence_after();
        for (int kb = t.kb0; kb < t.kb1; ++kb) {
          const bool second = SECOND && kb >= p.kb;
          if (OP == kFfHidden && kb == p.kb) {
            if (!mbar_wait(ab_empty, (it & 1) ^ 1u, abort_flag, &blocks_status, kDevTimeoutMma)) {
              ok = false;
              break;
            }
          }
          if (!mbar_wait(full(s), ph, abort_flag, &blocks_status, kDevTimeoutMma)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sa = base + s * kFfStageBytes, sb = sa + 16384;
          const bool b_mn = OP == kFfInput || OP == kFfWeights || (OP == kFfHidden && !second);
          const int n = OP == kFfHidden && !second ? p.bn / 2 : p.bn;
          const uint32_t idesc = umma_idesc(128 * G, n, A_MN, b_mn, fmt, fmt);
          const uint32_t d = OP == kFfHidden && second ? tmem : tmem + kAcc0 + acc * kAcc;
          const uint64_t da = A_MN ? umma_desc_mnmajor(sa, 8192) : umma_desc_kmajor(sa);
          const uint64_t db = b_mn ? umma_desc_mnmajor(sb, 8192) : umma_desc_kmajor(sb);
          const uint32_t ka = A_MN ? 128 : 2, kn = b_mn ? 128 : 2;  // 16-byte units per 16 of k
          const bool fresh = OP == kFfHidden ? kb == 0 || kb == p.kb : kb == t.kb0;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t more = fresh && k == 0 ? 0u : 1u;
            if constexpr (PAIR)
              umma_pair(d, da + k * ka, db + k * kn, idesc, more);
            else
              umma_bf16(d, da + k * ka, db + k * kn, idesc, more);
          }
          if constexpr (PAIR)
            umma_commit_pair(empty(s));
          else
            umma_commit(empty(s));
          if (++s == S) {
            s = 0;
            ph ^= 1u;
          }
        }
        if (ok) {
          if constexpr (PAIR)
            umma_commit_pair(acc_full(acc));
          else
            umma_commit(acc_full(acc));
        }
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue: a row per thread, a quarter of the tile's columns per
    // group of four warps. All of a thread's accumulators are read at once and handed back before the arithmetic (kFfHidden: those
    // of a and b, of which there is one set; dh has two).
    const int q = warp & 3, part = (warp - 2) >> 2;
    const uint32_t lanes = static_cast<uint32_t>(q * 32) << 16;
    int it = 0;
    for (int i = first; i < tiles; i += step, ++it) {
      const Tile t = tile_at(i);
      const int acc = it & 1;
      const int row = (t.m * G + static_cast<int>(rank)) * 128 + q * 32 + lane;
      const bool in = row < p.rows;
      if (!mbar_wait_warp(acc_full(acc), (it >> 1) & 1, abort_flag, &blocks_status, kDevTimeoutEpilogue)) break;
      tc_fence_after();
      auto release = [&](uint32_t bar) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (PAIR)
            mbar_arrive_leader(bar, rank);
          else
            mbar_arrive(bar);
        }
      };
      // 16 neighbours of a row of the output (multiples of 8 of them within the width)
      auto store16 = [&](void* out, int col, const float (&v)[16]) {
        if (!in || col >= p.cols) return;
        uint16_t* o = static_cast<uint16_t*>(out) + static_cast<size_t>(row) * p.ld + col;
        uint32_t w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = ff_pack<F16>(v[2 * j], v[2 * j + 1]);
        if (col + 16 <= p.cols)
          ff_store32(o, w);
        else
          *reinterpret_cast<uint4*>(o) = make_uint4(w[0], w[1], w[2], w[3]);
      };
      const uint32_t d = tmem + lanes + kAcc0 + acc * kAcc;
      if constexpr (OP == kFfUp || OP == kFfHidden) {
        constexpr int N = kUnits / 4;
        const uint32_t ab = (OP == kFfUp ? d : tmem + lanes) + part * N;
        uint32_t va[N / 16][16], vb[N / 16][16];
#pragma unroll
        for (int c = 0; c < N / 16; ++c) {
          tmem_ld16(ab + c * 16, va[c]);
          tmem_ld16(ab + kUnits + c * 16, vb[c]);
        }
        tmem_ld_wait();
        release(OP == kFfUp ? acc_empty(acc) : ab_empty);
#pragma unroll
        for (int c = 0; c < N / 16; ++c) {
          const int col = t.n * kUnits + part * N + c * 16;
          if constexpr (OP == kFfUp) {
            float v[16];
            ff_gate16(va[c], vb[c], ACT, v);
            store16(p.out[0], col, v);
          } else {
            uint32_t vd[16];
            tmem_ld16(d + part * N + c * 16, vd);
            tmem_ld_wait();
            if (c == N / 16 - 1) release(acc_empty(acc));
            float da[16], db[16], h[16];
            ff_gate_back16(va[c], vb[c], vd, ACT, da, db, h);
            store16(p.out[0], col, da);
            store16(p.out[1], col, db);
            store16(p.out[2], col, h);
          }
        }
      } else {
        const int n = p.bn / 4;
#pragma unroll 1
        for (int c = 0; c < n; c += 16) {
          uint32_t v[16];
          tmem_ld16(d + part * n + c, v);
          tmem_ld_wait();
          if (c + 16 >= n) release(acc_empty(acc));
          const int col = t.n * p.bn + part * n + c;
          float f[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) f[j] = __uint_as_float(v[j]);
          if constexpr (OP != kFfWeights) {
            store16(p.out[0], col, f);
          } else if (in && col < p.cols) {
            const int left = p.cols - col;
            if (p.partial != nullptr) {
              ff_put16(p.partial, ((static_cast<size_t>(t.split) * 3 + t.product) * p.rows + row) * p.cols + col, f, left, 1);
            } else if (void* const o = t.product == 0 ? p.out[0] : t.product == 1 ? p.out[1] : p.out[2]; o != nullptr) {
              if (t.product < 2) {
                ff_put16(o, static_cast<size_t>(row) * p.cols + col, f, left, p.type);
              } else {  // dW_s [D, H]: neighbouring lanes are neighbours in memory
#pragma unroll
                for (int j = 0; j < 16; ++j)
                  if (j < left) ff_put(o, static_cast<size_t>(col + j) * p.rows + row, f[j], p.type);
              }
            }
          }
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync_all();  // neither CTA leaves while the other may still signal its barriers or read its operands
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    if constexpr (PAIR)
      tmem_dealloc_pair(tmem, kTmemCols);
    else
      tmem_dealloc(tmem, kTmemCols);
  }
}

// Sums the parts of the weight gradients in the order of the rows and rounds once: dW_a, dW_b [H, D] as they lie, dW_s [D, H] from
// its transpose (through shared memory). A block takes 32 x 128 values of one product.
struct FfReduce {
  const float* partial;  // [splits][3][H][D]
  void* out[3];
  int splits, H, D;
  int type;  // 0 bf16, 1 fp32, 2 fp16
};
__global__ void __launch_bounds__(256) ff_reduce_kernel(const FfReduce p) {
  __shared__ float tile[32][129];
  grid_dependency_wait();
  grid_dependents_launch();
  void* out = blockIdx.z == 0 ? p.out[0] : blockIdx.z == 1 ? p.out[1] : p.out[2];
  if (out == nullptr) return;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int c = blockIdx.x * 128 + tx * 4;
  const size_t part = static_cast<size_t>(3) * p.H * p.D;
  float4 a[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) a[j] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k = 0; k < p.splits; ++k) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = blockIdx.y * 32 + ty + 8 * j;
      if (r >= p.H || c >= p.D) continue;
      const float4 v = __ldcg(reinterpret_cast<const float4*>(p.partial + k * part + (static_cast<size_t>(blockIdx.z) * p.H + r) * p.D + c));
      a[j].x += v.x;
      a[j].y += v.y;
      a[j].z += v.z;
      a[j].w += v.w;
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int r = blockIdx.y * 32 + ty + 8 * j;
    if (blockIdx.z < 2) {
      if (r >= p.H || c >= p.D) continue;
      const size_t i = static_cast<size_t>(r) * p.D + c;
      if (p.type == 1)
        reinterpret_cast<float4*>(static_cast<float*>(out) + i)[0] = a[j];
      else if (p.type == 0)
        reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + i)[0] = make_uint2(pack_bf16x2(a[j].x, a[j].y), pack_bf16x2(a[j].z, a[j].w));
      else
        reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + i)[0] =
            make_uint2(pack_f16x2(make_float2(a[j].x, a[j].y)), pack_f16x2(make_float2(a[j].z, a[j].w)));
    } else {
      float* s = &tile[ty + 8 * j][tx * 4];
      s[0] = a[j].x;
      s[1] = a[j].y;
      s[2] = a[j].z;
      s[3] = a[j].w;
    }
  }
  if (blockIdx.z < 2) return;
  __syncthreads();
  const int h = blockIdx.y * 32 + tx;
  for (int j = ty; j < 128; j += 8) {
    const int d = blockIdx.x * 128 + j;
    if (d < p.D && h < p.H) ff_put(out, static_cast<size_t>(d) * p.H + h, tile[tx][j], p.type);
  }
}

// fp32 master weights as operands (the type of x, saturating for fp16)
__global__ void __launch_bounds__(256) ff_cast_kernel(const float* a, const float* b, const float* s, uint4* out, long long n8, int f16) {
  grid_dependency_wait();
  grid_dependents_launch();
  for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < 3 * n8; i += static_cast<long long>(gridDim.x) * 256) {
    const int which = static_cast<int>(i / n8);
    const float4* w = reinterpret_cast<const float4*>((which == 0 ? a : which == 1 ? b : s) + (i - which * n8) * 8);
    const float4 u = __ldcg(w), v = __ldcg(w + 1);
    out[i] = f16 ? make_uint4(ff_pack<true>(u.x, u.y), ff_pack<true>(u.z, u.w), ff_pack<true>(v.x, v.y), ff_pack<true>(v.z, v.w))
                 : make_uint4(ff_pack<false>(u.x, u.y), ff_pack<false>(u.z, u.w), ff_pack<false>(v.x, v.y), ff_pack<false>(v.z, v.w));
  }
}

}  // namespace trimul
