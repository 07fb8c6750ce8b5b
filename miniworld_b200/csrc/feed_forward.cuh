// The gated feed-forward of any width (multiples of eight), x [M, D], W_a and W_b [H, D], W_s [D, H]:
//
//   a = x W_a^T,  b = x W_b^T,  h = act(a) b,  y = h W_s^T                        (act: SiLU, or GELU with the error function)
//   dh = dy W_s,  da = dh b act'(a),  db = dh act(a),  dx = da W_a + db W_b,  dW_a = da^T x,  dW_b = db^T x,  dW_s = dy^T h
//
// The backward forms a and b again from x (16 M D H multiply-adds in all instead of 12), or, where that costs more than writing and
// reading them (D >= 512 and many rows: the caller then keeps a buffer), takes them from the forward, as fp16 values with a power of two
// for 16 neighbours (10 to 11 bits of their values over fp32's range, see ff_keep16: kept in bf16 they would add more to the gradients'
// error than all other roundings, and plain fp16 loses what lies beyond its range). The products run on the tensor cores (fp32
// accumulators in tensor memory), by one kernel template; what is between two products of a row is done in the first one's epilogue, on
// the accumulators:
//
//   kFfUp       a | b side by side in one accumulator, h leaves              K = D
//   kFfDown     y = h W_s^T                                                   K = H
//   kFfHidden   dh, and a | b again: da, db and h leave                       K = D, D
//   kFfInput    dx = da W_a + db W_b, one accumulator over both               K = H, H
//   kFfGrad     dh with a and b from the forward: da and db leave             K = D
//   kFfWeights  dW_a, dW_b and dW_s^T = h^T dy: three products of one shape, the rows (K = M) split over the CTAs; fp32 partials
//
// Operands as they lie in memory: the weights' other orientation and the rows-as-K operands are read MN-major, so nothing is
// transposed. h, da and db are rounded to the type of x, each once, as operands of 16-bit products have to be (a finite h stays within fp16;
// da, db and the results go to infinity beyond it).
// The structure is the contraction's: persistent CTAs (pairs for large products: 256-row tiles, each CTA supplies its rows of the
// first operand and half of the second), one warp loads through TMA, one issues the MMAs, the others are the epilogue of the tile
// before. All waits are bounded; one that gives up leaves a code in blocks_status.
// M, D, H = 16384, 1024, 4096, bf16, each alone: up 168 us (204 with a and b kept), down 98, grad 145, input 191, weights 300, that is 1.64,
// 1.40, 0.95, 1.44 and 1.37 PFLOP/s (cuBLAS 8192^3: 1.64); forming a and b again (kFfHidden) 395 instead of grad's 145. The 256 x 256
// tiles wait for their loads (stamps: 610 to 730 cycles for a k block of 512 cycles of products).
#pragma once

#include "blocks_status.cuh"
#include "ptx.cuh"

namespace trimul {

enum FfOp : int { kFfUp = 0, kFfDown = 1, kFfHidden = 2, kFfInput = 3, kFfWeights = 4, kFfGrad = 5 };
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
  int splits, kb_split;  // kFfWeights, SPLIT: parts of the k range, k blocks of each
  const void* kept[2]; // kFfGrad: a and b of the forward, fp16: see ff_kept_at
  void* keep[2];       // kFfUp: where to leave them, or null
  int type;            // kFfWeights: of `out`, 0 bf16, 1 fp32, 2 fp16
};

constexpr int kFfStages = 6;
constexpr int kFfStageBytes = 32768;  // 128 rows of the first operand, up to 128 of the second, 64 deep
constexpr int kFfEpilogueWarps = 16;
constexpr int kFfThreads = 64 + 32 * kFfEpilogueWarps;
constexpr int kFfBoxBytes = 2048;     // 32 x 32 values of an output; one for each epilogue warp
constexpr int kFfSmemBytes = kFfStages * kFfStageBytes + kFfEpilogueWarps * kFfBoxBytes + 256 + 1024;

// Two values of a result, or of da and db: beyond fp16 they are infinite, so that gradients formed from them say so
template <bool F16>
__device__ __forceinline__ uint32_t ff_pack(float a, float b) {
  return F16 ? pack_f16x2(make_float2(a, b)) : pack_bf16x2(a, b);
}
// Two values of h, an operand whose finite ones stay within fp16: those beyond become +-65504, infinite ones stay. (v 2^-112 is below the
// half of a step there for a finite h, |h| < 2^104: 2^52 for each of a and b from fp16 rows of 2^20 elements.)
template <bool F16>
__device__ __forceinline__ uint32_t ff_pack_held(float a, float b) {
  if (!F16) return pack_bf16x2(a, b);
  const float2 v = make_float2(a, b);
  uint32_t r;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(pack_f16x2_sat(v)), "r"(pack_f16x2(__fmul2_rn(v, make_float2(0x1p-112f, 0x1p-112f)))));
  return r;
}

__device__ __forceinline__ float2 ff_f2(float v) { return make_float2(v, v); }
// 1 / (1 + 2^(-a log2 e)) of four values with one reciprocal, of the product of the four denominators (the special-function unit, four
// lanes a clock and scheduler, is what an epilogue of few products waits for). OPEN: all are numbers from kFfOpen on, and the product is
// finite. Otherwise the exponents are held below 31 for it, and where they were beyond, a < -21.5, the result is zero (it is less than
// 5e-10 there: a sigmoid(a) is off by 1e-8 at most, for any a). Which of the two is settled for 16 values of a warp's rows at a time:
// with the limits in every value 196608 x 64 x 256 took 33.2 us and the hidden gradients of 119736 x 120 x 320 20 us more.
constexpr float kFfOpen = -21.f;
template <bool OPEN>
__device__ __forceinline__ void ff_sigmoid4(float2 a, float2 b, float2& sa, float2& sb) {
  const float2 m = __fmul2_rn(a, ff_f2(-1.44269504f)), n = __fmul2_rn(b, ff_f2(-1.44269504f));
  const auto held = [](float v) { return OPEN ? v : fminf(v, 31.f); };
  float2 x, y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(x.x) : "f"(held(m.x)));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(x.y) : "f"(held(m.y)));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y.x) : "f"(held(n.x)));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y.y) : "f"(held(n.y)));
  x = __fadd2_rn(x, ff_f2(1.f));
  y = __fadd2_rn(y, ff_f2(1.f));
  const float px = x.x * x.y, py = y.x * y.y;
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(px * py));
  sa = __fmul2_rn(ff_f2(r * py), make_float2(x.y, x.x));
  sb = __fmul2_rn(ff_f2(r * px), make_float2(y.y, y.x));
  if (!OPEN) {
    sa = make_float2(m.x >= 31.f ? 0.f : sa.x, m.y >= 31.f ? 0.f : sa.y);
    sb = make_float2(n.x >= 31.f ? 0.f : sb.x, n.y >= 31.f ? 0.f : sb.y);
  }
}
// The least of three, NaN if one of them is
__device__ __forceinline__ float ff_least(float a, float b, float c) {
  float r;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// Whether the whole warp's values are open (GELU asks for nothing)
__device__ __forceinline__ bool ff_open(const uint32_t (&a)[16], int act) {
  if (act != kFfSilu) return true;
  float v = __uint_as_float(a[0]);
#pragma unroll
  for (int j = 1; j < 15; j += 2) v = ff_least(v, __uint_as_float(a[j]), __uint_as_float(a[j + 1]));
  v = ff_least(v, __uint_as_float(a[15]), 0.f);
  return __all_sync(0xFFFFFFFFu, v >= kFfOpen);
}
// The normal distribution's function and e^(-a^2 / 2) of four values: with z = |a| / sqrt 2 and t = 1 / (1 + 0.3275911 z),
// erfc(z) = (c1 t + ... + c5 t^5) e^(-z^2) to 1.5e-7 (Abramowitz and Stegun, Handbook of Mathematical Functions, 7.1.26), the
// reciprocals from one as above. z is held below 16, where erfc is zero in fp32.
__device__ __forceinline__ void ff_normal4(const float2 (&a)[2], float2 (&cdf)[2], float2 (&bell)[2]) {
  float2 x[2], z[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    z[k] = make_float2(fminf(fabsf(a[k].x) * 0.70710678f, 16.f), fminf(fabsf(a[k].y) * 0.70710678f, 16.f));
    x[k] = __ffma2_rn(z[k], ff_f2(0.3275911f), ff_f2(1.f));
    const float2 n = __fmul2_rn(__fmul2_rn(z[k], z[k]), ff_f2(-1.44269504f));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(bell[k].x) : "f"(n.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(bell[k].y) : "f"(n.y));
  }
  const float p0 = x[0].x * x[0].y, p1 = x[1].x * x[1].y;
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(p0 * p1));
  const float2 t[2] = {__fmul2_rn(ff_f2(r * p1), make_float2(x[0].y, x[0].x)), __fmul2_rn(ff_f2(r * p0), make_float2(x[1].y, x[1].x))};
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    float2 q = __ffma2_rn(t[k], ff_f2(0.5f * 1.061405429f), ff_f2(0.5f * -1.453152027f));
    q = __ffma2_rn(q, t[k], ff_f2(0.5f * 1.421413741f));
    q = __ffma2_rn(q, t[k], ff_f2(0.5f * -0.284496736f));
    q = __ffma2_rn(q, t[k], ff_f2(0.5f * 0.254829592f));
    q = __fmul2_rn(__fmul2_rn(q, t[k]), bell[k]);  // erfc(z) / 2
    cdf[k] = make_float2(a[k].x < 0.f ? q.x : 1.f - q.x, a[k].y < 0.f ? q.y : 1.f - q.y);
  }
}
__device__ __forceinline__ float2 ff_at(const uint32_t (&v)[16], int j) { return make_float2(__uint_as_float(v[j]), __uint_as_float(v[j + 1])); }
// act(a) and (where asked for) act'(a) of four values
template <bool SLOPE, bool OPEN>
__device__ __forceinline__ void ff_act4(const float2 (&a)[2], int act, float2 (&f)[2], float2 (&slope)[2]) {
  float2 s[2];
  if (act == kFfSilu) {
    ff_sigmoid4<OPEN>(a[0], a[1], s[0], s[1]);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      f[k] = __fmul2_rn(a[k], s[k]);
      if (SLOPE) slope[k] = __ffma2_rn(f[k], __fadd2_rn(ff_f2(1.f), make_float2(-s[k].x, -s[k].y)), s[k]);  // s (1 + a (1 - s))
    }
  } else {
    float2 bell[2];
    ff_normal4(a, s, bell);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      f[k] = __fmul2_rn(a[k], s[k]);
      if (SLOPE) slope[k] = __ffma2_rn(__fmul2_rn(a[k], ff_f2(0.39894228f)), bell[k], s[k]);  // cdf + a / sqrt(2 pi) e^(-a^2 / 2)
    }
  }
}
// Values of 16 neighbouring units: act(a) b
template <bool OPEN>
__device__ __forceinline__ void ff_gate16_of(const uint32_t (&a)[16], const uint32_t (&b)[16], int act, float (&h)[16]) {
#pragma unroll
  for (int j = 0; j < 16; j += 4) {
    const float2 v[2] = {ff_at(a, j), ff_at(a, j + 2)};
    float2 f[2], none[2];
    ff_act4<false, OPEN>(v, act, f, none);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float2 r = __fmul2_rn(f[k], ff_at(b, j + 2 * k));
      h[j + 2 * k] = r.x;
      h[j + 2 * k + 1] = r.y;
    }
  }
}
__device__ __forceinline__ void ff_gate16(const uint32_t (&a)[16], const uint32_t (&b)[16], int act, float (&h)[16]) {
  if (ff_open(a, act))
    ff_gate16_of<true>(a, b, act, h);
  else
    ff_gate16_of<false>(a, b, act, h);
}
// ... and of the backward: dh b act'(a), dh act(a), act(a) b
template <bool OPEN>
__device__ __forceinline__ void ff_gate_back16_of(const uint32_t (&a)[16], const uint32_t (&b)[16], const uint32_t (&d)[16], int act, float (&da)[16],
                                               float (&db)[16], float (&h)[16]) {
#pragma unroll
  for (int i = 0; i < 16; i += 4) {
    const float2 v[2] = {ff_at(a, i), ff_at(a, i + 2)};
    float2 f[2], slope[2];
    ff_act4<true, OPEN>(v, act, f, slope);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int j = i + 2 * k;
      const float2 vb = ff_at(b, j), vd = ff_at(d, j);
      const float2 x = __fmul2_rn(__fmul2_rn(vd, vb), slope[k]), y = __fmul2_rn(vd, f[k]), z = __fmul2_rn(f[k], vb);
      da[j] = x.x;
      da[j + 1] = x.y;
      db[j] = y.x;
      db[j + 1] = y.y;
      h[j] = z.x;
      h[j + 1] = z.y;
    }
  }
}
__device__ __forceinline__ void ff_gate_back16(const uint32_t (&a)[16], const uint32_t (&b)[16], const uint32_t (&d)[16], int act, float (&da)[16],
                                               float (&db)[16], float (&h)[16]) {
  if (ff_open(a, act))
    ff_gate_back16_of<true>(a, b, d, act, da, db, h);
  else
    ff_gate_back16_of<false>(a, b, d, act, da, db, h);
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

// Where the forward leaves a row's 16 neighbours of a or b for the backward: a warp's 32 rows of them lie together (1 KB), since the
// same threads hold them in both passes and no product reads them.
__device__ __forceinline__ size_t ff_kept_at(int row, int col, long long ld) {
  return (static_cast<size_t>(row >> 5) * (ld >> 4) + (col >> 4)) * 512 + (row & 31) * 16;
}
template <bool F16>
__device__ __forceinline__ void ff_pack16(const float (&v)[16], uint32_t (&w)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) w[j] = ff_pack<F16>(v[2 * j], v[2 * j + 1]);
}
// ... of h. (0 times each value adds up to a NaN where one is not finite: half an instruction a value instead of ff_pack_held's three a pair)
template <bool F16>
__device__ __forceinline__ void ff_pack16_held(const float (&v)[16], uint32_t (&w)[8]) {
  ff_pack16<F16>(v, w);
  if constexpr (F16) {
    uint32_t z = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) asm("fma.rn.f16x2 %0, %1, %2, %0;" : "+r"(z) : "r"(w[j]), "r"(0u));
    if ((z & 0x7FFF7FFFu) != 0) {
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = ff_pack_held<true>(v[2 * j], v[2 * j + 1]);
    }
  }
}
// 16 values in 32 bytes (p on such a boundary) that keep the range of fp32: fp16 values times 2^(138 - 4 q), q = E / 4 (at least 3) for the
// exponent field E of the largest finite one, which so lies in [2^11, 2^15). The six bits of q are the last bits of the first six
// values, which are rounded to 10 bits for it (Veltkamp's splitting: x C - (x C - x) with C = 2^14 + 1; Dekker, Numerische Mathematik 18,
// 1971); the others have 11. Both hold down to 2^-25 of the largest of the 16; what is smaller is a multiple of 2^-35 of it (2^-34 among
// the first six). An infinite value stays infinite or becomes a NaN.
__device__ __forceinline__ void ff_keep16(__half* p, const uint32_t (&v)[16]) {
  float most = 0.f;
#pragma unroll
  for (int j = 0; j < 16; ++j) most = fmaxf(most, fabsf(__uint_as_float(v[j])));  // (a NaN is left out)
  if (__float_as_uint(most) == 0x7F800000u) {
    most = 0.f;
#pragma unroll
    for (int j = 0; j < 16; ++j) most = fmaxf(most, (v[j] & 0x7FFFFFFFu) == 0x7F800000u ? 0.f : fabsf(__uint_as_float(v[j])));
  }
  const uint32_t q = max(__float_as_uint(most) >> 25, 3u);
  const float2 scale = ff_f2(__uint_as_float((265u - 4u * q) << 23));
  uint32_t w[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    float2 x = __fmul2_rn(ff_at(v, 2 * j), scale);
    if (j < 3) {
      const float2 c = __fmul2_rn(x, ff_f2(16385.f)), n = make_float2(-c.x, -c.y);
      x = __fadd2_rn(c, __fadd2_rn(x, n));
    }
    w[j] = pack_f16x2(x);
    if (j < 3) w[j] = (w[j] & 0xFFFEFFFEu) | (q >> 2 * j & 1u) | (q >> (2 * j + 1) & 1u) << 16;
  }
  ff_store32(p, w);
}
__device__ __forceinline__ void ff_kept16(const uint4 (&w)[2], uint32_t (&v)[16]) {
  uint32_t h[8] = {w[0].x, w[0].y, w[0].z, w[0].w, w[1].x, w[1].y, w[1].z, w[1].w};
  uint32_t q = 0;
#pragma unroll
  for (int j = 0; j < 3; ++j) {
    q |= (h[j] & 1u) << 2 * j | (h[j] >> 16 & 1u) << (2 * j + 1);
    h[j] &= 0xFFFEFFFEu;
  }
  const float2 scale = ff_f2(__uint_as_float((4u * q - 11u) << 23));  // 2^(4 q - 138)
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float2 f = __fmul2_rn(f16x2_to_float2(h[j]), scale);
    v[2 * j] = __float_as_uint(f.x);
    v[2 * j + 1] = __float_as_uint(f.y);
  }
}

// SPLIT: the k range of an output tile over the CTAs (pairs) of a cluster, for products of few tiles and a long k. Each leaves its fp32
// tile in the (by then idle) stages, and each adds up its share of the rows over the cluster's shared memory, in the order of k.
template <int OP, bool PAIR, bool F16, int ACT, bool SPLIT>
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
  const uint32_t box_base = base + S * kFfStageBytes;
  const uint32_t bar_base = box_base + kFfEpilogueWarps * kFfBoxBytes;
  auto full = [&](int s) { return bar_base + 8u * s; };
  auto empty = [&](int s) { return bar_base + 8u * (S + s); };
  auto acc_full = [&](int a) { return bar_base + 8u * (2 * S + a); };
  auto acc_empty = [&](int a) { return bar_base + 8u * (2 * S + 2 + a); };
  const uint32_t ab_empty = bar_base + 8u * (2 * S + 4);  // kFfHidden: a | b are in registers
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem_raw + (bar_base - smem_u32(smem_raw)) + 8 * (2 * S + 5));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t cluster_rank = PAIR || SPLIT ? cluster_ctarank() : 0;
  const uint32_t rank = PAIR ? cluster_rank & 1u : 0;   // in the pair; 0 leads
  const uint32_t leader = PAIR ? cluster_rank & ~1u : cluster_rank;
  const int ctas = SPLIT ? G * p.splits : G;            // of a tile
  const int first = blockIdx.x / ctas, step = gridDim.x / ctas;

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
      if (i == 0 || OP == kFfHidden || (i == 1 && OP != kFfDown && OP != kFfGrad)) prefetch_tmap(&maps.b[i]);
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
  if constexpr (PAIR || SPLIT) cluster_sync_all();  // barriers of both CTAs are initialised before any signal crosses
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  auto commit = [&](uint32_t bar) {
    if constexpr (PAIR)
      umma_commit_mask(bar, static_cast<uint16_t>(3u << leader));
    else
      umma_commit(bar);
  };
  auto arrive = [&](uint32_t bar) {  // (a barrier of the leader's)
    if (PAIR && rank != 0)
      mbar_arrive_cluster(map_to_cta(bar, leader));
    else
      mbar_arrive(bar);
  };

  const int per_split = p.m_tiles * p.n_tiles * (OP == kFfWeights ? 3 : 1);
  const int tiles = SPLIT ? per_split : per_split * p.splits;
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
    const int kb = p.kb + (SECOND ? p.kb_second : 0);
    t.kb0 = OP == kFfWeights ? t.split * p.kb_split : SPLIT ? static_cast<int>(cluster_rank) / G * p.kb_split : 0;
    t.kb1 = OP == kFfWeights || SPLIT ? min(kb, t.kb0 + p.kb_split) : kb;
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
              tma_load_2d_pair(dst, m, map_to_cta(full(s), leader), c0, c1);
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
          const bool b_mn = OP == kFfInput || OP == kFfWeights || OP == kFfGrad || (OP == kFfHidden && !second);
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
          commit(empty(s));
          if (++s == S) {
            s = 0;
            ph ^= 1u;
          }
        }
        if (ok) commit(acc_full(acc));
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue: a row per thread, a quarter of the tile's columns per
    // group of four warps. All of a thread's accumulators are read at once and handed back before the arithmetic (kFfHidden: those
    // of a and b, of which there is one set; dh has two).
    const bool boxes = OP == kFfUp || OP == kFfHidden ? PAIR : p.bn >= 128;  // 32 columns a warp and more
    const int q = warp & 3, part = (warp - 2) >> 2;
    const uint32_t lanes = static_cast<uint32_t>(q * 32) << 16;
    int it = 0;
    for (int i = first; i < tiles; i += step, ++it) {
      const Tile t = tile_at(i);
      const int acc = it & 1;
      const int row = (t.m * G + static_cast<int>(rank)) * 128 + q * 32 + lane;
      const bool in = row < p.rows;
      // kFfGrad: the forward's a and b, a piece ahead of the accumulators
      uint4 ka[2], kb[2];
      auto kept = [&](int col) {
        ka[0] = ka[1] = kb[0] = kb[1] = make_uint4(0u, 0u, 0u, 0u);
        if (!in || col >= p.cols) return;
        const size_t at = ff_kept_at(row, col, p.ld) * 2;
        ld_gpu_chunks(reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p.kept[0]) + at), true, ka);
        ld_gpu_chunks(reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p.kept[1]) + at), true, kb);
      };
      if constexpr (OP == kFfGrad) kept(t.n * p.bn + part * (p.bn / 4));
      if (!mbar_wait_warp(acc_full(acc), (it >> 1) & 1, abort_flag, &blocks_status, kDevTimeoutEpilogue)) break;
      tc_fence_after();
      auto release = [&](uint32_t bar) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive(bar);
      };
      // 16 neighbours of a row of output `which` (multiples of 8 of them within the width). Where a warp has 32 columns and more, two calls
      // fill a box of 32 rows x 32 columns in shared memory, and the warp stores it eight rows of 64 bytes at a time: 32 lanes that
      // store to 32 rows take the load-store unit two cycles a sector, and copies of such boxes by TMA take it from the loads, whose
      // rows of 128 bytes it moves in 2.7 cycles each (that is what bounds the wide products).
      auto store16 = [&](int which, int col, const uint32_t (&w)[8]) {
        void* const out = which == 0 ? p.out[0] : which == 1 ? p.out[1] : p.out[2];
        if (boxes) {
          const uint32_t box = box_base + (warp - 2) * kFfBoxBytes, mine = box + lane * 64;
          const uint32_t c = (col >> 3) & 2, swap = (lane >> 1) & 3;  // 16-byte piece of the row's 64 bytes
          if (c == 0) __syncwarp();                                     // the box before has been read
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(mine + ((c ^ swap) << 4)), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(mine + (((c + 1) ^ swap) << 4)), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
          if (c == 0) return;
          __syncwarp();
          const int row0 = row - lane, piece = lane & 3, at = col - 16 + piece * 8;
          uint16_t* o = static_cast<uint16_t*>(out) + static_cast<size_t>(row0) * p.ld + at;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int r = j * 8 + (lane >> 2);
            uint4 v;
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(box + r * 64 + ((piece ^ ((r >> 1) & 3)) << 4)) : "memory");
            if (row0 + r < p.rows && at < p.cols) *reinterpret_cast<uint4*>(o + static_cast<size_t>(r) * p.ld) = v;
          }
          return;
        }
        if (!in || col >= p.cols) return;
        uint16_t* o = static_cast<uint16_t*>(out) + static_cast<size_t>(row) * p.ld + col;
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
        const int col = t.n * kUnits + part * N;
        if constexpr (OP == kFfUp) {
#pragma unroll
          for (int c = 0; c < N / 16; ++c) {
            float v[16];
            uint32_t w[8];
            ff_gate16(va[c], vb[c], ACT, v);
            ff_pack16_held<F16>(v, w);
            store16(0, col + c * 16, w);
            if (p.keep[0] != nullptr && in && col + c * 16 < p.cols) {
              const size_t at = ff_kept_at(row, col + c * 16, p.ld);
              ff_keep16(static_cast<__half*>(p.keep[0]) + at, va[c]);
              ff_keep16(static_cast<__half*>(p.keep[1]) + at, vb[c]);
            }
          }
        } else {
          uint32_t w[3][N / 16][8];  // da, db, h: formed together, leaving one after the other
#pragma unroll
          for (int c = 0; c < N / 16; ++c) {
            uint32_t vd[16];
            tmem_ld16(d + part * N + c * 16, vd);
            tmem_ld_wait();
            if (c == N / 16 - 1) release(acc_empty(acc));
            float da[16], db[16], h[16];
            ff_gate_back16(va[c], vb[c], vd, ACT, da, db, h);
            ff_pack16<F16>(da, w[0][c]);
            ff_pack16<F16>(db, w[1][c]);
            ff_pack16_held<F16>(h, w[2][c]);
          }
#pragma unroll
          for (int o = 0; o < 3; ++o)
#pragma unroll
            for (int c = 0; c < N / 16; ++c) store16(o, col + c * 16, w[o][c]);
        }
      } else {
        const int n = p.bn / 4;
        if constexpr (OP == kFfGrad) {
          // 32 columns at a time: da of both halves leaves, then db
#pragma unroll 1
          for (int c = 0; c < n; c += 32) {
            const int col = t.n * p.bn + part * n + c;
            uint32_t wb[2][8];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              uint32_t va[16], vb[16], v[16], wa[8];
              tmem_ld16(d + part * n + c + 16 * k, v);
              tmem_ld_wait();
              if (k == 1 && c + 32 >= n) release(acc_empty(acc));
              ff_kept16(ka, va);
              ff_kept16(kb, vb);
              if (k == 0 || c + 32 < n) kept(col + 16 * (k + 1));
              float da[16], db[16], h[16];
              ff_gate_back16(va, vb, v, ACT, da, db, h);  // (h is the forward's)
              ff_pack16<F16>(da, wa);
              ff_pack16<F16>(db, wb[k]);
              store16(0, col + 16 * k, wa);
            }
            store16(1, col, wb[0]);
            store16(1, col + 16, wb[1]);
          }
          continue;
        }
#pragma unroll 1
        for (int c = 0; c < n; c += 16) {
          uint32_t v[16];
          tmem_ld16(d + part * n + c, v);
          tmem_ld_wait();
          if (!SPLIT && c + 16 >= n) release(acc_empty(acc));
          const int col = t.n * p.bn + part * n + c;
          if constexpr (SPLIT) {
            // fp32 rows of bn columns, 16-byte pieces in an order that spreads a column over the banks
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint32_t piece = static_cast<uint32_t>(part * n + c) / 4 + j;
              const uint32_t at = base + static_cast<uint32_t>(q * 32 + lane) * p.bn * 4 + ((piece ^ (lane & 7u)) << 4);
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v[4 * j]), "r"(v[4 * j + 1]), "r"(v[4 * j + 2]), "r"(v[4 * j + 3])
                           : "memory");
            }
            continue;
          }
          float f[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) f[j] = __uint_as_float(v[j]);
          if constexpr (OP != kFfWeights) {
            uint32_t w[8];
            ff_pack16<F16>(f, w);
            store16(0, col, w);
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

  if constexpr (SPLIT) {
    __syncwarp();
    cluster_sync_all();  // every CTA's tile is in its shared memory
    const Tile t = tile_at(first);
    const int share = 128 / p.splits;  // rows of this CTA
    const int r0 = static_cast<int>(cluster_rank) / G * share;
    const int pieces = p.bn / 8;
    for (int e = threadIdx.x; e < share * pieces; e += kFfThreads) {
      const int r = r0 + e / pieces, c = e % pieces;
      const int row = (t.m * G + static_cast<int>(rank)) * 128 + r, col = t.n * p.bn + c * 8;
      if (row >= p.rows || col >= p.cols) continue;
      float f[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = 0.f;
      for (int k = 0; k < p.splits; ++k) {
        const uint32_t tile = map_to_cta(base, k * G + rank) + static_cast<uint32_t>(r) * p.bn * 4;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float4 v;
          asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                       : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                       : "r"(tile + (((2u * c + j) ^ (r & 7u)) << 4)));
          f[4 * j] += v.x;
          f[4 * j + 1] += v.y;
          f[4 * j + 2] += v.z;
          f[4 * j + 3] += v.w;
        }
      }
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out[0]) + static_cast<size_t>(row) * p.ld + col) =
          make_uint4(ff_pack<F16>(f[0], f[1]), ff_pack<F16>(f[2], f[3]), ff_pack<F16>(f[4], f[5]), ff_pack<F16>(f[6], f[7]));
    }
  }

  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR || SPLIT) cluster_sync_all();  // no CTA leaves while another may still signal its barriers or read its memory
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
__global__ void __launch_bounds__(1024) ff_reduce_kernel(const FfReduce p) {
  __shared__ float tile[32][129];
  grid_dependency_wait();
  grid_dependents_launch();
  void* out = blockIdx.z == 0 ? p.out[0] : blockIdx.z == 1 ? p.out[1] : p.out[2];
  if (out == nullptr) return;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int c = blockIdx.x * 128 + tx * 4, r = blockIdx.y * 32 + ty;
  const bool in = r < p.H && c < p.D;
  const size_t part = static_cast<size_t>(3) * p.H * p.D;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  if (in) {
    const float* s = p.partial + (static_cast<size_t>(blockIdx.z) * p.H + r) * p.D + c;
#pragma unroll 8
    for (int k = 0; k < p.splits; ++k) {
      const float4 v = __ldcg(reinterpret_cast<const float4*>(s + k * part));
      a.x += v.x;
      a.y += v.y;
      a.z += v.z;
      a.w += v.w;
    }
  }
  if (blockIdx.z < 2) {
    if (!in) return;
    const size_t i = static_cast<size_t>(r) * p.D + c;
    if (p.type == 1)
      *reinterpret_cast<float4*>(static_cast<float*>(out) + i) = a;
    else if (p.type == 0)
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + i) = make_uint2(pack_bf16x2(a.x, a.y), pack_bf16x2(a.z, a.w));
    else
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + i) = make_uint2(pack_f16x2(make_float2(a.x, a.y)), pack_f16x2(make_float2(a.z, a.w)));
    return;
  }
  float* s = &tile[ty][tx * 4];
  s[0] = a.x;
  s[1] = a.y;
  s[2] = a.z;
  s[3] = a.w;
  __syncthreads();
  const int h = blockIdx.y * 32 + tx;
#pragma unroll
  for (int j = ty; j < 128; j += 32) {
    const int d = blockIdx.x * 128 + j;
    if (d < p.D && h < p.H) ff_put(out, static_cast<size_t>(d) * p.H + h, tile[tx][j], p.type);
  }
}

// A few rows (the single tokens of serving): every weight is read once and meets all rows, so the bytes of the weights bound it and
// tensor cores would idle on tiles of 128 rows. A warp takes a hidden unit (its rows of W_a and W_b) or a column of y (a row of W_s), a
// lane every 32nd piece of eight weights; the rows lie in shared memory in fp32. R: rows, rounded up to a power of two.
// (us a call, calls in a graph, this and tiles of tensor cores: 768 x 2048 one row 4.6, four 7.7, eight 11.6 and 12.8; 384 x 1536 eight
// 9.3 and 9.7; 1024 x 4096 two 11.0, eight 23.9 and 17.6)
constexpr int kFfVecRows = 4;
constexpr int kFfVecThreads = 256;
constexpr int kFfVecSmem = 96 * 1024;  // rows of the second product pass through it in parts

template <bool F16>
__device__ __forceinline__ float2 ff_two(uint32_t w) {
  return F16 ? f16x2_to_float2(w) : bf16x2_to_float2(w);
}
// rows [0, R) of n columns of a 16-bit matrix to fp32 [R][n], the halves of each piece of eight n / 2 apart (16-byte reads of
// a warp without bank conflicts); rows past `rows` are zero
template <bool F16, int R>
__device__ __forceinline__ void ff_vec_rows(float* to, const void* from, int rows, int ld, int n) {
  for (int c = threadIdx.x * 8; c < n; c += kFfVecThreads * 8) {
    uint4 w[R];
#pragma unroll
    for (int r = 0; r < R; ++r)
      w[r] = r < rows ? __ldcg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(from) + static_cast<size_t>(r) * ld + c)) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float2 a = ff_two<F16>(w[r].x), b = ff_two<F16>(w[r].y), d = ff_two<F16>(w[r].z), f = ff_two<F16>(w[r].w);
      float* o = to + r * n + c / 2;
      *reinterpret_cast<float4*>(o) = make_float4(a.x, a.y, b.x, b.y);
      *reinterpret_cast<float4*>(o + n / 2) = make_float4(d.x, d.y, f.x, f.y);
    }
  }
}
// acc[r] += the products of eight weights with the rows' eight values
template <bool F16, int R>
__device__ __forceinline__ void ff_vec_step(float2 (&acc)[R], const float* rows, int n, int c, const uint4& w) {
  const float2 v[4] = {ff_two<F16>(w.x), ff_two<F16>(w.y), ff_two<F16>(w.z), ff_two<F16>(w.w)};
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float4 a = *reinterpret_cast<const float4*>(rows + r * n + c / 2);
    const float4 b = *reinterpret_cast<const float4*>(rows + r * n + n / 2 + c / 2);
    acc[r] = __ffma2_rn(make_float2(a.x, a.y), v[0], acc[r]);
    acc[r] = __ffma2_rn(make_float2(a.z, a.w), v[1], acc[r]);
    acc[r] = __ffma2_rn(make_float2(b.x, b.y), v[2], acc[r]);
    acc[r] = __ffma2_rn(make_float2(b.z, b.w), v[3], acc[r]);
  }
}
__device__ __forceinline__ float ff_warp_sum(float2 v) {
  float s = v.x + v.y;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
  return s;
}

struct FfVec {
  const void *x, *w_a, *w_b, *w_s;
  float* h;     // [rows][hidden]: no product of tensor cores asks for 16 bits here
  void* y;
  int rows, d, hidden, act;
  int part;     // columns of h that are in shared memory at a time
};
template <bool F16, int R>
__global__ void __launch_bounds__(kFfVecThreads) ff_vec_up_kernel(const FfVec p) {
  extern __shared__ __align__(16) float vec_rows[];
  grid_dependency_wait();
  grid_dependents_launch();
  const int unit = blockIdx.x * (kFfVecThreads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const size_t row = static_cast<size_t>(min(unit, p.hidden - 1)) * p.d;
  const uint16_t* wa = static_cast<const uint16_t*>(p.w_a) + row;
  const uint16_t* wb = static_cast<const uint16_t*>(p.w_b) + row;
  // the first weights are on their way while the rows come in
  constexpr int kFirst = 4;
  uint4 fa[kFirst], fb[kFirst];
#pragma unroll
  for (int i = 0; i < kFirst; ++i) {
    const int c = lane * 8 + i * 256;
    fa[i] = c < p.d ? __ldcg(reinterpret_cast<const uint4*>(wa + c)) : make_uint4(0, 0, 0, 0);
    fb[i] = c < p.d ? __ldcg(reinterpret_cast<const uint4*>(wb + c)) : make_uint4(0, 0, 0, 0);
  }
  ff_vec_rows<F16, R>(vec_rows, p.x, p.rows, p.d, p.d);
  __syncthreads();
  if (unit >= p.hidden) return;
  float2 a[R], b[R];
#pragma unroll
  for (int r = 0; r < R; ++r) a[r] = b[r] = make_float2(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < kFirst; ++i) {
    const int c = lane * 8 + i * 256;
    if (c >= p.d) break;
    ff_vec_step<F16, R>(a, vec_rows, p.d, c, fa[i]);
    ff_vec_step<F16, R>(b, vec_rows, p.d, c, fb[i]);
  }
#pragma unroll 2
  for (int c = lane * 8 + kFirst * 256; c < p.d; c += 256) {
    const uint4 va = __ldcg(reinterpret_cast<const uint4*>(wa + c)), vb = __ldcg(reinterpret_cast<const uint4*>(wb + c));
    ff_vec_step<F16, R>(a, vec_rows, p.d, c, va);
    ff_vec_step<F16, R>(b, vec_rows, p.d, c, vb);
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float sa = ff_warp_sum(a[r]), sb = ff_warp_sum(b[r]);
    if (lane == r && r < p.rows) {
      const float f = p.act == kFfSilu ? __fdividef(sa, 1.0f + __expf(-sa)) : 0.5f * sa * (1.0f + erff(sa * 0.70710678f));
      p.h[static_cast<size_t>(r) * p.hidden + unit] = f * sb;
    }
  }
}
template <bool F16, int R>
__global__ void __launch_bounds__(kFfVecThreads) ff_vec_down_kernel(const FfVec p) {
  extern __shared__ __align__(16) float vec_rows[];
  const int col = blockIdx.x * (kFfVecThreads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const uint16_t* w = static_cast<const uint16_t*>(p.w_s) + static_cast<size_t>(col < p.d ? col : 0) * p.hidden;
  // The first weights before the wait: the launch before is ff_vec_up_kernel, which writes h alone and has itself waited for what wrote
  // the weights before it let this kernel begin.
  constexpr int kFirst = 8;
  uint4 first[kFirst];
#pragma unroll
  for (int i = 0; i < kFirst; ++i) {
    const int c = lane * 8 + i * 256;
    first[i] = c < p.hidden ? __ldcg(reinterpret_cast<const uint4*>(w + c)) : make_uint4(0, 0, 0, 0);
  }
  grid_dependency_wait();
  grid_dependents_launch();
  float2 acc[R];
#pragma unroll
  for (int r = 0; r < R; ++r) acc[r] = make_float2(0.f, 0.f);
  for (int k0 = 0; k0 < p.hidden; k0 += p.part) {
    const int n = min(p.part, p.hidden - k0);
    if (k0 != 0) __syncthreads();
#pragma unroll 2
    for (int c = threadIdx.x * 4; c < n; c += kFfVecThreads * 4) {
      float4 v[R];
#pragma unroll
      for (int r = 0; r < R; ++r)
        v[r] = r < p.rows ? __ldcg(reinterpret_cast<const float4*>(p.h + static_cast<size_t>(r) * p.hidden + k0 + c)) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int r = 0; r < R; ++r) *reinterpret_cast<float4*>(vec_rows + r * n + (c & 4) / 4 * (n / 2) + c / 8 * 4) = v[r];  // (the order of ff_vec_rows)
    }
    __syncthreads();
    int start = lane * 8;
    if (k0 == 0) {
#pragma unroll
      for (int i = 0; i < kFirst; ++i) {
        if (start >= n) break;
        ff_vec_step<F16, R>(acc, vec_rows, n, start, first[i]);
        start += 256;
      }
    }
#pragma unroll 4
    for (int c = start; c < n; c += 256) {
      const uint4 v = __ldcg(reinterpret_cast<const uint4*>(w + k0 + c));
      ff_vec_step<F16, R>(acc, vec_rows, n, c, v);
    }
  }
  if (col >= p.d) return;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float s = ff_warp_sum(acc[r]);
    if (lane == r && r < p.rows) static_cast<uint16_t*>(p.y)[static_cast<size_t>(r) * p.d + col] = static_cast<uint16_t>(ff_pack_held<F16>(s, 0.f));
  }
}

// fp32 master weights as operands: rounded to the type of x
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
