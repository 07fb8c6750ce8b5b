// The norms around a block, joined with its gate, residual scale and residual (all arithmetic in fp32, one rounding per output):
//
//   t = norm_post(u)                       u: the block's output          norm(v) = c rstd w + b,  c = v - mean v (layer) or v (rms),
//   y = x + valid * scale * sigmoid(g) * t x: the residual stream                  rstd = 1 / sqrt(mean c^2 + eps)
//   h = norm_pre(y)                        h: what the next block reads
//
// and, without u, the plain norm h = norm_pre(x). Every part may be absent. h is the norm of the unrounded y. Gradients, with
// J^T q = rstd (q w - [layer] mean(q w) - n mean(q w n)), n = c rstd, of a norm whose result has gradient q:
//
//   e = dy + J_pre^T dh;  dx = e;  dt = e valid scale sigmoid(g);  du = J_post^T dt;  dg = dt t (1 - sigmoid(g))
//   d scale = sum e valid sigmoid(g) t;  d w_post = sum dt n;  d b_post = sum dt;  d w_pre = sum dh n_y;  d b_pre = sum dh
//
// 20 and 50 operations per element against 10 and 16 bytes of a 16-bit type: both directions are bound by HBM, so each is one
// pass over the tensors with the row in registers. The backward takes x and not y: it forms the unrounded y again, so that the
// sums over the rows (fp32 results) do not see the rounding of y to 16 bits; it reads the same number of bytes.
#pragma once

#include "ptx.cuh"

namespace trimul {

enum NormKind : int { kNormNone = 0, kNormLayer = 1, kNormRms = 2 };

struct JoinParams {
  const void* x;
  const void* u;           // null: a plain norm
  const void* gate;        // logits, null: 1; one row of them for every `gate_rows` rows of x
  const uint8_t* mask;     // per row, null: all valid
  const float* scale;      // [d], null: 1
  const float* post_w;     // [d], null: 1 (with post_kind none: not read)
  const float* post_b;     // [d], null: 0
  const float* pre_w;
  const float* pre_b;
  void* y;                 // null with u == null
  void* h;                 // null with pre_kind none
  float2* post_stats;      // [rows] mean and 1 / sigma, null: not kept
  float2* pre_stats;
  // backward only
  const void* dy;          // null: 0
  const void* dh;          // null: 0
  void* dx;
  void* du;
  void* dgate;             // 16 or 32 bits, the type of x
  float* sums;             // [blocks][5][d]: d scale, d post_w, d post_b, d pre_w, d pre_b of a block's rows
  float* gate_part;        // [teams][2][d] (gate_rows > 1): see join_gate_kernel
  long long rows;
  long long gate_rows;
  long long rows_per_team;  // backward with gate_rows > 1: consecutive rows of a team
  int d;
  int team;                // threads per row: a power of two up to 32, or a multiple of 32
  int post_kind, pre_kind;
  float post_eps, pre_eps;
};

// ---------------------------------------------------------------- a row in registers
// Thread t of a team of R holds 8 NV elements of the row: pieces of eight neighbours, piece t of each run of R pieces (WIDE, for
// widths that are a multiple of eight on 16-byte boundaries: 16-byte requests), or single elements, every R-th one.
template <typename T>
struct Io;
template <>
struct Io<__nv_bfloat16> {
  static __device__ __forceinline__ float get(const __nv_bfloat16* p) { return __uint_as_float(static_cast<uint32_t>(__ldcg(reinterpret_cast<const unsigned short*>(p))) << 16); }
  static __device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
  static __device__ __forceinline__ float2 two(uint32_t w) { return bf16x2_to_float2(w); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack_bf16x2(a, b); }
};
template <>
struct Io<__half> {
  static __device__ __forceinline__ float get(const __half* p) {
    const unsigned short w = __ldcg(reinterpret_cast<const unsigned short*>(p));
    return __half2float(__ushort_as_half(w));
  }
  static __device__ __forceinline__ void put(__half* p, float v) { *p = __float2half_rn(v); }
  static __device__ __forceinline__ float2 two(uint32_t w) { return f16x2_to_float2(w); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack_f16x2(make_float2(a, b)); }
};
template <>
struct Io<float> {
  static __device__ __forceinline__ float get(const float* p) { return __ldcg(p); }
  static __device__ __forceinline__ void put(float* p, float v) { *p = v; }
};

// Column of element i (0 .. 8 NV - 1) of thread t. Past the width: no element.
template <bool WIDE>
__device__ __forceinline__ int join_col(int i, int t, int team) {
  return WIDE ? ((i >> 3) * team + t) * 8 + (i & 7) : i * team + t;
}

// Loads bypass L1: the launch before may have left older lines there (the rule at grid_dependency_wait).
template <typename T, bool WIDE, int NV>
__device__ __forceinline__ void load_row(const void* base, long long row, int d, int t, int team, bool on, float (&v)[8 * NV]) {
  const T* p = static_cast<const T*>(base) + row * d;
#pragma unroll
  for (int i = 0; i < 8 * NV; ++i) v[i] = 0.f;
  if (!on) return;
  if constexpr (WIDE) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * team + t) * 8;
      if (c >= d) continue;
      if constexpr (sizeof(T) == 2) {
        const uint4 w = __ldcg(reinterpret_cast<const uint4*>(p + c));
        const uint32_t q[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 f = Io<T>::two(q[k]);
          v[8 * j + 2 * k] = f.x;
          v[8 * j + 2 * k + 1] = f.y;
        }
      } else {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float4 f = __ldcg(reinterpret_cast<const float4*>(p + c) + k);
          v[8 * j + 4 * k] = f.x;
          v[8 * j + 4 * k + 1] = f.y;
          v[8 * j + 4 * k + 2] = f.z;
          v[8 * j + 4 * k + 3] = f.w;
        }
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8 * NV; ++i) {
      const int c = i * team + t;
      if (c < d) v[i] = Io<T>::get(p + c);
    }
  }
}

template <typename T, bool WIDE, int NV>
__device__ __forceinline__ void store_row(void* base, long long row, int d, int t, int team, const float (&v)[8 * NV]) {
  T* p = static_cast<T*>(base) + row * d;
  if constexpr (WIDE) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * team + t) * 8;
      if (c >= d) continue;
      if constexpr (sizeof(T) == 2) {
        uint4 w;
        w.x = Io<T>::pack(v[8 * j], v[8 * j + 1]);
        w.y = Io<T>::pack(v[8 * j + 2], v[8 * j + 3]);
        w.z = Io<T>::pack(v[8 * j + 4], v[8 * j + 5]);
        w.w = Io<T>::pack(v[8 * j + 6], v[8 * j + 7]);
        *reinterpret_cast<uint4*>(p + c) = w;
      } else {
#pragma unroll
        for (int k = 0; k < 2; ++k)
          reinterpret_cast<float4*>(p + c)[k] = make_float4(v[8 * j + 4 * k], v[8 * j + 4 * k + 1], v[8 * j + 4 * k + 2], v[8 * j + 4 * k + 3]);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8 * NV; ++i) {
      const int c = i * team + t;
      if (c < d) Io<T>::put(p + c, v[i]);
    }
  }
}

// A parameter vector ([d] fp32, any alignment); `none` where it is absent and past the width
template <bool WIDE, int NV>
__device__ __forceinline__ void load_param(const float* w, int d, int t, int team, float none, float (&v)[8 * NV]) {
#pragma unroll
  for (int i = 0; i < 8 * NV; ++i) {
    const int c = join_col<WIDE>(i, t, team);
    v[i] = w != nullptr && c < d ? __ldcg(w + c) : none;
  }
}

// Sums of two values over a team, the same bits in every thread. Teams of several warps meet at a named barrier of their own; the
// two halves of `scratch` are used in turn, so that one barrier a sum is enough.
struct TeamSum {
  float2* scratch;  // this team's: two halves of 16
  int warps, id, half;
  __device__ __forceinline__ float2 operator()(float2 v, int team) {
    const int width = team < 32 ? team : 32;
    for (int o = width >> 1; o > 0; o >>= 1) {
      v.x += __shfl_xor_sync(0xFFFFFFFFu, v.x, o);
      v.y += __shfl_xor_sync(0xFFFFFFFFu, v.y, o);
    }
    if (warps > 1) {
      float2* s = scratch + half * 16;
      half ^= 1;
      const int w = (threadIdx.x % team) >> 5;
      if ((threadIdx.x & 31) == 0) s[w] = v;
      named_bar_sync(1 + id, team);
      v = make_float2(0.f, 0.f);
      for (int i = 0; i < warps; ++i) {
        v.x += s[i].x;
        v.y += s[i].y;
      }
    }
    return v;
  }
};

// mean and 1 / sigma of a row whose elements past the width are zero: two passes over the registers
template <bool WIDE, int NV>
__device__ __forceinline__ float2 row_stats(const float (&v)[8 * NV], int kind, float eps, int d, int t, int team, TeamSum& sum) {
  const float inv = 1.0f / static_cast<float>(d);
  float mean = 0.f;
  if (kind == kNormLayer) {
    float a = 0.f;
#pragma unroll
    for (int i = 0; i < 8 * NV; ++i) a += v[i];
    mean = sum(make_float2(a, 0.f), team).x * inv;
  }
  float q = 0.f;
#pragma unroll
  for (int i = 0; i < 8 * NV; ++i) {
    const float c = v[i] - mean;
    if (join_col<WIDE>(i, t, team) < d) q = fmaf(c, c, q);
  }
  const float var = sum(make_float2(q, 0.f), team).x * inv;
  return make_float2(mean, 1.0f / sqrtf(var + eps));
}

__device__ __forceinline__ float sigmoid_fast(float g) { return __fdividef(1.0f, 1.0f + __expf(-g)); }

constexpr int kJoinForwardThreads = 256;
constexpr int kJoinBackwardThreads = 512;

// (single elements only: rows on 16-byte boundaries always fit the tiles of join_tiles.cuh)
template <typename T, int NV>
__global__ void __launch_bounds__(kJoinForwardThreads) join_forward_kernel(const JoinParams p) {
  __shared__ float2 scratch[kJoinForwardThreads / 64 * 32];
  const int team = p.team, t = threadIdx.x % team, id = threadIdx.x / team, teams = blockDim.x / team;
  TeamSum sum{scratch + (team > 32 ? id : 0) * 32, (team + 31) / 32, id, 0};
  const int d = p.d;
  grid_dependency_wait();
  grid_dependents_launch();
  for (long long first = static_cast<long long>(blockIdx.x) * teams; first < p.rows; first += static_cast<long long>(gridDim.x) * teams) {
    const long long row = first + id;
    const bool on = row < p.rows;
    float x[8 * NV];
    load_row<T, false, NV>(p.x, row, d, t, team, on, x);
    if (p.u != nullptr) {
      const bool valid = on && (p.mask == nullptr || __ldcg(p.mask + row) != 0);
      float u[8 * NV], g[8 * NV], w[8 * NV];
      load_row<T, false, NV>(p.u, row, d, t, team, valid, u);
      if (p.gate != nullptr) load_row<T, false, NV>(p.gate, p.gate_rows == 1 ? row : row / p.gate_rows, d, t, team, valid, g);
      if (p.post_kind != kNormNone) {
        const float2 st = row_stats<false, NV>(u, p.post_kind, p.post_eps, d, t, team, sum);
        if (on && t == 0 && p.post_stats != nullptr) p.post_stats[row] = st;
#pragma unroll
        for (int i = 0; i < 8 * NV; ++i) u[i] = (u[i] - st.x) * st.y;
        load_param<false, NV>(p.post_w, d, t, team, 1.f, w);
#pragma unroll
        for (int i = 0; i < 8 * NV; ++i) u[i] *= w[i];
        load_param<false, NV>(p.post_b, d, t, team, 0.f, w);
#pragma unroll
        for (int i = 0; i < 8 * NV; ++i) u[i] += w[i];
      }
      if (p.gate != nullptr)
#pragma unroll
        for (int i = 0; i < 8 * NV; ++i) u[i] *= sigmoid_fast(g[i]);
      load_param<false, NV>(p.scale, d, t, team, 1.f, w);
      if (valid)
#pragma unroll
        for (int i = 0; i < 8 * NV; ++i)
          if (join_col<false>(i, t, team) < d) x[i] = fmaf(u[i], w[i], x[i]);
      if (on) store_row<T, false, NV>(p.y, row, d, t, team, x);
    }
    if (p.pre_kind != kNormNone) {
      const float2 st = row_stats<false, NV>(x, p.pre_kind, p.pre_eps, d, t, team, sum);
      if (on && t == 0 && p.pre_stats != nullptr) p.pre_stats[row] = st;
      float w[8 * NV], b[8 * NV];
      load_param<false, NV>(p.pre_w, d, t, team, 1.f, w);
      load_param<false, NV>(p.pre_b, d, t, team, 0.f, b);
#pragma unroll
      for (int i = 0; i < 8 * NV; ++i) x[i] = fmaf((x[i] - st.x) * st.y, w[i], b[i]);
      if (on) store_row<T, false, NV>(p.h, row, d, t, team, x);
    }
  }
}

// A gate row that several rows share: a team walks `rows_per_team` consecutive rows, adds up the gradient of the current gate row in
// registers and leaves it when the gate row changes: as it is where no other team has a part of it, else in fp32 in the team's place
// 0 (the gate row of its first row) or 1 (of its last), which join_gate_kernel adds up in the teams' order.
// The sums over all rows stay in registers to the end; a block adds up its teams in shared memory and join_sums_kernel the blocks, each in a fixed
// order: the results are the same bits in every call.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(kJoinBackwardThreads, 1) join_backward_kernel(const JoinParams p) {
  __shared__ float2 scratch[kJoinBackwardThreads / 64 * 32];
  extern __shared__ float block_sums[];  // [teams][d]
  const int team = p.team, t = threadIdx.x % team, id = threadIdx.x / team, teams = blockDim.x / team;
  TeamSum sum{scratch + (team > 32 ? id : 0) * 32, (team + 31) / 32, id, 0};
  const int d = p.d;
  const float inv = 1.0f / static_cast<float>(d);
  grid_dependency_wait();
  grid_dependents_launch();
  const bool shared_gate = p.gate != nullptr && p.gate_rows > 1;
  const long long team_index = static_cast<long long>(blockIdx.x) * teams + id;
  const long long step = shared_gate ? 1 : static_cast<long long>(gridDim.x) * teams;
  const long long first = shared_gate ? team_index * p.rows_per_team : team_index;
  const long long last = shared_gate ? (first + p.rows_per_team < p.rows ? first + p.rows_per_team : p.rows) : p.rows;
  // every team of a block makes the same number of rounds (warps hold several teams)
  const long long rounds = shared_gate ? p.rows_per_team : (p.rows + step - 1) / step;
  float s_scale[8], s_pw[8], s_pb[8], s_nw[8], s_nb[8], s_gate[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) s_scale[i] = s_pw[i] = s_pb[i] = s_nw[i] = s_nb[i] = s_gate[i] = 0.f;
  for (long long k = 0; k < rounds; ++k) {
    const long long row = first + k * step;
    const bool on = row < last;
    float x[8], dh[8], e[8];
    load_row<T, WIDE, 1>(p.x, row, d, t, team, on && p.pre_kind != kNormNone, x);
    load_row<T, WIDE, 1>(p.dy, row, d, t, team, on && p.dy != nullptr, e);
    load_row<T, WIDE, 1>(p.dh, row, d, t, team, on && p.dh != nullptr, dh);
    float n[8], tt[8], sg[8], w[8];  // n: normalised u; tt: its affine image; sg: valid scale sigmoid
    bool valid = false;
    float2 post = make_float2(0.f, 0.f);
    float gate[8];
    if (p.u != nullptr) {
      valid = on && (p.mask == nullptr || __ldcg(p.mask + row) != 0);
      load_row<T, WIDE, 1>(p.u, row, d, t, team, valid, n);
      load_row<T, WIDE, 1>(p.gate, p.gate_rows == 1 ? row : row / p.gate_rows, d, t, team, valid && p.gate != nullptr, gate);
      if (p.post_kind != kNormNone && valid) post = __ldcg(p.post_stats + row);
      load_param<WIDE, 1>(p.scale, d, t, team, 1.f, sg);
      if (p.post_kind != kNormNone) {
#pragma unroll
        for (int i = 0; i < 8; ++i) n[i] = (n[i] - post.x) * post.y;
        load_param<WIDE, 1>(p.post_w, d, t, team, 1.f, w);
        load_param<WIDE, 1>(p.post_b, d, t, team, 0.f, tt);
#pragma unroll
        for (int i = 0; i < 8; ++i) tt[i] = fmaf(n[i], w[i], tt[i]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) tt[i] = n[i];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        gate[i] = p.gate != nullptr ? sigmoid_fast(gate[i]) : 1.f;
        const bool in = valid && join_col<WIDE>(i, t, team) < d;
        if (!in) sg[i] = tt[i] = n[i] = 0.f;
        x[i] = fmaf(tt[i] * gate[i], sg[i], x[i]);
      }
    }
    if (p.pre_kind != kNormNone) {
      const float2 st = on ? __ldcg(p.pre_stats + row) : make_float2(0.f, 0.f);
      float pw[8];
      load_param<WIDE, 1>(p.pre_w, d, t, team, 1.f, pw);
      float c1 = 0.f, c2 = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = join_col<WIDE>(i, t, team) < d ? (x[i] - st.x) * st.y : 0.f;
        s_nw[i] = fmaf(dh[i], x[i], s_nw[i]);
        s_nb[i] += dh[i];
        dh[i] *= pw[i];
        c1 += dh[i];
        c2 = fmaf(dh[i], x[i], c2);
      }
      const float2 c = sum(make_float2(c1, c2), team);
      const float m1 = p.pre_kind == kNormLayer ? c.x * inv : 0.f, m2 = c.y * inv;
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = fmaf(st.y, dh[i] - m1 - x[i] * m2, e[i]);
    }
    if (on && p.dx != nullptr) store_row<T, WIDE, 1>(p.dx, row, d, t, team, e);
    if (p.u == nullptr) continue;
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (!valid || join_col<WIDE>(i, t, team) >= d) e[i] = 0.f;
      const float eg = e[i] * gate[i];
      s_scale[i] = fmaf(eg, tt[i], s_scale[i]);
      const float dt = eg * sg[i];
      s_pw[i] = fmaf(dt, n[i], s_pw[i]);
      s_pb[i] += dt;
      gate[i] = dt * tt[i] * (1.f - gate[i]);  // gradient of the gate's logits
      e[i] = p.post_kind != kNormNone ? dt * w[i] : dt;
      s1 += e[i];
      s2 = fmaf(e[i], n[i], s2);
    }
    if (p.post_kind != kNormNone) {
      const float2 c = sum(make_float2(s1, s2), team);
      const float m1 = p.post_kind == kNormLayer ? c.x * inv : 0.f, m2 = c.y * inv;
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = post.y * (e[i] - m1 - n[i] * m2);
    }
    if (on && p.du != nullptr) store_row<T, WIDE, 1>(p.du, row, d, t, team, e);
    if (p.gate != nullptr && p.dgate != nullptr && on) {
      if (!shared_gate) {
        store_row<T, WIDE, 1>(p.dgate, row, d, t, team, gate);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) s_gate[i] += gate[i];
        const long long group = row / p.gate_rows, begin = group * p.gate_rows, end = begin + p.gate_rows;
        if (row + 1 == last || row + 1 == end) {
          if (begin >= first && end <= last) {
            store_row<T, WIDE, 1>(p.dgate, group, d, t, team, s_gate);
          } else {
            store_row<float, false, 1>(p.gate_part, team_index * 2 + (first >= begin ? 0 : 1), 8 * team, t, team, s_gate);
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) s_gate[i] = 0.f;
        }
      }
    }
  }
  if (p.sums == nullptr) return;
  // the block's teams, one sum after the other
#pragma unroll
  for (int s = 0; s < 5; ++s) {
    const float(&v)[8] = s == 0 ? s_scale : s == 1 ? s_pw : s == 2 ? s_pb : s == 3 ? s_nw : s_nb;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = join_col<WIDE>(i, t, team);
      if (c < d) block_sums[id * d + c] = v[i];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < d; c += blockDim.x) {
      float a = 0.f;
      for (int j = 0; j < teams; ++j) a += block_sums[j * d + c];
      p.sums[(static_cast<size_t>(blockIdx.x) * 5 + s) * d + c] = a;
    }
  }
}

// The blocks' sums, eight chains a column
struct JoinSums {
  const float* sums;
  float* out[5];  // null: not asked for
  int blocks, d;
};
__global__ void __launch_bounds__(256) join_sums_kernel(const JoinSums p) {
  __shared__ float part[8][32];
  grid_dependency_wait();
  grid_dependents_launch();
  float* out = p.out[blockIdx.y];
  if (out == nullptr) return;
  const int c = blockIdx.x * 32 + (threadIdx.x & 31), chain = threadIdx.x >> 5;
  float a = 0.f;
  if (c < p.d)
    for (int b = chain; b < p.blocks; b += 8) a += __ldcg(p.sums + (static_cast<size_t>(b) * 5 + blockIdx.y) * p.d + c);
  part[chain][threadIdx.x & 31] = a;
  __syncthreads();
  if (chain == 0 && c < p.d) {
    a = 0.f;
    for (int k = 0; k < 8; ++k) a += part[k][threadIdx.x];
    out[c] = a;
  }
}

// Gate rows of which several teams have a part
template <typename T, bool WIDE>
__global__ void __launch_bounds__(256) join_gate_kernel(const JoinParams p) {
  grid_dependency_wait();
  grid_dependents_launch();
  const long long groups = p.rows / p.gate_rows;
  for (long long group = blockIdx.x; group < groups; group += gridDim.x) {
    const long long begin = group * p.gate_rows, end = begin + p.gate_rows;
    const long long t0 = begin / p.rows_per_team, t1 = (end - 1) / p.rows_per_team;
    if (t0 == t1) continue;
    for (int c = threadIdx.x; c < p.d; c += blockDim.x) {
      // place of column c in a team's eight elements per thread
      const int i = WIDE ? c & 7 : c / p.team, t = WIDE ? c >> 3 : c % p.team;
      float a = 0.f;
      for (long long k = t0; k <= t1; ++k) {
        const long long slot = k * 2 + (k * p.rows_per_team >= begin ? 0 : 1);
        a += __ldcg(p.gate_part + slot * (8 * p.team) + i * p.team + t);
      }
      Io<T>::put(static_cast<T*>(p.dgate) + group * p.d + c, a);
    }
  }
}

}  // namespace trimul
