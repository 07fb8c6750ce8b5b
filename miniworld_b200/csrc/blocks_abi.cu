// C-ABI entry points of the block operators (see include/b200_blocks.h): argument checks, tensor maps, the choice of a variant and
// launches; all arithmetic is in the kernels.
#include "../../include/b200_blocks.h"

#include <algorithm>
#include <numeric>
#include <utility>

#include "feed_forward.cuh"
#include "feed_forward_narrow.cuh"
#include "host_util.cuh"
#include "join.cuh"
#include "join_tiles.cuh"

namespace trimul {

static size_t up(size_t v, size_t a) { return (v + a - 1) / a * a; }

constexpr int kMaxSms = 160;

// ---------------------------------------------------------------- join
// Threads of a row (up to 32 reduce by shuffles alone; wider rows take four warps) and 8-element pieces of each: the fewest idle lanes,
// then two pieces (us, forward of 2^24 elements with every part, one, two and four pieces: 16 bits, 64 wide 42.6, 40.7, 42.8, 256 wide
// 41.7, 39.1, 39.3, 200 wide 55, 53, 50, 250 wide 57, 50, 50, 101 wide 84, 77, 85, 203 wide 119, 83, 87; fp32, 256 wide 57, 61, 95, 203
// wide 84, 69, 111). Three pieces only where they leave fewer lanes idle: 384 wide 36.7. One piece is left to rows of up to eight elements,
// whatever the type (fp32 of 256 would gain 4 us with one, of 203 lose 15).
struct JoinShape {
  int team, nv;
};
static JoinShape join_forward_shape(int d) {
  JoinShape best{0, 0};
  int waste = 0;
  for (int nv : {2, 1, 4, 3})
    for (int team : {1, 2, 4, 8, 16, 32, 64, 128}) {
      const int have = team * nv * 8;
      if (have < d || (team > 32 && nv < 4)) continue;
      if (best.team == 0 || have - d < waste) {
        best = {team, nv};
        waste = have - d;
      }
      break;
    }
  return best;
}
static int join_backward_team(int d) {
  int team = 1;
  while (team < 32 && team * 8 < d) team *= 2;
  if (team * 8 < d) team = (d + 255) / 256 * 32;
  return team;
}
struct JoinGrid {
  int team, teams, blocks;
  long long rows_per_team;  // with a shared gate
};
static JoinGrid join_backward_grid(long long rows, int d, bool shared_gate, int sms) {
  JoinGrid g;
  g.team = join_backward_team(d);
  g.teams = kJoinBackwardThreads / g.team;
  g.blocks = static_cast<int>(std::min<long long>(sms, (rows + g.teams - 1) / g.teams));
  g.rows_per_team = 0;
  if (shared_gate) g.rows_per_team = (rows + static_cast<long long>(g.blocks) * g.teams - 1) / (static_cast<long long>(g.blocks) * g.teams);
  return g;
}

static int check_join(long long rows, int d, long long gate_rows, int dtype, int post_kind, int pre_kind) {
  if (rows < 0 || d < 1 || gate_rows < 1) return B200_TRIMUL_E_SHAPE;
  if (rows > (1ll << 40) / d || rows % gate_rows != 0) return B200_TRIMUL_E_SHAPE;
  if (d > B200_NORM_MAX_WIDTH || dtype < 0 || dtype > 2 || post_kind < 0 || post_kind > 2 || pre_kind < 0 || pre_kind > 2)
    return B200_TRIMUL_E_UNSUPPORTED;
  return B200_TRIMUL_OK;
}
static bool all_aligned16(std::initializer_list<const void*> ps) {
  for (const void* q : ps)
    if (!aligned(q, 16)) return false;
  return true;
}

// Tiles of a call (see join_tiles.cuh): rows to a tile, stages and their places. False where the tensors do not start on 16 bytes
// or a row takes more warps than there are or two stages do not fit: the kernels of join.cuh
// then run.
constexpr int kTileRounds = 4;  // most rounds of a tile
static bool plan_tiles(JoinTileParams* p, const void* const* tensors, int count, int size, int nv, int params, int blocks_most, int smem) {
  for (int i = 0; i < count; ++i)
    if (!aligned(tensors[i], 16)) return false;
  const JoinParams& j = p->j;
  if (j.team > kTileWarps * 32) return false;
  const int unit = 16 / static_cast<int>(std::gcd(16, j.d * size));  // rows whose bytes are a multiple of 16
  const int teams = j.team > 32 ? std::min(kTileTeams, kTileWarps * 32 / j.team) : kTileWarps * 32 / j.team;
  p->workers = teams * j.team;
  p->params = 8 * nv * j.team;
  const int fixed = params * p->params * 4 + kTileScratch + kTileTail;
  auto place = [&](int rows) {
    p->slot = static_cast<int>(up(static_cast<size_t>(rows) * j.d * size, 128));
    p->stages = std::min(kTileMaxStages, (smem - fixed) / (p->slot * p->slots));
    return p->stages;
  };
  // The fewest rounds of the teams in all, then the smallest tile: the rows of a tile are a multiple of `unit`, so that where that does not
  // divide the teams the last round of a tile leaves some idle, and tiles of several rounds leave fewer (while four stages fit).
  const long long share = (j.rows + blocks_most - 1) / blocks_most;
  const int most = static_cast<int>(up(static_cast<size_t>(std::min<long long>(kTileRounds * teams, share)), unit));
  int rows = 0;
  long long best = 0;
  for (int r = unit; r <= most; r += unit) {
    if (place(r) < (r > teams ? 4 : 2)) break;
    const long long tiles = (j.rows + r - 1) / r, rounds = (tiles + blocks_most - 1) / blocks_most * ((r + teams - 1) / teams);
    if (rows == 0 || rounds < best) best = rounds, rows = r;
  }
  if (rows == 0) return false;
  place(rows);
  p->tile_rows = rows;
  const long long tiles = (j.rows + rows - 1) / rows;
  if (tiles > 0x7FFFFFFF) return false;
  p->tiles = static_cast<int>(tiles);
  p->stages = static_cast<int>(std::min<long long>(p->stages, std::max<long long>(2, (tiles + blocks_most - 1) / blocks_most)));
  return true;
}
static int tile_smem(const JoinTileParams& p, int params) {
  // (the backward's sums pass through the stages)
  return params * p.params * 4 + kTileScratch + kTileTail + std::max(p.stages * p.slots * p.slot, params == 3 ? p.workers * 8 * 4 : 0);
}
using TileKernel = void (*)(JoinTileParams);
template <typename T>
constexpr int kOdd = sizeof(T) == 2 ? 3 : 1;
template <typename T, int VEC, bool EXACT>
static TileKernel tile_forward_kernel(int nv) {
  if constexpr (VEC != 8 || EXACT)  // (one piece: widths of up to eight, of which eight is exact)
    if (nv == 1) return join_tile_forward_kernel<T, VEC, 1, EXACT>;
  switch (nv) {
    case 2: return join_tile_forward_kernel<T, VEC, 2, EXACT>;
    case 3: return join_tile_forward_kernel<T, VEC, 3, EXACT>;
    default: return join_tile_forward_kernel<T, VEC, 4, EXACT>;
  }
}
template <typename T, bool JOIN>
static TileKernel tile_backward_kernel(int vec, bool exact) {
  if (exact) return join_tile_backward_kernel<T, 8, true, JOIN>;
  return vec == 8 ? join_tile_backward_kernel<T, 8, false, JOIN> : vec == 2 ? join_tile_backward_kernel<T, 2, false, JOIN> : join_tile_backward_kernel<T, kOdd<T>, false, JOIN>;
}
// elements of a row that a thread reads at once
static int join_vec(int d, size_t size) { return d % 8 == 0 ? 8 : d % 2 == 0 ? 2 : size == 2 ? 3 : 1; }  // (see tile_col)

template <typename T>
static int launch_join_forward(const JoinParams& p0, const DeviceInfo& info, cudaStream_t stream) {
  JoinTileParams q = {};
  q.j = p0;
  const JoinShape s = join_forward_shape(p0.d);
  q.j.team = s.team;
  q.slot_of[0] = q.slots++;
  q.slot_of[1] = p0.u != nullptr ? q.slots++ : -1;
  q.slot_of[2] = p0.gate != nullptr && p0.gate_rows == 1 ? q.slots++ : -1;
  q.slot_of[3] = q.slot_of[4] = -1;
  q.out_slot[0] = p0.y != nullptr ? 0 : -1;
  q.out_slot[1] = p0.h != nullptr ? (p0.u != nullptr ? 1 : 0) : -1;
  q.out_slot[2] = -1;
  const void* tensors[] = {p0.x, p0.u, p0.gate, p0.y, p0.h};
  const int per_sm = s.nv == 1 ? 2 : 1;
  if (plan_tiles(&q, tensors, 5, sizeof(T), s.nv, 4, per_sm * info.sms, per_sm == 2 ? kTileSmemHalf : kTileSmem)) {
    const int vec = join_vec(p0.d, sizeof(T));
    const TileKernel kernel = p0.d == 8 * s.nv * s.team ? tile_forward_kernel<T, 8, true>(s.nv)
                              : vec == 8                ? tile_forward_kernel<T, 8, false>(s.nv)
                              : vec == 2                ? tile_forward_kernel<T, 2, false>(s.nv)
                                                        : tile_forward_kernel<T, kOdd<T>, false>(s.nv);
    const int rc = set_smem(kernel, kTileSmem, info.device);
    if (rc != 0) return rc;
    TRIMUL_CUDA(launch_overlapped(kernel, dim3(std::min(per_sm * info.sms, q.tiles)), q.workers + 32, tile_smem(q, 4), stream, q));
    return B200_TRIMUL_OK;
  }
  JoinParams p = p0;
  p.team = s.team;
  const int teams = kJoinForwardThreads / s.team;
  const int blocks = static_cast<int>(std::min<long long>((p.rows + teams - 1) / teams, 8ll * info.sms));
  void (*kernel)(JoinParams) = nullptr;
  switch (s.nv) {
    case 1: kernel = join_forward_kernel<T, 1>; break;
    case 2: kernel = join_forward_kernel<T, 2>; break;
    case 3: kernel = join_forward_kernel<T, 3>; break;
    default: kernel = join_forward_kernel<T, 4>; break;
  }
  TRIMUL_CUDA(launch_overlapped(kernel, dim3(blocks), kJoinForwardThreads, 0, stream, p));
  return B200_TRIMUL_OK;
}

constexpr long long kSharedGateRows = 256;  // gate rows of fewer rows take the kernels of join.cuh: less scratch a gate row

template <typename T>
static int launch_join_backward(const JoinParams& p, bool wide, const JoinGrid& g, const JoinSums& sums, const DeviceInfo& info,
                                cudaStream_t stream) {
  JoinTileParams q = {};
  q.j = p;
  const bool shared_gate = p.gate != nullptr && p.gate_rows > 1;
  q.slot_of[0] = p.pre_kind != kNormNone ? q.slots++ : -1;
  q.slot_of[1] = p.u != nullptr ? q.slots++ : -1;
  q.slot_of[2] = p.gate != nullptr && !shared_gate ? q.slots++ : -1;
  q.slot_of[3] = p.dy != nullptr ? q.slots++ : -1;
  q.slot_of[4] = p.dh != nullptr ? q.slots++ : -1;
  q.out_slot[0] = p.dx == nullptr ? -1 : q.slot_of[0] >= 0 ? q.slot_of[0] : q.slot_of[3] >= 0 ? q.slot_of[3] : q.slots++;
  q.out_slot[1] = p.du != nullptr ? q.slot_of[1] : -1;
  q.out_slot[2] = p.dgate != nullptr && !shared_gate ? q.slot_of[2] : -1;
  const bool join = p.u != nullptr;
  const int most = std::min(info.sms, kMaxSms) * (join ? 1 : 2);
  const void* tensors[] = {p.x, p.u, p.gate, p.dy, p.dh, p.dx, p.du, q.out_slot[2] >= 0 ? p.dgate : nullptr};
  if (q.slots > 0 && (!shared_gate || p.gate_rows >= kSharedGateRows) && plan_tiles(&q, tensors, 8, sizeof(T), 1, 3, most, join ? kTileSmem : kTileSmemHalf)) {
    const int blocks = std::min(most, q.tiles);
    if (shared_gate) {
      q.block_tiles = (q.tiles + blocks - 1) / blocks;
      q.group_slots = static_cast<int>(static_cast<long long>(q.block_tiles) * q.tile_rows / p.gate_rows) + 2;
    }
    const int vec = join_vec(p.d, sizeof(T));
    const TileKernel kernel = join ? tile_backward_kernel<T, true>(vec, p.d == 8 * p.team) : tile_backward_kernel<T, false>(vec, p.d == 8 * p.team);
    const int rc = set_smem(kernel, kTileSmem, info.device);
    if (rc != 0) return rc;
    TRIMUL_CUDA(launch_overlapped(kernel, dim3(blocks), q.workers + 32, tile_smem(q, 3), stream, q));
    if (p.sums != nullptr) {
      JoinTileSums t = {p.sums, p.scale, p.post_w, p.post_b, {}, blocks, p.d, p.post_kind};
      for (int i = 0; i < 5; ++i) t.out[i] = sums.out[i];
      TRIMUL_CUDA(launch_overlapped(join_tile_sums_kernel, dim3((p.d + 31) / 32, 2), 1024, 0, stream, t));
    }
    if (p.dgate != nullptr && shared_gate) {
      auto last = vec == 8 ? join_tile_gate_kernel<T, 8> : vec == 2 ? join_tile_gate_kernel<T, 2> : join_tile_gate_kernel<T, kOdd<T>>;
      // (kSharedGateRows rows a gate row and more: memory ends long before the grid does)
      TRIMUL_CUDA(launch_overlapped(last, dim3(static_cast<unsigned>(p.rows / p.gate_rows), (8 * p.team + 31) / 32), 1024, 0, stream, q));
    }
    return B200_TRIMUL_OK;
  }
  const int smem = p.sums != nullptr ? g.teams * p.d * 4 : 0;
  TRIMUL_CUDA(launch_overlapped(wide ? join_backward_kernel<T, true> : join_backward_kernel<T, false>, dim3(g.blocks), g.team * g.teams, smem,
                                stream, p));
  if (p.sums != nullptr) TRIMUL_CUDA(launch_overlapped(join_sums_kernel, dim3((p.d + 31) / 32, 5), 256, 0, stream, sums));
  if (p.dgate != nullptr && p.gate_rows > 1) {
    const int blocks = static_cast<int>(std::min<long long>(p.rows / p.gate_rows, 1024));
    TRIMUL_CUDA(launch_overlapped(wide ? join_gate_kernel<T, true> : join_gate_kernel<T, false>, dim3(blocks), 256, 0, stream, p));
  }
  return B200_TRIMUL_OK;
}

// (a norm's two blocks an SM leave two of the four sums: up to eight in all)
static size_t join_sums_bytes(int d) { return up(static_cast<size_t>(kMaxSms) * 8 * d * 4, 1024); }

// ---------------------------------------------------------------- feed-forward
// The current device, whose context is then the calling thread's: a thread that has not used the GPU yet (autograd's, on its first
// backward) has none, and tensor maps are made by the driver.
static int ff_device(DeviceInfo* info) {
  const int rc = device_info(info);
  if (rc != 0) return rc;
  info->sms = std::min(info->sms, kMaxSms);  // (workspaces are sized for these)
  TRIMUL_CUDA(cudaSetDevice(info->device));
  return B200_TRIMUL_OK;
}

static int ff_ld(int hidden) { return static_cast<int>(up(hidden, 64)); }  // rows of h, da and db: whole 128-byte lines

// Rows [rows][cols] of 16-bit elements, `ld` elements apart, in boxes of 64 columns by `box` rows
static int ff_map(CUtensorMap* m, const void* base, long long rows, int cols, long long ld, int box) {
  const uint64_t dims[2] = {static_cast<uint64_t>(cols), static_cast<uint64_t>(rows)};
  const uint64_t strides[1] = {static_cast<uint64_t>(ld) * 2};
  const uint32_t b[2] = {64, static_cast<uint32_t>(box)};
  return make_map(m, base, 2, dims, strides, b);
}

struct FfProblem {
  long long rows;
  int d, hidden, ld;
  bool f16;
  int act;
  const void *w_a, *w_b, *w_s;  // operands, in the type of x
  DeviceInfo info;
  cudaStream_t stream;
};

template <int OP, bool PAIR, bool F16, int ACT, bool SPLIT>
static int ff_launch_kernel(const FfMaps& maps, const FfParams& p, const DeviceInfo& info, cudaStream_t stream) {
  const auto kernel = ff_kernel<OP, PAIR, F16, ACT, SPLIT>;
  const int rc = set_smem(kernel, kFfSmemBytes, info.device);
  if (rc != B200_TRIMUL_OK) return rc;
  const long long tiles = static_cast<long long>(p.m_tiles) * p.n_tiles * (OP == kFfWeights ? 3 * p.splits : 1);
  const int cluster = (PAIR ? 2 : 1) * (SPLIT ? p.splits : 1);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(SPLIT ? tiles : std::min<long long>(tiles, info.sms / cluster)) * cluster);
  cfg.blockDim = dim3(kFfThreads);
  cfg.dynamicSmemBytes = kFfSmemBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  TRIMUL_CUDA(cudaLaunchKernelEx(&cfg, kernel, maps, p));
  return B200_TRIMUL_OK;
}
template <int OP, bool PAIR, bool F16>
static int ff_launch_variant(const FfMaps& maps, const FfParams& p, int act, const DeviceInfo& info, cudaStream_t stream) {
  if constexpr (OP == kFfUp || OP == kFfHidden || OP == kFfGrad)
    if (act == kFfGelu) return ff_launch_kernel<OP, PAIR, F16, kFfGelu, false>(maps, p, info, stream);
  if constexpr (OP == kFfDown || OP == kFfInput)
    if (p.splits > 1) return ff_launch_kernel<OP, PAIR, F16, kFfSilu, true>(maps, p, info, stream);
  return ff_launch_kernel<OP, PAIR, F16, kFfSilu, false>(maps, p, info, stream);
}
template <int OP>
static int ff_launch(const FfMaps& maps, const FfParams& p, bool pair, const FfProblem& f) {
  if (pair) return f.f16 ? ff_launch_variant<OP, true, true>(maps, p, f.act, f.info, f.stream) : ff_launch_variant<OP, true, false>(maps, p, f.act, f.info, f.stream);
  return f.f16 ? ff_launch_variant<OP, false, true>(maps, p, f.act, f.info, f.stream) : ff_launch_variant<OP, false, false>(maps, p, f.act, f.info, f.stream);
}

static int blocks_of(long long n, int b) { return static_cast<int>((n + b - 1) / b); }

// CTA pairs where their 256-row tiles still occupy most of the GPU, single CTAs below
static bool ff_pair(long long rows, long long n_tiles, int sms) { return rows > 128 && blocks_of(rows, 256) * n_tiles >= sms / 2 * 3 / 4; }

// h = act(x W_a^T) * (x W_b^T), or with dy the backward's da, db, h
static int ff_hidden(const FfProblem& f, const void* x, const void* dy, void* const out[3], void* const keep[2] = nullptr) {
  const bool pair = ff_pair(f.rows, blocks_of(f.hidden, 128), f.info.sms);
  const int units = pair ? 128 : 64;
  FfMaps maps = {};
  int rc = ff_map(&maps.a[dy != nullptr ? 1 : 0], x, f.rows, f.d, f.d, 128);
  if (rc == 0) rc = ff_map(&maps.b[0], f.w_a, f.hidden, f.d, f.d, units);
  if (rc == 0) rc = ff_map(&maps.b[1], f.w_b, f.hidden, f.d, f.d, units);
  if (rc == 0 && dy != nullptr) rc = ff_map(&maps.a[0], dy, f.rows, f.d, f.d, 128);
  if (rc == 0 && dy != nullptr) rc = ff_map(&maps.b[2], f.w_s, f.d, f.hidden, f.hidden, 64);
  if (rc != 0) return rc;
  FfParams p = {};
  for (int i = 0; i < 3; ++i) p.out[i] = out[i];
  if (keep != nullptr) p.keep[0] = keep[0], p.keep[1] = keep[1];
  p.ld = f.ld;
  p.rows = static_cast<int>(f.rows);
  p.cols = f.hidden;
  p.m_tiles = blocks_of(f.rows, pair ? 256 : 128);
  p.n_tiles = blocks_of(f.hidden, units);
  p.kb = p.kb_second = blocks_of(f.d, 64);
  p.bn = 2 * units;
  p.splits = 1;
  return dy != nullptr ? ff_launch<kFfHidden>(maps, p, pair, f) : ff_launch<kFfUp>(maps, p, pair, f);
}

// da and db from dy with the forward's a and b
static int ff_grad(const FfProblem& f, const void* dy, const void* const kept[2], void* da, void* db) {
  const bool pair = ff_pair(f.rows, blocks_of(f.hidden, 256), f.info.sms);
  const int bn = pair ? 256 : 128;
  FfMaps maps = {};
  int rc = ff_map(&maps.a[0], dy, f.rows, f.d, f.d, 128);
  if (rc == 0) rc = ff_map(&maps.b[0], f.w_s, f.d, f.hidden, f.hidden, 64);
  if (rc != 0) return rc;
  FfParams p = {};
  p.out[0] = da;
  p.out[1] = db;
  p.kept[0] = kept[0];
  p.kept[1] = kept[1];
  p.ld = f.ld;
  p.rows = static_cast<int>(f.rows);
  p.cols = f.hidden;
  p.m_tiles = blocks_of(f.rows, pair ? 256 : 128);
  p.n_tiles = blocks_of(f.hidden, bn);
  p.kb = blocks_of(f.d, 64);
  p.bn = bn;
  p.splits = 1;
  return ff_launch<kFfGrad>(maps, p, pair, f);
}

// Tiles of y = h W_s^T or dx = da W_a + db W_b (`input`): k blocks are far more than tiles where there are few rows. Pairs (tiles of 256
// rows) read half as much of the second operand a product as single CTAs do, and what a single CTA's smaller tile reads from L2 is
// what bounds it, so pairs are taken where, with their k range split over a cluster of up to eight CTAs, they still occupy half the GPU.
// CTAs (pairs) that clusters of `splits` of them occupy at a time: a cluster lies within one of the GPU's processing clusters, of
// which clusters of four leave a ninth and clusters of eight a fifth of the SMs idle (33 and 15 of them on 148 SMs).
static long long ff_split_units(bool pair, int splits, int sms) {
  const int cluster = splits * (pair ? 2 : 1);
  const int ctas = cluster <= 2 ? sms : cluster == 4 ? sms * 33 / 37 : sms * 30 / 37;
  return ctas / (pair ? 2 : 1);
}
struct FfProject {
  bool pair;
  int bn, m_tiles, n_tiles, kb, splits, kb_split;
};
static FfProject ff_project_plan(long long rows, int d, int hidden, bool input, int sms) {
  FfProject best = {};
  const int kb_all = blocks_of(hidden, 64) * (input ? 2 : 1);
  for (int pair = 1; pair >= 0; --pair) {
    if (pair && rows <= 128) continue;
    FfProject q = {};
    q.pair = pair != 0;
    q.bn = pair ? 256 : 128;
    while (q.bn > (pair && input ? 128 : 64) && blocks_of(d, q.bn / 2) * (q.bn / 2) < blocks_of(d, q.bn) * q.bn) q.bn /= 2;
    const int units = pair ? sms / 2 : sms;
    q.m_tiles = blocks_of(rows, pair ? 256 : 128);
    while (q.bn > (pair && input ? 128 : 64) && static_cast<long long>(q.m_tiles) * blocks_of(d, q.bn) * (pair ? 4 : 8) < units) q.bn /= 2;
    q.n_tiles = blocks_of(d, q.bn);
    q.kb = blocks_of(hidden, 64);
    const long long tiles = static_cast<long long>(q.m_tiles) * q.n_tiles;
    // parts of at least two k blocks, a power of two of them, in one round of tiles
    q.splits = 1;
    while (q.splits < (pair ? 4 : 8) && tiles * q.splits * 2 <= ff_split_units(pair != 0, q.splits * 2, sms) && kb_all >= q.splits * 4) q.splits *= 2;
    q.kb_split = blocks_of(kb_all, q.splits);
    while ((q.splits - 1) * q.kb_split >= kb_all) q.splits /= 2, q.kb_split = blocks_of(kb_all, q.splits);  // (no part empty)
    best = q;
    if (tiles * q.splits * 2 >= units) break;
  }
  return best;
}

// y = h W_s^T, or (two operands) dx = da W_a + db W_b
static int ff_project(const FfProblem& f, const void* first, const void* second, void* out) {
  const bool input = second != nullptr;
  const FfProject plan = ff_project_plan(f.rows, f.d, f.hidden, input, f.info.sms);
  const bool pair = plan.pair;
  const int bn = plan.bn;
  FfMaps maps = {};
  int rc = ff_map(&maps.a[0], first, f.rows, f.hidden, f.ld, 128);
  if (input) {
    if (rc == 0) rc = ff_map(&maps.a[1], second, f.rows, f.hidden, f.ld, 128);
    if (rc == 0) rc = ff_map(&maps.b[0], f.w_a, f.hidden, f.d, f.d, 64);
    if (rc == 0) rc = ff_map(&maps.b[1], f.w_b, f.hidden, f.d, f.d, 64);
  } else if (rc == 0) {
    rc = ff_map(&maps.b[0], f.w_s, f.d, f.hidden, f.hidden, pair ? bn / 2 : bn);
  }
  if (rc != 0) return rc;
  FfParams p = {};
  p.out[0] = out;
  p.ld = f.d;
  p.rows = static_cast<int>(f.rows);
  p.cols = f.d;
  p.m_tiles = plan.m_tiles;
  p.n_tiles = plan.n_tiles;
  p.kb = p.kb_second = plan.kb;
  p.bn = bn;
  p.splits = plan.splits;
  p.kb_split = plan.kb_split;
  return input ? ff_launch<kFfInput>(maps, p, pair, f) : ff_launch<kFfDown>(maps, p, pair, f);
}

// Narrow tensors in one kernel, where its tiles of 256 rows occupy most of the GPU
static bool ff_narrow(long long rows, int d, int sms) { return d <= 128 && blocks_of(rows, 256) >= sms / 2 * 3 / 4; }
template <bool F16, int ACT, int HALVES>
static int ff_narrow_launch(const FfProblem& f, const void* x, void* y) {
  const auto kernel = ff_narrow_kernel<F16, ACT, HALVES>;
  int rc = set_smem(kernel, kNwSmemBytes, f.info.device);
  FfMaps maps = {};
  if (rc == 0) rc = ff_map(&maps.a[0], x, f.rows, f.d, f.d, 128);
  if (rc == 0) rc = ff_map(&maps.b[0], f.w_a, f.hidden, f.d, f.d, 64);
  if (rc == 0) rc = ff_map(&maps.b[1], f.w_b, f.hidden, f.d, f.d, 64);
  if (rc == 0) rc = ff_map(&maps.b[2], f.w_s, f.d, f.hidden, f.hidden, 32 * HALVES);
  if (rc != 0) return rc;
  const FfNarrowParams p = {y, f.rows, f.d, blocks_of(f.rows, 256), blocks_of(f.hidden, 64)};
  TRIMUL_CUDA(launch_overlapped(kernel, dim3(2 * std::min(p.num_tiles, f.info.sms / 2)), kNwThreads, kNwSmemBytes, f.stream, maps, p));
  return 0;
}
static int ff_narrow_forward(const FfProblem& f, const void* x, void* y) {
  const bool wide = f.d > 64, gelu = f.act == kFfGelu;
  if (f.f16) {
    if (gelu) return wide ? ff_narrow_launch<true, kFfGelu, 2>(f, x, y) : ff_narrow_launch<true, kFfGelu, 1>(f, x, y);
    return wide ? ff_narrow_launch<true, kFfSilu, 2>(f, x, y) : ff_narrow_launch<true, kFfSilu, 1>(f, x, y);
  }
  if (gelu) return wide ? ff_narrow_launch<false, kFfGelu, 2>(f, x, y) : ff_narrow_launch<false, kFfGelu, 1>(f, x, y);
  return wide ? ff_narrow_launch<false, kFfSilu, 2>(f, x, y) : ff_narrow_launch<false, kFfSilu, 1>(f, x, y);
}

template <bool F16, int R>
static int ff_vec_launch(const FfProblem& f, FfVec v) {
  const int rc0 = set_smem(ff_vec_up_kernel<F16, R>, kFfVecSmem, f.info.device);
  if (rc0 != 0) return rc0;
  const int rc1 = set_smem(ff_vec_down_kernel<F16, R>, kFfVecSmem, f.info.device);
  if (rc1 != 0) return rc1;
  const int warps = kFfVecThreads / 32;
  TRIMUL_CUDA(launch_overlapped(ff_vec_up_kernel<F16, R>, dim3(blocks_of(f.hidden, warps)), kFfVecThreads, R * f.d * 4, f.stream, v));
  v.part = std::min(f.hidden, kFfVecSmem / (R * 4) / 256 * 256);
  TRIMUL_CUDA(launch_overlapped(ff_vec_down_kernel<F16, R>, dim3(blocks_of(f.d, warps)), kFfVecThreads, R * v.part * 4, f.stream, v));
  return 0;
}
static int ff_vec_rows_up(long long rows) { return rows <= 1 ? 1 : rows <= 2 ? 2 : 4; }
static bool ff_vec(long long rows, int d) { return rows <= kFfVecRows && ff_vec_rows_up(rows) * static_cast<long long>(d) * 4 <= kFfVecSmem; }
template <bool F16>
static int ff_vec_forward(const FfProblem& f, const void* x, void* h, void* y) {
  const FfVec v = {x, f.w_a, f.w_b, f.w_s, static_cast<float*>(h), y, static_cast<int>(f.rows), f.d, f.hidden, f.act, 0};
  switch (ff_vec_rows_up(f.rows)) {
    case 1: return ff_vec_launch<F16, 1>(f, v);
    case 2: return ff_vec_launch<F16, 2>(f, v);
    default: return ff_vec_launch<F16, 4>(f, v);
  }
}

// Tiles and parts of the weight gradients' products [hidden, d]: as many parts as fill the GPU in one round of tiles (more parts would
// take more rounds and cost the fp32 partials' traffic), of at least eight k blocks
struct FfSplit {
  bool pair;
  int bn, m_tiles, n_tiles, kb, splits, kb_split;
  int most;  // parts before they are made equal: no fewer than `splits` for any smaller number of SMs
};
static FfSplit ff_split(long long rows, int d, int hidden, int sms) {
  FfSplit s;
  s.kb = std::max(1, blocks_of(rows, 64));
  s.pair = hidden > 128 && d > 64 && static_cast<long long>(hidden) * d >= 512 * 128;
  s.bn = s.pair ? 256 : 128;
  while (s.bn > (s.pair ? 128 : 64) && blocks_of(d, s.bn / 2) * (s.bn / 2) < blocks_of(d, s.bn) * s.bn) s.bn /= 2;
  s.m_tiles = blocks_of(hidden, s.pair ? 256 : 128);
  s.n_tiles = blocks_of(d, s.bn);
  const long long tiles = 3ll * s.m_tiles * s.n_tiles, units = s.pair ? sms / 2 : sms;
  long long parts = units / tiles;
  parts = std::max<long long>(1, std::min<long long>(parts, s.kb / 8));
  s.most = static_cast<int>(parts);
  s.kb_split = blocks_of(s.kb, static_cast<int>(parts));
  s.splits = blocks_of(s.kb, s.kb_split);
  return s;
}

static int ff_weight_gradients(const FfProblem& f, const void* x, const void* dy, void* const hidden3[3], float* partial, void* dw_a,
                               void* dw_b, void* dw_s, int weight_dtype) {
  const FfSplit s = ff_split(f.rows, f.d, f.hidden, f.info.sms);
  FfMaps maps = {};
  int rc = 0;
  for (int i = 0; i < 3 && rc == 0; ++i) rc = ff_map(&maps.a[i], hidden3[i], f.rows, f.hidden, f.ld, 64);
  if (rc == 0) rc = ff_map(&maps.b[0], x, f.rows, f.d, f.d, 64);
  if (rc == 0) rc = ff_map(&maps.b[1], dy, f.rows, f.d, f.d, 64);
  if (rc != 0) return rc;
  FfParams p = {};
  if (s.splits > 1) p.partial = partial;
  p.out[0] = dw_a;
  p.out[1] = dw_b;
  p.out[2] = dw_s;
  p.type = weight_dtype;
  p.rows = f.hidden;
  p.cols = f.d;
  p.m_tiles = s.m_tiles;
  p.n_tiles = s.n_tiles;
  p.kb = s.kb;
  p.bn = s.bn;
  p.splits = s.splits;
  p.kb_split = s.kb_split;
  rc = ff_launch<kFfWeights>(maps, p, s.pair, f);
  if (rc != 0 || s.splits == 1) return rc;
  FfReduce r = {};
  r.partial = partial;
  r.out[0] = dw_a;
  r.out[1] = dw_b;
  r.out[2] = dw_s;
  r.splits = s.splits;
  r.H = f.hidden;
  r.D = f.d;
  r.type = weight_dtype;
  TRIMUL_CUDA(launch_overlapped(ff_reduce_kernel, dim3(blocks_of(f.d, 128), blocks_of(f.hidden, 32), 3), 1024, 0, f.stream, r));
  return 0;
}

static int check_ff(long long rows, int d, int hidden, int weight_dtype, int dtype = 0) {
  if (rows < 0 || rows > 0x7FFFFFFFll - 256 || d < 1 || hidden < 1) return B200_TRIMUL_E_SHAPE;
  if (d % 8 != 0 || hidden % 8 != 0 || d > (1 << 20) || hidden > (1 << 20)) return B200_TRIMUL_E_UNSUPPORTED;
  if (dtype != B200_BLOCKS_BF16 && dtype != B200_BLOCKS_F16) return B200_TRIMUL_E_UNSUPPORTED;
  if (weight_dtype < 0 || weight_dtype > 2) return B200_TRIMUL_E_UNSUPPORTED;
  return B200_TRIMUL_OK;
}

// What the forward keeps for the backward: h in x's type, a and b as ff_keep16 packs them, [rows][ld] values of 16 bits each; nothing where forming a and b again is
// cheaper. Writing and reading them costs 8 bytes a value, forming them 4 D operations: 0.0012 against 0.0027 D picoseconds at
// 6.5 TB/s and 1.5 PFLOP/s, equal at D = 460; calls of few rows are bound by latency either way and keep nothing.
// (16384 x 1024 x 4096: kernels of a training step, each alone, 1151 -> 938 us.)
static size_t ff_kept_bytes(long long rows, int d, int hidden) {
  if (d < 512 || rows < 1024) return 0;
  return 3 * up(up(static_cast<size_t>(rows), 32) * ff_ld(hidden) * 2, 1024);
}

struct FfRegions {
  size_t weights, hidden[3], partial, total;
};
static FfRegions ff_regions(long long rows, int d, int hidden, int weight_dtype, bool backward) {
  FfRegions r = {};
  size_t at = 0;
  r.weights = at;
  if (weight_dtype == B200_BLOCKS_F32) at += up(static_cast<size_t>(3) * hidden * d * 2, 1024);
  for (int i = 0; i < (backward ? 3 : 1); ++i) {
    r.hidden[i] = at;
    at += up(static_cast<size_t>(rows) * ff_ld(hidden) * (rows <= kFfVecRows ? 4 : 2), 1024);  // (fp32 where tensor cores take no part)
  }
  r.partial = at;
  const int parts = backward ? ff_split(rows, d, hidden, kMaxSms).most : 0;
  if (parts > 1) at += up(static_cast<size_t>(parts) * 3 * hidden * d * 4, 1024);
  r.total = at;
  return r;
}

// The problem of a call, its weights cast if they are fp32
static int ff_problem(FfProblem* f, const void* w_a, const void* w_b, const void* w_s, long long rows, int d, int hidden, int dtype,
                      int weight_dtype, int activation, uint8_t* cast_to, void* cuda_stream) {
  f->rows = rows;
  f->d = d;
  f->hidden = hidden;
  f->ld = ff_ld(hidden);
  f->f16 = dtype == B200_BLOCKS_F16;
  f->act = activation;
  f->stream = static_cast<cudaStream_t>(cuda_stream);
  f->w_a = w_a;
  f->w_b = w_b;
  f->w_s = w_s;
  if (weight_dtype != B200_BLOCKS_F32) return 0;
  const long long n = static_cast<long long>(hidden) * d;
  f->w_a = cast_to;
  f->w_b = cast_to + n * 2;
  f->w_s = cast_to + n * 4;
  const int blocks = static_cast<int>(std::min<long long>((3 * n / 8 + 255) / 256, 8 * f->info.sms));
  TRIMUL_CUDA(launch_overlapped(ff_cast_kernel, dim3(blocks), 256, 0, f->stream, static_cast<const float*>(w_a), static_cast<const float*>(w_b),
                                static_cast<const float*>(w_s), reinterpret_cast<uint4*>(cast_to), n / 8, static_cast<int>(f->f16)));
  return 0;
}

}  // namespace trimul

using namespace trimul;

extern "C" {

int b200_block_join_forward(const void* x, const void* u, const void* gate, const uint8_t* mask, const float* scale, const float* post_w,
                            const float* post_b, const float* pre_w, const float* pre_b, void* y, void* h, float* post_stats,
                            float* pre_stats, long long rows, int d, long long gate_rows, int dtype, int post_kind, int pre_kind,
                            float post_eps, float pre_eps, void* cuda_stream) {
  int rc = check_join(rows, d, gate_rows, dtype, post_kind, pre_kind);
  if (rc != 0) return rc;
  if (rows == 0) return B200_TRIMUL_OK;
  if (x == nullptr || (u != nullptr) != (y != nullptr) || (pre_kind != kNormNone) != (h != nullptr)) return B200_TRIMUL_E_NULL;
  if (u == nullptr && (pre_kind == kNormNone || post_kind != kNormNone || gate != nullptr || mask != nullptr || scale != nullptr))
    return B200_TRIMUL_E_NULL;
  DeviceInfo info;
  rc = device_info(&info);
  if (rc != 0) return rc;
  JoinParams p = {};
  p.x = x;
  p.u = u;
  p.gate = gate;
  p.mask = mask;
  p.scale = scale;
  p.post_w = post_kind != kNormNone ? post_w : nullptr;  // (parameters of a norm that is not there are not read)
  p.post_b = post_kind != kNormNone ? post_b : nullptr;
  p.pre_w = pre_kind != kNormNone ? pre_w : nullptr;
  p.pre_b = pre_kind != kNormNone ? pre_b : nullptr;
  p.y = y;
  p.h = h;
  p.post_stats = reinterpret_cast<float2*>(post_stats);
  p.pre_stats = reinterpret_cast<float2*>(pre_stats);
  p.rows = rows;
  p.gate_rows = gate_rows;
  p.d = d;
  p.post_kind = post_kind;
  p.pre_kind = pre_kind;
  p.post_eps = post_eps;
  p.pre_eps = pre_eps;
  const int size = dtype == B200_BLOCKS_F32 ? 4 : 2;
  if (!aligned(x, size) || !aligned(u, size) || !aligned(gate, size) || !aligned(y, size) || !aligned(h, size) ||
      !aligned(post_stats, 8) || !aligned(pre_stats, 8))
    return B200_TRIMUL_E_ALIGN;
  const cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  if (dtype == B200_BLOCKS_BF16) return launch_join_forward<__nv_bfloat16>(p, info, stream);
  if (dtype == B200_BLOCKS_F16) return launch_join_forward<__half>(p, info, stream);
  return launch_join_forward<float>(p, info, stream);
}

int b200_block_join_workspace_bytes(long long rows, int d, long long gate_rows, size_t* out_bytes) {
  if (out_bytes == nullptr) return B200_TRIMUL_E_NULL;
  const int rc = check_join(rows, d, gate_rows, 0, 0, 0);
  if (rc != 0) return rc;
  *out_bytes = join_sums_bytes(d);
  if (gate_rows > 1) {
    const int team = join_backward_team(d);
    // the kernels of join.cuh: two gate rows a team; on tiles: the gate rows that the blocks' rows touch (see launch_join_backward)
    const size_t plain = static_cast<size_t>(kMaxSms) * (kJoinBackwardThreads / team) * 2 * 8 * team * 4;
    const long long most = gate_rows >= kSharedGateRows ? 2 * (rows + kTileRounds * kTileWarps * 32 + 16) / gate_rows + 3 * kMaxSms : 0;
    *out_bytes += std::max(plain, static_cast<size_t>(most) * (kTileWarps * 32 / team) * 8 * team * 4);
  }
  return B200_TRIMUL_OK;
}

int b200_block_join_backward(const void* dy, const void* dh, const void* x, const void* u, const void* gate, const uint8_t* mask,
                             const float* scale, const float* post_w, const float* post_b, const float* pre_w, const float* pre_b,
                             const float* post_stats, const float* pre_stats, void* dx, void* du, void* dgate, float* d_scale,
                             float* d_post_w, float* d_post_b, float* d_pre_w, float* d_pre_b, void* workspace, size_t workspace_bytes,
                             long long rows, int d, long long gate_rows, int dtype, int post_kind, int pre_kind, void* cuda_stream) {
  int rc = check_join(rows, d, gate_rows, dtype, post_kind, pre_kind);
  if (rc != 0) return rc;
  const cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  if (rows == 0) {
    for (float* s : {d_scale, d_post_w, d_post_b, d_pre_w, d_pre_b})
      if (s != nullptr) TRIMUL_CUDA(cudaMemsetAsync(s, 0, static_cast<size_t>(d) * 4, stream));
    return B200_TRIMUL_OK;
  }
  if (x == nullptr || workspace == nullptr || (post_kind != kNormNone && post_stats == nullptr) || (pre_kind != kNormNone && pre_stats == nullptr))
    return B200_TRIMUL_E_NULL;
  if (u == nullptr && (pre_kind == kNormNone || post_kind != kNormNone || gate != nullptr || mask != nullptr || scale != nullptr))
    return B200_TRIMUL_E_NULL;
  // (sums of a block's output or of a norm that is not there: no kernel forms them)
  if ((u == nullptr && (d_scale != nullptr || d_post_w != nullptr || d_post_b != nullptr)) ||
      (post_kind == kNormNone && (d_post_w != nullptr || d_post_b != nullptr)))
    return B200_TRIMUL_E_NULL;
  if ((pre_kind == kNormNone && dh != nullptr) || (u == nullptr && (dy != nullptr || du != nullptr)) || (gate == nullptr && dgate != nullptr))
    return B200_TRIMUL_E_NULL;
  if (!aligned(workspace, 1024)) return B200_TRIMUL_E_ALIGN;
  size_t need = 0;
  rc = b200_block_join_workspace_bytes(rows, d, gate_rows, &need);
  if (rc != 0) return rc;
  if (workspace_bytes < need) return B200_TRIMUL_E_WORKSPACE;
  DeviceInfo info;
  rc = device_info(&info);
  if (rc != 0) return rc;
  const JoinGrid g = join_backward_grid(rows, d, gate != nullptr && gate_rows > 1, std::min(info.sms, kMaxSms));
  JoinParams p = {};
  p.x = x;
  p.u = u;
  p.gate = gate;
  p.mask = mask;
  p.scale = scale;
  p.post_w = post_kind != kNormNone ? post_w : nullptr;  // (parameters of a norm that is not there are not read)
  p.post_b = post_kind != kNormNone ? post_b : nullptr;
  p.pre_w = pre_kind != kNormNone ? pre_w : nullptr;
  p.pre_b = pre_kind != kNormNone ? pre_b : nullptr;
  p.post_stats = reinterpret_cast<float2*>(const_cast<float*>(post_stats));
  p.pre_stats = reinterpret_cast<float2*>(const_cast<float*>(pre_stats));
  p.dy = dy;
  p.dh = dh;
  p.dx = dx;
  p.du = du;
  p.dgate = dgate;
  p.rows = rows;
  p.gate_rows = gate_rows;
  p.rows_per_team = g.rows_per_team;
  p.d = d;
  p.team = g.team;
  p.post_kind = post_kind;
  p.pre_kind = pre_kind;
  JoinSums sums = {};
  float* const outs[5] = {d_scale, d_post_w, d_post_b, d_pre_w, d_pre_b};
  bool any = false;
  for (int i = 0; i < 5; ++i) {
    sums.out[i] = outs[i];
    any = any || outs[i] != nullptr;
  }
  p.sums = any ? static_cast<float*>(workspace) : nullptr;
  p.gate_part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + join_sums_bytes(d));
  sums.sums = p.sums;
  sums.blocks = g.blocks;
  sums.d = d;
  const int size = dtype == B200_BLOCKS_F32 ? 4 : 2;
  for (const void* q : {x, u, gate, dy, dh, static_cast<const void*>(dx), static_cast<const void*>(du), static_cast<const void*>(dgate)})
    if (!aligned(q, size)) return B200_TRIMUL_E_ALIGN;
  if (!aligned(post_stats, 8) || !aligned(pre_stats, 8)) return B200_TRIMUL_E_ALIGN;
  const bool wide = d % 8 == 0 && all_aligned16({x, u, gate, dy, dh, dx, du, dgate});
  if (dtype == B200_BLOCKS_BF16) return launch_join_backward<__nv_bfloat16>(p, wide, g, sums, info, stream);
  if (dtype == B200_BLOCKS_F16) return launch_join_backward<__half>(p, wide, g, sums, info, stream);
  return launch_join_backward<float>(p, wide, g, sums, info, stream);
}

int b200_ff_workspace_bytes(long long rows, int d, int hidden, int weight_dtype, int backward, size_t* out_bytes) {
  if (out_bytes == nullptr) return B200_TRIMUL_E_NULL;
  const int rc = check_ff(rows, d, hidden, weight_dtype);
  if (rc != 0) return rc;
  *out_bytes = std::max<size_t>(ff_regions(rows, d, hidden, weight_dtype, backward != 0).total, 1024);
  return B200_TRIMUL_OK;
}

int b200_ff_kept_bytes(long long rows, int d, int hidden, size_t* out_bytes) {
  if (out_bytes == nullptr) return B200_TRIMUL_E_NULL;
  const int rc = check_ff(rows, d, hidden, 0);
  if (rc != 0) return rc;
  *out_bytes = ff_kept_bytes(rows, d, hidden);
  return B200_TRIMUL_OK;
}

int b200_ff_forward(const void* x, const void* w_a, const void* w_b, const void* w_s, void* y, void* kept, void* workspace,
                    size_t workspace_bytes, long long rows, int d, int hidden, int dtype, int weight_dtype, int activation, void* cuda_stream) {
  int rc = check_ff(rows, d, hidden, weight_dtype, dtype);
  if (rc != 0) return rc;
  if (weight_dtype != B200_BLOCKS_F32 && weight_dtype != dtype) return B200_TRIMUL_E_UNSUPPORTED;
  if (activation != B200_ACT_SILU && activation != B200_ACT_GELU) return B200_TRIMUL_E_UNSUPPORTED;
  if (rows == 0) return B200_TRIMUL_OK;
  if (x == nullptr || w_a == nullptr || w_b == nullptr || w_s == nullptr || y == nullptr || workspace == nullptr) return B200_TRIMUL_E_NULL;
  if (!all_aligned16({x, w_a, w_b, w_s, y}) || !aligned(workspace, 1024) || !aligned(kept, 1024)) return B200_TRIMUL_E_ALIGN;
  FfProblem f;
  rc = ff_device(&f.info);
  if (rc != 0) return rc;
  const FfRegions r = ff_regions(rows, d, hidden, weight_dtype, false);
  if (workspace_bytes < r.total) return B200_TRIMUL_E_WORKSPACE;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  rc = ff_problem(&f, w_a, w_b, w_s, rows, d, hidden, dtype, weight_dtype, activation, ws + r.weights, cuda_stream);
  if (rc != 0) return rc;
  const size_t keep = kept != nullptr ? ff_kept_bytes(rows, d, hidden) / 3 : 0;
  if (keep != 0) {
    uint8_t* k = static_cast<uint8_t*>(kept);
    void* const all[3] = {k, nullptr, nullptr};
    void* const ab[2] = {k + keep, k + 2 * keep};
    rc = ff_hidden(f, x, nullptr, all, ab);
    return rc != 0 ? rc : ff_project(f, k, nullptr, y);
  }
  void* const out[3] = {ws + r.hidden[0], nullptr, nullptr};
  if (ff_narrow(rows, d, f.info.sms)) return ff_narrow_forward(f, x, y);
  if (ff_vec(rows, d)) return f.f16 ? ff_vec_forward<true>(f, x, out[0], y) : ff_vec_forward<false>(f, x, out[0], y);
  rc = ff_hidden(f, x, nullptr, out);
  return rc != 0 ? rc : ff_project(f, out[0], nullptr, y);
}

int b200_ff_backward(const void* dy, const void* x, const void* w_a, const void* w_b, const void* w_s, const void* kept, void* dx, void* dw_a, void* dw_b,
                     void* dw_s, void* workspace, size_t workspace_bytes, long long rows, int d, int hidden, int dtype, int weight_dtype,
                     int activation, void* cuda_stream) {
  int rc = check_ff(rows, d, hidden, weight_dtype, dtype);
  if (rc != 0) return rc;
  if (weight_dtype != B200_BLOCKS_F32 && weight_dtype != dtype) return B200_TRIMUL_E_UNSUPPORTED;
  if (activation != B200_ACT_SILU && activation != B200_ACT_GELU) return B200_TRIMUL_E_UNSUPPORTED;
  const size_t weight_bytes = static_cast<size_t>(hidden) * d * (weight_dtype == B200_BLOCKS_F32 ? 4 : 2);
  if (rows == 0) {
    for (void* w : {dw_a, dw_b, dw_s})
      if (w != nullptr) TRIMUL_CUDA(cudaMemsetAsync(w, 0, weight_bytes, static_cast<cudaStream_t>(cuda_stream)));
    return B200_TRIMUL_OK;
  }
  if (dy == nullptr || x == nullptr || w_a == nullptr || w_b == nullptr || w_s == nullptr || workspace == nullptr) return B200_TRIMUL_E_NULL;
  if (!all_aligned16({dy, x, w_a, w_b, w_s, dx, dw_a, dw_b, dw_s}) || !aligned(workspace, 1024) || !aligned(kept, 1024)) return B200_TRIMUL_E_ALIGN;
  FfProblem f;
  rc = ff_device(&f.info);
  if (rc != 0) return rc;
  const FfRegions r = ff_regions(rows, d, hidden, weight_dtype, true);
  if (workspace_bytes < r.total) return B200_TRIMUL_E_WORKSPACE;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  rc = ff_problem(&f, w_a, w_b, w_s, rows, d, hidden, dtype, weight_dtype, activation, ws + r.weights, cuda_stream);
  if (rc != 0) return rc;
  void* hidden3[3] = {ws + r.hidden[0], ws + r.hidden[1], ws + r.hidden[2]};
  const size_t keep = kept != nullptr ? ff_kept_bytes(rows, d, hidden) / 3 : 0;
  if (keep != 0) {
    uint8_t* k = static_cast<uint8_t*>(const_cast<void*>(kept));
    const void* const ab[2] = {k + keep, k + 2 * keep};
    hidden3[2] = k;
    rc = ff_grad(f, dy, ab, hidden3[0], hidden3[1]);
  } else {
    rc = ff_hidden(f, x, dy, hidden3);
  }
  if (rc == 0 && dx != nullptr) rc = ff_project(f, hidden3[0], hidden3[1], dx);
  if (rc == 0 && (dw_a != nullptr || dw_b != nullptr || dw_s != nullptr))
    rc = ff_weight_gradients(f, x, dy, hidden3, reinterpret_cast<float*>(ws + r.partial), dw_a, dw_b, dw_s, weight_dtype);
  return rc;
}

int b200_blocks_read_status(void* cuda_stream, int* code) {
  if (code == nullptr) return B200_TRIMUL_E_NULL;
  const cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  *code = 0;
  TRIMUL_CUDA(cudaMemcpyFromSymbolAsync(code, blocks_status, sizeof(int), 0, cudaMemcpyDeviceToHost, stream));
  TRIMUL_CUDA(cudaStreamSynchronize(stream));
  if (*code != 0) {
    const int zero = 0;
    TRIMUL_CUDA(cudaMemcpyToSymbolAsync(blocks_status, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, stream));
    TRIMUL_CUDA(cudaStreamSynchronize(stream));
  }
  return B200_TRIMUL_OK;
}

}  // extern "C"
