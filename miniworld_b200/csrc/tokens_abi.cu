// C-ABI entry points of the token operators (see include/b200_tokens.h): argument checks, the choice of a variant and launches; all
// arithmetic is in the kernels.
#include "../../include/b200_tokens.h"

#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include "attention_backward.cuh"
#include "attention_forward.cuh"
#include "dropout.cuh"
#include "host_util.cuh"
#include "position.cuh"

namespace trimul {

static size_t up(size_t v, size_t a) { return (v + a - 1) / a * a; }
static long long blocks_for(long long n, long long b) { return (n + b - 1) / b; }
static size_t size_of(int dtype) { return dtype == B200_BLOCKS_F32 ? 4 : 2; }
static bool all_aligned16(std::initializer_list<const void*> ps) {
  for (const void* q : ps)
    if (!aligned(q, 16)) return false;
  return true;
}
// As many as an SM's memory is planned for
constexpr int kMaxSms = 160;
static int tokens_device(DeviceInfo* info) {
  const int rc = device_info(info);
  if (rc != 0) return rc;
  info->sms = std::min(info->sms, kMaxSms);
  TRIMUL_CUDA(cudaSetDevice(info->device));  // (a thread that has not used the GPU yet has no context)
  return B200_TRIMUL_OK;
}

// ---------------------------------------------------------------- attention
static int check_attention(const b200_attention_call* c) {
  if (c == nullptr) return B200_TRIMUL_E_NULL;
  if (c->rows < 0 || c->rows > 0x7FFFFFFFll - 1024 || c->sequences < 0 || c->heads < 1 || c->kv_heads < 1 || c->heads % c->kv_heads != 0) return B200_TRIMUL_E_SHAPE;
  if (c->offsets == nullptr && (c->length < 0 || static_cast<long long>(c->sequences) * c->length != c->rows)) return B200_TRIMUL_E_SHAPE;
  if (c->offsets != nullptr && c->sequences < 1) return B200_TRIMUL_E_SHAPE;
  if (c->d < 8 || c->d > B200_ATTENTION_MAX_WIDTH || c->d % 8 != 0 || c->heads > 32768) return B200_TRIMUL_E_UNSUPPORTED;
  if (c->dtype != B200_BLOCKS_BF16 && c->dtype != B200_BLOCKS_F16) return B200_TRIMUL_E_UNSUPPORTED;
  if (c->rows * c->heads > (1ll << 40) / c->d) return B200_TRIMUL_E_SHAPE;
  if (attention_places(c->offsets, c->rows, c->sequences, c->length, kAtTile) * c->heads > 0x7FFFFFFFll) return B200_TRIMUL_E_SHAPE;  // (blocks)
  if (!(c->scale == c->scale) || c->scale - c->scale != 0.f) return B200_TRIMUL_E_UNSUPPORTED;
  if (c->table != nullptr) {
    if (c->bucket_of == nullptr) return B200_TRIMUL_E_NULL;
    if (c->buckets < 1 || c->reach < 0) return B200_TRIMUL_E_SHAPE;
    if (c->buckets > B200_POSITION_MAX_BUCKETS || c->reach > B200_POSITION_MAX_REACH) return B200_TRIMUL_E_UNSUPPORTED;
    if (c->table_dtype != c->dtype && c->table_dtype != B200_BLOCKS_F32) return B200_TRIMUL_E_UNSUPPORTED;
  }
  return B200_TRIMUL_OK;
}
static int check_attention_tensor(const b200_attention_tensor* t) {
  if (t == nullptr || t->data == nullptr) return B200_TRIMUL_E_NULL;
  if (!aligned(t->data, 16) || t->row_stride % 8 != 0 || t->head_stride % 8 != 0) return B200_TRIMUL_E_ALIGN;
  return t->row_stride < 0 || t->head_stride < 0 ? B200_TRIMUL_E_SHAPE : B200_TRIMUL_OK;
}
static AttentionTensor attention_tensor(const b200_attention_tensor* t) { return {t->data, t->row_stride, t->head_stride}; }
static AttentionParams attention_params(const b200_attention_call* c, const b200_attention_tensor* q, const b200_attention_tensor* k,
                                        const b200_attention_tensor* v) {
  AttentionParams p = {};
  p.q = attention_tensor(q);
  p.k = attention_tensor(k);
  p.v = attention_tensor(v);
  p.offsets = c->offsets;
  p.mask = c->mask;
  p.table = c->table;
  p.bucket_of = c->bucket_of;
  p.rows = c->rows;
  p.sequences = c->sequences;
  p.length = c->length;
  p.heads = c->heads;
  p.kv_heads = c->kv_heads;
  p.d = c->d;
  p.buckets = c->buckets;
  p.reach = c->table != nullptr ? c->reach : 0;
  p.causal = c->causal != 0;
  p.wide_table = c->table_dtype == B200_BLOCKS_F32;
  p.scale = c->scale;
  return p;
}
// [rows][heads][d] in boxes of 128 rows of 64 elements
static int attention_map(CUtensorMap* m, const AttentionTensor& t, long long rows, int heads, int d) {
  const uint64_t dims[3] = {static_cast<uint64_t>(d), static_cast<uint64_t>(heads), static_cast<uint64_t>(rows)};
  const uint64_t strides[2] = {static_cast<uint64_t>(heads == 1 ? d : t.head) * 2, static_cast<uint64_t>(rows == 1 ? static_cast<long long>(heads) * d : t.row) * 2};
  const uint32_t box[3] = {64, 1, kAtTile};
  return make_map(m, t.base, 3, dims, strides, box);
}
// The warps that take registers wait until others have given them up: the sum of their shares must be what the block is launched with,
// whatever the compiler has made of the launch bounds (asked once a kernel).
template <auto KERNEL, int WARPGROUPS, int MANY, int FEW>
static int check_registers() {
  static const int registers = [] {
    cudaFuncAttributes a = {};
    return cudaFuncGetAttributes(&a, KERNEL) == cudaSuccess ? a.numRegs : 0;
  }();
  return registers * WARPGROUPS >= (WARPGROUPS - 1) * MANY + FEW ? B200_TRIMUL_OK : B200_TRIMUL_E_UNSUPPORTED;
}
template <bool F16, int HALVES>
static int launch_attention_forward(const AttentionMaps& maps, AttentionParams p, const DeviceInfo& info, cudaStream_t stream) {
  using C = AtForward<HALVES>;
  const auto kernel = attention_forward_kernel<F16, HALVES>;
  int rc = set_smem(kernel, C::smem(true, B200_POSITION_MAX_REACH), info.device);
  if (rc == 0) rc = check_registers<attention_forward_kernel<F16, HALVES>, C::kThreads / 128, C::kMany, C::kFew>();
  if (rc != 0) return rc;
  p.places = attention_places(p.offsets, p.rows, p.sequences, p.length, C::kTiles * kAtTile);
  TRIMUL_CUDA(launch_overlapped(kernel, dim3(static_cast<unsigned>(p.places * p.heads)), C::kThreads, C::smem(p.table != nullptr, p.reach), stream, maps, p));
  return B200_TRIMUL_OK;
}
static int attention_delta_blocks(long long rows, int d) {
  int team = 1;
  while (team * 8 < d) team *= 2;
  return static_cast<int>(std::min<long long>(kAtDeltaBlocks, blocks_for(rows, kAtDeltaThreads / team)));
}
template <bool F16, int HALVES>
static int launch_attention_backward(const AttentionMaps& maps, const AttentionParams& p, const DeviceInfo& info, cudaStream_t stream) {
  using T = std::conditional_t<F16, __half, __nv_bfloat16>;
  const auto dq = attention_dq_kernel<F16, HALVES>;
  const auto dkv = attention_dkv_kernel<F16, HALVES>;
  int rc = set_smem(dq, AtDq<HALVES>::smem(true, B200_POSITION_MAX_REACH), info.device);
  if (rc == 0) rc = set_smem(dkv, AtDkv<HALVES>::smem(true, B200_POSITION_MAX_REACH), info.device);
  if (rc == 0) rc = check_registers<attention_dq_kernel<F16, HALVES>, kAtBackThreads / 128, kAtBackMany, kAtBackFew>();
  if (rc == 0) rc = check_registers<attention_dkv_kernel<F16, HALVES>, kAtBackThreads / 128, kAtBackMany, kAtBackFew>();
  if (rc != 0) return rc;
  const bool table = p.table != nullptr;
  TRIMUL_CUDA(launch_overlapped(attention_delta_kernel<T>, dim3(p.delta_blocks, p.kv_heads), kAtDeltaThreads, 0, stream, p));
  TRIMUL_CUDA(launch_overlapped(dq, dim3(static_cast<unsigned>(p.places * p.heads)), kAtBackThreads, AtDq<HALVES>::smem(table, p.reach), stream, maps, p));
  TRIMUL_CUDA(launch_overlapped(dkv, dim3(static_cast<unsigned>(p.places * p.kv_heads)), kAtBackThreads, AtDkv<HALVES>::smem(table, p.reach), stream, maps, p));
  if (p.partial != nullptr)
    TRIMUL_CUDA(launch_overlapped(p.wide_table ? attention_table_kernel<float> : attention_table_kernel<T>, dim3(p.heads), 1024, 0, stream, p));
  return B200_TRIMUL_OK;
}
struct AttentionRegions {
  size_t delta, most, partial, total;
};
static AttentionRegions attention_regions(const b200_attention_call* c) {
  AttentionRegions r;
  r.delta = 0;
  r.most = up(static_cast<size_t>(c->rows) * c->heads * 4, 1024);
  r.partial = r.most + up(static_cast<size_t>(c->kv_heads) * attention_delta_blocks(c->rows, c->d) * 8, 1024);
  const size_t places = static_cast<size_t>(attention_places(c->offsets, c->rows, c->sequences, c->length, kAtTile));
  r.total = r.partial + (c->table != nullptr ? up(places * c->heads * (2 * c->reach + 1) * 4, 1024) : 0);
  return r;
}

// ---------------------------------------------------------------- relative position
static int check_position(int b, int n, int c, int buckets) {
  if (b < 0 || n < 0 || c < 1 || buckets < 1) return B200_TRIMUL_E_SHAPE;
  if (buckets > B200_POSITION_MAX_BUCKETS || c > B200_NORM_MAX_WIDTH) return B200_TRIMUL_E_UNSUPPORTED;
  return static_cast<long long>(b) * n > 0x7FFFFFFFll || static_cast<double>(b) * n * n * c > 0x1p40 ? B200_TRIMUL_E_SHAPE : B200_TRIMUL_OK;
}
constexpr size_t kPositionSmem = 220 * 1024;
struct PositionGrid {
  int warps, chunks, blocks;
};
// As many warps to a block as tables of sums fit into shared memory, up to 13; blocks: one an SM in all chunks together, and no more than
// there is work for.
static PositionGrid position_grid(int b, int n, int c, int buckets, int sms) {
  PositionGrid g;
  g.warps = static_cast<int>(std::min<size_t>(kPositionWarps, kPositionSmem / (static_cast<size_t>(buckets) * kPositionChunk * 4)));
  g.chunks = static_cast<int>(blocks_for(c, kPositionChunk));
  const long long units = static_cast<long long>(b) * n * blocks_for(n, 32);
  g.blocks = static_cast<int>(std::max<long long>(1, std::min<long long>(std::max(1, sms / g.chunks), blocks_for(units, g.warps))));
  return g;
}
static size_t position_bytes(const PositionGrid& g, int buckets) {
  return up(static_cast<size_t>(g.chunks) * g.blocks * buckets * kPositionChunk * 4, 1024);
}

template <typename T, int V>
static int launch_position_forward(PositionParams p, const DeviceInfo& info, cudaStream_t stream) {
  const long long cells = static_cast<long long>(p.b) * p.n * p.n;
  const int pieces = p.c / V;
  // tiles of about 64 KB, smaller where that leaves SMs without one
  long long tile = std::max<long long>(1, std::min<long long>(kPositionMostCells, 65536 / (static_cast<long long>(p.c) * sizeof(T))));
  while (tile > 8 && blocks_for(cells, tile) < 4ll * info.sms) tile /= 2;
  p.cells = static_cast<int>(tile);
  p.magic = pieces == 1 ? 0 : static_cast<uint32_t>(((1ull << 32) + pieces - 1) / pieces);
  // the table in shared memory where a block reads it often enough to have it copied
  const size_t table = static_cast<size_t>(p.buckets) * p.c * 4;
  p.table_in_smem = table <= 100 * 1024 && cells / (4 * info.sms) > 2 * p.buckets;
  const int smem = p.table_in_smem ? static_cast<int>(table) : 0;
  const int per_sm = table <= 50 * 1024 || !p.table_in_smem ? 4 : 2;
  const auto kernel = position_forward_kernel<T, V>;
  const int rc = set_smem(kernel, 100 * 1024, info.device);
  if (rc != 0) return rc;
  TRIMUL_CUDA(launch_overlapped(kernel, dim3(static_cast<unsigned>(std::min<long long>(blocks_for(cells, tile), per_sm * info.sms))), kPositionThreads, smem, stream, p));
  return B200_TRIMUL_OK;
}
template <typename T>
static int position_forward(const PositionParams& p, const DeviceInfo& info, cudaStream_t stream) {
  constexpr int kWhole = 16 / sizeof(T);
  auto fits = [&](int v) { return p.c % v == 0 && aligned(p.z, v * sizeof(T)) && aligned(p.y, v * sizeof(T)) && aligned(p.table, std::min(v, 4) * 4); };
  if (fits(kWhole)) return launch_position_forward<T, kWhole>(p, info, stream);
  if (fits(kWhole / 2)) return launch_position_forward<T, kWhole / 2>(p, info, stream);
  if constexpr (kWhole / 4 > 1)
    if (fits(kWhole / 4)) return launch_position_forward<T, kWhole / 4>(p, info, stream);
  return launch_position_forward<T, 1>(p, info, stream);
}
template <typename T>
static int position_backward(const PositionParams& p, const PositionGrid& g, const DeviceInfo& info, cudaStream_t stream) {
  const auto kernel = p.c % 2 == 0 && aligned(p.dy, 2 * sizeof(T)) ? position_backward_kernel<T, 2> : position_backward_kernel<T, 1>;
  const int smem = g.warps * p.buckets * kPositionChunk * 4;
  const int rc = set_smem(kernel, kPositionSmem, info.device);
  if (rc != 0) return rc;
  TRIMUL_CUDA(launch_overlapped(kernel, dim3(g.chunks * g.blocks), g.warps * 32, smem, stream, p));
  TRIMUL_CUDA(launch_overlapped(position_sums_kernel, dim3(p.buckets, g.chunks), 256, 0, stream, p));
  return B200_TRIMUL_OK;
}

// ---------------------------------------------------------------- dropout
template <typename T>
static int dropout(DropoutParams p, const DeviceInfo& info, cudaStream_t stream) {
  const bool residual = p.x != nullptr, whole = all_aligned16({p.x, p.u, p.y});
  const long long n = p.outer * p.inner, groups = blocks_for(n, 8);
  if (whole && p.shared == 1) {
    const auto kernel = residual ? dropout_kernel<T, true> : dropout_kernel<T, false>;
    TRIMUL_CUDA(launch_overlapped(kernel, dim3(static_cast<unsigned>(blocks_for(groups, kDropoutThreads * kDropoutFlight))), kDropoutThreads, 0, stream, p));
    return B200_TRIMUL_OK;
  }
  const bool eights = whole && p.inner % 8 == 0;
  const long long threads = eights ? groups : n;
  // rows that share a mask are cut into runs, as long as there are enough threads to fill the GPU
  p.chunk = std::max<long long>(std::min<long long>(p.shared, 8), blocks_for(p.shared * threads, 2048ll * info.sms));
  p.chunk = std::max(p.chunk, blocks_for(p.shared, 65535));
  const dim3 grid(static_cast<unsigned>(std::min<long long>(blocks_for(threads, kDropoutThreads), 1 << 30)), static_cast<unsigned>(blocks_for(p.shared, p.chunk)));
  void (*kernel)(DropoutParams) = eights ? (residual ? dropout_shared_kernel<T, true> : dropout_shared_kernel<T, false>)
                                         : (residual ? dropout_single_kernel<T, true> : dropout_single_kernel<T, false>);
  TRIMUL_CUDA(launch_overlapped(kernel, grid, kDropoutThreads, 0, stream, p));
  return B200_TRIMUL_OK;
}

}  // namespace trimul

using namespace trimul;

extern "C" {

int b200_token_attention_forward(const b200_attention_call* call, const b200_attention_tensor* q, const b200_attention_tensor* k,
                                 const b200_attention_tensor* v, void* o, void* rest, float* lse, void* cuda_stream) {
  int rc = check_attention(call);
  if (rc != 0) return rc;
  if (call->rows == 0) return B200_TRIMUL_OK;
  for (const b200_attention_tensor* t : {q, k, v})
    if ((rc = check_attention_tensor(t)) != 0) return rc;
  if (o == nullptr || (rest == nullptr) != (lse == nullptr)) return B200_TRIMUL_E_NULL;
  if (!all_aligned16({o, rest})) return B200_TRIMUL_E_ALIGN;
  DeviceInfo info;
  if ((rc = tokens_device(&info)) != 0) return rc;
  AttentionParams p = attention_params(call, q, k, v);
  p.o = o;
  p.rest = rest;
  p.lse = lse;
  AttentionMaps maps = {};
  rc = attention_map(&maps.q, p.q, p.rows, p.heads, p.d);
  if (rc == 0) rc = attention_map(&maps.k, p.k, p.rows, p.kv_heads, p.d);
  if (rc == 0) rc = attention_map(&maps.v, p.v, p.rows, p.kv_heads, p.d);
  if (rc != 0) return rc;
  const cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  if (call->dtype == B200_BLOCKS_F16) return p.d <= 64 ? launch_attention_forward<true, 1>(maps, p, info, stream) : launch_attention_forward<true, 2>(maps, p, info, stream);
  return p.d <= 64 ? launch_attention_forward<false, 1>(maps, p, info, stream) : launch_attention_forward<false, 2>(maps, p, info, stream);
}

int b200_token_attention_workspace_bytes(const b200_attention_call* call, size_t* out_bytes) {
  if (out_bytes == nullptr) return B200_TRIMUL_E_NULL;
  const int rc = check_attention(call);
  if (rc != 0) return rc;
  *out_bytes = std::max<size_t>(attention_regions(call).total, 1024);
  return B200_TRIMUL_OK;
}

int b200_token_attention_backward(const b200_attention_call* call, const b200_attention_tensor* q, const b200_attention_tensor* k,
                                  const b200_attention_tensor* v, const void* o, const void* rest, const float* lse,
                                  const b200_attention_tensor* d_o, void* dq,
                                  void* dk, void* dv, void* dtable, void* workspace, size_t workspace_bytes, void* cuda_stream) {
  int rc = check_attention(call);
  if (rc != 0) return rc;
  const cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  if (dtable != nullptr && call->table == nullptr) return B200_TRIMUL_E_NULL;
  if (call->rows == 0) {
    if (dtable != nullptr)
      TRIMUL_CUDA(cudaMemsetAsync(dtable, 0, static_cast<size_t>(call->buckets) * call->heads * size_of(call->table_dtype), stream));
    return B200_TRIMUL_OK;
  }
  for (const b200_attention_tensor* t : {q, k, v, d_o})
    if ((rc = check_attention_tensor(t)) != 0) return rc;
  if (o == nullptr || rest == nullptr || lse == nullptr || dq == nullptr || dk == nullptr || dv == nullptr || workspace == nullptr) return B200_TRIMUL_E_NULL;
  if (!all_aligned16({o, rest, dq, dk, dv}) || !aligned(workspace, 1024)) return B200_TRIMUL_E_ALIGN;
  const AttentionRegions regions = attention_regions(call);
  if (workspace_bytes < (dtable != nullptr ? regions.total : regions.partial)) return B200_TRIMUL_E_WORKSPACE;
  DeviceInfo info;
  if ((rc = tokens_device(&info)) != 0) return rc;
  AttentionParams p = attention_params(call, q, k, v);
  p.dout = attention_tensor(d_o);
  p.o = const_cast<void*>(o);
  p.rest = const_cast<void*>(rest);
  p.lse = const_cast<float*>(lse);
  p.dq = dq;
  p.dk = dk;
  p.dv = dv;
  p.dtable = dtable;
  uint8_t* const ws = static_cast<uint8_t*>(workspace);
  p.delta = reinterpret_cast<float*>(ws + regions.delta);
  p.most = reinterpret_cast<float*>(ws + regions.most);
  p.partial = dtable != nullptr ? reinterpret_cast<float*>(ws + regions.partial) : nullptr;
  p.places = attention_places(p.offsets, p.rows, p.sequences, p.length, kAtTile);
  p.delta_blocks = attention_delta_blocks(p.rows, p.d);
  AttentionMaps maps = {};
  rc = attention_map(&maps.q, p.q, p.rows, p.heads, p.d);
  if (rc == 0) rc = attention_map(&maps.k, p.k, p.rows, p.kv_heads, p.d);
  if (rc == 0) rc = attention_map(&maps.v, p.v, p.rows, p.kv_heads, p.d);
  if (rc == 0) rc = attention_map(&maps.dout, p.dout, p.rows, p.heads, p.d);
  if (rc != 0) return rc;
  if (call->dtype == B200_BLOCKS_F16) return p.d <= 64 ? launch_attention_backward<true, 1>(maps, p, info, stream) : launch_attention_backward<true, 2>(maps, p, info, stream);
  return p.d <= 64 ? launch_attention_backward<false, 1>(maps, p, info, stream) : launch_attention_backward<false, 2>(maps, p, info, stream);
}

int b200_relative_position_forward(const void* z, const float* table, const void* index, const void* chain, const int* bucket_of, void* y,
                                   int b, int n, int c, int buckets, int reach, int wide, int dtype, void* cuda_stream) {
  int rc = check_position(b, n, c, buckets);
  if (rc != 0) return rc;
  if (reach < 0) return B200_TRIMUL_E_SHAPE;
  if (reach > B200_POSITION_MAX_REACH || dtype < 0 || dtype > 2) return B200_TRIMUL_E_UNSUPPORTED;
  if (b == 0 || n == 0) return B200_TRIMUL_OK;
  if (z == nullptr || table == nullptr || index == nullptr || bucket_of == nullptr || y == nullptr) return B200_TRIMUL_E_NULL;
  DeviceInfo info;
  if ((rc = tokens_device(&info)) != 0) return rc;
  PositionParams p = {};
  p.z = z;
  p.table = table;
  p.index = index;
  p.chain = chain;
  p.bucket_of = bucket_of;
  p.y = y;
  p.b = b;
  p.n = n;
  p.c = c;
  p.buckets = buckets;
  p.reach = reach;
  p.wide = wide != 0;
  const cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  if (dtype == B200_BLOCKS_BF16) return position_forward<__nv_bfloat16>(p, info, stream);
  if (dtype == B200_BLOCKS_F16) return position_forward<__half>(p, info, stream);
  return position_forward<float>(p, info, stream);
}

int b200_relative_position_workspace_bytes(int b, int n, int c, int buckets, size_t* out_bytes) {
  if (out_bytes == nullptr) return B200_TRIMUL_E_NULL;
  const int rc = check_position(b, n, c, buckets);
  if (rc != 0) return rc;
  *out_bytes = position_bytes(position_grid(b, n, c, buckets, kMaxSms), buckets);
  return B200_TRIMUL_OK;
}

int b200_relative_position_backward(const void* dy, const void* index, const void* chain, const int* bucket_of, float* dtable,
                                    void* workspace, size_t workspace_bytes, int b, int n, int c, int buckets, int reach, int wide,
                                    int dtype, void* cuda_stream) {
  int rc = check_position(b, n, c, buckets);
  if (rc != 0) return rc;
  if (reach < 0) return B200_TRIMUL_E_SHAPE;
  if (reach > B200_POSITION_MAX_REACH || dtype < 0 || dtype > 2) return B200_TRIMUL_E_UNSUPPORTED;
  if (dtable == nullptr) return B200_TRIMUL_E_NULL;
  const cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  if (b == 0 || n == 0) {
    TRIMUL_CUDA(cudaMemsetAsync(dtable, 0, static_cast<size_t>(buckets) * c * 4, stream));
    return B200_TRIMUL_OK;
  }
  if (dy == nullptr || index == nullptr || bucket_of == nullptr || workspace == nullptr) return B200_TRIMUL_E_NULL;
  if (!aligned(workspace, 1024)) return B200_TRIMUL_E_ALIGN;
  DeviceInfo info;
  if ((rc = tokens_device(&info)) != 0) return rc;
  const PositionGrid g = position_grid(b, n, c, buckets, info.sms);
  if (workspace_bytes < position_bytes(g, buckets)) return B200_TRIMUL_E_WORKSPACE;
  PositionParams p = {};
  p.dy = dy;
  p.index = index;
  p.chain = chain;
  p.bucket_of = bucket_of;
  p.partial = static_cast<float*>(workspace);
  p.dtable = dtable;
  p.b = b;
  p.n = n;
  p.c = c;
  p.buckets = buckets;
  p.reach = reach;
  p.wide = wide != 0;
  p.chunks = g.chunks;
  p.blocks = g.blocks;
  if (dtype == B200_BLOCKS_BF16) return position_backward<__nv_bfloat16>(p, g, info, stream);
  if (dtype == B200_BLOCKS_F16) return position_backward<__half>(p, g, info, stream);
  return position_backward<float>(p, g, info, stream);
}

int b200_block_dropout(const void* x, const void* u, const long long* key, unsigned long long call, void* y, long long outer, long long shared,
                       long long inner, int threshold, int dtype, void* cuda_stream) {
  if (outer < 0 || shared < 0 || inner < 0 || (outer > 0 && shared > 0 && inner > (1ll << 40) / outer / shared)) return B200_TRIMUL_E_SHAPE;
  if (outer > (1ll << 40) || shared > (1ll << 40)) return B200_TRIMUL_E_SHAPE;
  if (threshold < 0 || threshold > 65536 || dtype < 0 || dtype > 2) return B200_TRIMUL_E_UNSUPPORTED;
  if (outer == 0 || shared == 0 || inner == 0) return B200_TRIMUL_OK;
  if (u == nullptr || key == nullptr || y == nullptr) return B200_TRIMUL_E_NULL;
  DeviceInfo info;
  const int rc = tokens_device(&info);
  if (rc != 0) return rc;
  DropoutParams p = {};
  p.x = x;
  p.u = u;
  p.y = y;
  p.key = key;
  p.call = call;
  p.outer = outer;
  p.inner = inner;
  p.shared = shared;
  p.threshold = static_cast<uint32_t>(threshold);
  p.scale = threshold < 65536 ? 65536.f / static_cast<float>(65536 - threshold) : 0.f;
  const cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  if (dtype == B200_BLOCKS_BF16) return dropout<__nv_bfloat16>(p, info, stream);
  if (dtype == B200_BLOCKS_F16) return dropout<__half>(p, info, stream);
  return dropout<float>(p, info, stream);
}

int b200_tokens_read_status(void* cuda_stream, int* code) {
  if (code == nullptr) return B200_TRIMUL_E_NULL;
  const cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  *code = 0;
  TRIMUL_CUDA(cudaMemcpyFromSymbolAsync(code, tokens_status, sizeof(int), 0, cudaMemcpyDeviceToHost, stream));
  TRIMUL_CUDA(cudaStreamSynchronize(stream));
  if (*code != 0) {
    const int zero = 0;
    TRIMUL_CUDA(cudaMemcpyToSymbolAsync(tokens_status, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, stream));
    TRIMUL_CUDA(cudaStreamSynchronize(stream));
  }
  return B200_TRIMUL_OK;
}

}  // extern "C"
