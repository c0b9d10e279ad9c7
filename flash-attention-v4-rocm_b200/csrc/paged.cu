// Host side of the paged key/value cache entries of include/fav4_bshd.h: argument checks, workspace
// layout and launches. Nothing is allocated and the host never synchronises.
#include <cuda_runtime.h>

#include <climits>
#include <cmath>
#include <cstdint>
#include <mutex>

#include "fav4_bshd.h"
#include "host_status.h"
#include "paged.cuh"
#include "paged_tile_sm100.cuh"
#include "tensor_map.h"

namespace fav4 {
namespace {

constexpr int kMaxDevices = 64;
constexpr int kMaxSms = 160;         // bound on the SMs that the workspace is laid out for (a B200 has 148)
constexpr long long kKeyMargin = 8192;  // the kernels' key indexes go this far past a sequence's length at most
constexpr int kPagedPerSm = 2;       // blocks of paged_attn_kernel per SM
constexpr int kMaxGrid = kMaxSms * kPagedPerSm;

// Launch as a programmatic dependent (see wait_for_predecessor).
template <typename... Params, typename... Args>
int launch(void (*kernel)(Params...), unsigned grid, unsigned block, size_t smem, cudaStream_t stream, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }
bool stride_ok(long long s) { return s >= 0 && s % 8 == 0; }
size_t round256(size_t n) { return (n + 255) & ~size_t(255); }

// SM count, and the kernels' shared-memory limit set once per device.
int sm_count(int* sms) {
  static std::mutex mu;
  static int count[kMaxDevices] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
  std::lock_guard<std::mutex> lock(mu);
  if (count[dev] == 0) {
    int n = 0;
    e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return e;
    for (auto kernel : {paged_attn_kernel<false>, paged_attn_kernel<true>}) {
      e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kPagedSmem);
      if (e != cudaSuccess) return e;
    }
    e = cudaFuncSetAttribute(paged_tile_kernel<1>, cudaFuncAttributeMaxDynamicSharedMemorySize, PagedTileLayout<1>::kAlloc);
    if (e != cudaSuccess) return e;
    e = cudaFuncSetAttribute(paged_tile_kernel<2>, cudaFuncAttributeMaxDynamicSharedMemorySize, PagedTileLayout<2>::kAlloc);
    if (e != cudaSuccess) return e;
    count[dev] = n < kMaxSms ? n : kMaxSms;
  }
  *sms = count[dev];
  return 0;
}

bool cache_valid(const Fav4PagedCache& c) {
  return c.k && c.v && c.page_table && c.seq_lens && aligned16(c.k) && aligned16(c.v) && aligned4(c.page_table) &&
         aligned4(c.seq_lens) && stride_ok(c.page_stride) && stride_ok(c.token_stride) && stride_ok(c.head_stride) &&
         c.batch > 0 && c.batch < INT_MAX && c.kv_heads > 0 && c.num_pages > 0 && c.page_size >= 16 &&
         c.page_size % 16 == 0 && c.max_pages > 0 && c.table_stride >= 0 &&
         static_cast<long long>(c.max_pages) * c.page_size <= INT_MAX - kKeyMargin;
}

PagedCacheView view_of(const Fav4PagedCache& c) {
  PagedCacheView v;
  v.k = static_cast<__nv_bfloat16*>(c.k);
  v.v = static_cast<__nv_bfloat16*>(c.v);
  v.page_stride = c.page_stride;
  v.token_stride = c.token_stride;
  v.head_stride = c.head_stride;
  v.table = c.page_table;
  v.table_stride = c.table_stride;
  v.lens = c.seq_lens;
  v.num_pages = c.num_pages;
  v.page_size = c.page_size;
  v.max_pages = c.max_pages;
  v.kv_heads = c.kv_heads;
  v.batch = c.batch;
  return v;
}

bool append_valid(const Fav4PagedAppendArgs* a) {
  if (!a || !cache_valid(a->cache) || a->heads <= 0 || a->heads > INT_MAX / 256 || a->cache.kv_heads > INT_MAX / 256 ||
      a->total_q < 0 || !a->cu_seqlens_q || !aligned4(a->cu_seqlens_q) || a->rotary_dim < 0 || a->rotary_dim > 128 ||
      a->rotary_dim % 16 || (a->interleaved != 0 && a->interleaved != 1) || !aligned4(a->offsets))
    return false;
  if (a->total_q == 0) return true;
  if (!a->q || !a->k || !a->v || !a->q_out || !aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) ||
      !aligned16(a->q_out) || !stride_ok(a->q_token_stride) || !stride_ok(a->q_head_stride) ||
      !stride_ok(a->k_token_stride) || !stride_ok(a->k_head_stride) || !stride_ok(a->v_token_stride) ||
      !stride_ok(a->v_head_stride))
    return false;
  // the tables' rows are rotary_dim / 2 floats, a multiple of 32 bytes
  return a->rotary_dim == 0 ||
         (a->cos_table && a->sin_table && aligned16(a->cos_table) && aligned16(a->sin_table) && a->table_rows > 0);
}

bool paged_valid(const Fav4PagedArgs* a) {
  if (!a || !cache_valid(a->cache) || a->heads <= 0 || a->heads > INT_MAX / 256 || a->heads % a->cache.kv_heads ||
      a->total_q < 0 || a->max_sq < 0 || a->max_sq > a->total_q || !a->cu_seqlens_q || !aligned4(a->cu_seqlens_q) ||
      !std::isfinite(a->scale) || a->scale <= 0 || (a->prefix_pages == nullptr) != (a->prefix_len == nullptr))
    return false;
  if (a->prefix_pages &&
      (!aligned4(a->prefix_pages) || !aligned4(a->prefix_len) || a->max_prefix_pages <= 0 ||
       static_cast<long long>(a->max_prefix_pages) * a->cache.page_size > INT_MAX - kKeyMargin))
    return false;
  if (a->total_q == 0) return true;
  return a->max_sq > 0 && a->q && a->o && aligned16(a->q) && aligned16(a->o) && aligned4(a->lse) &&
         stride_ok(a->q_token_stride) && stride_ok(a->q_head_stride);
}

// Workspace: counters first (their place never changes, so that any call may follow any other), then the
// pieces of units that paged_attn_kernel cuts (a prefixed call's two launches overlap, and have their own),
// those of paged_tile_kernel, then the first of a prefixed call's two results. Sized by the rows alone: a
// server's batch and tables change from step to step, and its workspace has to do for all of them.
struct PagedSpace {
  size_t part, tile_o, tile_ml, cut, first_o, first_lse, total;
  static constexpr size_t kCounters = 4096;
  static constexpr size_t kPartO = size_t(2) * kMaxGrid * kPagedRows * 128 * sizeof(float);
  static constexpr size_t kPart = kPartO + size_t(2) * kMaxGrid * kPagedRows * 2 * sizeof(float);
};
static_assert(2 * kMaxGrid * sizeof(uint32_t) <= PagedSpace::kCounters, "two calls' counters");
static_assert(kTileRows == kBlockM, "q_tiles counts in the rows of a Q tile");
static_assert(kMaxSms <= 256, "paged_join_kernel reads one cut unit per thread");
PagedSpace paged_space(const Fav4PagedArgs& a) {
  const int tiles = q_tiles_bound(a.prefix_pages ? a.total_q : a.max_sq, a.heads);
  PagedSpace s;
  s.part = PagedSpace::kCounters;
  s.tile_o = s.part + (a.prefix_pages ? 2 : 1) * PagedSpace::kPart;
  s.tile_ml = s.tile_o + size_t(2) * kMaxSms * tiles * kBlockM * 128 * sizeof(float);
  s.cut = s.tile_ml + size_t(2) * kMaxSms * tiles * kBlockM * 2 * sizeof(float);
  s.first_o = s.cut + round256(kMaxSms * sizeof(int4));
  s.first_lse = s.total = s.first_o;
  if (a.prefix_pages) {
    const size_t rows = static_cast<size_t>(a.total_q) * a.heads;
    s.first_lse = s.first_o + round256(rows * 128 * sizeof(float));
    s.total = s.first_lse + round256(rows * sizeof(float));
  }
  return s;
}

bool encode_cache(CUtensorMap* map, const __nv_bfloat16* base, const PagedCacheView& c, int box_rows) {
  const cuuint64_t dims[4] = {128, static_cast<cuuint64_t>(c.kv_heads), static_cast<cuuint64_t>(c.page_size),
                              static_cast<cuuint64_t>(c.num_pages)};
  const long long strides[4] = {1, c.head_stride, c.token_stride, c.page_stride};
  const cuuint32_t box[4] = {64, 1, static_cast<cuuint32_t>(box_rows), 1};
  return encode_rows(map, base, 4, dims, strides, box);
}

template <int QTiles>
int launch_tiles(const PagedParams& p, const PagedSpace& sp, uint8_t* ws, int sms, cudaStream_t stream) {
  PagedTileParams t;
  t.p = p;
  t.p.part_o = reinterpret_cast<float*>(ws + sp.tile_o);
  t.p.part_ml = reinterpret_cast<float*>(ws + sp.tile_ml);
  t.cut = reinterpret_cast<int4*>(ws + sp.cut);
  t.tile_tokens = kBlockM / p.group;
  t.box_rows = 16;  // the largest power of two up to 128 that divides the page size
  while (t.box_rows < kTileKeys && p.c.page_size % (2 * t.box_rows) == 0) t.box_rows *= 2;
  t.status = pipeline_status_word();
  t.wait_limit_ns = pipeline_wait_limit_ns();
  if (!t.status) return cudaErrorInvalidDevice;
  CUtensorMap tq, tk, tv;
  const cuuint64_t dims[3] = {128, static_cast<cuuint64_t>(p.heads), static_cast<cuuint64_t>(p.total_q)};
  const long long strides[3] = {1, p.q_hs, p.q_ts};
  const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(p.group), static_cast<cuuint32_t>(t.tile_tokens)};
  if (!encode_rows(&tq, p.q, 3, dims, strides, box) || !encode_cache(&tk, p.c.k, p.c, t.box_rows) ||
      !encode_cache(&tv, p.c.v, p.c, t.box_rows))
    return cudaErrorInvalidValue;
  const int rc = launch(paged_tile_kernel<QTiles>, sms, 384, PagedTileLayout<QTiles>::kAlloc, stream, tq, tk, tv, t);
  if (rc) return rc;
  return launch(paged_join_kernel<QTiles>, kJoinPerSm * sms, 256, 0, stream, t, sms);
}

long long key_capacity(const PagedParams& p) { return static_cast<long long>(p.c.max_pages) * p.c.page_size; }

int tiles_of(const PagedParams& p) {
  // a cache expanded over heads or pages (stride 0) has no tensor map
  const bool mapped = (p.c.head_stride > 0 || p.c.kv_heads == 1) && (p.c.page_stride > 0 || p.c.num_pages == 1) &&
                      p.c.token_stride > 0 && (p.q_hs > 0 || p.heads == 1) && (p.q_ts > 0 || p.total_q == 1);
  return mapped ? q_tiles(p.max_sq, p.c.batch, p.group, p.c.kv_heads, key_capacity(p)) : 0;
}

// One attention of all rows over one set of page tables; per_sm: blocks of paged_attn_kernel.
int launch_rows(const PagedParams& p, const PagedSpace& sp, uint8_t* ws, int sms, int per_sm, cudaStream_t stream) {
  const int tiles = tiles_of(p);
  if (tiles == 1) return launch_tiles<1>(p, sp, ws, sms, stream);
  if (tiles == 2) return launch_tiles<2>(p, sp, ws, sms, stream);
  return launch(p.add_o ? paged_attn_kernel<true> : paged_attn_kernel<false>, sms * per_sm, kPagedWarps * 32, kPagedSmem,
                stream, p);
}

int launch_paged(const Fav4PagedArgs& a, int causal, uint8_t* ws, cudaStream_t stream) {
  int sms = 0;
  int rc = sm_count(&sms);
  if (rc) return rc;
  const PagedSpace sp = paged_space(a);
  PagedParams p = {};
  p.c = view_of(a.cache);
  p.q = static_cast<const __nv_bfloat16*>(a.q);
  p.q_ts = a.q_token_stride;
  p.q_hs = a.q_head_stride;
  p.part_o = reinterpret_cast<float*>(ws + sp.part);
  p.part_ml = reinterpret_cast<float*>(ws + sp.part + PagedSpace::kPartO);
  p.arrived = reinterpret_cast<uint32_t*>(ws);
  p.heads = a.heads;
  p.group = a.heads / a.cache.kv_heads;
  p.total_q = a.total_q;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.cu = a.cu_seqlens_q;
  p.max_sq = a.max_sq;
  p.causal = causal;
  p.o = static_cast<__nv_bfloat16*>(a.o);
  p.lse = a.lse;
  if (!a.prefix_pages) return launch_rows(p, sp, ws, sms, kPagedPerSm, stream);
  // every row of the batch against the prefix, as one sequence without a mask, into the workspace in FP32;
  // then the sequences' own keys, joined with it (rows of no sequence are never written)
  PagedParams first = p;
  first.c.table = a.prefix_pages;
  first.c.lens = a.prefix_len;
  first.c.max_pages = a.max_prefix_pages;
  first.c.batch = 1;
  first.cu = nullptr;
  first.max_sq = a.total_q;
  first.causal = 0;
  first.o = nullptr;
  first.o32 = reinterpret_cast<float*>(ws + sp.first_o);
  first.lse = reinterpret_cast<float*>(ws + sp.first_lse);
  first.part_o = reinterpret_cast<float*>(ws + sp.part + PagedSpace::kPart);
  first.part_ml = reinterpret_cast<float*>(ws + sp.part + PagedSpace::kPart + PagedSpace::kPartO);
  first.arrived += kMaxGrid;
  rc = launch_rows(first, sp, ws, sms, kPagedPerSm, stream);
  if (rc) return rc;
  p.add_o = first.o32;
  p.add_lse = first.lse;
  // Behind paged_attn_kernel, whose blocks leave the SMs one by one, the own keys take one block per SM while their
  // tables are not much wider than the prefix's: 8 sequences, 8 heads, of up to 100 keys behind 1000 13.2 us against
  // 15.3, behind 32768 37.0 against 39.5, 1000 to 4000 behind 32768 52.5 against 54.9; but up to 4000 behind 300 25.1
  // against 23.3, and behind the tile kernel 64 of up to 2048 behind 32768 51.2 against 45.7.
  const bool few = tiles_of(first) == 0 && p.c.batch * key_capacity(p) <= 2 * key_capacity(first);
  return launch_rows(p, sp, ws, sms, few ? 1 : kPagedPerSm, stream);
}

int forward_paged(const Fav4PagedArgs* a, int causal, void* workspace, size_t bytes, cudaStream_t stream,
                  bool prefix) {
  if (!paged_valid(a) || (causal != 0 && causal != 1) || (a->prefix_pages != nullptr) != prefix)
    return cudaErrorInvalidValue;
  if (a->total_q == 0) return 0;
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255) || bytes < paged_space(*a).total)
    return cudaErrorInvalidValue;
  return launch_paged(*a, causal, static_cast<uint8_t*>(workspace), stream);
}

}  // namespace
}  // namespace fav4

extern "C" int fav4_bshd_paged_append(const Fav4PagedAppendArgs* a, cudaStream_t stream) {
  if (!fav4::append_valid(a)) return cudaErrorInvalidValue;
  if (a->total_q == 0) return 0;
  fav4::AppendParams p;
  p.c = fav4::view_of(a->cache);
  p.q = static_cast<const __nv_bfloat16*>(a->q);
  p.k = static_cast<const __nv_bfloat16*>(a->k);
  p.v = static_cast<const __nv_bfloat16*>(a->v);
  p.q_out = static_cast<__nv_bfloat16*>(a->q_out);
  p.cu = a->cu_seqlens_q;
  p.cos_t = a->cos_table;
  p.sin_t = a->sin_table;
  p.offsets = a->offsets;
  p.q_ts = a->q_token_stride;
  p.q_hs = a->q_head_stride;
  p.k_ts = a->k_token_stride;
  p.k_hs = a->k_head_stride;
  p.v_ts = a->v_token_stride;
  p.v_hs = a->v_head_stride;
  p.heads = a->heads;
  p.total_q = a->total_q;
  p.rotary = a->rotary_dim;
  p.table_rows = a->table_rows;
  const long long per_token = (a->heads + 2ll * a->cache.kv_heads + fav4::kAppendRows - 1) / fav4::kAppendRows;
  const long long blocks = (a->total_q * per_token + 7) / 8;
  if (blocks > INT_MAX) return cudaErrorInvalidValue;
  return fav4::launch(a->interleaved ? fav4::paged_append_kernel<true> : fav4::paged_append_kernel<false>,
                      static_cast<unsigned>(blocks), 256, 0, stream, p);
}

extern "C" size_t fav4_bshd_paged_workspace_bytes(const Fav4PagedArgs* a) {
  return fav4::paged_valid(a) ? fav4::paged_space(*a).total : 0;
}

extern "C" int fav4_bshd_forward_paged(const Fav4PagedArgs* a, int causal, void* workspace, size_t workspace_bytes,
                                       cudaStream_t stream) {
  return fav4::forward_paged(a, causal, workspace, workspace_bytes, stream, false);
}

extern "C" int fav4_bshd_forward_shared_prefix(const Fav4PagedArgs* a, int causal, void* workspace,
                                               size_t workspace_bytes, cudaStream_t stream) {
  return fav4::forward_paged(a, causal, workspace, workspace_bytes, stream, true);
}
