// Paged key/value cache: the kernels around its pages (no reference counterpart; the reference has
// no cache).
//
// A cache is two BF16 arrays of num_pages pages of page_size keys. Key s of sequence b lives in slot
// s % page_size of page table[b][s / page_size]. Queries are packed rows: sequence b owns
// [cu[b], cu[b+1]), and its row i stands at position len_b - sq_b + i, so its last row is its newest
// key.
#pragma once
#include <cuda_bf16.h>
#include <cstdint>
#include "paged_schedule.h"
#include "sm100.cuh"

namespace fav4 {

// Every kernel here is launched as a programmatic dependent of whatever precedes it on its stream: it may be
// scheduled while that still runs, waits here before it reads or writes any memory that others use, and
// lets its own successor be scheduled at once.
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_launch_dependents() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void wait_for_predecessor() {
  grid_wait();
  grid_launch_dependents();
}

struct PagedCacheView {
  __nv_bfloat16 *k, *v;
  int64_t page_stride, token_stride, head_stride;  // elements
  const int* table;                                // [batch][table_stride]
  int64_t table_stride;
  const int* lens;  // keys per sequence, this step's included
  int num_pages, page_size, max_pages, kv_heads, batch;
};

// A load through L1 (the ordinary case) or past it. Never the non-coherent path: that is for memory which stays as it
// is for as long as the kernel runs, and these kernels are resident while their predecessor still writes, append's
// queries before an attention for one.
template <bool PastL1, typename T>
__device__ __forceinline__ T load(const T* p) {
  return PastL1 ? __ldcg(p) : *p;
}

// Offsets, lengths and rows of sequence b, clamped so that malformed ones can give wrong rows but no access
// outside the tensors. Rows past max_sq are not computed; with a mask, nor are the keys that only they see
// (the last row's key stays the last one, so the others keep their places; the length may become negative).
template <bool PastL1 = false>
__device__ __forceinline__ SeqView seq_view(const PagedCacheView& c, const int* cu, int total_q, int max_sq,
                                            int causal, int b) {
  SeqView s;
  const int64_t cap = static_cast<int64_t>(c.max_pages) * c.page_size;
  s.len = static_cast<int>(min(static_cast<int64_t>(max(load<PastL1>(c.lens + b), 0)), cap));
  if (cu != nullptr) {
    s.q0 = min(max(load<PastL1>(cu + b), 0), total_q);
    const int rows = min(max(load<PastL1>(cu + b + 1), s.q0), total_q) - s.q0;
    s.sq = min(rows, max_sq);
    if (causal) s.len -= rows - s.sq;
  } else {  // one sequence of all rows
    s.q0 = 0;
    s.sq = total_q;
  }
  return s;
}

// ------------------------------------------------------------------------------------------------
// Append: q' = R(pos) q, and k' = R(pos) k, v into their slots.
//
// R turns each pair (x_i, y_i), i < rotary/2, by the angle of row pos of the cos / sin tables:
// (x cos - y sin, y cos + x sin). Pairs are (i, i + rotary/2), or (2i, 2i + 1) when interleaved;
// elements from `rotary` on pass unchanged. The arithmetic is FP32 and each result is rounded once.
//
// Bandwidth: every row (one head of one token, 256 bytes) is read once and written once. A warp takes
// 8 rows of one token, 8 lanes per row; a lane holds the two 16-byte pieces that contain 8 whole
// pairs, and because both pairings put pairs 8s..8s+7 into lane s, the lane's slice of cos / sin is
// the same 32 bytes either way and is loaded once for its rows. 32 x 4096 tokens of 8 + 8 + 8 heads: 259 us,
// 6.2 TB/s (0.95 of the copy rate); 128 single tokens: 4.6 us on the device.
// ------------------------------------------------------------------------------------------------
struct AppendParams {
  PagedCacheView c;
  const __nv_bfloat16 *q, *k, *v;
  __nv_bfloat16* q_out;  // [total_q, heads, 128]
  const int* cu;
  const float *cos_t, *sin_t;  // [table_rows, rotary/2]
  const int* offsets;          // rotation position = cache position + offsets[b]; may be null
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;  // strides in elements
  int heads, total_q, rotary, table_rows;
};

// The sequence of packed row t, i.e. the number of b with cu[b+1] <= t, by 32 probes a step; the last step
// brings what the caller needs of the sequence along, so that a warp waits once less. False: t belongs to no
// sequence.
struct AppendSeq {
  int b, begin, end, len, offset;
};
__device__ __forceinline__ bool find_sequence(const PagedCacheView& c, const int* cu, const int* offsets, int t,
                                              int lane, AppendSeq* out) {
  int lo = 0, hi = c.batch;  // the answer is in [lo, hi]
  while (hi - lo > 31) {
    const int step = (hi - lo + 31) / 32;
    const int64_t i = lo + static_cast<int64_t>(lane) * step + step - 1;
    const bool before = i < hi && load<false>(cu + i + 1) <= t;
    lo += __popc(__ballot_sync(0xffffffffu, before)) * step;
    hi = min(hi, lo + step - 1);
  }
  const int i = lo + lane;
  const bool any = i < c.batch;
  AppendSeq s;
  s.begin = any ? load<false>(cu + i) : 0;
  s.end = any ? load<false>(cu + i + 1) : 0;
  s.len = any ? load<false>(c.lens + i) : 0;
  s.offset = any && offsets != nullptr ? load<false>(offsets + i) : 0;
  const int at = __popc(__ballot_sync(0xffffffffu, i < hi && s.end <= t));
  out->b = lo + at;
  out->begin = __shfl_sync(0xffffffffu, s.begin, at);
  out->end = __shfl_sync(0xffffffffu, s.end, at);
  out->len = __shfl_sync(0xffffffffu, s.len, at);
  out->offset = __shfl_sync(0xffffffffu, s.offset, at);
  return out->b < c.batch && out->begin <= t && t < out->end;  // offsets out of order: no sequence
}

__device__ __forceinline__ void rotate_pairs(uint32_t& a, uint32_t& b, float2 c, float2 s) {
  // two pairs: (a.lo, b.lo) by (c.x, s.x) and (a.hi, b.hi) by (c.y, s.y)
  const float2 x = __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&a));
  const float2 y = __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&b));
  a = pack_bf16x2(x.x * c.x - y.x * s.x, x.y * c.y - y.y * s.y);
  b = pack_bf16x2(y.x * c.x + x.x * s.x, y.y * c.y + x.y * s.y);
}

constexpr int kAppendRows = 8;  // rows of one token per warp

template <bool Interleaved>
__global__ void __launch_bounds__(256) paged_append_kernel(const __grid_constant__ AppendParams p) {
  const int lane = threadIdx.x % 32;
  const int hk = p.c.kv_heads, rows = p.heads + 2 * hk;
  const int per_token = (rows + kAppendRows - 1) / kAppendRows;
  const int64_t item = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) / 32;
  wait_for_predecessor();
  if (item >= static_cast<int64_t>(p.total_q) * per_token) return;
  const int t = static_cast<int>(item / per_token);
  const int r0 = static_cast<int>(item - static_cast<int64_t>(t) * per_token) * kAppendRows;
  const int slot = lane % 8;  // pairs 8 slot .. 8 slot + 7
  const bool turned = slot < p.rotary / 16;
  // 16-byte pieces of this lane within a row
  int pa, pb;
  if (Interleaved) {
    pa = 2 * slot;
    pb = pa + 1;
  } else if (turned) {
    pa = slot;
    pb = slot + p.rotary / 16;
  } else {
    pa = 2 * slot;  // past the rotated elements: rotary/8 + 2 (slot - rotary/16)
    pb = pa + 1;
  }
  // the rows do not depend on the sequence: their loads go out first
  uint4 a[2], b[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int r = r0 + u * 4 + lane / 8;
    const __nv_bfloat16* src = nullptr;
    if (r < p.heads) src = p.q + t * p.q_ts + r * p.q_hs;
    else if (r < p.heads + hk) src = p.k + t * p.k_ts + (r - p.heads) * p.k_hs;
    else if (r < rows) src = p.v + t * p.v_ts + (r - p.heads - hk) * p.v_hs;
    if (src != nullptr) {
      a[u] = *reinterpret_cast<const uint4*>(src + pa * 8);
      b[u] = *reinterpret_cast<const uint4*>(src + pb * 8);
    }
  }
  AppendSeq seq;
  if (!find_sequence(p.c, p.cu, p.offsets, t, lane, &seq)) return;
  const int64_t pos = static_cast<int64_t>(seq.len) - seq.end + t;
  float4 cs[2], sn[2];
  if (turned) {
    const int64_t at = pos + seq.offset;
    const int64_t row = min(max(at, int64_t(0)), static_cast<int64_t>(p.table_rows) - 1);
    const float4* cp = reinterpret_cast<const float4*>(p.cos_t + row * (p.rotary / 2) + slot * 8);
    const float4* sp = reinterpret_cast<const float4*>(p.sin_t + row * (p.rotary / 2) + slot * 8);
    cs[0] = load<false>(cp);
    cs[1] = load<false>(cp + 1);
    sn[0] = load<false>(sp);
    sn[1] = load<false>(sp + 1);
  }
  int64_t dst_kv = -1;  // a position without a slot (negative, past the table, no such page) is not written
  if (r0 + kAppendRows > p.heads && pos >= 0 && pos < static_cast<int64_t>(p.c.max_pages) * p.c.page_size) {
    const int idx = static_cast<int>(pos) / p.c.page_size;
    const int page = load<false>(p.c.table + seq.b * p.c.table_stride + idx);
    if (page >= 0 && page < p.c.num_pages)
      dst_kv = page * p.c.page_stride + (static_cast<int>(pos) - idx * p.c.page_size) * p.c.token_stride;
  }
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int r = r0 + u * 4 + lane / 8;
    __nv_bfloat16* dst = nullptr;
    if (r < p.heads) {
      dst = p.q_out + (static_cast<int64_t>(t) * p.heads + r) * 128;
    } else if (r < rows && dst_kv >= 0) {
      const bool is_k = r < p.heads + hk;
      dst = (is_k ? p.c.k : p.c.v) + dst_kv + (r - p.heads - (is_k ? 0 : hk)) * p.c.head_stride;
    }
    if (turned && r < p.heads + hk) {
      uint32_t* x = reinterpret_cast<uint32_t*>(&a[u]);
      uint32_t* y = reinterpret_cast<uint32_t*>(&b[u]);
      const float* c = reinterpret_cast<const float*>(cs);
      const float* s = reinterpret_cast<const float*>(sn);
      if (Interleaved) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // word e of each piece is one pair
          uint32_t lo = __byte_perm(x[e], y[e], 0x5410), hi = __byte_perm(x[e], y[e], 0x7632);
          rotate_pairs(lo, hi, make_float2(c[e], c[e + 4]), make_float2(s[e], s[e + 4]));
          x[e] = __byte_perm(lo, hi, 0x5410);
          y[e] = __byte_perm(lo, hi, 0x7632);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          rotate_pairs(x[e], y[e], make_float2(c[2 * e], c[2 * e + 1]), make_float2(s[2 * e], s[2 * e + 1]));
      }
    }
    if (dst != nullptr) {
      *reinterpret_cast<uint4*>(dst + pa * 8) = a[u];
      *reinterpret_cast<uint4*>(dst + pb * 8) = b[u];
    }
  }
}

// ------------------------------------------------------------------------------------------------
// Attention over the pages, 16 rows at a time.
//
// O = softmax(scale Q K^T + mask) V and LSE, with the running maximum m and sum l of the softmax kept
// per row in FP32 (base 2: scores times scale log2 e).
//
// For the next tokens of a batch every key and value is read once and 4 sq G FLOP are done per element
// read, so HBM bounds it: what counts is that all SMs read all the time, whatever the lengths. The
// rows of all sq new tokens and all G query heads of one K/V head share its keys: row r of a unit is
// token r / G, head r % G. The work of the launch is one line of 64-key tiles (sequence, K/V head, 16
// rows, tile), and each block takes an equal stretch of it, so a batch of any lengths is balanced to a
// tile; a unit that a boundary cuts leaves its pieces in the workspace, and the block that finishes
// last joins them in the order of their keys (the sum does not depend on who that is).
//
// Inside a block the four warps never wait on one another within a piece: each takes every fourth 16-key
// group with its own ring of asynchronous copies, its own m, l and O (16 x 128 in registers, mma.sync
// m16n8k16), and they are joined at the end of the piece, through the ring slots that they have just
// used, while the copies of the next piece are under way. 16 rows keep the legacy tensor path busy well
// below its rate at HBM speed: 32 instructions of 2048 multiply-adds for each 8 KiB (the pipe is 20 % busy).
// 64 sequences of 8192 to 24576 keys, 8 heads: 625 us, 6.9 TB/s; 32 of 1 to 32767, 2 heads: 89 us, 6.0 TB/s; one of
// 8192, 8 heads: 12.6 us, where the keys take 3 and the rest is start, joins and one wait after another.
// ------------------------------------------------------------------------------------------------
struct PagedParams {
  PagedCacheView c;
  const __nv_bfloat16* q;
  int64_t q_ts, q_hs;
  const int* cu;       // null: one sequence of all rows
  __nv_bfloat16* o;    // [total_q, heads, 128]; null: o32
  float* o32;          // FP32 [total_q, heads, 128], for a result that is joined with another
  float* lse;          // [heads, total_q] or null
  const float* add_o;  // another normalised result of the same rows (FP32) with its LSE, joined in; or null
  const float* add_lse;
  float* part_o;       // workspace: [2 grid][16][128] and [2 grid][16][2] (m, l)
  float* part_ml;
  uint32_t* arrived;   // [grid], zero between launches
  int heads, group, max_sq, total_q;
  int causal;
  float scale_log2;
};

constexpr int kPagedTile = 64;  // keys per tile: one 16-key group per warp
constexpr int kPagedWarps = 4;
constexpr int kPagedStages = 3;
constexpr int kPagedStageBytes = 2 * 16 * 256;  // 16 keys and 16 values
constexpr int kPagedRing = kPagedStages * kPagedStageBytes;
// Room on the line before each unit's tiles for what it costs beside them: 128 sequences of 10 to 300 keys, 8 K/V
// heads, take 38.8 us without, 29.3 with 1, 26.9 with 2 and 3; 256 of 1 to 100 keys, 2 heads, 16.2, 16.1, 13.0, 13.4;
// one of 8192 keys 12.5, 14.1, 12.9, 12.9.
constexpr int kRowExtra = 2;
constexpr int kPagedList = 64;   // pieces that are listed at a time
constexpr int kPagedSmem = kPagedWarps * kPagedRing;
static_assert(kPagedRows * 128 * 4 <= kPagedStageBytes, "a warp's O is left in one ring slot");

__device__ __forceinline__ uint32_t add_acq_rel(uint32_t* p) {
  uint32_t old;
  asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(old) : "l"(p) : "memory");
  return old;
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Tiles of one (row block, K/V head) of a sequence; a sequence without keys keeps one, which writes its
// zero rows.
__device__ __forceinline__ int paged_tiles(const SeqView& s) {
  return max((s.len + kPagedTile - 1) / kPagedTile, 1);
}
__device__ __forceinline__ int64_t paged_seq_work(const PagedParams& p, const SeqView& s) {
  if (s.sq == 0) return 0;
  const int64_t blocks = (static_cast<int64_t>(s.sq) * p.group + kPagedRows - 1) / kPagedRows;
  return blocks * p.c.kv_heads * (kRowExtra + paged_tiles(s));
}

// Row `r` of a unit to its place in the tensors; false past the last row.
struct RowPlace {
  int token, head;
};
__device__ __forceinline__ bool row_place(const PagedParams& p, const SeqView& s, int h, int64_t r, RowPlace* out) {
  if (r >= static_cast<int64_t>(s.sq) * p.group) return false;
  const int i = static_cast<int>(quotient(r, p.group));
  out->token = s.q0 + i;
  out->head = h * p.group + static_cast<int>(r - static_cast<int64_t>(i) * p.group);
  return true;
}

// One finished row: columns 4 lane .. 4 lane + 3 of sum / l, joined with the other result if there is one.
__device__ __forceinline__ void finish_row(const PagedParams& p, const RowPlace& at, float4 acc, float m, float l,
                                           int lane) {
  const int64_t row = static_cast<int64_t>(at.token) * p.heads + at.head;
  const int64_t lse_at = static_cast<int64_t>(at.head) * p.total_q + at.token;
  if (p.add_o != nullptr) {
    const float other = __ldcg(p.add_lse + lse_at) * 1.4426950408889634f;  // base 2; -inf where that result saw no key
    // relative to 0 where neither saw a key: a NaN of either still goes through
    const float top = fmaxf(m, other), zero = top == -INFINITY ? 0.f : top;
    const float w = exp2f(m - zero), x = exp2f(other - zero);
    const float4 b = __ldcg(reinterpret_cast<const float4*>(p.add_o + row * 128 + lane * 4));
    // where x is 0 the other row is zero
    acc = make_float4(acc.x * w + b.x * x, acc.y * w + b.y * x, acc.z * w + b.z * x, acc.w * w + b.w * x);
    l = l * w + x;
    m = top;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;  // l is 0 when no key was seen; NaN goes through
  acc = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
  if (p.o != nullptr)
    *reinterpret_cast<uint2*>(p.o + row * 128 + lane * 4) =
        make_uint2(pack_bf16x2(acc.x, acc.y), pack_bf16x2(acc.z, acc.w));
  else
    *reinterpret_cast<float4*>(p.o32 + row * 128 + lane * 4) = acc;
  if (p.lse != nullptr && lane == 0) p.lse[lse_at] = l == 0.f ? -INFINITY : m * 0.6931471805599453f + logf(l);
}

// A stretch of one unit, as this block takes it.
struct PagedPiece {
  int b, h, r0, sq;               // sequence, K/V head, first row, tokens
  int q0, len, key_begin, groups; // first packed row, keys; the piece's first key and its 16-key groups
  int tile0, cnt, n, c0;          // tiles [tile0, tile0 + cnt) of n; blocks c0..c1 hold the unit
  int c1, pad[3];
};
static_assert(sizeof(PagedPiece) == 64, "four 16-byte words");

// Inclusive sum over the block's threads; *sum is the total. Ends with every thread past its reads of `tmp`.
template <typename T>
__device__ __forceinline__ T block_scan(T v, T* tmp, T* sum) {
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const T up = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += up;
  }
  if (lane == 31) tmp[warp] = v;
  __syncthreads();
  T all = 0;
#pragma unroll
  for (int w = 0; w < kPagedWarps; ++w) {
    if (w < warp) v += tmp[w];
    all += tmp[w];
  }
  *sum = all;
  __syncthreads();
  return v;
}

// Byte offset of 4-column piece c of row r of a 16 x 128 FP32 tile in a ring slot, spread over the banks.
__device__ __forceinline__ int tile_at(int r, int c) { return r * 512 + ((c ^ (r & 7)) * 16); }

// Joined: the result is joined with another one (add_o), which the predecessor computes from the same inputs.
// That kernel let this one be scheduled only after its own wait, so everything but its result (and the
// outputs, whose last reader may have been before it) is there already and only the rows' ends wait: the
// launch, the first copies and the products overlap with it (64 sequences behind 32768 keys: 64 -> 54 us).
// The inputs are then read through L2, past lines that an SM may hold from before; that costs a short launch
// 1 us, so the ordinary kernel keeps L1.
template <bool Joined>
__global__ void __launch_bounds__(kPagedWarps * 32, 2) paged_attn_kernel(const __grid_constant__ PagedParams p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ __align__(16) PagedPiece list[kPagedList];
  __shared__ int64_t scan64[kPagedWarps];
  __shared__ int scan32[kPagedWarps];
  __shared__ float piece_ml[kPagedWarps][kPagedRows][2];
  __shared__ int free_slot[kPagedWarps];
  __shared__ uint32_t last_one;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int g = lane / 4, t4 = lane % 4;     // mma fragments: rows g and g + 8, columns 2 t4 and 2 t4 + 1 of eight
  const int mi = lane / 8, mr = lane % 8;    // ldmatrix: matrix and row that this lane addresses
  const int cl = lane % 16, rl = lane / 16;  // copies: 16-byte piece cl of rows rl + 2 j
  const uint32_t ring = smem_addr(smem) + warp * kPagedRing;
  if (Joined) grid_launch_dependents();
  else wait_for_predecessor();

  int64_t total = 0, per = 0, begin = 0, end = 0;
  for (int round = 0;; ++round) {
    // ---- the pieces of this block's stretch [begin, end) of the line of tiles, kPagedList at a time ----
    int pieces = 0;  // of the whole stretch
    for (int pass = round == 0 ? 0 : 1; pass < 2; ++pass) {
      int64_t base = 0;
      pieces = 0;
      for (int b0 = 0; b0 < p.c.batch; b0 += kPagedWarps * 32) {
        const int b = b0 + tid;
        SeqView s = {0, 0, 0};
        if (b < p.c.batch) s = seq_view<Joined>(p.c, p.cu, p.total_q, p.max_sq, p.causal, b);
        const int64_t work = paged_seq_work(p, s);
        int64_t sum;
        const int64_t first_tile = base + block_scan(work, scan64, &sum) - work;  // of this sequence
        if (p.c.batch <= kPagedWarps * 32) pass = 1;  // one step sees the whole batch
        if (round == 0 && p.c.batch <= kPagedWarps * 32) {
          total = sum;
          per = quotient(total + gridDim.x - 1, gridDim.x);
          begin = blockIdx.x * per;
          end = min(total, begin + per);
        }
        if (pass == 1) {
          const int64_t lo = max(begin, first_tile), hi = min(end, first_tile + work);
          const int n = paged_tiles(s);
          int mine = 0;
          int64_t u = 0;
          if (lo < hi) {
            u = quotient(lo - first_tile, kRowExtra + n);
            mine = static_cast<int>(quotient(hi - 1 - first_tile, kRowExtra + n) - u) + 1;
          }
          int listed;
          int at = pieces + block_scan(mine, scan32, &listed) - mine - round * kPagedList;
          pieces += listed;
          const int64_t rows = static_cast<int64_t>(s.sq) * p.group;
          const int64_t blocks = (rows + kPagedRows - 1) / kPagedRows;
          for (; mine > 0; --mine, ++u, ++at) {
            if (at < 0 || at >= kPagedList) continue;
            PagedPiece w;
            w.b = b;
            w.h = static_cast<int>(quotient(u, blocks));
            w.r0 = static_cast<int>(u - w.h * blocks) * kPagedRows;
            w.sq = s.sq;
            w.q0 = s.q0;
            w.len = s.len;
            const int64_t tile1 = first_tile + u * (kRowExtra + n) + kRowExtra;  // its first tile's place on the line
            w.tile0 = steps_before(begin - tile1, n);
            w.cnt = steps_before(end - tile1, n) - w.tile0;
            w.n = n;
            w.c0 = static_cast<int>(quotient(tile1, per));
            w.c1 = static_cast<int>(quotient(tile1 + n - 1, per));
            w.key_begin = w.tile0 * kPagedTile;
            int64_t key_end = min((w.tile0 + static_cast<int64_t>(w.cnt)) * kPagedTile, static_cast<int64_t>(s.len));
            if (p.causal)  // the last key that the block's last row sees
              key_end = min(key_end, static_cast<int64_t>(s.len) - s.sq + 1 +
                                         quotient(min(static_cast<int64_t>(w.r0) + kPagedRows, rows) - 1, p.group));
            w.groups = static_cast<int>(max(key_end - w.key_begin + 15, int64_t(0)) / 16);
            list[at] = w;
          }
        }
        base += sum;
      }
      if (pass == 0) {
        total = base;
        per = quotient(total + gridDim.x - 1, gridDim.x);
        begin = blockIdx.x * per;
        end = min(total, begin + per);
      }
    }
    const int listed = min(pieces - round * kPagedList, kPagedList);
    if (listed <= 0) break;
    __syncthreads();
    // a stretch that ends before its last unit's first tile has nothing of it
    const int count = list[listed - 1].cnt == 0 ? listed - 1 : listed;

    // ---- copies: this warp's 16-key groups of all listed pieces, kPagedStages - 1 ahead of their use ----
    // A stretch of up to 32 groups of a piece has its page numbers in the lanes; those of the stretch after it
    // are loaded when it begins.
    auto steps_of = [&](int i) { return (list[i].groups - warp + kPagedWarps - 1) / kPagedWarps; };
    auto pages_from = [&](int i, int s0) -> int {
      if (i >= count || s0 + lane >= steps_of(i)) return 0;
      const int key = list[i].key_begin + (warp + kPagedWarps * (s0 + lane)) * 16;
      const int page = load<Joined>(p.c.table + list[i].b * p.c.table_stride + key / p.c.page_size);
      return min(max(page, 0), p.c.num_pages - 1);
    };
    auto skip_empty = [&](int i) {
      while (i < count && steps_of(i) <= 0) ++i;
      return i;
    };
    int li = skip_empty(0), ls = 0;  // next group to copy: step ls of piece li
    int l_stop = 0, l_key = 0, l_len = 0, n_piece = 0, n_from = 0;
    int64_t l_head = 0;
    int pages = pages_from(li, 0), pages_next = 0;
    auto open = [&]() {  // the stretch that holds step ls of piece li begins; the one after it is looked up
      if (li >= count) return;
      const int steps = steps_of(li);
      l_stop = min(steps, ls + 32);
      l_key = list[li].key_begin + warp * 16;
      l_len = list[li].len;
      l_head = list[li].h * p.c.head_stride + cl * 8;
      n_piece = l_stop < steps ? li : skip_empty(li + 1);
      n_from = l_stop < steps ? l_stop : 0;
      pages_next = pages_from(n_piece, n_from);
    };
    open();
    int slot_in = 0;  // ring slot of the next copy
    auto issue = [&]() {
      if (li < count) {
        const int key = l_key + ls * (kPagedWarps * 16);
        const int64_t page = __shfl_sync(0xffffffffu, pages, ls % 32);
        const int64_t off = page * p.c.page_stride + (key % p.c.page_size + rl) * p.c.token_stride + l_head;
        const __nv_bfloat16* ks = p.c.k + off;
        const __nv_bfloat16* vs = p.c.v + off;
        const uint32_t dst = ring + slot_in * kPagedStageBytes + rl * 256;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int row = rl + 2 * j;
          const int bytes = key + row < l_len ? 16 : 0;  // slots past the end may hold anything: zeros instead
          const uint32_t d = dst + j * 512 + ((cl ^ (row & 7)) * 16);
          cp_async16(d, ks + 2 * j * p.c.token_stride, bytes);
          cp_async16(d + 4096, vs + 2 * j * p.c.token_stride, bytes);
        }
        if (++ls == l_stop) {
          li = n_piece;
          ls = n_from;
          pages = pages_next;
          open();
        }
      }
      cp_async_commit();
      slot_in = slot_in == kPagedStages - 1 ? 0 : slot_in + 1;
    };
#pragma unroll 1
    for (int i = 0; i < kPagedStages - 1; ++i) issue();

    uint32_t qf[8][4];
    auto load_q = [&](int i) {
      const PagedPiece& w = list[i];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int r = w.r0 + g + 8 * u, token = r / p.group;
        const bool live = token < w.sq;
        const __nv_bfloat16* src =
            p.q + (w.q0 + token) * p.q_ts + (w.h * p.group + r - token * p.group) * p.q_hs + t4 * 2;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          qf[k][u] = live ? load<Joined>(reinterpret_cast<const uint32_t*>(src + k * 16)) : 0u;
          qf[k][u + 2] = live ? load<Joined>(reinterpret_cast<const uint32_t*>(src + k * 16 + 8)) : 0u;
        }
      }
    };
    if (count > 0) load_q(0);

    int slot = 0;  // ring slot of the next group to use
    for (int i = 0; i < count; ++i) {
      const int len = list[i].len, sq = list[i].sq, r0 = list[i].r0;
      const int steps = steps_of(i);
      // last visible key of this thread's rows (g and g + 8), and of the first row of all
      int lim[2];
#pragma unroll
      for (int u = 0; u < 2; ++u)
        lim[u] = p.causal ? len - sq + min((r0 + g + 8 * u) / p.group, sq - 1) : len - 1;
      const int lim_min = p.causal ? len - sq + r0 / p.group : len - 1;
      int key = list[i].key_begin + warp * 16;

      float o[16][4];
#pragma unroll
      for (int j = 0; j < 16; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
      float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
      for (int st_i = 0; st_i < steps; ++st_i, key += kPagedWarps * 16) {
        cp_async_wait<kPagedStages - 2>();
        __syncwarp();  // this group has arrived, and every lane is done with the one before
        const uint32_t st = ring + slot * kPagedStageBytes;
        slot = slot == kPagedStages - 1 ? 0 : slot + 1;
        float sc[2][4] = {}, sc_odd[2][4] = {};  // two chains each: a chain of eight products would show
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          uint32_t kb[4];
          ldsm4(st + ((mi / 2) * 8 + mr) * 256 + (((2 * k + (mi & 1)) ^ mr) * 16), kb);
          mma16816(k & 1 ? sc_odd[0] : sc[0], qf[k], kb[0], kb[1]);
          mma16816(k & 1 ? sc_odd[1] : sc[1], qf[k], kb[2], kb[3]);
        }
        issue();  // behind the products
#pragma unroll
        for (int e = 0; e < 8; ++e) sc[e / 4][e % 4] += sc_odd[e / 4][e % 4];
        if (key + 15 > lim_min) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int col = key + (e / 4) * 8 + t4 * 2 + (e & 1);
            if (col > lim[(e / 2) & 1]) sc[e / 4][e % 4] = -INFINITY;
          }
        }
        bool grow = false;
        float cand[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float mx = fmaxf(fmaxf(sc[0][2 * u], sc[0][2 * u + 1]), fmaxf(sc[1][2 * u], sc[1][2 * u + 1]));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          cand[u] = fmaxf(m[u], mx * p.scale_log2);
          grow |= cand[u] > m[u] + 8.f;  // the sums are rescaled only when a maximum grows by 2^8
        }
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const float a = cand[u] == -INFINITY ? 1.f : ex2_mufu(m[u] - cand[u]);
            m[u] = cand[u];
            l[u] *= a;
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              o[j][2 * u] *= a;
              o[j][2 * u + 1] *= a;
            }
          }
        }
        uint32_t pf[4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const float mb = m[u] == -INFINITY ? 0.f : m[u];
          const float p0 = ex2_mufu(fmaf(sc[0][2 * u], p.scale_log2, -mb));
          const float p1 = ex2_mufu(fmaf(sc[0][2 * u + 1], p.scale_log2, -mb));
          const float p2 = ex2_mufu(fmaf(sc[1][2 * u], p.scale_log2, -mb));
          const float p3 = ex2_mufu(fmaf(sc[1][2 * u + 1], p.scale_log2, -mb));
          l[u] += (p0 + p1) + (p2 + p3);
          pf[u] = pack_bf16x2(p0, p1);  // P in BF16 for the second product; l sums the unrounded values
          pf[u + 2] = pack_bf16x2(p2, p3);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          uint32_t vb[4];
          ldsm4_t(st + 4096 + ((mi & 1) * 8 + mr) * 256 + (((2 * j + mi / 2) ^ mr) * 16), vb);
          mma16816(o[2 * j], pf, vb[0], vb[1]);
          mma16816(o[2 * j + 1], pf, vb[2], vb[3]);
        }
      }
      if (i + 1 < count) load_q(i + 1);  // arrives while this piece is joined

      // ---- join the four warps: each leaves its O in the ring slot that no copy is under way to ----
      const int spare = slot == 0 ? kPagedStages - 1 : slot - 1;
      __syncwarp();
      uint8_t* mine = smem + warp * kPagedRing + spare * kPagedStageBytes;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        l[u] += __shfl_xor_sync(0xffffffffu, l[u], 1);
        l[u] += __shfl_xor_sync(0xffffffffu, l[u], 2);
        if (t4 == 0) {
          piece_ml[warp][g + 8 * u][0] = m[u];
          piece_ml[warp][g + 8 * u][1] = l[u];
        }
#pragma unroll
        for (int j = 0; j < 16; ++j)
          *reinterpret_cast<float2*>(mine + tile_at(g + 8 * u, 2 * j + t4 / 2) + (t4 & 1) * 8) =
              make_float2(o[j][2 * u], o[j][2 * u + 1]);
      }
      if (lane == 0) free_slot[warp] = spare;
      __syncthreads();
      if (Joined) grid_wait();  // the other result is complete
      const PagedPiece& w = list[i];
      const int rows = static_cast<int>(min(static_cast<int64_t>(kPagedRows), static_cast<int64_t>(sq) * p.group - r0));
      const bool whole = w.cnt == w.n;
      const SeqView s = {w.q0, sq, len};
      const int part = 2 * blockIdx.x + (w.tile0 == 0 ? 1 : 0);  // a piece that opens its unit, or one that carries on
      for (int r = warp; r < rows; r += kPagedWarps) {
        float top = piece_ml[0][r][0];
#pragma unroll
        for (int x = 1; x < kPagedWarps; ++x) top = fmaxf(top, piece_ml[x][r][0]);
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        float sum = 0.f;
#pragma unroll
        for (int x = 0; x < kPagedWarps; ++x) {
          const float mx = piece_ml[x][r][0];
          const float a = mx == -INFINITY ? 0.f : exp2f(mx - top);
          const float4 v = *reinterpret_cast<const float4*>(smem + x * kPagedRing + free_slot[x] * kPagedStageBytes +
                                                            tile_at(r, lane));
          acc = make_float4(acc.x + a * v.x, acc.y + a * v.y, acc.z + a * v.z, acc.w + a * v.w);
          sum += a * piece_ml[x][r][1];
        }
        if (whole) {
          RowPlace at;
          row_place(p, s, w.h, r0 + r, &at);
          finish_row(p, at, acc, top, sum, lane);
        } else {
          *reinterpret_cast<float4*>(p.part_o + (static_cast<int64_t>(part) * kPagedRows + r) * 128 + lane * 4) = acc;
          if (lane == 0)
            *reinterpret_cast<float2*>(p.part_ml + (static_cast<int64_t>(part) * kPagedRows + r) * 2) =
                make_float2(top, sum);
        }
      }
      if (!whole) {
        __syncthreads();
        if (tid == 0) {
          // after the barrier, this thread's release and acquire stand for the whole block's
          const uint32_t before = add_acq_rel(p.arrived + w.c0);
          last_one = before == static_cast<uint32_t>(w.c1 - w.c0);
          if (last_one) p.arrived[w.c0] = 0u;  // ready for the next launch
        }
        __syncthreads();
        if (last_one) {
          // this block is the last of the unit's: it adds the pieces up in the order of their keys. With fewer
          // rows than warps, the warps share a row's pieces.
          const int share = rows == 1 ? 4 : rows == 2 ? 2 : 1;
          const int turn = warp % share, parts = w.c1 - w.c0 + 1;
          const int x_begin = parts * turn / share, x_end = parts * (turn + 1) / share;
          for (int r = warp / share; r < rows; r += kPagedWarps / share) {
            auto part_row = [&](int x) { return static_cast<int64_t>(2 * (w.c0 + x) + (x == 0 ? 1 : 0)) * kPagedRows + r; };
            float top = -INFINITY, sum = 0.f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int x0 = x_begin; x0 < x_end; x0 += 8) {
              float4 v[8];
              float2 ml[8];
#pragma unroll
              for (int x = 0; x < 8; ++x) {
                ml[x] = make_float2(-INFINITY, 0.f);
                v[x] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (x0 + x < x_end) {
                  v[x] = __ldcg(reinterpret_cast<const float4*>(p.part_o + part_row(x0 + x) * 128 + lane * 4));
                  ml[x] = __ldcg(reinterpret_cast<const float2*>(p.part_ml + part_row(x0 + x) * 2));
                }
              }
              float next = top;
#pragma unroll
              for (int x = 0; x < 8; ++x) next = fmaxf(next, ml[x].x);
              // relative to 0 while no piece has seen a key: NaN sums still go through
              const float zero = next == -INFINITY ? 0.f : next, a = exp2f(top - zero);
              acc = make_float4(acc.x * a, acc.y * a, acc.z * a, acc.w * a);
              sum *= a;
              top = next;
#pragma unroll
              for (int x = 0; x < 8; ++x) {
                const float c = exp2f(ml[x].x - zero);
                acc = make_float4(acc.x + c * v[x].x, acc.y + c * v[x].y, acc.z + c * v[x].z, acc.w + c * v[x].w);
                sum += c * ml[x].y;
              }
            }
            if (share > 1) {
              float* sums = reinterpret_cast<float*>(smem + warp * kPagedRing + spare * kPagedStageBytes);
              reinterpret_cast<float4*>(sums)[lane] = acc;
              if (lane == 0) {
                piece_ml[warp][0][0] = top;
                piece_ml[warp][0][1] = sum;
              }
              named_sync(1 + r, share * 32);
              if (turn > 0) continue;
              for (int x = 1; x < share; ++x) top = fmaxf(top, piece_ml[warp + x][0][0]);
              acc = make_float4(0.f, 0.f, 0.f, 0.f);
              sum = 0.f;
              const float zero = top == -INFINITY ? 0.f : top;
              for (int x = 0; x < share; ++x) {
                const float c = exp2f(piece_ml[warp + x][0][0] - zero);
                const float4 v = *reinterpret_cast<const float4*>(smem + (warp + x) * kPagedRing +
                                                                  free_slot[warp + x] * kPagedStageBytes + lane * 16);
                acc = make_float4(acc.x + c * v.x, acc.y + c * v.y, acc.z + c * v.z, acc.w + c * v.w);
                sum += c * piece_ml[warp + x][0][1];
              }
            }
            RowPlace at;
            row_place(p, s, w.h, r0 + r, &at);
            finish_row(p, at, acc, top, sum, lane);
          }
        }
      }
      __syncthreads();  // the slots that hold the O tiles are the next to be copied to
    }
    cp_async_wait<0>();
    if (pieces - round * kPagedList <= kPagedList) break;
    __syncthreads();  // the list is written anew
  }
  if (Joined) grid_wait();  // no block ends before its predecessor has: the successor waits for this grid only
}

}  // namespace fav4
