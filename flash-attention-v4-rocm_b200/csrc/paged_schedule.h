// The arithmetic of the paged attention's schedules and the choice of its kernel, for the kernels, their launches
// and a host compiler.
#pragma once
#include <cstdint>

#ifdef __CUDACC__
#define FAV4_HD __host__ __device__ __forceinline__
#define FAV4_HD_CALL __host__ __device__ __noinline__ inline
#else
#define FAV4_HD inline
#define FAV4_HD_CALL inline
#endif

namespace fav4 {

// One sequence: its first row of Q, its rows, its keys.
struct SeqView {
  int q0, sq, len;
};

// a / b for a >= 0, b > 0. Work counts are 64-bit, but nearly always small: a 64-bit division costs several
// times a 32-bit one, and the schedules wait for theirs. The long way is kept out of line: code that a kernel
// fetches once, at its start, costs it more than the arithmetic.
FAV4_HD_CALL int64_t divide64(int64_t a, int64_t b) { return a / b; }
FAV4_HD int64_t quotient(int64_t a, int64_t b) {
  if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
  return divide64(a, b);
}

// paged_tile_kernel: a unit is `bt` tokens of a sequence (the last one: what is left) and takes a step for
// each 128-key tile up to its last visible key; one that sees no key keeps a step, which writes its zero rows.
constexpr int kTileKeys = 128;

// sum over j < n of floor((a j + c) / 128), for a, c >= 0, by the steps of Euclid's algorithm. Blocks wait
// for it, so the first step (by 128) has no division and the others one each: their c and a are below 128.
FAV4_HD_CALL int64_t floor_sum128(int64_t n, int64_t a, int64_t c) {
  if (n <= 0) return 0;
  int64_t s = n * (n - 1) / 2 * (a >> 7) + n * (c >> 7);
  int m = 128, r = static_cast<int>(a & 127), d = static_cast<int>(c & 127);
  while (true) {
    const int64_t y = r * n + d;
    if (y < m) break;
    const int64_t k = m == 128 ? y >> 7 : quotient(y, m);
    d = static_cast<int>(y - k * m);
    n = k;
    const int q = static_cast<int>(static_cast<unsigned>(m) / static_cast<unsigned>(r));  // r > 0: y >= m > d
    const int e = static_cast<int>(static_cast<unsigned>(d) / static_cast<unsigned>(r));
    s += n * (n - 1) / 2 * q + n * e;
    const int t = m - q * r;
    d -= e * r;
    m = r;
    r = t;
  }
  return s;
}

FAV4_HD int steps_up_to(int64_t keys) {
  return keys <= 0 ? 1 : static_cast<int>((keys + kTileKeys - 1) / kTileKeys);
}
// Steps of unit r of a sequence, and of units 0 .. r - 1.
FAV4_HD int unit_steps(const SeqView& s, int causal, int bt, int r) {
  const int64_t full = (static_cast<int64_t>(r) + 1) * bt;
  const int64_t last = full < s.sq ? full : s.sq;
  return steps_up_to(causal ? static_cast<int64_t>(s.len) - s.sq + last : s.len);
}
FAV4_HD_CALL int64_t units_steps(SeqView s, int causal, int bt, int64_t r) {
  if (r <= 0) return 0;
  if (!causal) return r * steps_up_to(s.len);
  const int64_t units = quotient(static_cast<int64_t>(s.sq) + bt - 1, bt);
  int64_t sum = 0;
  if (r == units) {  // the last one ends with the sequence, the others after a whole number of bt tokens
    sum = steps_up_to(s.len);
    --r;
  }
  const int64_t past = static_cast<int64_t>(s.len) - s.sq;
  int64_t ones = past <= kTileKeys ? quotient(kTileKeys - past, bt) : 0;  // units that end within the first tile
  if (ones > r) ones = r;
  // units ones .. r - 1: ceil((past + (j + 1) bt) / 128)
  return sum + ones + floor_sum128(r - ones, bt, past + (ones + 1) * bt + kTileKeys - 1);
}
// The line on which the blocks share the work has room for kUnitExtra steps before each unit's own: what a unit
// costs beside them (its first loads, the end of the pipeline, its rows' ends). Without it a block of many
// short units ends last: 4 prompts of 4096 tokens, 8 heads on 2, 199 us, with 2 152, 3 155, 4 155; 3 ragged chunks
// 37.9, 32.3, 31.4, 33.9; 8 prompts of 1000 tokens, 8 heads, 56, 57, 50, 52.
constexpr int kUnitExtra = 3;
FAV4_HD int64_t units_cost(const SeqView& s, int causal, int bt, int64_t r) {
  return units_steps(s, causal, bt, r) + kUnitExtra * r;
}
FAV4_HD int64_t tile_seq_work(const SeqView& s, int causal, int bt) {
  return s.sq == 0 ? 0 : units_cost(s, causal, bt, quotient(static_cast<int64_t>(s.sq) + bt - 1, bt));
}

// How many of a unit's n steps lie before a boundary `at` places after its first one.
FAV4_HD int steps_before(int64_t at, int n) { return at <= 0 ? 0 : at >= n ? n : static_cast<int>(at); }

constexpr int kPagedRows = 16;  // rows of a unit of paged_attn_kernel
constexpr int kTileRows = 128;  // and of a Q tile of paged_tile_kernel

// Q tiles per block for `batch` sequences of at most `tokens` new tokens each behind page tables for `capacity`
// keys; 0 for paged_attn_kernel. `rows` of a sequence share a K/V head; lengths are not known here.
//   16-row kernel or tiles. Up to 16 rows the former reads at HBM speed with half the start-up: 32 sequences
//   of up to 32767 keys take 89 us against 103 with 4 rows, 58 against 62 with 16 (and with 24: 79 against 62).
//   But the last block of a unit joins its pieces alone, and with few units there are many: with 8 rows, one
//   unit of 8000 keys 27 us against 17, four units 20 against 17, eight 18 against 19, 64 units of 500 to 1500
//   keys 15 against 21. With 16 rows 16 units of 100 to 1000 keys 15 against 14, 32 of 8000 34 against 39.
//   One tile or two. Two tiles read each key half as often and have half the units; one makes smaller pieces and
//   less padding and has both warpgroups on every step. Long chunks take two: 4096 tokens behind 28672 keys (16384
//   rows) 474 us against 504, 3 ragged ones of up to 2000 rows 31 against 33, 8 of 1024 rows behind 8000 keys 87
//   against 93 (but one of 2048 rows behind 8000 35 against 33); and so do prompts that begin their sequence, whose
//   units have few steps, as tables not much wider than the chunk tell: 4 of 4096 tokens 155 against 167, 8 of 512
//   rows (8 heads) 23 against 32, 8 of 257 24 against 26. The others take one: 32 of 600 rows behind 1000 keys 49
//   against 55, 4 of 600 (8 heads) behind 600 32 against 39, 256 rows on 32768 keys 27 against 32.
inline int q_tiles(long long tokens, int batch, int group, int kv_heads, long long capacity) {
  const long long rows = tokens * group, units = static_cast<long long>(batch) * kv_heads;
  if (group > kTileRows || (rows <= kPagedRows && rows < 2 * units && (rows <= 8 || units >= 32))) return 0;
  return rows >= 1024 || (rows > kTileRows && capacity < 2 * tokens) ? 2 : 1;
}

// A bound on q_tiles over every batch, K/V head count and page table that `tokens` rows of `heads` can meet.
inline int q_tiles_bound(long long tokens, int heads) {
  return tokens * (heads < kTileRows ? heads : kTileRows) > kTileRows ? 2 : 1;
}

}  // namespace fav4
