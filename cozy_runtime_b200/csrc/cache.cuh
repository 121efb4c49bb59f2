// What the kernels of the 8-bit paged cache share: its numbers (e4m3 codes under power-of-two
// block scales), and how a step's attention is cut into units of work.
//
// A block is one page of one head: `page` rows of head_dim codes, value = code · 2^e with one
// int8 exponent e a block. A power of two costs a floating-point code no precision (the codes
// keep their 4 significant bits at any scale), growing it shifts the codes without loss down to
// e4m3's subnormals, and it folds into an exponent: 2^s · 2^e = 2^(s + e).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/cozy_ulysses.h"

namespace cozy {

// Exponents: the floor keeps 2^(s - m + e) of the attention above fp32's smallest normal for
// every key within 2^-26 of its row's largest term, whatever mixture of scales a row meets
// (floor to ceiling is a factor of 2^100); magnitudes up to 2^-70 are stored as zero, those over
// 448 · 2^40 (infinities among them) as NaN.
constexpr int kExponentFloor = -60;
constexpr int kExponentCeiling = 40;
constexpr float kLargestStored = 448.0f * 1099511627776.0f;  // 448 · 2^40

// Bits of CozyCachePlan::status.
enum : int {
  kPlanNoPages = 1,     // fewer free pages than the requests need
  kPlanNarrow = 2,      // a request longer than its table row
  kPlanTokens = 4,      // more new tokens than `tokens`, or than `longest` in one request
  kPlanLengths = 8,     // a negative length, new < -1, or a ring whose cursor is not possible
  kPlanBadPage = 16,    // a page number outside [0, pages): its tokens are left out; among pages
                        // to be released: the step is refused
  kPlanTimeout = 32,    // an on-chip wait of a call of this step ran past its limit
};

// 2^e of an exponent byte; any byte is valid (uninitialised blocks behind a sequence are read).
__host__ __device__ __forceinline__ float exponent_scale(int e) {
  const uint32_t bits = static_cast<uint32_t>((e < -126 ? -126 : e) + 127) << 23;
#ifdef __CUDA_ARCH__
  return __uint_as_float(bits);
#else
  float f;
  __builtin_memcpy(&f, &bits, 4);
  return f;
#endif
}

// a / b of counts: the 64-bit division is many times the 32-bit one, which mostly does.
__host__ __device__ __forceinline__ long long quotient(long long a, long long b) {
  if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
  return a / b;
}

// Σ floor((a·i + b) / 128) for i in [0, n), 0 ≤ a ≤ 256, 0 ≤ b, n < 2^24: the floor sum of lattice
// points under a line by its well-known recursion, which swaps the divisor and a as Euclid's
// algorithm does; behind its first step everything is below 2^31.
__host__ __device__ inline long long floor_sum_128(uint32_t n, uint32_t a, long long b) {
  if (n == 0) return 0;
  long long sum = static_cast<long long>(n) * (n - 1) / 2 * (a >> 7) + n * (b >> 7);
  uint32_t m = 128, c = static_cast<uint32_t>(b) & 127u;
  a &= 127u;
  for (;;) {
    const uint32_t top = a * n + c;
    if (top < m) return sum;
    n = top / m;  // at least 1
    c = top - n * m;
    const uint32_t old = a;
    a = m;
    m = old;
    sum += static_cast<long long>(n) * (n - 1) / 2 * (a / m) + static_cast<long long>(n) * (c / m);
    a %= m;
    c %= m;
  }
}

// ------------------------------------------------------------------------ the attention's work
// A request's new tokens × the group's query heads are the rows that read one key/value head. Each
// request goes by its own rows: up to kFewItems items of kRowsFew rows walk the keys in chunks of
// kChunkKeys; more rows are cut into items of kRowsMany (whole tokens) whose keys are walked in
// tiles of kTileKeys. A unit is one chunk or tile; a plan counts the units of one key/value head
// before each request, of either kind. An item of few rows reads its keys again, mostly from L2:
// on a B200 16 requests of 8000 keys and 8 heads took 110 us with 20 rows as three such items,
// 244 with 48 rows as six, and 127 as one item of many whatever its rows.
constexpr int kRowsFew = 8;
constexpr int kFewItems = 3;
constexpr int kChunkKeys = 64;
constexpr int kRowsMany = 256;
constexpr int kTileKeys = 128;

__host__ __device__ __forceinline__ bool few_rows(int group, long long added) {
  return group * added <= kRowsFew * kFewItems;
}

// Units before item `item` of a request with `cached` tokens before its new ones: the tiles of
// keys of each item (item i's last token sees cached + (i + 1) · tokens_of_item keys, the last
// item of a request fewer) and kItemUnits for its start and end.
constexpr int kItemUnits = 3;

__host__ __device__ __forceinline__ long long units_before(int group, long long cached,
                                                           long long item) {
  const int per = kRowsMany / group;
  return floor_sum_128(static_cast<uint32_t>(item), per, cached + per + kTileKeys - 1) +
         kItemUnits * item;
}

// Units of one key/value head of a request: of few rows, or of many.
__host__ __device__ __forceinline__ long long attention_units(int group, long long cached,
                                                              long long added) {
  if (added == 0) return 0;
  if (few_rows(group, added)) {
    return quotient(added * group + kRowsFew - 1, kRowsFew) * ((cached + added + kChunkKeys - 1) / kChunkKeys);
  }
  const int per = kRowsMany / group;
  const long long items = quotient(added + per - 1, per);
  return units_before(group, cached, items - 1) + (cached + added + kTileKeys - 1) / kTileKeys +
         kItemUnits;
}

}  // namespace cozy
