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
// (floor to ceiling is a factor of 2^100); magnitudes under 2^-69 are stored as zero, those over
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
  kPlanBadPage = 16,    // a page number outside [0, pages): its tokens are left out
  kPlanTimeout = 32,    // an on-chip wait of a call of this step ran past its limit
};
constexpr int kPlanRefused = kPlanNoPages | kPlanNarrow | kPlanTokens | kPlanLengths;

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

// Σ floor((a·i + b) / m) for i in [0, n), a, b ≥ 0 (the Euclid-like recursion on a and m).
__host__ __device__ inline long long floor_sum(long long n, long long m, long long a, long long b) {
  long long sum = 0;
  while (n > 0) {
    sum += (n - 1) * n / 2 * (a / m) + n * (b / m);
    a %= m;
    b %= m;
    const long long top = a * n + b;
    if (top < m) break;
    n = top / m;
    b = top % m;
    const long long t = a;
    a = m;
    m = t;
  }
  return sum;
}

// ------------------------------------------------------------------------ the attention's work
// A request's new tokens × the group's query heads are the rows that read one key/value head.
// Up to kRowsFew of them share one pass over the keys in chunks of kChunkKeys; more are cut into
// items of kRowsMany rows (whole tokens) whose keys are walked in tiles of kTileKeys. A unit is
// one chunk or tile; `units[n]` of a plan counts the units of one key/value head before request n.
constexpr int kRowsFew = 16;
constexpr int kChunkKeys = 64;
constexpr int kRowsMany = 256;
constexpr int kTileKeys = 128;

__host__ __device__ __forceinline__ bool few_rows(int group, int longest) {
  return static_cast<long long>(group) * longest <= kRowsFew;
}

// Tiles before item `item` of a request with `cached` tokens before its new ones: item i's last
// token sees cached + (i + 1) · tokens_of_item keys (the last item of a request fewer).
__host__ __device__ __forceinline__ long long tiles_before(int group, long long cached,
                                                           long long item) {
  const int per = kRowsMany / group;
  return floor_sum(item, kTileKeys, per, cached + per + kTileKeys - 1);
}

__host__ __device__ __forceinline__ long long attention_units(int group, int longest,
                                                              long long cached, long long added) {
  if (few_rows(group, longest)) return (cached + added + kChunkKeys - 1) / kChunkKeys;
  const int per = kRowsMany / group;
  const long long items = (added + per - 1) / per;
  return tiles_before(group, cached, items - 1) + (cached + added + kTileKeys - 1) / kTileKeys;
}

}  // namespace cozy
