// Attention over the 8-bit paged cache.
//
// Few rows a key/value head (a decode step): `attend_few`. All units of work (chunks of 64 keys
// of one head of one request) stand in one order, requests outermost, and every warp of the GPU
// takes an equal run of them, whatever the lengths are. A run that covers an item (one head of
// one request) writes its output; pieces of items leave fp32 rows and (max, sum) in the
// workspace, and a second kernel joins them in order: no atomics, the same bits every time. The
// join is launched while the first kernel runs, which hides the launch; its blocks start as SMs
// come free, since the first leaves none the registers (8192 of an SM with heads of 128, and a
// join's block takes 12288).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "../../include/cozy_ulysses.h"
#include "cache.cuh"
#include "sm100.cuh"

namespace cozy {

int cache_plan_check(const CozyCachePlan& p);
int cache_store_check(const CozyCacheStore& c, const CozyCachePlan& p);

// What both kernels read: the plan's answers, the pool and the call.
struct CacheArgs {
  const int* table;
  long long table_stride;
  const int* starts;
  const int* lengths;
  const long long* units_few;   // [requests + 1] units of one head before each request
  const long long* units_many;  // (a request has units of one kind only)
  int* status;
  int requests, pages, page, page_shift, group, heads_kv;
  const int8_t* key_exponent;
  const int8_t* value_exponent;
  const __nv_bfloat16* query;
  long long q_token, q_head;
  __nv_bfloat16* out;
  long long o_token, o_head;
  float* lse;
  uint32_t per_group;  // ceil(2^16 / group): r · per_group >> 16 is r / group for rows r < 256
  float scale_log2;  // softmax scale · log2(e)
  float* ws_o;       // [worker][2][rows][HD]
  float2* ws_ml;     // [worker][2][rows]
  int workers;
};

// 2^15 over a row's reference: P ≤ 2^15 in f16, normal down to 2^-29 of the row's largest term.
constexpr float kFewBias = 15.0f;

__device__ __forceinline__ void tma_load_2d(void* dst, const void* tmap, uint64_t* bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(tmap)), "r"(smem_u32(bar)), "r"(x), "r"(y)
      : "memory");
}

// A bounded wait that reports through the plan's status word.
__device__ __noinline__ bool cache_wait_slow(uint64_t* bar, uint32_t parity, int* status) {
  const uint64_t start = global_timer_ns();
  for (uint32_t spin = 1;; ++spin) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((spin & 63u) == 0 && global_timer_ns() - start > kWaitLimitNs) {
      atomicOr(status, kPlanTimeout);
      return false;
    }
  }
}

__device__ __forceinline__ bool cache_wait(uint64_t* bar, uint32_t parity, int* status) {
  return mbar_try_wait(bar, parity) || cache_wait_slow(bar, parity, status);
}

__device__ __forceinline__ uint4 lds128(uint32_t at) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "r"(at));
  return r;
}

__device__ __forceinline__ uint2 lds64(uint32_t at) {
  uint2 r;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "r"(at));
  return r;
}

// Four codes to two pairs of f16 (exact).
__device__ __forceinline__ void widen4(uint32_t codes, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(codes));
}

// D[16 × 8] += A[16 × 16] · B[16 × 8], f16 in, fp32 accumulators.
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7},"
      " {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t f16_pair(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Bytes of `codes` that are e4m3's NaN (0x7f or 0xff), as 0xff.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t codes) {
  return __vcmpeq4(codes & 0x7f7f7f7fu, 0x7f7f7f7fu);
}

// The request whose units hold `u` (units of all its heads), by all lanes together: 32 places
// of the search range are read at once, so 8192 requests take three rounds.
__device__ __forceinline__ int request_of(const CacheArgs& a, const long long* units, long long u) {
  const int lane = threadIdx.x & 31;
  int low = 0, count = a.requests;  // the answer is in [low, low + count)
  while (count > 1) {
    const int step = (count + 31) / 32;
    const int at = low + lane * step;
    const bool before = lane * step < count && units[at] * a.heads_kv <= u;
    const int last = 31 - __clz(__ballot_sync(0xffffffffu, before));
    const int used = last * step;
    low += used;
    count = min(step, count - used);
  }
  return low;
}

// ------------------------------------------------------------------------------- few rows
// HBM bounds this: a chunk is 2 · 64 · HD bytes (64 requests of 2000 to 16384 keys, 32/8 heads of
// 128: 1.16 GB in 199 us, 0.89 of the measured copy rate). The matrix instructions are mma.sync m16n8k16
// with the keys as their 16 rows and the 8 query rows of an item as their columns (queries as the
// 16 rows left half of every instruction, weight and accumulator of a decode step unused: 64
// requests of 10000 keys 223 against 211 us in a loop under the power cap, 10 requests of 1800
// keys and 24 heads 37 against 32). Codes are widened to f16 in registers (exact) straight from the
// swizzled tile that TMA wrote. The operand layouts are chosen so that no transposing load is needed: the
// contraction over channels may run in any order, so a thread's 16 consecutive channels of a key
// serve four instructions; the keys of a tile may be taken in any order (row c is
// (c & 1 ? c + 4 : c) mod 8 of 8, which keeps the 16-byte reads of both K and V free of bank
// conflicts); V's pairs of keys are joined by byte permutes before widening; and movmatrix turns
// the weights from a thread a key to a thread a row.
template <int HD>
struct Few {
  static constexpr int kWarps = HD == 128 ? 8 : 12;
  static constexpr int kSlotBytes = kChunkKeys * HD;
  static constexpr int kSlots = 196608 / kWarps / kSlotBytes;  // rings of 192 KB an SM
  static constexpr int kMeta = 8;                              // chunks whose scales are kept
  static constexpr int kBarOffset = kWarps * kSlots * kSlotBytes;
  static constexpr int kMetaOffset = kBarOffset + kWarps * kSlots * 8;
  static constexpr int kAlloc = kMetaOffset + kWarps * kMeta * 32 + 1024;
};

// A position in the order of units, moved on chunk by chunk.
struct FewAt {
  int n, h, item, j;  // request, head, rows of it, chunk of keys
  int items, chunks;  // items of a head, chunks of an item
  int keys;           // the request's tokens
};

__device__ __forceinline__ void few_request(const CacheArgs& a, FewAt& at, int n) {
  at.n = n;
  at.keys = a.lengths[n];
  at.items = a.units_few[n + 1] == a.units_few[n]
                 ? 0
                 : ((a.starts[n + 1] - a.starts[n]) * a.group + kRowsFew - 1) / kRowsFew;
  at.chunks = (at.keys + kChunkKeys - 1) / kChunkKeys;
}

__device__ __forceinline__ FewAt few_at(const CacheArgs& a, long long u) {
  FewAt at;
  few_request(a, at, request_of(a, a.units_few, u));
  const long long within = u - a.units_few[at.n] * a.heads_kv;
  const long long item = quotient(within, at.chunks);
  at.j = static_cast<int>(within - item * at.chunks);
  at.h = static_cast<int>(quotient(item, at.items));
  at.item = static_cast<int>(item - static_cast<long long>(at.h) * at.items);
  return at;
}

// To the next chunk; true when it belongs to another item.
__device__ __forceinline__ bool few_next(const CacheArgs& a, FewAt& at) {
  if (++at.j < at.chunks) return false;
  at.j = 0;
  if (++at.item < at.items) return true;
  at.item = 0;
  if (++at.h == a.heads_kv) {
    at.h = 0;
    do few_request(a, at, at.n + 1);
    while (at.items == 0);  // only reached while units remain
  }
  return true;
}

__device__ __forceinline__ uint32_t transposed(uint32_t pair) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(pair));
  return r;
}

template <int HD>
__global__ void __launch_bounds__(Few<HD>::kWarps * 32, 1)
    attend_few(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
               const CacheArgs a) {
  using L = Few<HD>;
  constexpr int KSTEPS = HD / 16;  // k16 steps of K·Q
  constexpr int XT = HD / 16;      // 16-channel tiles of the output
  extern __shared__ uint8_t few_smem[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(few_smem) + 1023) & ~static_cast<uintptr_t>(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  uint8_t* ring = smem + warp * (L::kSlots * L::kSlotBytes);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kBarOffset) + warp * L::kSlots;
  // scales of a chunk's up to four pages: {2^key exponent, value exponent}
  float2* meta = reinterpret_cast<float2*>(smem + L::kMetaOffset) + warp * L::kMeta * 4;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  const long long total = a.units_few[a.requests] * a.heads_kv;
  const int workers = static_cast<int>(min(static_cast<long long>(a.workers), total));
  const int worker = warp * gridDim.x + blockIdx.x;
  if (worker >= workers) return;  // warps share nothing
  const long long u0 = quotient(worker * total, workers), u1 = quotient((worker + 1) * total, workers);
  if (lane == 0) {
    for (int i = 0; i < L::kSlots; ++i) mbar_init(&full[i], 1);
    fence_barrier_init();
  }
  __syncwarp();

  // ---- the loads: fill f is the keys (even) or values (odd) of unit u0 + f / 2
  const int box_shift = min(a.page_shift, 6), box = 1 << box_shift, per_chunk = kChunkKeys >> box_shift;
  const unsigned units = static_cast<unsigned>(u1 - u0), fills = 2 * units;
  FewAt to = few_at(a, u0);  // the chunk to load next
  FewAt at = to;             // the chunk to compute
  int batch = 0, id = -1, ids = 0;  // a lane's page number among 32 of the item's, of the chunk's
  int key_e = 0, value_e = 0;       // its page's exponents
  bool fresh_pages = true, fresh_scales = true;
  auto load = [&](unsigned f) {
    if (f >= fills) return;
    const unsigned slot = f % L::kSlots;
    const int first = to.j * kChunkKeys >> a.page_shift;
    const int offset = to.j * kChunkKeys & (a.page - 1);
    const int count = min(per_chunk, (to.keys - to.j * kChunkKeys + box - 1) >> box_shift);
    const bool keys = (f & 1) == 0;
    if (keys) {
      const bool other = first < batch || first + per_chunk > batch + 32;
      if (fresh_pages || other) {
        batch = first;
        id = -1;
        const int index = first + lane;
        if (index * static_cast<long long>(a.page) < to.keys) {
          id = a.table[to.n * a.table_stride + index];
          if (id < 0 || id >= a.pages) {
            id = -1;
            atomicOr(a.status, kPlanBadPage);
          }
        }
      }
      ids = __shfl_sync(0xffffffffu, id, (first - batch + (lane & 3)) & 31);
      if (lane >= count) ids = -1;
      fresh_scales |= fresh_pages || other;
      fresh_pages = false;
    }
    const unsigned there = __ballot_sync(0xffffffffu, lane < per_chunk && ids >= 0);
    if (lane == 0) mbar_expect_tx(&full[slot], __popc(there) * box * HD);
    __syncwarp();
    if (lane < per_chunk && ids >= 0)
      tma_load_2d(ring + slot * L::kSlotBytes + lane * box * HD, keys ? &tm_k : &tm_v, &full[slot],
                  0, (ids * a.heads_kv + to.h) * a.page + offset);
    if (keys) {
      if (fresh_scales) {  // asked for here, looked at when the chunk's values are loaded
        fresh_scales = false;
        key_e = value_e = 0;
        if (id >= 0) {
          const long long block = static_cast<long long>(id) * a.heads_kv + to.h;
          key_e = a.key_exponent[block];
          value_e = a.value_exponent[block];
        }
      }
    } else {
      // the chunk's scales; a page that is not there has a scale of zero
      const int from = (first - batch + (lane & 3)) & 31;
      const int ke = __shfl_sync(0xffffffffu, key_e, from), ve = __shfl_sync(0xffffffffu, value_e, from);
      if (lane < per_chunk)
        meta[(f >> 1) % L::kMeta * 4 + lane] =
            make_float2(ids < 0 ? 0.f : exponent_scale(ke), static_cast<float>(ve));
      __syncwarp();
      if (f + 1 < fills) {
        const int was = to.n;
        if (few_next(a, to)) {
          fresh_scales = true;
          fresh_pages = to.n != was;  // a request's heads share its pages
        }
      }
    }
  };
  for (unsigned f = 0; f < L::kSlots; ++f) load(f);

  const int order = (g & 1) ? ((g + 4) & 7) : g;  // row of this lane's column of K
  const uint32_t base = smem_u32(ring);
  uint32_t k_off[HD / 64];
#pragma unroll
  for (int c = 0; c < HD / 64; ++c)
    k_off[c] = HD == 128 ? order * 128 + (((t + 4 * c) ^ order) << 4)
                         : order * 64 + ((t ^ ((order >> 1) & 3)) << 4);
  const int row0 = 2 * t, row1 = (2 * t + 5) & 7;  // rows of columns 2t and 2t + 1
  uint32_t v_off[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = i ? row1 : row0;
    v_off[i] = HD == 128 ? r * 128 + ((g ^ r) << 4)
                         : r * 64 + (((g >> 1) ^ ((r >> 1) & 3)) << 4) + (g & 1) * 8;
  }

  bool ok = true;
  unsigned u = 0;
  while (u < units && ok) {
    // ---- an item, or the part of it that this worker has
    const int first_token = a.starts[at.n], added = a.starts[at.n + 1] - first_token;
    const int first_row = at.item * kRowsFew;
    const int rows = min(kRowsFew, added * a.group - first_row);
    const int seen0 = at.keys - added + first_row / a.group;  // keys before the first row's own
    const int cached = at.keys - added;
    const int j0 = at.j;
    const int steps = static_cast<int>(min(units - u, static_cast<unsigned>(at.chunks - at.j)));
    // Query row g times a power of two that puts their largest value in [2^14, 2^15),
    // as the columns of K · Q; scores and outputs come to this thread for rows 2t and 2t + 1.
    uint32_t q[KSTEPS][2];
    float mul[2];
    int last[2], last_g;  // the last key that a row sees
    const int row = g;
    last_g = cached + (first_row + min(row, rows - 1)) / a.group;
    uint4 x[HD / 64][2];
    float amax = 0.f;
#pragma unroll
    for (int c = 0; c < HD / 64; ++c) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        x[c][k] = make_uint4(0, 0, 0, 0);
        if (row < rows)
          x[c][k] = *reinterpret_cast<const uint4*>(
              a.query + (first_token + (first_row + row) / a.group) * a.q_token +
              (at.h * a.group + (first_row + row) % a.group) * a.q_head + (t + 4 * c) * 16 + k * 8);
        const uint32_t w[4] = {x[c][k].x, x[c][k].y, x[c][k].z, x[c][k].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          amax = fmaxf(amax, fabsf(__uint_as_float(w[e] << 16)));
          amax = fmaxf(amax, fabsf(__uint_as_float(w[e] & 0xffff0000u)));
        }
      }
    }
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    const int up = min(100, 14 + 127 - static_cast<int>(__float_as_uint(amax) >> 23));
    // scores of an infinity have no softmax: under a scale of zero it is NaN, and its row with it
    const float s = amax == INFINITY ? 0.f : exponent_scale(up), back = a.scale_log2 * exponent_scale(-up);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      mul[i] = __shfl_sync(0xffffffffu, back, 4 * (2 * t + i));
      last[i] = __shfl_sync(0xffffffffu, last_g, 4 * (2 * t + i));
    }
#pragma unroll
    for (int c = 0; c < HD / 64; ++c) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint32_t w[4] = {x[c][k].x, x[c][k].y, x[c][k].z, x[c][k].w};
#pragma unroll
        for (int e = 0; e < 4; ++e)  // words 2i, 2i + 1 of the 8 a chunk are step i's two registers
          q[c * 4 + (k * 4 + e) / 2][e & 1] =
              f16_pair(__uint_as_float(w[e] << 16) * s, __uint_as_float(w[e] & 0xffff0000u) * s);
      }
    }
    float o[XT][4];
#pragma unroll
    for (int x = 0; x < XT; ++x)
      o[x][0] = o[x][1] = o[x][2] = o[x][3] = 0.f;
    float m[2], l[2];
    m[0] = m[1] = -INFINITY;
    l[0] = l[1] = 0.f;

    for (int step = 0; step < steps; ++step, ++u) {
      const unsigned f = 2 * u;
      unsigned slot = f % L::kSlots;
      if (!(ok = __all_sync(0xffffffffu, cache_wait(&full[slot], (f / L::kSlots) & 1, a.status)))) break;
      const float2* scales = meta + (f >> 1) % L::kMeta * 4;
      const int key0 = (j0 + step) * kChunkKeys;
      // ---- scores: tile kt of 16 keys; s[..][0, 1]: this lane's key of 8 for rows 2t, 2t + 1;
      // [2, 3]: the key 8 behind
      float s[4][4];
#pragma unroll
      for (int kt = 0; kt < 4; ++kt) {
        s[kt][0] = s[kt][1] = s[kt][2] = s[kt][3] = 0.f;
#pragma unroll
        for (int c = 0; c < HD / 64; ++c) {
          const uint32_t from = base + slot * L::kSlotBytes + kt * 16 * HD + k_off[c];
          const uint4 lo = lds128(from), hi = lds128(from + 8 * HD);
          const uint32_t w0[4] = {lo.x, lo.y, lo.z, lo.w}, w1[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t k[4];
            widen4(w0[e], k[0], k[2]);
            widen4(w1[e], k[1], k[3]);
            mma16816(s[kt], k, q[c * 4 + e][0], q[c * 4 + e][1]);
          }
        }
      }
      __syncwarp();
      // the scales are read before the ring of chunks moves on
      float2 sc[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) sc[i] = scales[i >> (box_shift - 4)];
      __syncwarp();
      load(f + L::kSlots);
      bool whole = key0 + kChunkKeys <= seen0 + 1;  // every row sees every key
#pragma unroll
      for (int i = 0; i < 4; ++i) whole = whole && sc[i].x != 0.f;
      float top[2];
      bool grew = false;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float most = m[i];
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) {
          const float f0 = mul[i] * sc[kt].x;
          float& near = s[kt][i];
          float& far = s[kt][2 + i];
          near = fmaf(near, f0, sc[kt].y);
          far = fmaf(far, f0, sc[kt].y);
          if (!whole) {
            const int key = key0 + kt * 16 + order;
            const bool gone = sc[kt].x == 0.f;
            if (gone || key > last[i]) near = -INFINITY;
            if (gone || key + 8 > last[i]) far = -INFINITY;
          }
          most = fmaxf(most, fmaxf(near, far));
        }
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
        top[i] = most;
        grew |= most > m[i];
      }
      if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float w = m[i] == -INFINITY ? 0.f : ex2_approx(m[i] - top[i]);
          l[i] *= w;
          m[i] = top[i];
#pragma unroll
          for (int x = 0; x < XT; ++x) {
            o[x][i] *= w;
            o[x][2 + i] *= w;
          }
        }
      }
      // weights 2^(s + e - m), their sum without the value's 2^e; p: a thread a row (g)
      uint32_t p[4][2];
      const float r0 = (m[0] == -INFINITY ? 0.f : m[0]) - kFewBias;
      const float r1 = (m[1] == -INFINITY ? 0.f : m[1]) - kFewBias;
#pragma unroll
      for (int kt = 0; kt < 4; ++kt) {
        const float back = exponent_scale(-static_cast<int>(sc[kt].y));
        const float p0 = ex2_approx(s[kt][0] - r0), p1 = ex2_approx(s[kt][1] - r1);
        const float p2 = ex2_approx(s[kt][2] - r0), p3 = ex2_approx(s[kt][3] - r1);
        l[0] = fmaf(p0 + p2, back, l[0]);
        l[1] = fmaf(p1 + p3, back, l[1]);
        p[kt][0] = transposed(f16_pair(p0, p1));
        p[kt][1] = transposed(f16_pair(p2, p3));
      }
      // ---- values
      slot = (f + 1) % L::kSlots;
      if (!(ok = __all_sync(0xffffffffu, cache_wait(&full[slot], ((f + 1) / L::kSlots) & 1, a.status)))) break;
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        constexpr int WORDS = HD / 32;  // words of 4 channels a thread and key
        uint32_t v[4][WORDS];
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // keys row0, row1, 8 + row0, 8 + row1 of 16
          const uint32_t from = base + slot * L::kSlotBytes + (kk * 16 + (i >> 1) * 8) * HD + v_off[i & 1];
          if constexpr (HD == 128) {
            const uint4 x = lds128(from);
            v[i][0] = x.x; v[i][1] = x.y; v[i][2] = x.z; v[i][3] = x.w;
          } else {
            const uint2 x = lds64(from);
            v[i][0] = x.x; v[i][1] = x.y;
          }
        }
        if (!whole) {
          // Codes behind the last key of the request and in pages that are not there are whatever
          // they are, and a NaN that some row does not see must not reach it as 0 · NaN: both
          // become zeros here, and rows that do see a NaN get it by a product of ones.
          uint32_t any = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int at16 = kk * 16 + (i >> 1) * 8 + ((i & 1) ? row1 : row0);
            const bool gone = sc[kk].x == 0.f || key0 + at16 >= at.keys;
#pragma unroll
            for (int w = 0; w < WORDS; ++w) {
              if (gone) v[i][w] = 0;
              any |= nan_bytes(v[i][w]);
            }
          }
          if (__any_sync(0xffffffffu, any != 0)) {
            const int k = key0 + kk * 16, to_row = last_g;
            const uint32_t see0 = f16_pair(k + row0 <= to_row ? 1.f : 0.f, k + row1 <= to_row ? 1.f : 0.f);
            const uint32_t see1 = f16_pair(k + 8 + row0 <= to_row ? 1.f : 0.f, k + 8 + row1 <= to_row ? 1.f : 0.f);
#pragma unroll
            for (int x = 0; x < XT; ++x) {
              auto one = [&](int i, int c) { return (nan_bytes(v[i][c / 4]) >> (c & 3) * 8 & 0xffu) ? 0x3c00u : 0u; };
              const uint32_t n[4] = {one(0, 2 * x) | one(1, 2 * x) << 16, one(0, 2 * x + 1) | one(1, 2 * x + 1) << 16,
                                     one(2, 2 * x) | one(3, 2 * x) << 16, one(2, 2 * x + 1) | one(3, 2 * x + 1) << 16};
              float hit[4] = {0.f, 0.f, 0.f, 0.f};
              mma16816(hit, n, see0, see1);
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (hit[i] > 0.f) o[x][i] = __uint_as_float(0x7fc00000u);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int w = 0; w < WORDS; ++w) v[i][w] &= ~nan_bytes(v[i][w]);
          }
        }
#pragma unroll
        for (int w = 0; w < WORDS; ++w) {
          uint32_t x0[4], x1[4];  // channels 4w, 4w + 1 and 4w + 2, 4w + 3 of this lane's
          widen4(__byte_perm(v[0][w], v[1][w], 0x5140), x0[0], x0[1]);
          widen4(__byte_perm(v[2][w], v[3][w], 0x5140), x0[2], x0[3]);
          widen4(__byte_perm(v[0][w], v[1][w], 0x7362), x1[0], x1[1]);
          widen4(__byte_perm(v[2][w], v[3][w], 0x7362), x1[2], x1[3]);
          mma16816(o[2 * w], x0, p[kk][0], p[kk][1]);
          mma16816(o[2 * w + 1], x1, p[kk][0], p[kk][1]);
        }
      }
      __syncwarp();
      load(f + 1 + L::kSlots);
    }
    if (!ok) break;
    // ---- the item's end: this thread has channels [g · HD / 8, + HD / 8) of rows 2t and 2t + 1
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float sum = l[i];
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      const int row = 2 * t + i;
      if (row >= rows) continue;
      if (steps == at.chunks) {
        const int token = first_token + (first_row + row) / a.group;
        const int head = at.h * a.group + (first_row + row) % a.group;
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        uint4* to_row = reinterpret_cast<uint4*>(a.out + token * a.o_token + head * a.o_head + g * (HD / 8));
#pragma unroll
        for (int x = 0; x < XT; x += 4)
          to_row[x / 4] = make_uint4(
              pack_bf16x2(o[x][i] * inv, o[x][2 + i] * inv),
              pack_bf16x2(o[x + 1][i] * inv, o[x + 1][2 + i] * inv),
              pack_bf16x2(o[x + 2][i] * inv, o[x + 2][2 + i] * inv),
              pack_bf16x2(o[x + 3][i] * inv, o[x + 3][2 + i] * inv));
        if (a.lse != nullptr && g == 0)
          a.lse[static_cast<long long>(token) * a.heads_kv * a.group + head] =
              sum == 0.f ? -INFINITY : 0.6931471805599453f * (m[i] - kFewBias + __log2f(sum));
      } else {
        const long long part = (2LL * worker + (j0 == 0 ? 1 : 0)) * kRowsFew + row;
        float4* to_row = reinterpret_cast<float4*>(a.ws_o + part * HD + g * (HD / 8));
#pragma unroll
        for (int x = 0; x < XT; x += 2)
          to_row[x / 2] = make_float4(o[x][i], o[x][2 + i], o[x + 1][i], o[x + 1][2 + i]);
        if (g == 0) a.ws_ml[part] = make_float2(m[i], sum);
      }
    }
    at.j += steps - 1;
    if (u < units) few_next(a, at);
  }
  if (!ok) {  // copies in flight land before the warp leaves
    const unsigned f = 2 * u;
    for (unsigned i = f; i < f + 2 * L::kSlots && i < fills; ++i)
      cache_wait_slow(&full[i % L::kSlots], (i / L::kSlots) & 1, a.status);
  }
}

// Joins the parts of an item that several workers had: block (item, row). The parts' references
// and sums are read at once, a thread a part; then 8 warps add the parts up, in a fixed order.
constexpr int kMostParts = 2048;  // workers: 8 or 12 warps an SM

template <int HD>
__global__ void __launch_bounds__(256) join_few(const CacheArgs a) {
  constexpr int PER = HD / 32;  // channels a lane
  __shared__ float weight[kMostParts];
  __shared__ float sum_o[8][HD];
  __shared__ float warp_top[8], warp_sum[8];
  const int n = blockIdx.x / a.heads_kv, h = blockIdx.x % a.heads_kv;
  const int item = blockIdx.y / kRowsFew, row = blockIdx.y % kRowsFew;
  const int start = a.starts[n], next = a.starts[n + 1], length = a.lengths[n];
  const long long before = a.units_few[n], behind = a.units_few[n + 1], all = a.units_few[a.requests];
  const int rows = behind == before ? 0 : (next - start) * a.group;
  const int items = (rows + kRowsFew - 1) / kRowsFew;
  const long long chunks = (length + kChunkKeys - 1) / kChunkKeys;
  const long long total = all * a.heads_kv;
  const long long workers = min(static_cast<long long>(a.workers), total);
  const long long u0 = before * a.heads_kv + (static_cast<long long>(h) * items + item) * chunks;
  const int first = total == 0 ? 0 : static_cast<int>(quotient((u0 + 1) * workers - 1, total));
  const int last = total == 0 ? 0 : static_cast<int>(quotient((u0 + chunks) * workers - 1, total));
  const bool split = static_cast<int>(blockIdx.y) < rows && first != last;
  // one block at least waits, so that this grid does not end before the one it follows
  if (split || (blockIdx.x == 0 && blockIdx.y == 0)) asm volatile("griddepcontrol.wait;" ::: "memory");
  if (!split) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, parts = last - first + 1;
  auto place = [&](int p) { return (2LL * (first + p) + (p == 0 ? 1 : 0)) * kRowsFew + row; };
  // the loads of the parts' rows do not wait for their weights
  constexpr int AHEAD = 4;
  float x[AHEAD][PER] = {};
#pragma unroll
  for (int i = 0; i < AHEAD; ++i)
#pragma unroll
    for (int c = 0; c < PER; ++c)
      if (warp + 8 * i < parts) x[i][c] = __ldcg(&a.ws_o[place(warp + 8 * i) * HD + c * 32 + lane]);
  float top = -INFINITY;
  for (int p = threadIdx.x; p < parts; p += 256) top = fmaxf(top, __ldcg(&a.ws_ml[place(p)]).x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) warp_top[warp] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) top = fmaxf(top, warp_top[i]);
  float sum = 0.f;
  for (int p = threadIdx.x; p < parts; p += 256) {
    const float2 ml = __ldcg(&a.ws_ml[place(p)]);
    // a part without a key has zeros; one whose scores are NaN has a sum of NaN
    const float w = ml.x == -INFINITY ? 1.f : ex2_approx(ml.x - top);
    weight[p] = w;
    sum += ml.y * w;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) warp_sum[warp] = sum;
  __syncthreads();
  float o[PER];
#pragma unroll
  for (int c = 0; c < PER; ++c) o[c] = 0.f;
  for (int p = warp; p < parts; p += 8 * AHEAD) {
    float y[AHEAD][PER] = {};  // the next ones, meanwhile
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
#pragma unroll
      for (int c = 0; c < PER; ++c)
        if (p + 8 * (AHEAD + i) < parts)
          y[i][c] = __ldcg(&a.ws_o[place(p + 8 * (AHEAD + i)) * HD + c * 32 + lane]);
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      if (p + 8 * i < parts) {
        const float w = weight[p + 8 * i];
#pragma unroll
        for (int c = 0; c < PER; ++c) o[c] = fmaf(x[i][c], w, o[c]);
      }
#pragma unroll
      for (int c = 0; c < PER; ++c) x[i][c] = y[i][c];
    }
  }
#pragma unroll
  for (int c = 0; c < PER; ++c) sum_o[warp][c * 32 + lane] = o[c];
  __syncthreads();
  const int d = threadIdx.x;
  if (d >= HD) return;
  float value = 0.f;
  sum = 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    value += sum_o[w][d];
    sum += warp_sum[w];
  }
  const int token = start + blockIdx.y / a.group, head = h * a.group + blockIdx.y % a.group;
  a.out[token * a.o_token + head * a.o_head + d] = __float2bfloat16(sum == 0.f ? 0.f : value / sum);
  if (a.lse != nullptr && d == 0)
    a.lse[static_cast<long long>(token) * a.heads_kv * a.group + head] =
        sum == 0.f ? -INFINITY : 0.6931471805599453f * (top - kFewBias + __log2f(sum));
}

// ------------------------------------------------------------------------------ many rows
// Items of up to 256 query rows (whole tokens of one head's group) over tiles of 128 keys, on
// the 5th-generation tensor cores: two query tiles of 128 rows take turns, so that one's softmax
// runs while the other's products do. Every CTA takes an equal run of all units, item after item
// (one head's items are neighbours and share its keys in L2).
//
//   warps 0-3, 4-7  softmax of query tile 0, 1 (a thread a row, a TMEM lane)
//   warp  8         page numbers, scales, and TMA of K and V codes into their rings
//   warps 9, 10     the matrix instructions of query tile 0, 1
//   warps 12-15     V's codes widened to f16 (exact); they also see K's next tile in, so that
//                   the issuer waits once for both
//
// S = Q·Kᵀ runs in 8 bits on K's codes as they are stored, with Q split into two e4m3 parts
// under one power of two a row that puts its largest value in (224, 448]: q = hi + lo holds all 8
// bits of a bf16 from 2^-2 on, which is at most 2^-9.8 of the largest, and a smaller one to half of
// e4m3's smallest step, 2^-10: 2^-17.8 of the largest or less. Two 8-bit products cost what one
// 16-bit product costs, and K needs neither widening nor more than its stored bytes of shared
// memory. P stays in f16 (11 bits; two 8-bit parts would lose the weights under 2^-17 of a row's
// largest, which a long context has many of), so V is widened.
//
// A tile of keys is taken in two halves of 64 with a buffer of S each, so that the next half's
// Q·Kᵀ is done when a half's softmax ends: neither the tensor cores nor the softmax wait for the
// other's round trip. (With one buffer of 128 a unit took 3823 clocks, 2129 of them on the tensor
// cores.) A chunk of 1024 tokens behind 130047 keys (32/8 heads of 128) takes 4.1 M clocks: 2.12 ms
// at 1965 MHz, and in a loop under the power cap 2.48 ms at 1657 MHz, 885 TFLOP/s, 0.53 of the
// measured bf16 rate. That is 4650 clocks a unit, of which the exponentials take 2092 and the matrix
// instructions 2448: as much as both, one after the other. Tensor memory: S/P of tile s, half b at column 128 s + 64 b, O at 256 + HD s.
template <int HD>
struct Many {
  static constexpr int kThreads = 512;
  static constexpr int kKStages = 3, kV8Stages = 2, kV16Stages = 2;
  static constexpr int kScaleRing = 8;
  static constexpr int kCodeTile = 128 * HD;      // 128 rows of codes
  static constexpr int kQOffset = 0;              // [tile][hi, lo]
  static constexpr int kKOffset = 4 * kCodeTile;
  static constexpr int kV8Offset = kKOffset + kKStages * kCodeTile;
  static constexpr int kV16Offset = kV8Offset + kV8Stages * kCodeTile;
  static constexpr int kPoisonOffset = kV16Offset + kV16Stages * 2 * kCodeTile;  // [256 rows][16]
  static constexpr int kNanOffset = kPoisonOffset + 256 * 16;  // [V16 slot][128 keys][16 bytes]
  static constexpr int kScaleOffset = kNanOffset + kV16Stages * 128 * 16;
  // [ring]{2^key exponent [8], value exponent [8], 2^-value exponent [8], gone groups, pad}
  static constexpr int kScaleBytes = 112;
  static constexpr int kBarOffset = kScaleOffset + kScaleRing * kScaleBytes;
  static constexpr int kBars = 2 + 2 * kKStages + 2 * kV8Stages + 2 * kV16Stages + 4 + 4 + 4 +
                               kScaleRing + 1;
  static constexpr int kMiscOffset = kBarOffset + kBars * 8;
  static constexpr int kAtOffset = kMiscOffset + 32;  // each softmax warp's place in its run
  static constexpr int kAlloc = kAtOffset + 8 * 64 + 1024;
};
// Registers: 512 threads start with 128 each; 256 · 168 + 256 · 88 = 65536, what they started with.
constexpr int kManySoftmaxRegs = 168;
constexpr int kManyOtherRegs = 88;
constexpr int kWideners = 128;  // threads that widen V: a warp on each sub-partition

// P = 2^(s - m + 7) against a reference that may lie 2^8 below the row's largest (O is rescaled
// only when the maximum grew by more): at most 2^15 in f16, normal down to 2^-21 of the reference.
constexpr float kManyBias = 7.0f;
constexpr float kManySlack = 8.0f;

// A group's multiplier of scores: never zero, so that a hidden score's -inf stays one (products
// below 2^-120 are scores of nothing either way).
__device__ __forceinline__ float group_mul(float mul, float key_scale) {
  return fmaxf(mul * key_scale, 7.52316385e-37f);
}

// A worker's part of an item. Its units are the item's kItemUnits, then its tiles of keys.
struct ManyAt {
  int n, h, item;    // request, head, item
  int j, steps;      // first tile of keys, tiles
  int items, tiles;  // items of the request's head, tiles of this item
  int keys, cached, added, first_token;
  int left, units;  // units left to the worker from this part on; units of the part
};

// The part of the item that begins at its unit `unit`; the run ends where a part has no tile.
__device__ __forceinline__ void many_part(const CacheArgs& a, ManyAt& at, int unit) {
  const int per = kRowsMany / a.group;
  at.tiles = (at.cached + min((at.item + 1) * per, at.added) + kTileKeys - 1) / kTileKeys;
  at.j = max(0, unit - kItemUnits);
  at.units = min(at.left, kItemUnits + at.tiles - unit);
  at.steps = unit + at.units - kItemUnits - at.j;
}

__device__ __forceinline__ void many_request(const CacheArgs& a, ManyAt& at, int n) {
  const int per = kRowsMany / a.group;
  at.n = n;
  at.first_token = a.starts[n];
  at.added = a.starts[n + 1] - at.first_token;
  at.keys = a.lengths[n];
  at.cached = at.keys - at.added;
  at.items = a.units_many[n + 1] == a.units_many[n] ? 0 : (at.added + per - 1) / per;
}

__device__ __forceinline__ ManyAt many_at(const CacheArgs& a, long long u, int left) {
  ManyAt at;
  at.left = left;
  many_request(a, at, request_of(a, a.units_many, u));
  const long long units = a.units_many[at.n + 1] - a.units_many[at.n];
  const long long within = u - a.units_many[at.n] * a.heads_kv;
  at.h = static_cast<int>(quotient(within, units));
  const long long rest = within - at.h * units;
  const int lane = threadIdx.x & 31;
  int low = 0, count = at.items;  // 32 places of the search range at once
  while (count > 1) {
    const int step = (count + 31) / 32;
    const bool before = lane * step < count && units_before(a.group, at.cached, low + lane * step) <= rest;
    const int used = (31 - __clz(__ballot_sync(0xffffffffu, before))) * step;
    low += used;
    count = min(step, count - used);
  }
  at.item = low;
  many_part(a, at, static_cast<int>(rest - units_before(a.group, at.cached, low)));
  return at;
}

// To the worker's part of the next item.
__device__ __forceinline__ void many_next(const CacheArgs& a, ManyAt& at) {
  at.left -= at.units;
  if (at.left <= 0) {
    at.steps = 0;
    return;
  }
  if (++at.item == at.items) {
    at.item = 0;
    if (++at.h == a.heads_kv) {
      at.h = 0;
      do many_request(a, at, at.n + 1);
      while (at.items == 0);  // only reached while units remain
    }
  }
  many_part(a, at, 0);
}

// A warp's place in shared memory: what the loop over tiles does not need stands there, not in
// registers (128 scores and 16 weights a thread leave few).
__device__ __forceinline__ void many_put(volatile int* to, const ManyAt& at) {
  __syncwarp();
  const int v[13] = {at.n, at.h, at.item, at.j, at.steps, at.items, at.tiles, at.keys, at.cached,
                     at.added, at.first_token, at.left, at.units};
#pragma unroll
  for (int i = 0; i < 13; ++i) to[i] = v[i];
  __syncwarp();
}

__device__ __forceinline__ ManyAt many_get(const volatile int* from) {
  return {from[0], from[1], from[2], from[3], from[4], from[5], from[6], from[7], from[8], from[9],
          from[10], from[11], from[12]};
}

// Halves of the part's tiles: the last tile of an item may need only one.
__device__ __forceinline__ int many_halves(const CacheArgs& a, const ManyAt& at) {
  const int keys = at.cached + min((at.item + 1) * (kRowsMany / a.group), at.added);
  return min(2 * at.steps, (keys - at.j * kTileKeys + 63) / 64);
}

// The token of an item's row, and its head of the group.
__device__ __forceinline__ int row_token(const CacheArgs& a, int row) {
  return static_cast<int>(row * a.per_group >> 16);
}

__device__ __forceinline__ int many_rows(const CacheArgs& a, const ManyAt& at) {
  const int per = kRowsMany / a.group;
  return min(per, at.added - at.item * per) * a.group;
}

__device__ __forceinline__ bool many_wait(uint64_t* bar, uint32_t parity, volatile int* abort,
                                          int* status) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t start = global_timer_ns();
  for (uint32_t spin = 1;; ++spin) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((spin & 63u) == 0) {
      if (*abort) return false;
      if (global_timer_ns() - start > kWaitLimitNs) {
        *abort = 1;
        atomicOr(status, kPlanTimeout);
        return false;
      }
    }
  }
}

__device__ __forceinline__ bool many_warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort,
                                               int* status) {
  return __all_sync(0xffffffffu, many_wait(bar, parity, abort, status));
}

__device__ __forceinline__ bool elect_one() {
  uint32_t pred;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(pred));
  return pred != 0;
}

__device__ __forceinline__ void fence_async_smem() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

__device__ __forceinline__ void tie(uint32_t (&r)[32]) {
  asm volatile(""
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                 "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                 "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]),
                 "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                 "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                 "+r"(r[30]), "+r"(r[31]));
}

__device__ __forceinline__ void sts128(uint32_t at, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z),
               "r"(v.w)
               : "memory");
}

__device__ __forceinline__ void sts64(uint32_t at, uint32_t lo, uint32_t hi) {
  asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(at), "r"(lo), "r"(hi) : "memory");
}

// Matrix descriptors (the layout that sm100.cuh states), kept as their low words: the start
// address, and LBO where it counts. The high words are constants.
__host__ __device__ constexpr uint32_t desc_high(uint32_t stride_bytes, uint32_t layout) {
  return stride_bytes >> 4 | 1u << 14 | layout << 29;
}

__device__ __forceinline__ uint32_t desc_low(uint32_t at, uint32_t lbo_bytes) {
  return (at & 0x3FFFFu) >> 4 | lbo_bytes >> 4 << 16;
}

__device__ __forceinline__ uint64_t desc(uint32_t low, uint32_t high) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(low), "r"(high));
  return d;
}

// Sixteen scores (under one scale) to weights 2^(s · mul + add) in f16 pairs, summed into acc.
__device__ __forceinline__ void weigh16(const uint32_t* r, float mul, float add, float2& acc,
                                        uint32_t* pk) {
  const float2 m2 = make_float2(mul, mul), a2 = make_float2(add, add);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 s = make_float2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
    const float2 x = __ffma2_rn(s, m2, a2);
    const float2 e = make_float2(ex2_approx(x.x), ex2_approx(x.y));
    acc = __fadd2_rn(acc, e);
    pk[i] = f16_pair(e.x, e.y);
  }
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

__device__ __forceinline__ float max16(const uint32_t* r) {
  float a = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  float b = fmaxf(__uint_as_float(r[2]), __uint_as_float(r[3]));
#pragma unroll
  for (int i = 4; i < 16; i += 4) {
    a = max3(a, __uint_as_float(r[i]), __uint_as_float(r[i + 1]));
    b = max3(b, __uint_as_float(r[i + 2]), __uint_as_float(r[i + 3]));
  }
  return fmaxf(a, b);
}

// Columns past `limit` (relative to the chunk; may be negative) and of groups that are not
// there (bits 0 and 1 of `gone`) become -inf.
__device__ __forceinline__ void hide32(uint32_t (&r)[32], int limit, int gone) {
#pragma unroll
  for (int i = 0; i < 32; ++i)
    if (i > limit || (gone >> (i / 16) & 1)) r[i] = 0xff800000u;
}

// GROUPS: scales that 64 keys can have (64 / page, at least 1).
template <int HD, int GROUPS>
__global__ void __launch_bounds__(512, 1)
    attend_many(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                const CacheArgs a) {
  using L = Many<HD>;
  extern __shared__ uint8_t many_smem[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(many_smem) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + L::kBarOffset);
  uint64_t* q_ready = bar;
  uint64_t* k_full = q_ready + 2;
  uint64_t* k_empty = k_full + L::kKStages;
  uint64_t* v8_full = k_empty + L::kKStages;
  uint64_t* v8_empty = v8_full + L::kV8Stages;
  uint64_t* v16_full = v8_empty + L::kV8Stages;
  uint64_t* v16_empty = v16_full + L::kV16Stages;
  uint64_t* s_full = v16_empty + L::kV16Stages;
  uint64_t* p_ready = s_full + 4;
  uint64_t* pv_done = p_ready + 4;  // these three [tile][half]
  uint64_t* scale_full = pv_done + 4;
  uint64_t* drain = scale_full + L::kScaleRing;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kMiscOffset);
  volatile int* abort = reinterpret_cast<volatile int*>(smem + L::kMiscOffset + 4);
  volatile int* nan_tile = reinterpret_cast<volatile int*>(smem + L::kMiscOffset + 8);  // [slot]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  const long long total = a.units_many[a.requests] * a.heads_kv;
  const int workers = static_cast<int>(min(static_cast<long long>(a.workers), total));
  if (static_cast<int>(blockIdx.x) >= workers) return;
  const long long u0 = quotient(blockIdx.x * total, workers), u1 = quotient((blockIdx.x + 1) * total, workers);
  const int units = static_cast<int>(u1 - u0);

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_ready[i], 128);
      mbar_init(&s_full[2 * i], 1);
      mbar_init(&s_full[2 * i + 1], 1);
      mbar_init(&p_ready[2 * i], 128);
      mbar_init(&p_ready[2 * i + 1], 128);
      mbar_init(&pv_done[2 * i], 1);
      mbar_init(&pv_done[2 * i + 1], 1);
    }
    for (int i = 0; i < L::kKStages; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 2);
    }
    for (int i = 0; i < L::kV8Stages; ++i) {
      mbar_init(&v8_full[i], 1);
      mbar_init(&v8_empty[i], kWideners);
    }
    for (int i = 0; i < L::kV16Stages; ++i) {
      mbar_init(&v16_full[i], kWideners);
      mbar_init(&v16_empty[i], 2);
      nan_tile[i] = 0;
    }
    for (int i = 0; i < L::kScaleRing; ++i) mbar_init(&scale_full[i], 1);
    mbar_init(drain, 2);
    *abort = 0;
    fence_barrier_init();
  }
  if (warp == 8) {
    tmem_alloc(tmem_slot, 512);
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp < 8) {
    // ------------------------------------------------------------------------------ softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kManySoftmaxRegs));
    const int s = warp >> 2;
    const int row128 = threadIdx.x & 127;
    const uint32_t lane_bits = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + lane_bits + static_cast<uint32_t>(s * 128);
    const uint32_t tO = tmem + lane_bits + 256u + static_cast<uint32_t>(s * HD);
    uint4* poison = reinterpret_cast<uint4*>(smem + L::kPoisonOffset) + threadIdx.x;
    int block = 0;       // tiles of keys seen
    uint32_t phase = 0;  // bit b: parity of half b's next scores (its last product has the other)
    bool ok = true;
    volatile int* place = reinterpret_cast<volatile int*>(smem + L::kAtOffset) + warp * 16;
    many_put(place, many_at(a, u0, units));
    while (ok && place[4] > 0) {
      int steps, halves, last, first_seen, key0;
      bool here;
      float mul = 0.f;
      {
        const ManyAt at = many_get(place);
        steps = at.steps;
        halves = many_halves(a, at);
        key0 = at.j * kTileKeys;
        const int rows = many_rows(a, at);
        here = s * 128 < rows;
        const int per = kRowsMany / a.group;
        const int row = min(s * 128 + row128, rows - 1);
        const int token = at.item * per + row_token(a, row);  // of the request
        last = at.cached + token;                         // the last key it sees
        first_seen = at.cached + at.item * per;           // the item's first token's last key
        if (here) {
          // ---- this warp's 32 rows of Q as two e4m3 parts, HD / 8 lanes a row (rows behind the
          // last repeat it)
          constexpr int LANES = HD / 8, ROWS = 32 / LANES;
          const int sub = lane / LANES, d0 = lane % LANES * 8;
          const uint32_t hi_at = smem_u32(smem + L::kQOffset + s * 2 * L::kCodeTile);
          // Four rows' loads and exchanges side by side, the next four's loads ahead. A loop, not
          // straight code: run once an item, that would come from memory instruction by instruction.
          auto load = [&](int g, uint4 (&v)[4]) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int r = min(s * 128 + (warp & 3) * 32 + (g * 4 + i) * ROWS + sub, rows - 1);
              const int of = row_token(a, r);
              v[i] = *reinterpret_cast<const uint4*>(
                  a.query + (at.first_token + at.item * per + of) * a.q_token +
                  (at.h * a.group + r - of * a.group) * a.q_head + d0);
            }
          };
          uint4 x[4];
          load(0, x);
#pragma unroll 1
          for (int g = 0; g < LANES / 4; ++g) {
            uint4 y[4];
            load(min(g + 1, LANES / 4 - 1), y);
            float amax[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
              amax[i] = 0.f;
#pragma unroll
              for (int k = 0; k < 4; ++k)
                amax[i] = max3(amax[i], fabsf(__uint_as_float(w[k] << 16)), fabsf(__uint_as_float(w[k] & 0xffff0000u)));
            }
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1)
#pragma unroll
              for (int i = 0; i < 4; ++i) amax[i] = fmaxf(amax[i], __shfl_xor_sync(0xffffffffu, amax[i], o));
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int r128 = (warp & 3) * 32 + (g * 4 + i) * ROWS + sub;
              const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
              // the largest value in [224, 448]: 448 = 1.75 · 2^8
              const int e = max(-100, static_cast<int>((__float_as_uint(amax[i]) + 0x1fffffu) >> 23) - 127 - 8);
              const float up = exponent_scale(-e);
              const float mine = a.scale_log2 * exponent_scale(e);
              const float given = __shfl_sync(0xffffffffu, mine, lane % ROWS * LANES);
              if (lane / ROWS == g * 4 + i) mul = given;
              uint32_t hi[2], lo[2];
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                float f0 = __uint_as_float(w[k] << 16) * up, f1 = __uint_as_float(w[k] & 0xffff0000u) * up;
                // an infinity has no parts: its row is NaN, as its softmax is
                if (!(fabsf(f0) <= 448.f)) f0 = __uint_as_float(0x7fc00000u);
                if (!(fabsf(f1) <= 448.f)) f1 = __uint_as_float(0x7fc00000u);
                uint16_t h, l;
                asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(h) : "f"(f0), "f"(f1));
                uint32_t back;
                asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(back) : "h"(h));
                const float2 g = __half22float2(*reinterpret_cast<const __half2*>(&back));
                asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(l) : "f"(f0 - g.x), "f"(f1 - g.y));
                hi[k >> 1] = (k & 1) ? hi[k >> 1] | static_cast<uint32_t>(h) << 16 : h;
                lo[k >> 1] = (k & 1) ? lo[k >> 1] | static_cast<uint32_t>(l) << 16 : l;
              }
              const int c = d0 / 16;
              const uint32_t off = (HD == 128 ? r128 * 128 + ((c ^ (r128 & 7)) << 4)
                                              : r128 * 64 + ((c ^ ((r128 >> 1) & 3)) << 4)) + d0 % 16;
              sts64(hi_at + off, hi[0], hi[1]);
              sts64(hi_at + L::kCodeTile + off, lo[0], lo[1]);
              x[i] = y[i];
            }
          }
          *poison = make_uint4(0, 0, 0, 0);
          fence_async_smem();
          mbar_arrive(&q_ready[s]);
        }
      }
      if (here) {
        float m = -INFINITY, l = 0.f;
        for (int h = 0; h < halves; ++h) {
          const int b = h & 1, tile = block + (h >> 1), slot = tile % L::kScaleRing;
          const int tile_key0 = key0 + (h >> 1) * kTileKeys, half_key0 = tile_key0 + b * 64;
          // The scales are there long before the scores. Not so for an item's first tile: rows that
          // skipped items may be far ahead of the copies, and a parity two phases ahead reads as
          // complete; its scores have arrived only behind its scales.
          if (h == 0 && !many_wait(&s_full[2 * s], phase & 1, abort, a.status)) {
            ok = false;
            break;
          }
          const float* scales =
              reinterpret_cast<const float*>(smem + L::kScaleOffset + slot * L::kScaleBytes) + b * 4;
          if (b == 0 && !many_wait(&scale_full[slot], (tile / L::kScaleRing) & 1, abort, a.status)) {
            ok = false;
            break;
          }
          float mul_of[GROUPS], add_of[GROUPS], back_of[GROUPS];
#pragma unroll
          for (int c = 0; c < GROUPS; ++c) {
            mul_of[c] = group_mul(mul, scales[c * (4 / GROUPS)]);
            add_of[c] = scales[8 + c * (4 / GROUPS)];
            back_of[c] = scales[16 + c * (4 / GROUPS)];
          }
          const int gone = reinterpret_cast<const int*>(scales)[24 - b * 4];
          if (h > 0 && !many_wait(&s_full[2 * s + b], phase >> b & 1, abort, a.status)) {
            ok = false;
            break;
          }
          phase ^= 1u << b;
          tc_fence_after();
          uint32_t r[2][32];
          tmem_ld32(tS + b * 64, r[0]);
          tmem_ld32(tS + b * 64 + 32, r[1]);
          tmem_wait_ld();
          tie(r[0]);
          tie(r[1]);
          // some row of the item does not see the whole tile
          const bool partial = tile_key0 + kTileKeys > first_seen + 1 || gone != 0;
          if (partial) {
            hide32(r[0], last - half_key0, gone >> (4 * b));
            hide32(r[1], last - half_key0 - 32, gone >> (4 * b + 2));
          }
          float top = -INFINITY;
#pragma unroll
          for (int c = 0; c < GROUPS; ++c) {
            float most = -INFINITY;
#pragma unroll
            for (int e = 0; e < 4 / GROUPS; ++e) {
              const int of = c * (4 / GROUPS) + e;
              most = fmaxf(most, max16(&r[of >> 1][(of & 1) * 16]));
            }
            top = fmaxf(top, fmaf(most, mul_of[c], add_of[c]));
          }
          const float m_new = fmaxf(m, top);
          if (__any_sync(0xffffffffu, m != -INFINITY && m_new > m + kManySlack)) {
            // O is this warp's own once the last half's product has been added to it
            if (!many_wait(&pv_done[2 * s + (b ^ 1)], (phase >> (b ^ 1) & 1) ^ 1, abort, a.status)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const float w = m == -INFINITY ? 0.f : ex2_approx(m - m_new);
            l *= w;
#pragma unroll
            for (int c = 0; c < HD / 32; ++c) {
              uint32_t o[32];
              tmem_ld32(tO + c * 32, o);
              tmem_wait_ld();
              tie(o);
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * w);
              tmem_st32(tO + c * 32, o);
            }
            m = m_new;
          }
          if (m == -INFINITY) m = m_new;
          const float ref = (m == -INFINITY ? 0.f : m) - kManyBias;
          uint32_t pk[32];
          float2 acc = make_float2(0.f, 0.f);
#pragma unroll
          for (int of = 0; of < 4; ++of) {
            const int group = of * GROUPS / 4;
            if (of % (4 / GROUPS) == 0) acc = make_float2(0.f, 0.f);
            weigh16(&r[of / 2][of % 2 * 16], mul_of[group], add_of[group] - ref, acc, pk + 8 * of);
            if ((of + 1) % (4 / GROUPS) == 0) l = fmaf(acc.x + acc.y, back_of[group], l);
          }
          tmem_st32(tS + b * 64, pk);
          if (partial) {
            // values that are NaN in a tile that some row does not see whole: the rows that see
            // the key take the NaN, in its channels, at the end
            const int v = tile % L::kV16Stages;
            if (!many_wait(&v16_full[v], (tile / L::kV16Stages) & 1, abort, a.status)) ok = false;
            else if (nan_tile[v] == tile + 1) {
              const uint4* bits = reinterpret_cast<const uint4*>(smem + L::kNanOffset) + v * 128 + b * 64;
              uint4 p = *poison;
              for (int k = 0; k < 64 && half_key0 + k <= last; ++k) {
                p.x |= bits[k].x;
                p.y |= bits[k].y;
                p.z |= bits[k].z;
                p.w |= bits[k].w;
              }
              *poison = p;
            }
          }
          tmem_wait_st();
          tc_fence_before();
          mbar_arrive(&p_ready[2 * s + b]);
        }
        const int b = (halves - 1) & 1;
        if (ok) ok = many_wait(&pv_done[2 * s + b], (phase >> b & 1) ^ 1, abort, a.status);
        tc_fence_after();
        if (!ok) break;
        block += steps;
        // ---- the item's end, or this worker's part of it
        const ManyAt at = many_get(place);
        const int rows = many_rows(a, at), row = s * 128 + row128;
        const int first_token = at.first_token + at.item * (kRowsMany / a.group);
        const int token = first_token + row_token(a, row);
        const bool whole = steps == at.tiles;
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const long long part = 2LL * blockIdx.x + (at.j == 0 ? 1 : 0);
        const int head = at.h * a.group + row - (token - first_token) * a.group;
        // Whole rows leave through the tile's Q (free now, and of the same size), HD / 8 lanes a
        // row. A row takes the bytes of its own two parts, which only its warp writes: the tile's
        // other warps may be at the next item's Q already, or still at this one's rows. Chunk j
        // stands where Q has it, so no two lanes of eight meet in a bank.
        const uint32_t stage = smem_u32(smem + L::kQOffset + s * 2 * L::kCodeTile);
        auto staged = [&](int r128, int j) {
          constexpr int CODES = HD / 16;  // chunks of a row of codes
          const uint32_t at = stage + (j / CODES) * L::kCodeTile + r128 * HD;
          return at + (((j % CODES) ^ (HD == 128 ? r128 & 7 : r128 >> 1 & 3)) << 4);
        };
        float4* ws = reinterpret_cast<float4*>(a.ws_o) + part * (HD / 4) * kRowsMany + row;
        const uint4 p = *poison;
        const bool nan = (p.x | p.y | p.z | p.w) != 0;
#pragma unroll
        for (int c = 0; c < HD / 32; ++c) {
          uint32_t o[32];
          tmem_ld32(tO + c * 32, o);
          tmem_wait_ld();
          tie(o);
          if (nan) {
            const uint32_t bits = c == 0 ? p.x : c == 1 ? p.y : c == 2 ? p.z : p.w;
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (bits >> i & 1) o[i] = 0x7fc00000u;
          }
          if (whole) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t w[4];
#pragma unroll
              for (int k = 0; k < 4; ++k)
                w[k] = pack_bf16x2(__uint_as_float(o[8 * i + 2 * k]) * inv,
                                   __uint_as_float(o[8 * i + 2 * k + 1]) * inv);
              sts128(staged(row128, c * 4 + i), make_uint4(w[0], w[1], w[2], w[3]));
            }
          } else if (row < rows) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              ws[(c * 8 + i) * kRowsMany] =
                  make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]),
                              __uint_as_float(o[4 * i + 2]), __uint_as_float(o[4 * i + 3]));
          }
        }
        tc_fence_before();
        if (whole) {
          constexpr int LANES = HD / 8, ROWS = 32 / LANES;
          __syncwarp();
#pragma unroll 4
          for (int i = 0; i < LANES; ++i) {
            const int r128 = (warp & 3) * 32 + i * ROWS + lane / LANES, j = lane % LANES;
            const int r = s * 128 + r128;
            const uint4 v = lds128(staged(r128, j));
            const int of = row_token(a, r);
            if (r < rows)
              *reinterpret_cast<uint4*>(a.out + (first_token + of) * a.o_token +
                                        (at.h * a.group + r - of * a.group) * a.o_head + j * 8) = v;
          }
          __syncwarp();
        }
        if (row < rows) {
          if (!whole) a.ws_ml[part * kRowsMany + row] = make_float2(m, l);
          else if (a.lse != nullptr)
            a.lse[static_cast<long long>(token) * a.heads_kv * a.group + head] =
                l == 0.f ? -INFINITY : 0.6931471805599453f * (m - kManyBias + __log2f(l));
        }
      } else {
        block += steps;
      }
      ManyAt at = many_get(place);
      many_next(a, at);
      many_put(place, at);
    }
  } else if (warp == 8) {
    // -------------------------------------------------------------- page numbers and copies
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kManyOtherRegs));
    const int box = a.page, per_tile = kTileKeys >> a.page_shift;
    int block = 0;
    bool ok = true;
    for (ManyAt at = many_at(a, u0, units); at.steps > 0; many_next(a, at)) {
      const int steps = at.steps;
      int batch = 0, id = -1;
      float key_scale = 1.f, value_e = 0.f;
      for (int step = 0; step < steps; ++step, ++block) {
        const int key0 = (at.j + step) * kTileKeys;
        const int first = key0 >> a.page_shift;
        if (step == 0 || first + per_tile > batch + 32) {  // 32 pages' numbers and scales at once
          batch = first;
          id = -1;
          key_scale = 1.f;
          value_e = 0.f;
          const int index = first + lane;
          if (index * static_cast<long long>(a.page) < at.keys) {
            id = a.table[at.n * a.table_stride + index];
            if (id < 0 || id >= a.pages) {
              id = -1;
              atomicOr(a.status, kPlanBadPage);
            } else {
              const long long at_block = static_cast<long long>(id) * a.heads_kv + at.h;
              key_scale = exponent_scale(a.key_exponent[at_block]);
              value_e = static_cast<float>(a.value_exponent[at_block]);
            }
          }
        }
        // groups of 16 keys: lane's group is in page (key0 + 16 · lane) / page
        const int from = ((key0 + (lane & 7) * 16 >> a.page_shift) - batch) & 31;
        const float ks = __shfl_sync(0xffffffffu, key_scale, from);
        const float ve = __shfl_sync(0xffffffffu, value_e, from);
        const int group_id = __shfl_sync(0xffffffffu, id, from);
        const unsigned gone = __ballot_sync(
            0xffffffffu, lane < 8 && group_id < 0 && key0 + (lane & 7) * 16 < at.keys);
        const int page_id = __shfl_sync(0xffffffffu, id, (first - batch + lane) & 31);
        const bool load = lane < per_tile && page_id >= 0 && key0 + lane * box < at.keys;
        const int bytes = __popc(__ballot_sync(0xffffffffu, load)) * box * HD;
        const int ks_stage = block % L::kKStages, v_stage = block % L::kV8Stages;
        if (block >= L::kKStages &&
            !(ok = many_warp_wait(&k_empty[ks_stage], (block / L::kKStages - 1) & 1, abort, a.status)))
          break;
        float* scales = reinterpret_cast<float*>(smem + L::kScaleOffset +
                                                 (block % L::kScaleRing) * L::kScaleBytes);
        if (lane < 8) {
          scales[lane] = ks;
          scales[8 + lane] = ve;
          scales[16 + lane] = exponent_scale(-static_cast<int>(ve));
        }
        if (lane == 0) reinterpret_cast<int*>(scales)[24] = static_cast<int>(gone);
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&scale_full[block % L::kScaleRing]);
          mbar_expect_tx(&k_full[ks_stage], bytes);
        }
        __syncwarp();
        const int y = (page_id * a.heads_kv + at.h) * a.page;
        if (load)
          tma_load_2d(smem + L::kKOffset + ks_stage * L::kCodeTile + lane * box * HD, &tm_k,
                      &k_full[ks_stage], 0, y);
        if (block >= L::kV8Stages &&
            !(ok = many_warp_wait(&v8_empty[v_stage], (block / L::kV8Stages - 1) & 1, abort, a.status))) {
          // this tile's K was asked for without its V: counted below as K only
          many_warp_wait(&k_full[ks_stage], (block / L::kKStages) & 1, abort, a.status);
          break;
        }
        if (lane == 0) mbar_expect_tx(&v8_full[v_stage], bytes);
        __syncwarp();
        if (load)
          tma_load_2d(smem + L::kV8Offset + v_stage * L::kCodeTile + lane * box * HD, &tm_v,
                      &v8_full[v_stage], 0, y);
      }
      if (!ok) break;
    }
    // every copy lands before the CTA unwinds
    volatile int never = 0;
    for (int b = max(0, block - L::kKStages); b < block; ++b)
      many_wait(&k_full[b % L::kKStages], (b / L::kKStages) & 1, &never, a.status);
    for (int b = max(0, block - L::kV8Stages); b < block; ++b)
      many_wait(&v8_full[b % L::kV8Stages], (b / L::kV8Stages) & 1, &never, a.status);
    __syncwarp();
  } else if (warp < 11) {
    // ------------------------------------------------------------------ matrix instructions
    // A warp for each query tile: a wait of a warp with products in flight takes about 300
    // clocks even where its barrier is long complete (traced with clock64), and the queue of
    // products is short, so one warp for both left the tensor cores idle between its turns.
    const int s = warp - 9;
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kManyOtherRegs));
    constexpr uint32_t kIdescQK = idesc_e4m3_f32(128, 64, false);
    constexpr uint32_t kIdescPV = idesc_e4m3_f32(128, HD, true);  // f16 has the same code, 0
    // K-major codes in the swizzle of a row's width, 8 rows an atom; V in 128-byte boxes
    constexpr uint32_t kCodes = desc_high(8 * HD, HD == 128 ? 2 : 4), kValues = desc_high(1024, 2);
    const uint32_t q0 = desc_low(smem_u32(smem + L::kQOffset) + s * 2 * L::kCodeTile, 16);
    const uint32_t k0 = desc_low(smem_u32(smem + L::kKOffset), 16);
    const uint32_t v0 = desc_low(smem_u32(smem + L::kV16Offset), 128 * 128);
    constexpr uint32_t kTile = L::kCodeTile >> 4;
    const uint32_t ts = tmem + s * 128, to = tmem + 256u + s * HD;
    auto issue_qk = [&](int b, int stage) {  // a half: 64 rows of K
      const uint32_t k = k0 + stage * kTile + b * (kTile / 2);
#pragma unroll
      for (int part = 0; part < 2; ++part)
#pragma unroll
        for (int kk = 0; kk < HD / 32; ++kk)
          mma_ss_f8(ts + b * 64, desc(q0 + part * kTile + kk * 2, kCodes), desc(k + kk * 2, kCodes),
                    kIdescQK, part + kk > 0 ? 1u : 0u);
      mma_commit(&s_full[2 * s + b]);
    };
    auto issue_pv = [&](int b, int slot, uint32_t accumulate) {
      const uint32_t v = v0 + slot * 2 * kTile + ((b * 64 * 128) >> 4);
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
        mma_ts(to, ts + b * 64 + kk * 8, desc(v + ((kk * 16 * 128) >> 4), kValues), kIdescPV,
               kk > 0 ? 1u : accumulate);
      mma_commit(&pv_done[2 * s + b]);
    };
    int block = 0;
    uint32_t q_phase = 0, p_phase = 0;  // parities of q_ready, and of p_ready by half
    bool ok = true;
    for (ManyAt at = many_at(a, u0, units); at.steps > 0; many_next(a, at)) {
      const int steps = at.steps;
      const int halves = many_halves(a, at);
      const bool here = s * 128 < many_rows(a, at);
      if (here) {
        ok = many_warp_wait(&q_ready[s], q_phase, abort, a.status);
        q_phase ^= 1;
      }
      const int stage0 = block % L::kKStages;
      if (!ok || !(ok = many_warp_wait(&k_full[stage0], (block / L::kKStages) & 1, abort, a.status))) break;
      tc_fence_after();
      if (here && elect_one()) {
        for (int b = 0; b < min(2, halves); ++b) issue_qk(b, stage0);
        mma_commit(&k_empty[stage0]);
      }
      if (!here && lane == 0) mbar_arrive(&k_empty[stage0]);
      __syncwarp();
      for (int h = 0; h < halves; ++h) {
        const int b = h & 1, tile = block + (h >> 1), slot = tile % L::kV16Stages;
        const int stage = (tile + 1) % L::kKStages;
        const bool more = h + 2 < halves;
        // this tile's V and the next one's K
        if (b == 0 && !(ok = many_warp_wait(&v16_full[slot], (tile / L::kV16Stages) & 1, abort, a.status)))
          break;
        if (here) {
          if (!(ok = many_warp_wait(&p_ready[2 * s + b], p_phase >> b & 1, abort, a.status))) break;
          p_phase ^= 1u << b;
          tc_fence_after();
          if (elect_one()) {
            issue_pv(b, slot, h > 0 ? 1u : 0u);
            if (more) issue_qk(b, stage);
            if (b == 1 || h + 1 == halves) mma_commit(&v16_empty[slot]);
            if (more && (b == 1 || h + 3 == halves)) mma_commit(&k_empty[stage]);
          }
        } else if (b == 0 && lane == 0) {  // no rows here: only the tiles are given back
          mbar_arrive(&v16_empty[slot]);
          if (more) mbar_arrive(&k_empty[stage]);
        }
        __syncwarp();
      }
      block += steps;
      if (!ok) break;
    }
    // every product completes before tensor memory is given back
    if (elect_one()) mma_commit(drain);
    __syncwarp();
    volatile int never = 0;
    many_wait(drain, 0, &never, a.status);
    __syncwarp();
  } else if (warp == 11) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kManyOtherRegs));
  } else {
    // ----------------------------------------------------------------- V's codes to f16
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kManyOtherRegs));
    constexpr int CH = HD / 16;  // 16-byte chunks of a row of codes
    const int tid = threadIdx.x - 384;
    int block = 0;
    bool ok = true;
    for (ManyAt at = many_at(a, u0, units); at.steps > 0; many_next(a, at)) {
      const int steps = at.steps;
      const int first_seen = at.cached + at.item * (kRowsMany / a.group);
      for (int step = 0; step < steps; ++step, ++block) {
        const int in = block % L::kV8Stages, slot = block % L::kV16Stages;
        if (!(ok = many_wait(&v8_full[in], (block / L::kV8Stages) & 1, abort, a.status))) break;
        if (block >= L::kV16Stages &&
            !(ok = many_wait(&v16_empty[slot], (block / L::kV16Stages - 1) & 1, abort, a.status)))
          break;
        const int key0 = (at.j + step) * kTileKeys;
        // written before this tile's copies were asked for
        const int gone = *reinterpret_cast<const volatile int*>(
            smem + L::kScaleOffset + (block % L::kScaleRing) * L::kScaleBytes + 96);
        const bool partial = key0 + kTileKeys > first_seen + 1 || gone != 0;
        const uint32_t from = smem_u32(smem + L::kV8Offset + in * L::kCodeTile);
        const uint32_t to = smem_u32(smem + L::kV16Offset + slot * 2 * L::kCodeTile);
#pragma unroll 4
        for (int i = 0; i < 128 * CH / kWideners; ++i) {
          const int index = i * kWideners + tid, row = index / CH, c = index % CH;
          uint4 v = lds128(from + index * 16);
          if (partial) {
            if (key0 + row >= at.keys || (gone >> (row / 16) & 1)) v = make_uint4(0, 0, 0, 0);
            const uint32_t n[4] = {nan_bytes(v.x), nan_bytes(v.y), nan_bytes(v.z), nan_bytes(v.w)};
            uint32_t bits = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k)
              bits |= ((n[k] & 1) | (n[k] >> 7 & 2) | (n[k] >> 14 & 4) | (n[k] >> 21 & 8)) << (4 * k);
            *reinterpret_cast<uint16_t*>(smem + L::kNanOffset + (slot * 128 + row) * 16 + c * 2) =
                static_cast<uint16_t>(bits);
            if (bits) {
              nan_tile[slot] = block + 1;
              v.x &= ~n[0];
              v.y &= ~n[1];
              v.z &= ~n[2];
              v.w &= ~n[3];
            }
          }
          uint4 w0, w1;
          widen4(v.x, w0.x, w0.y);
          widen4(v.y, w0.z, w0.w);
          widen4(v.z, w1.x, w1.y);
          widen4(v.w, w1.z, w1.w);
          // 64 channels (128 bytes) a box; the upper box's writers take their two chunks in
          // the other order, so that 8 lanes never meet in a bank
          const uint32_t box = to + (c >> 2) * (128 * 128) + row * 128;
          const int j = 2 * (c & 3), turn = c >> 2;
          sts128(box + (((j + turn) ^ (row & 7)) << 4), turn ? w1 : w0);
          sts128(box + (((j + 1 - turn) ^ (row & 7)) << 4), turn ? w0 : w1);
        }
        fence_async_smem();
        mbar_arrive(&v8_empty[in]);
        if (step + 1 < steps &&
            !(ok = many_wait(&k_full[(block + 1) % L::kKStages], ((block + 1) / L::kKStages) & 1, abort, a.status)))
          break;
        mbar_arrive(&v16_full[slot]);
      }
      if (!ok) break;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the parts of an item that a boundary between workers cuts (the first such boundary has
// it): block (boundary, 32 rows), a lane a row, 8 warps over the channels.
template <int HD>
__global__ void __launch_bounds__(256) join_many(const CacheArgs a) {
  constexpr int PER = HD / 32;  // float4 columns a warp
  const long long total = a.units_many[a.requests] * a.heads_kv;
  const long long workers = min(static_cast<long long>(a.workers), total);
  const int w = blockIdx.x + 1;
  bool split = w < workers;
  ManyAt at;
  int last = 0, rows = 0;
  if (split) {
    const long long u = quotient(w * total, workers);
    at = many_at(a, u, 1 << 30);
    // cut behind its first tile, and the worker before has that one
    const long long u0 = u - kItemUnits - at.j;
    rows = many_rows(a, at);
    split = at.j > 0 && quotient((w - 1) * total, workers) <= u0 + kItemUnits &&
            static_cast<int>(blockIdx.y) * 32 < rows;
    last = static_cast<int>(quotient((u0 + kItemUnits + at.tiles) * workers - 1, total));
  }
  if (split || (blockIdx.x == 0 && blockIdx.y == 0)) asm volatile("griddepcontrol.wait;" ::: "memory");
  if (!split) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = blockIdx.y * 32 + lane;
  if (row >= rows) return;
  float top = -INFINITY;
  for (int p = w - 1; p <= last; ++p)
    top = fmaxf(top, __ldcg(&a.ws_ml[(2LL * p + (p == w - 1)) * kRowsMany + row]).x);
  float sum = 0.f;
  float4 o[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int p = w - 1; p <= last; ++p) {
    const long long part = 2LL * p + (p == w - 1);
    const float2 ml = __ldcg(&a.ws_ml[part * kRowsMany + row]);
    // a part without a key has zeros; one whose scores are NaN has a sum of NaN
    const float f = ml.x == -INFINITY ? 1.f : ex2_approx(ml.x - top);
    sum += ml.y * f;
    const float4* from = reinterpret_cast<const float4*>(a.ws_o) +
                         (part * (HD / 4) + warp * PER) * kRowsMany + row;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const float4 x = __ldcg(from + i * kRowsMany);
      o[i].x = fmaf(x.x, f, o[i].x);
      o[i].y = fmaf(x.y, f, o[i].y);
      o[i].z = fmaf(x.z, f, o[i].z);
      o[i].w = fmaf(x.w, f, o[i].w);
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int token = at.first_token + at.item * (kRowsMany / a.group) + row / a.group;
  const int head = at.h * a.group + row % a.group;
  uint2* to = reinterpret_cast<uint2*>(a.out + token * a.o_token + head * a.o_head) + warp * PER;
#pragma unroll
  for (int i = 0; i < PER; ++i)
    to[i] = make_uint2(pack_bf16x2(o[i].x * inv, o[i].y * inv), pack_bf16x2(o[i].z * inv, o[i].w * inv));
  if (a.lse != nullptr && warp == 0)
    a.lse[static_cast<long long>(token) * a.heads_kv * a.group + head] =
        sum == 0.f ? -INFINITY : 0.6931471805599453f * (top - kManyBias + __log2f(sum));
}

// ------------------------------------------------------------------------------- host side
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                 const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiled encode_tiled() {
  static EncodeTiled fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) !=
            cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      ptr = nullptr;
    return reinterpret_cast<EncodeTiled>(ptr);
  }();
  return fn;
}

// A pool's codes as rows of one head's channels; a box is `rows` rows, swizzled over a row's
// width or not.
static int code_map(CUtensorMap* map, const void* base, const CozyCacheStore& c, int rows,
                    bool swizzled) {
  EncodeTiled fn = encode_tiled();
  if (fn == nullptr) return cudaErrorNotSupported;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(c.head_dim),
                              static_cast<cuuint64_t>(c.pages) * c.heads_kv * c.page};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(c.head_dim)};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(c.head_dim), static_cast<cuuint32_t>(rows)};
  const cuuint32_t elem[2] = {1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims,
                        strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        !swizzled           ? CU_TENSOR_MAP_SWIZZLE_NONE
                        : c.head_dim == 128 ? CU_TENSOR_MAP_SWIZZLE_128B
                                            : CU_TENSOR_MAP_SWIZZLE_64B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

static int device_sms() {
  static int counts[64] = {};
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return 0;
  if (counts[device] == 0)
    cudaDeviceGetAttribute(&counts[device], cudaDevAttrMultiProcessorCount, device);
  return counts[device];
}

static long long few_workers(int head_dim) {
  return std::min(device_sms() * (head_dim == 128 ? Few<128>::kWarps : Few<64>::kWarps), kMostParts);
}

// Bytes of partial results that the kernels of a call may leave: two parts a worker.
static size_t few_bytes(int head_dim) {
  return few_workers(head_dim) * 2 * kRowsFew * (head_dim * sizeof(float) + sizeof(float2));
}

static size_t many_bytes(int head_dim) {
  return static_cast<size_t>(device_sms()) * 2 * kRowsMany * (head_dim * sizeof(float) + sizeof(float2));
}

// Which kernels a step needs, as far as the host knows: some request may have few rows, or many.
static bool may_be_few(const CozyCachePlan& p) { return few_rows(p.group, 1); }
static bool may_be_many(const CozyCachePlan& p) { return !few_rows(p.group, p.longest); }

long long cache_workspace(const CozyCachePlan& p, const CozyCacheStore& c) {
  return (may_be_few(p) ? few_bytes(c.head_dim) : 0) + (may_be_many(p) ? many_bytes(c.head_dim) : 0);
}

// A join is launched while its attention runs and waits for that one's end on the device.
static int join_launch(void (*kernel)(CacheArgs), dim3 grid, const CacheArgs& a, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

template <int HD>
static int few_launch(const CozyCacheStore& c, CacheArgs& a, int rows, cudaStream_t stream) {
  using L = Few<HD>;
  static bool configured[64] = {};
  int device = 0;
  cudaGetDevice(&device);
  if (device < 64 && !configured[device]) {
    const cudaError_t e = cudaFuncSetAttribute(
        attend_few<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kAlloc);
    if (e != cudaSuccess) return e;
    configured[device] = true;
  }
  CUtensorMap mk, mv;
  const int box = c.page < kChunkKeys ? c.page : kChunkKeys;
  int e = code_map(&mk, c.key, c, box, true);
  if (e || (e = code_map(&mv, c.value, c, box, true))) return e;
  attend_few<HD><<<device_sms(), L::kWarps * 32, L::kAlloc, stream>>>(mk, mv, a);
  if ((e = cudaGetLastError())) return e;
  return join_launch(join_few<HD>, dim3(a.requests * a.heads_kv, rows), a, stream);
}

template <int HD, int GROUPS>
static int many_launch(const CozyCacheStore& c, CacheArgs& a, cudaStream_t stream) {
  using L = Many<HD>;
  static bool configured[64] = {};
  int device = 0;
  cudaGetDevice(&device);
  if (device < 64 && !configured[device]) {
    const cudaError_t e = cudaFuncSetAttribute(
        attend_many<HD, GROUPS>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kAlloc);
    if (e != cudaSuccess) return e;
    configured[device] = true;
  }
  CUtensorMap mk, mv;
  const int box = c.page < kTileKeys ? c.page : kTileKeys;
  int e = code_map(&mk, c.key, c, box, true);
  if (e || (e = code_map(&mv, c.value, c, box, false))) return e;
  attend_many<HD, GROUPS><<<a.workers, L::kThreads, L::kAlloc, stream>>>(mk, mv, a);
  if ((e = cudaGetLastError())) return e;
  if (a.workers < 2) return cudaSuccess;
  return join_launch(join_many<HD>, dim3(a.workers - 1, kRowsMany / 32), a, stream);
}

int cache_attention(const CozyCachePlan& p, const CozyCacheStore& c, const CozyCacheAttend& x,
                    cudaStream_t stream) {
  int e = cache_plan_check(p);
  if (e || (e = cache_store_check(c, p))) return e;
  if (!(x.scale > 0.f) || x.scale > 2.0e38f) return cudaErrorInvalidValue;
  if (p.tokens == 0 || p.longest == 0) return cudaSuccess;  // nobody brings a token
  const void* ptrs[] = {x.query, x.out};
  for (const void* ptr : ptrs)
    if (ptr == nullptr || reinterpret_cast<uintptr_t>(ptr) % 16) return cudaErrorInvalidValue;
  for (int i = 0; i < 2; ++i)
    if (x.query_strides[i] < 0 || x.query_strides[i] % 8 || x.out_strides[i] < 0 ||
        x.out_strides[i] % 8)
      return cudaErrorInvalidValue;
  if (x.workspace == nullptr || reinterpret_cast<uintptr_t>(x.workspace) % 256 ||
      x.workspace_bytes < cache_workspace(p, c))
    return cudaErrorInvalidValue;
  CacheArgs a = {};
  a.table = p.table;
  a.table_stride = p.table_stride;
  a.starts = p.starts;
  a.lengths = p.lengths_after;
  a.units_few = p.units;
  a.units_many = p.units + p.requests + 1;
  a.status = p.status;
  a.requests = p.requests;
  a.pages = p.pages;
  a.page = p.page;
  a.page_shift = p.page == 16 ? 4 : p.page == 32 ? 5 : p.page == 64 ? 6 : 7;
  a.group = p.group;
  a.per_group = (65536u + p.group - 1) / p.group;
  a.heads_kv = c.heads_kv;
  a.key_exponent = static_cast<const int8_t*>(c.key_exponent);
  a.value_exponent = static_cast<const int8_t*>(c.value_exponent);
  a.query = static_cast<const __nv_bfloat16*>(x.query);
  a.q_token = x.query_strides[0];
  a.q_head = x.query_strides[1];
  a.out = static_cast<__nv_bfloat16*>(x.out);
  a.o_token = x.out_strides[0];
  a.o_head = x.out_strides[1];
  a.lse = x.lse;
  a.scale_log2 = x.scale * 1.4426950408889634f;
  uint8_t* space = static_cast<uint8_t*>(x.workspace);
  if (may_be_few(p)) {
    if (static_cast<long long>(p.requests) * c.heads_kv > 0x7fffffffLL) return cudaErrorInvalidValue;
    a.workers = static_cast<int>(few_workers(c.head_dim));
    a.ws_o = reinterpret_cast<float*>(space);
    a.ws_ml = reinterpret_cast<float2*>(a.ws_o + few_workers(c.head_dim) * 2 * kRowsFew * c.head_dim);
    space += few_bytes(c.head_dim);
    const int rows = static_cast<int>(std::min(static_cast<long long>(p.group) * p.longest,
                                               static_cast<long long>(kRowsFew * kFewItems)));
    const int r = c.head_dim == 64 ? few_launch<64>(c, a, rows, stream) : few_launch<128>(c, a, rows, stream);
    if (r) return r;
  }
  if (!may_be_many(p)) return cudaSuccess;
  a.workers = device_sms();
  a.ws_o = reinterpret_cast<float*>(space);
  a.ws_ml = reinterpret_cast<float2*>(a.ws_o + static_cast<size_t>(device_sms()) * 2 * kRowsMany * c.head_dim);
  if (c.head_dim == 64)
    return c.page >= 64   ? many_launch<64, 1>(c, a, stream)
           : c.page == 32 ? many_launch<64, 2>(c, a, stream)
                          : many_launch<64, 4>(c, a, stream);
  return c.page >= 64   ? many_launch<128, 1>(c, a, stream)
         : c.page == 32 ? many_launch<128, 2>(c, a, stream)
                        : many_launch<128, 4>(c, a, stream);
}

}  // namespace cozy
