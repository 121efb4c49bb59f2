// The 8-bit paged cache's bookkeeping: a step's plan (block tables and slot maps from request
// lengths) and the append (per-head RMSNorm and RoPE of the step's queries and keys, keys and
// values into e4m3 blocks).
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/cozy_ulysses.h"
#include "cache.cuh"
#include "norm_rope.cuh"

namespace cozy {

namespace cg = cooperative_groups;

// ---------------------------------------------------------------------------------- the plan
// One cluster. Every CTA scans all requests (a few loads a thread, two barriers a round: cheaper
// than handing the sums over), keeps the running sums in shared memory, and then takes its share
// of the tokens, fresh pages, released pages and touched blocks, each found by bisection.
// Nothing here is bandwidth: a step of 4 requests moves 112 bytes (6.1 us), one of 1000 requests
// 170 KB (13.3 us, 1 us of it the look at released page numbers); the time is the launch, one load
// of the lengths, the scan and the bisection's chain.
constexpr int kPlanThreads = 1024;

struct PlanSums {
  long long tokens, need, back, blocks, few, many;
};

__device__ __forceinline__ PlanSums operator+(PlanSums a, const PlanSums& b) {
  a.tokens += b.tokens;
  a.need += b.need;
  a.back += b.back;
  a.blocks += b.blocks;
  a.few += b.few;
  a.many += b.many;
  return a;
}

__device__ __forceinline__ PlanSums shifted(const PlanSums& a, int by) {
  PlanSums r;
  r.tokens = __shfl_up_sync(0xffffffffu, a.tokens, by);
  r.need = __shfl_up_sync(0xffffffffu, a.need, by);
  r.back = __shfl_up_sync(0xffffffffu, a.back, by);
  r.blocks = __shfl_up_sync(0xffffffffu, a.blocks, by);
  r.few = __shfl_up_sync(0xffffffffu, a.few, by);
  r.many = __shfl_up_sync(0xffffffffu, a.many, by);
  return r;
}

__device__ __forceinline__ long long pages_of(long long length, int page) {
  return (length + page - 1) / page;
}

// Pages that a request's row holds before the step: those of its length, or of the length that it
// was set back from.
__device__ __forceinline__ long long held_pages(const CozyCachePlan& p, const int* reached, int n) {
  return pages_of(reached == nullptr ? p.lengths[n] : max(p.lengths[n], reached[n]), p.page);
}

// Pages that it holds behind the step.
__device__ __forceinline__ long long kept_pages(const CozyCachePlan& p, int n) {
  const long long added = p.added[n];
  return added < 0 ? 0 : pages_of(p.lengths[n] + added, p.page);
}

// One request's part of the sums, and the status bits it raises.
__device__ __forceinline__ PlanSums request_sums(const CozyCachePlan& p, const int* reached, int n,
                                                 int* flags) {
  const long long length = p.lengths[n], added = p.added[n];
  PlanSums s = {};
  if (length < 0 || added < -1 || (reached != nullptr && reached[n] < 0)) {
    *flags |= kPlanLengths;
    return s;
  }
  const long long held = held_pages(p, reached, n), want = kept_pages(p, n);
  if (held > p.width || want > p.width) *flags |= kPlanNarrow;
  s.back = max(0LL, held - want);
  if (added < 0) return s;
  if (added > p.longest) *flags |= kPlanTokens;
  s.tokens = added;
  s.need = max(0LL, want - held);
  if (added > 0) {
    s.blocks = want - length / p.page;
    const long long units = attention_units(p.group, length, added);
    if (few_rows(p.group, added)) s.few = units;
    else s.many = units;
  }
  return s;
}

__device__ __forceinline__ int ring_at(long long at, int pages) {
  return static_cast<int>(at % pages);
}

// The request whose span [starts[n], starts[n + 1]) holds `at`.
__device__ __forceinline__ int span_of(const int* starts, int n, int at) {
  int low = 0, high = n - 1;
  while (low < high) {
    const int mid = (low + high + 1) >> 1;
    if (starts[mid] <= at) low = mid;
    else high = mid - 1;
  }
  return low;
}

// Released page number `i` of the step: its request's table entries behind what it keeps.
__device__ __forceinline__ int released_page(const CozyCachePlan& p, const int* backs, int i) {
  const int n = span_of(backs, p.requests, i);
  return p.table[n * p.table_stride + kept_pages(p, n) + (i - backs[n])];
}

__global__ void __launch_bounds__(kPlanThreads)
    cache_plan_kernel(const CozyCachePlan p, const int* reached) {
  extern __shared__ int plan_smem[];
  __shared__ PlanSums warp_sums[32];
  __shared__ int any_flags, bad_release;
  const int n1 = p.requests + 1;
  int* starts = plan_smem;        // [requests + 1] each: tokens, fresh pages, released pages, blocks
  int* needs = starts + n1;
  int* backs = needs + n1;
  int* blocks = backs + n1;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool lead = blockIdx.x == 0;
  if (threadIdx.x == 0) any_flags = bad_release = 0;
  __syncthreads();
  cg::cluster_group cluster = cg::this_cluster();
  const bool alone = gridDim.x == 1;
  if (!alone) cluster.barrier_arrive();

  // checks first: a step that cannot be served gets nothing at all
  int flags = 0;
  PlanSums carry = {};
  for (int base = 0; base < p.requests; base += kPlanThreads) {
    const int n = base + threadIdx.x;
    PlanSums mine = n < p.requests ? request_sums(p, reached, n, &flags) : PlanSums{};
    PlanSums upto = mine;
#pragma unroll
    for (int by = 1; by < 32; by <<= 1) {
      const PlanSums other = shifted(upto, by);
      if (lane >= by) upto = upto + other;
    }
    if (lane == 31) warp_sums[warp] = upto;
    __syncthreads();
    if (warp == 0) {
      PlanSums w = warp_sums[lane];
#pragma unroll
      for (int by = 1; by < 32; by <<= 1) {
        const PlanSums other = shifted(w, by);
        if (lane >= by) w = w + other;
      }
      warp_sums[lane] = w;
    }
    __syncthreads();
    PlanSums before = carry;
    if (warp > 0) before = before + warp_sums[warp - 1];
    const PlanSums end = before + upto;
    if (n < p.requests) {
      // sums past 2^31 - 1 only occur in steps that are refused below
      starts[n + 1] = static_cast<int>(end.tokens);
      needs[n + 1] = static_cast<int>(end.need);
      backs[n + 1] = static_cast<int>(end.back);
      blocks[n + 1] = static_cast<int>(end.blocks);
      if (lead) {
        p.units[n + 1] = end.few;
        p.units[n1 + n + 1] = end.many;
      }
    }
    carry = carry + warp_sums[31];
    __syncthreads();
  }
  const long long head = p.cursor[0], tail = p.cursor[1];
  if (head < 0 || tail < head || tail - head > p.pages) flags |= kPlanLengths;
  else if (carry.need > tail - head) flags |= kPlanNoPages;
  else if (tail - head + carry.back > p.pages) flags |= kPlanLengths;
  if (carry.tokens > p.tokens) flags |= kPlanTokens;
  if (flags) atomicOr(&any_flags, flags);
  if (threadIdx.x == 0) {
    starts[0] = needs[0] = backs[0] = blocks[0] = 0;
    if (lead) p.units[0] = p.units[n1] = 0;
  }
  __syncthreads();
  int status = any_flags;  // alike in all CTAs
  if (lead && threadIdx.x == 0) *p.status = status;
  const int first = blockIdx.x * kPlanThreads + threadIdx.x, step = gridDim.x * kPlanThreads;
  // A number outside the pool must not come into the ring, from where another request would be
  // given it: each CTA looks at its share and tells all. A thread's first numbers stay in registers.
  constexpr int kGiven = 4;
  int given[kGiven];
  if (!alone) cluster.barrier_wait();  // every bad_release is set
  if (status == 0 && carry.back > 0) {
    bool out = false;
    auto look = [&](int i) {
      const int id = i < carry.back ? released_page(p, backs, i) : 0;
      out |= id < 0 || id >= p.pages;
      return id;
    };
#pragma unroll
    for (int j = 0; j < kGiven; ++j) given[j] = look(first + j * step);
    for (int i = first + kGiven * step; i < carry.back; i += step) look(i);
    if (out)
      for (unsigned r = 0; r < gridDim.x; ++r) *cluster.map_shared_rank(&bad_release, r) = 1;
  }
  // the status word is also set before any CTA adds the bad-page bit to it
  if (alone) __syncthreads();
  else cluster.sync();
  if (bad_release) {
    status = kPlanBadPage;
    if (lead && threadIdx.x == 0) *p.status = status;  // nobody adds to it: the step has no rows
  }
  const bool refused = status != 0;
  if (refused) {
    for (int n = threadIdx.x; n < n1; n += kPlanThreads) {
      starts[n] = 0;
      if (lead) p.units[n] = p.units[n1 + n] = 0;
    }
    __syncthreads();
    carry = PlanSums{};
  }
  if (lead && threadIdx.x == 0) {
    p.cursor_after[0] = head + carry.need;
    p.cursor_after[1] = tail + carry.back;
  }

  for (int n = first; n < n1; n += step) {
    p.starts[n] = starts[n];
    if (n < p.requests) {
      const int length = p.lengths[n], added = p.added[n];
      p.lengths_after[n] = refused ? max(length, 0) : added < 0 ? 0 : length + added;
    }
  }
  // the page of block `b` of request n: fresh ones straight from the ring
  bool bad = false;
  auto page_of = [&](int n, int b) {
    const int held = static_cast<int>(held_pages(p, reached, n));
    const int id = b < held ? p.table[n * p.table_stride + b]
                            : p.free_ring[ring_at(head + needs[n] + (b - held), p.pages)];
    if (id >= 0 && id < p.pages) return id;
    bad = true;
    return -1;
  };
  const int tokens = static_cast<int>(carry.tokens);
  for (int t = first; t < p.tokens; t += step) {
    int position = -1;
    long long slot = -1;
    if (t < tokens) {
      const int n = span_of(starts, p.requests, t);
      position = p.lengths[n] + (t - starts[n]);
      const int id = page_of(n, position / p.page);
      if (id >= 0) slot = static_cast<long long>(id) * p.page + position % p.page;
      else position = -1;
    }
    p.positions[t] = position;
    p.slots[t] = slot;
  }
  for (int i = first; i < p.max_blocks; i += step) {
    int4 entry = make_int4(-1, 0, 0, 0);  // page, first row, rows, first token
    if (i < carry.blocks) {
      const int n = span_of(blocks, p.requests, i);
      const int length = p.lengths[n], added = p.added[n];
      const int b = length / p.page + (i - blocks[n]);
      const int low = max(length, b * p.page);
      const int high = static_cast<int>(min(static_cast<long long>(length) + added,
                                            (b + 1LL) * p.page));
      entry = make_int4(page_of(n, b), low - b * p.page, high - low, starts[n] + low - length);
    }
    reinterpret_cast<int4*>(p.blocks)[i] = entry;
  }
  if (bad) atomicOr(p.status, kPlanBadPage);
#pragma unroll
  for (int j = 0; j < kGiven; ++j)
    if (first + j * step < carry.back) p.free_ring[ring_at(tail + first + j * step, p.pages)] = given[j];
  for (int i = first + kGiven * step; i < carry.back; i += step)
    p.free_ring[ring_at(tail + i, p.pages)] = released_page(p, backs, i);
  for (int i = first; i < carry.need; i += step) {
    const int n = span_of(needs, p.requests, i);
    const long long held = held_pages(p, reached, n);
    p.table[n * p.table_stride + held + (i - needs[n])] = p.free_ring[ring_at(head + i, p.pages)];
  }
}

int cache_plan_check(const CozyCachePlan& p) {
  if (p.requests < 1 || p.requests > COZY_CACHE_MAX_REQUESTS || p.width < 1 || p.pages < 1)
    return cudaErrorInvalidValue;
  if (p.page != 16 && p.page != 32 && p.page != 64 && p.page != 128) return cudaErrorNotSupported;
  if (p.tokens < 0 || p.longest < 0 || p.group < 1 || p.table_stride < p.width)
    return cudaErrorInvalidValue;
  // positions, and those up to a tile behind them, in 31 bits; rows, and those a grid behind them
  if (static_cast<long long>(p.width) * p.page > (1LL << 30)) return cudaErrorInvalidValue;
  if (p.pages > 0x7fffffff / p.page) return cudaErrorInvalidValue;  // what no pool can hold
  if (p.tokens > COZY_CACHE_MAX_TOKENS || p.max_blocks > COZY_CACHE_MAX_TOKENS)
    return cudaErrorInvalidValue;
  if (p.group > COZY_CACHE_MAX_GROUP) return cudaErrorNotSupported;
  const void* ptrs[] = {p.lengths, p.added, p.table, p.free_ring, p.cursor, p.lengths_after,
                        p.starts, p.cursor_after, p.units, p.status};
  for (const void* ptr : ptrs)
    if (ptr == nullptr) return cudaErrorInvalidValue;
  if (p.tokens > 0 && (!p.positions || !p.slots || !p.blocks)) return cudaErrorInvalidValue;
  if (reinterpret_cast<uintptr_t>(p.blocks) % 16) return cudaErrorInvalidValue;
  // every block that `tokens` tokens of `requests` requests can touch has an entry
  const long long most = static_cast<long long>(p.tokens) / p.page + 2LL * p.requests;
  if (p.max_blocks < (most < p.tokens ? most : p.tokens)) return cudaErrorInvalidValue;
  return cudaSuccess;
}

int cache_plan(const CozyCachePlan& p, const int* reached, cudaStream_t stream) {
  const int e = cache_plan_check(p);
  if (e) return e;
  const size_t smem = 4 * sizeof(int) * (static_cast<size_t>(p.requests) + 1);
  static bool configured[64] = {};
  int device = 0;
  cudaGetDevice(&device);
  if (device < 64 && !configured[device]) {
    const cudaError_t r = cudaFuncSetAttribute(
        cache_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
        static_cast<int>(4 * sizeof(int) * (COZY_CACHE_MAX_REQUESTS + 1)));
    if (r != cudaSuccess) return r;
    configured[device] = true;
  }
  // one CTA up to a thread for each token, else the portable cluster of 8
  cudaLaunchConfig_t cfg = {};
  const unsigned ctas = p.tokens <= kPlanThreads ? 1 : 8;
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kPlanThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, cache_plan_kernel, p, reached);
}

// -------------------------------------------------------------------------------- the append
// A unit is one touched block of one head of K or V: its new rows are read once (held as bf16 in
// registers), normed and rotated, their largest magnitude sets or grows the block's exponent,
// and their codes are written. WARPS warps share a unit. Queries take CTAs of the same launch.
// HBM bounds the long form: a token reads (Hq + 2 Hkv) · D bf16 and writes Hq · D bf16 and
// 2 · Hkv · D codes. 8192 tokens (32/8 heads of 128) take 42.8 us, 0.67 of the measured copy rate
// (32.4 us, 0.84, without a rotation: each head's keys read the tables from L2 again).
struct AppendTensor {
  int normalize, wide;  // wide: the weights can be read 16 bytes at a time
  const float* norm_weight;
  float norm_offset, norm_eps;
};

struct AppendArgs {
  const int4* blocks;
  const int* positions;
  const int* used;  // tokens of the step's requests: rows from there on belong to nobody
  int max_blocks, tokens;
  int pages, page, heads_q, heads_kv;
  const __nv_bfloat16* src[3];  // query, key, value
  long long src_token[3], src_head[3];
  __nv_bfloat16* out;  // rotated queries
  long long out_token, out_head;
  uint8_t* codes[2];
  int8_t* exponents[2];
  AppendTensor t[3];
  CozyRope rope;
  int rotate, wide;  // wide: the tables' rows can be read 16 bytes at a time
  unsigned query_ctas;
};

// The 8 channels of a row that a thread holds: 4 at `low` and 4 at `high`. Split halves: each
// channel's partner of the rotation beside it, so no shuffle is needed (eight a row and thread
// cost 7 us of a prompt's 49). Otherwise 8 in a row, in one 16-byte access.
struct Piece {
  int low, high, turned;  // turned: rotated pairs, {i, 4 + i} or {2i, 2i + 1}
};

// APART: split halves are rotated, a row takes two accesses a thread.
template <bool APART>
__device__ __forceinline__ Piece piece_at(const AppendArgs& a, int chunk, bool rotate) {
  const int rotary = rotate ? a.rope.rotary : 0;
  if constexpr (APART) {
    if (chunk * 8 < rotary) return {chunk * 4, chunk * 4 + rotary / 2, 4};
    return {chunk * 8, chunk * 8 + 4, 0};
  }
  return {chunk * 8, chunk * 8 + 4, max(0, min(4, rotary / 2 - chunk * 4))};
}

template <bool APART>
__device__ __forceinline__ uint4 load_piece(const __nv_bfloat16* row, const Piece& p) {
  if constexpr (!APART) return *reinterpret_cast<const uint4*>(row + p.low);
  const uint2 low = *reinterpret_cast<const uint2*>(row + p.low);
  const uint2 high = *reinterpret_cast<const uint2*>(row + p.high);
  return make_uint4(low.x, low.y, high.x, high.y);
}

template <bool APART>
__device__ __forceinline__ void store_piece(__nv_bfloat16* row, const Piece& p, uint4 v) {
  if constexpr (APART) {
    *reinterpret_cast<uint2*>(row + p.low) = make_uint2(v.x, v.y);
    *reinterpret_cast<uint2*>(row + p.high) = make_uint2(v.z, v.w);
  } else {
    *reinterpret_cast<uint4*>(row + p.low) = v;
  }
}

template <bool APART>
__device__ __forceinline__ void store_piece(uint8_t* row, const Piece& p, uint2 v) {
  if constexpr (APART) {
    *reinterpret_cast<uint32_t*>(row + p.low) = v.x;
    *reinterpret_cast<uint32_t*>(row + p.high) = v.y;
  } else {
    *reinterpret_cast<uint2*>(row + p.low) = v;
  }
}

// Four values of a table or a weight.
__device__ __forceinline__ void load4(float* to, const float* from, long long stride, bool wide) {
  if (wide) {
    const float4 v = __ldg(reinterpret_cast<const float4*>(from));
    to[0] = v.x; to[1] = v.y; to[2] = v.z; to[3] = v.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) to[i] = __ldg(from + i * stride);
  }
}

// A thread's part of the rotation by one position: cos and sin of its 8 channels (split halves),
// or of its 4 pairs (interleaved, the first 4). Read once for all heads of a token.
struct Turn {
  float c[8], s[8];
};

template <bool APART>
__device__ __forceinline__ Turn turn_at(const AppendArgs& a, long long position, const Piece& p) {
  Turn t;
  const CozyRope& r = a.rope;
  const float* cs = r.cos + position * r.stride_token;
  const float* sn = r.sin + position * r.stride_token;
  if constexpr (APART) {
    if (p.turned) {
      load4(t.c, cs + p.low * r.stride_channel, r.stride_channel, a.wide);
      load4(t.s, sn + p.low * r.stride_channel, r.stride_channel, a.wide);
      load4(t.c + 4, cs + p.high * r.stride_channel, r.stride_channel, a.wide);
      load4(t.s + 4, sn + p.high * r.stride_channel, r.stride_channel, a.wide);
    }
  } else if (p.turned == 4) {
    load4(t.c, cs + p.low / 2 * r.stride_channel, r.stride_channel, a.wide);
    load4(t.s, sn + p.low / 2 * r.stride_channel, r.stride_channel, a.wide);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      t.c[i] = i < p.turned ? __ldg(cs + (p.low / 2 + i) * r.stride_channel) : 1.f;
      t.s[i] = i < p.turned ? __ldg(sn + (p.low / 2 + i) * r.stride_channel) : 0.f;
    }
  }
  return t;
}

// A norm's weights of a thread's channels, the offset in them.
struct Weights {
  float w[8];
};

__device__ __forceinline__ Weights weights_at(const AppendTensor& t, const Piece& p) {
  Weights w;
  if (t.normalize && t.norm_weight != nullptr) {
    load4(w.w, t.norm_weight + p.low, 1, t.wide);
    load4(w.w + 4, t.norm_weight + p.high, 1, t.wide);
#pragma unroll
    for (int i = 0; i < 8; ++i) w.w[i] += t.norm_offset;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) w.w[i] = 1.f;
  }
  return w;
}

// Per-head RMSNorm, then the rotation, of a row held 8 channels a thread (the laws of
// norm_rope.cuh, with the tables' values given): fp32, rounded by the caller.
template <int HD, bool APART>
__device__ __forceinline__ void ready_row(float (&x)[8], const Piece& p, unsigned mask, const AppendTensor& t,
                                          const AppendArgs& a, const Turn& turn, const Weights& w) {
  constexpr int CHUNKS = HD / 8;
  if (t.normalize) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
    for (int o = CHUNKS / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
    const float inv = rsqrtf(ss / HD + t.norm_eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = x[i] * inv * w.w[i];
  }
  if constexpr (APART) {
    if (p.turned) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float lo = x[i], hi = x[4 + i];
        x[i] = lo * turn.c[i] - hi * turn.s[i];
        x[4 + i] = hi * turn.c[4 + i] + lo * turn.s[4 + i];
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i >= p.turned) break;  // channels of their own: an infinity stays in its place
      const float lo = x[2 * i], hi = x[2 * i + 1];
      x[2 * i] = lo * turn.c[i] - hi * turn.s[i];
      x[2 * i + 1] = hi * turn.c[i] + lo * turn.s[i];
    }
  }
}

__device__ __forceinline__ void widen8(uint4 v, float (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ uint4 narrow8(const float (&x)[8]) {
  return make_uint4(bf16_pair(x[0], x[1]), bf16_pair(x[2], x[3]), bf16_pair(x[4], x[5]),
                    bf16_pair(x[6], x[7]));
}

// Eight values to e4m3 codes (round to nearest even; NaN stays NaN).
__device__ __forceinline__ uint2 encode8(const float (&x)[8]) {
  uint16_t h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(h[i]) : "f"(x[2 * i]), "f"(x[2 * i + 1]));
  return make_uint2(h[0] | static_cast<uint32_t>(h[1]) << 16, h[2] | static_cast<uint32_t>(h[3]) << 16);
}

__device__ __forceinline__ void decode8(uint2 c, float (&x)[8]) {
  const uint32_t w[2] = {c.x, c.y};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint16_t pair = static_cast<uint16_t>(w[i >> 1] >> ((i & 1) * 16));
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(pair));
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}

// The smallest exponent e ≥ the floor with amax ≤ 448 · 2^e: 448 = 1.75 · 2^8, so the fraction
// bits carry into the exponent field exactly when they are above 0.75.
__device__ __forceinline__ int exponent_of(float amax) {
  const int e = static_cast<int>((__float_as_uint(amax) + 0x1fffffu) >> 23) - 127 - 8;
  return max(e, kExponentFloor);
}

// Heads of a token that a thread group readies: the tables' values are read once for them.
constexpr int kHeadsAThread = 4;

template <int HD, bool APART>
__device__ __forceinline__ void append_query(const AppendArgs& a) {
  constexpr int CHUNKS = HD / 8, ROWS = 32 / CHUNKS;  // threads a row, rows a warp
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int chunk = lane % CHUNKS, sub = lane / CHUNKS;
  const unsigned mask = row_group_mask<CHUNKS>();
  const int sets = (a.heads_q + kHeadsAThread - 1) / kHeadsAThread;
  const unsigned at = (blockIdx.x * 8 + warp) * ROWS + sub;
  const int token = at / sets, head0 = at % sets * kHeadsAThread;
  if (token >= a.tokens) return;
  const int position = a.positions[token];
  const Piece p = piece_at<APART>(a, chunk, a.rotate);
  uint4 v[kHeadsAThread];
#pragma unroll
  for (int i = 0; i < kHeadsAThread; ++i)
    if (head0 + i < a.heads_q)
      v[i] = load_piece<APART>(a.src[0] + token * a.src_token[0] + (head0 + i) * a.src_head[0], p);
  // a token of a page outside the pool has no place: its query is zero (a branch of its own for
  // the zeros took 44.5 us instead of 42.6 for a prompt of 8192)
  const bool lost = position < 0;
  if (lost && token >= *a.used) return;
  Turn turn = {};
  if (a.rotate) turn = turn_at<APART>(a, max(position, 0), p);
  const Weights w = weights_at(a.t[0], p);
#pragma unroll
  for (int i = 0; i < kHeadsAThread; ++i) {
    if (head0 + i >= a.heads_q) break;
    float x[8];
    widen8(v[i], x);
    ready_row<HD, APART>(x, p, mask, a.t[0], a, turn, w);
    store_piece<APART>(a.out + token * a.out_token + (head0 + i) * a.out_head, p, lost ? make_uint4(0, 0, 0, 0) : narrow8(x));
  }
}

// READY: the rows are normed or rotated first (keys).
template <int HD, int WARPS, int PASSES, bool READY, bool APART>
__device__ __forceinline__ void append_unit(const AppendArgs& a, int which, int head, int4 entry,
                                            float* largest) {
  constexpr int CHUNKS = HD / 8;         // threads a row
  constexpr int ROWS = 32 / CHUNKS;      // rows a warp and pass
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int chunk = lane % CHUNKS, slot = (warp % WARPS) * ROWS + lane / CHUNKS;
  const unsigned mask = row_group_mask<CHUNKS>();
  const AppendTensor& t = a.t[1 + which];
  const __nv_bfloat16* src = a.src[1 + which] + entry.w * a.src_token[1 + which] +
                             head * a.src_head[1 + which];
  const Piece p = piece_at<APART>(a, chunk, READY && a.rotate);
  const long long block = static_cast<long long>(entry.x) * a.heads_kv + head;
  int8_t* exponent = a.exponents[which] + block;
  const int before = entry.y > 0 ? *exponent : kExponentFloor;
  uint4 held[PASSES];
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int r = slot + i * (WARPS * ROWS);
    if (r < entry.z) held[i] = load_piece<APART>(src + r * a.src_token[1 + which], p);
  }
  float amax = 0.f;
  int position = 0;
  Weights w;
  if constexpr (READY) {
    position = a.positions[entry.w];
    w = weights_at(t, p);
  }
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int r = slot + i * (WARPS * ROWS);
    if (r < entry.z) {
      float x[8];
      widen8(held[i], x);
      if constexpr (READY) {
        Turn turn = {};
        if (a.rotate) turn = turn_at<APART>(a, position + r, p);
        ready_row<HD, APART>(x, p, mask, t, a, turn, w);
        held[i] = narrow8(x);
        widen8(held[i], x);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float m = fabsf(x[k]);
        if (m <= kLargestStored) amax = fmaxf(amax, m);
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  if constexpr (WARPS > 1) {
    if (lane == 0) largest[warp] = amax;
    // the unit's own barrier: other units of the CTA may have left
    asm volatile("bar.sync %0, %1;" ::"r"(1 + warp / WARPS), "n"(WARPS * 32) : "memory");
#pragma unroll
    for (int i = 0; i < WARPS; ++i) amax = fmaxf(amax, largest[warp / WARPS * WARPS + i]);
  } else {
    __syncwarp();
  }
  const int e = max(before, exponent_of(amax));
  if (chunk == 0 && slot == 0) *exponent = static_cast<int8_t>(e);
  uint8_t* codes = a.codes[which] + block * a.page * HD;
  const float scale = exponent_scale(-e);
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int r = slot + i * (WARPS * ROWS);
    if (r < entry.z) {
      float x[8];
      widen8(held[i], x);
#pragma unroll
      for (int k = 0; k < 8; ++k)
        x[k] = fabsf(x[k]) <= kLargestStored ? x[k] * scale : __uint_as_float(0x7fc00000u);
      store_piece<APART>(codes + (entry.y + r) * HD, p, encode8(x));
    }
  }
  if (e > before && entry.y > 0) {  // the scale grew: shift what the block holds already
    const float shift = exponent_scale(max(before - e, -126));
    for (int r = slot; r < entry.y; r += WARPS * ROWS) {
      uint2* row = reinterpret_cast<uint2*>(codes + r * HD + chunk * 8);
      float x[8];
      decode8(*row, x);
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] *= shift;
      *row = encode8(x);
    }
  }
}

template <int HD, int WARPS, int PASSES, bool APART>
__global__ void __launch_bounds__(256, 4) cache_append_kernel(const AppendArgs a) {
  constexpr int UNITS = 8 / WARPS;       // units a CTA
  __shared__ float largest[8];
  if (blockIdx.x < a.query_ctas) {  // queries: some heads of a token a group of threads
    append_query<HD, APART>(a);
    return;
  }
  const int warp = threadIdx.x >> 5;
  const long long unit = static_cast<long long>(blockIdx.x - a.query_ctas) * UNITS + warp / WARPS;
  const int which = static_cast<int>(unit & 1);  // 0 keys, 1 values
  const int head = static_cast<int>((unit >> 1) % a.heads_kv);
  const long long at = (unit >> 1) / a.heads_kv;
  const int4 entry = at < a.max_blocks ? a.blocks[at] : make_int4(-1, 0, 0, 0);
  if (entry.x < 0) return;  // all warps of the unit alike
  if (which == 0 && (a.t[1].normalize || a.rotate))
    append_unit<HD, WARPS, PASSES, true, APART>(a, 0, head, entry, largest);
  else
    append_unit<HD, WARPS, PASSES, false, false>(a, which, head, entry, largest);
}

template <int HD>
static int append_launch(AppendArgs& a, int longest, cudaStream_t stream) {
  constexpr int kRows = 32 / (HD / 8);
  const long long sets = (a.heads_q + kHeadsAThread - 1) / kHeadsAThread;
  const long long rows = a.out != nullptr ? a.tokens * sets : 0;
  if (rows > 0x7fffffffLL) return cudaErrorInvalidValue;
  const long long query_ctas = (rows + 8 * kRows - 1) / (8 * kRows);
  const long long units = 2LL * a.heads_kv * a.max_blocks;
  // Four passes of rows a warp, and as many warps a unit as its rows then take (a page of 128 rows
  // of 128 channels: eight passes of 8 warps); two passes of twice the warps took 49.4 us for 8192
  // tokens instead of 42.8. A decode step has one row a unit: one pass, 4.9 us for 256 tokens
  // instead of 5.7 (device time; 32/8 heads of 128, pages of 64).
  const int most = longest < a.page ? longest : a.page;
  const int warps = most <= 4 * kRows ? 1 : most <= 8 * kRows ? 2 : most <= 16 * kRows ? 4 : 8;
  const long long ctas = query_ctas + (units * warps + 7) / 8;
  if (ctas > 0x7fffffffLL) return cudaErrorInvalidValue;
  a.query_ctas = static_cast<unsigned>(query_ctas);
  const unsigned grid = static_cast<unsigned>(ctas);
  const bool apart = a.rotate && !a.rope.interleaved && a.rope.rotary > 0;
  const auto launch = [&](auto* split, auto* whole) { (apart ? split : whole)<<<grid, 256, 0, stream>>>(a); };
  if (most <= kRows) launch(cache_append_kernel<HD, 1, 1, true>, cache_append_kernel<HD, 1, 1, false>);
  else if (warps == 1) launch(cache_append_kernel<HD, 1, 4, true>, cache_append_kernel<HD, 1, 4, false>);
  else if (warps == 2) launch(cache_append_kernel<HD, 2, 4, true>, cache_append_kernel<HD, 2, 4, false>);
  else if (warps == 4) launch(cache_append_kernel<HD, 4, 4, true>, cache_append_kernel<HD, 4, 4, false>);
  else if (most <= 32 * kRows)
    launch(cache_append_kernel<HD, 8, 4, true>, cache_append_kernel<HD, 8, 4, false>);
  else
    launch(cache_append_kernel<HD, 8, 128 / 8 / kRows, true>,
           cache_append_kernel<HD, 8, 128 / 8 / kRows, false>);
  return cudaGetLastError();
}

int cache_store_check(const CozyCacheStore& c, const CozyCachePlan& p) {
  if (c.head_dim != 64 && c.head_dim != 128) return cudaErrorNotSupported;
  if (c.heads_kv < 1 || c.pages != p.pages || c.page != p.page) return cudaErrorInvalidValue;
  // rows of a pool are counted in 31 bits (tensor-map coordinates)
  if (static_cast<long long>(c.pages) * c.heads_kv > 0x7fffffffLL / c.page)
    return cudaErrorInvalidValue;
  if (!c.key || !c.value || !c.key_exponent || !c.value_exponent) return cudaErrorInvalidValue;
  if (reinterpret_cast<uintptr_t>(c.key) % 128 || reinterpret_cast<uintptr_t>(c.value) % 128)
    return cudaErrorInvalidValue;
  return cudaSuccess;
}

int cache_append(const CozyCachePlan& p, const CozyCacheStore& c, const CozyCacheAppend& x,
                 cudaStream_t stream) {
  int e = cache_plan_check(p);
  if (e || (e = cache_store_check(c, p))) return e;
  if (p.tokens == 0 || p.longest == 0) return cudaSuccess;  // nobody brings a token
  AppendArgs a = {};
  a.blocks = reinterpret_cast<const int4*>(p.blocks);
  a.positions = p.positions;
  a.used = p.starts + p.requests;
  a.max_blocks = p.max_blocks;
  a.tokens = p.tokens;
  a.pages = c.pages;
  a.page = c.page;
  a.heads_q = c.heads_kv * p.group;
  a.heads_kv = c.heads_kv;
  const void* src[3] = {x.query, x.key, x.value};
  const long long* strides[3] = {x.query_strides, x.key_strides, x.value_strides};
  for (int i = 0; i < 3; ++i) {
    if (i == 0 && src[0] == nullptr) continue;
    if (src[i] == nullptr || reinterpret_cast<uintptr_t>(src[i]) % 16) return cudaErrorInvalidValue;
    if (strides[i][0] < 0 || strides[i][1] < 0 || strides[i][0] % 8 || strides[i][1] % 8)
      return cudaErrorInvalidValue;
    a.src[i] = static_cast<const __nv_bfloat16*>(src[i]);
    a.src_token[i] = strides[i][0];
    a.src_head[i] = strides[i][1];
  }
  if (src[0] != nullptr) {
    if (x.out == nullptr || reinterpret_cast<uintptr_t>(x.out) % 16 || x.out_strides[0] % 8 ||
        x.out_strides[1] % 8 || x.out_strides[0] < 0 || x.out_strides[1] < 0)
      return cudaErrorInvalidValue;
    a.out = static_cast<__nv_bfloat16*>(x.out);
    a.out_token = x.out_strides[0];
    a.out_head = x.out_strides[1];
  }
  a.codes[0] = static_cast<uint8_t*>(c.key);
  a.codes[1] = static_cast<uint8_t*>(c.value);
  a.exponents[0] = static_cast<int8_t*>(c.key_exponent);
  a.exponents[1] = static_cast<int8_t*>(c.value_exponent);
  for (int i = 0; i < 2; ++i) {
    a.t[i].normalize = x.normalize[i];
    a.t[i].norm_weight = x.norm_weight[i];
    a.t[i].norm_offset = x.norm_offset[i];
    a.t[i].norm_eps = x.norm_eps[i];
    a.t[i].wide = reinterpret_cast<uintptr_t>(x.norm_weight[i]) % 16 == 0;
  }
  if (x.rope != nullptr) {
    a.rope = *x.rope;
    if (!a.rope.cos || !a.rope.sin || a.rope.rotary < 0 || a.rope.rotary > c.head_dim ||
        a.rope.rotary % 2)
      return cudaErrorInvalidValue;
    if (!a.rope.interleaved && a.rope.rotary % 16) return cudaErrorNotSupported;
    a.rotate = 1;
    a.wide = a.rope.stride_channel == 1 && a.rope.stride_token % 4 == 0 &&
             reinterpret_cast<uintptr_t>(a.rope.cos) % 16 == 0 &&
             reinterpret_cast<uintptr_t>(a.rope.sin) % 16 == 0;
  }
  return c.head_dim == 64 ? append_launch<64>(a, p.longest, stream)
                          : append_launch<128>(a, p.longest, stream);
}

}  // namespace cozy
