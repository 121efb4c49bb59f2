// Attention over the 8-bit paged cache (the plain form: a warp a query row and head).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/cozy_ulysses.h"
#include "cache.cuh"

namespace cozy {

int cache_store_check(const CozyCacheStore& c, const CozyCachePlan& p);

template <int HD>
__global__ void __launch_bounds__(128) cache_attend_plain(const CozyCachePlan p,
                                                          const CozyCacheStore c,
                                                          const CozyCacheAttend a) {
  constexpr int PER = HD / 32;
  const int lane = threadIdx.x & 31;
  const int heads_q = c.heads_kv * p.group;
  const long long row = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (row >= static_cast<long long>(p.tokens) * heads_q) return;
  const int token = static_cast<int>(row / heads_q), hq = static_cast<int>(row % heads_q);
  if (token >= p.starts[p.requests]) return;
  int n = 0;
  for (int low = 0, high = p.requests - 1; low <= high;) {
    const int mid = (low + high) >> 1;
    if (p.starts[mid] <= token) { n = mid; low = mid + 1; }
    else high = mid - 1;
  }
  const int h = hq / p.group;
  const int keys = p.lengths_after[n] - (p.starts[n + 1] - token) + 1;
  const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(a.query) +
                           token * a.query_strides[0] + hq * a.query_strides[1] + lane * PER;
  float qv[PER], o[PER];
  for (int i = 0; i < PER; ++i) {
    qv[i] = __bfloat162float(q[i]) * a.scale;
    o[i] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int k = 0; k < keys; ++k) {
    const int page = p.table[n * p.table_stride + k / p.page];
    if (page < 0 || page >= p.pages) {
      if (lane == 0) atomicOr(p.status, kPlanBadPage);
      continue;
    }
    const long long block = static_cast<long long>(page) * c.heads_kv + h;
    const long long at = (block * p.page + k % p.page) * HD + lane * PER;
    const float ks = exponent_scale(static_cast<const int8_t*>(c.key_exponent)[block]);
    const float vs = exponent_scale(static_cast<const int8_t*>(c.value_exponent)[block]);
    float s = 0.f, v[PER];
    for (int i = 0; i < PER; i += 2) {
      uint32_t hk, hv;
      asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(hk) : "h"(*reinterpret_cast<const uint16_t*>(static_cast<const uint8_t*>(c.key) + at + i)));
      asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(hv) : "h"(*reinterpret_cast<const uint16_t*>(static_cast<const uint8_t*>(c.value) + at + i)));
      const float2 fk = __half22float2(*reinterpret_cast<const __half2*>(&hk));
      const float2 fv = __half22float2(*reinterpret_cast<const __half2*>(&hv));
      s = fmaf(qv[i], fk.x, fmaf(qv[i + 1], fk.y, s));
      v[i] = fv.x * vs;
      v[i + 1] = fv.y * vs;
    }
    for (int b = 16; b > 0; b >>= 1) s += __shfl_xor_sync(0xffffffffu, s, b);
    s *= ks;
    const float top = fmaxf(m, s), w = m == -INFINITY ? 0.f : __expf(m - top), e = __expf(s - top);
    l = l * w + e;
    for (int i = 0; i < PER; ++i) o[i] = fmaf(e, v[i], o[i] * w);
    m = top;
  }
  __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out) + token * a.out_strides[0] +
                       hq * a.out_strides[1] + lane * PER;
  for (int i = 0; i < PER; ++i) out[i] = __float2bfloat16(l > 0.f || l != l ? o[i] / l : 0.f);
  if (a.lse != nullptr && lane == 0) a.lse[row] = m + logf(l);
}

long long cache_workspace(const CozyCachePlan& p, const CozyCacheStore& c) { return 0; }

int cache_attention(const CozyCachePlan& p, const CozyCacheStore& c, const CozyCacheAttend& a,
                    cudaStream_t stream) {
  const int e = cache_store_check(c, p);
  if (e) return e;
  if (p.tokens == 0) return cudaSuccess;
  if (!(a.scale > 0.f) || a.scale > 3.0e38f) return cudaErrorInvalidValue;
  const void* ptrs[] = {a.query, a.out};
  for (const void* ptr : ptrs)
    if (ptr == nullptr || reinterpret_cast<uintptr_t>(ptr) % 16) return cudaErrorInvalidValue;
  for (int i = 0; i < 2; ++i)
    if (a.query_strides[i] < 0 || a.query_strides[i] % 8 || a.out_strides[i] < 0 ||
        a.out_strides[i] % 8)
      return cudaErrorInvalidValue;
  const long long rows = static_cast<long long>(p.tokens) * c.heads_kv * p.group;
  const long long ctas = (rows + 3) / 4;
  if (ctas > 0x7fffffffLL) return cudaErrorInvalidValue;
  if (c.head_dim == 64) cache_attend_plain<64><<<static_cast<unsigned>(ctas), 128, 0, stream>>>(p, c, a);
  else cache_attend_plain<128><<<static_cast<unsigned>(ctas), 128, 0, stream>>>(p, c, a);
  return cudaGetLastError();
}

}  // namespace cozy
