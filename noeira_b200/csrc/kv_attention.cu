// Attention of new tokens over the paged 8-bit cache: o = softmax(c q K^T) V over the keys up to each token's own position.
#include "common.cuh"
#include "kv_cache.h"

namespace {
using namespace nb;

__device__ __forceinline__ float2 values_of(uint16_t two) {
  uint32_t h2;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"(two));
  return __half22float2(*reinterpret_cast<__half2*>(&h2));
}

// One warp per (new token, query head): a lane holds D / 32 dimensions, one pass over the keys with a running maximum.
template <int D>
__global__ void __launch_bounds__(128) kv_attn_warp_kernel(KvAttn p) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31, h = blockIdx.y;
  const int t = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (t >= p.starts[p.rows] || t >= p.tokens) return;
  int a = 0, b = p.rows;
  while (b - a > 1) {
    const int m = (a + b) >> 1;
    if (p.starts[m] <= t) a = m; else b = m;
  }
  const int end = min(p.ends[a], p.width * p.block);
  const int last = min(end, p.ends[a] - (p.starts[a + 1] - t) + 1);   // keys [0, last)
  const int hk = h / (p.hq / p.hk);
  const __nv_bfloat16* q = (const __nv_bfloat16*)p.q + t * p.q_token + h * p.q_head + lane * E;
  float qv[E], o[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < E; ++i) { qv[i] = __bfloat162float(q[i]) * p.scale_log2; o[i] = 0.f; }
  for (int j = 0; j < last; ++j) {
    const int id = p.tables[(long long)a * p.width + j / p.block];
    if (id < 0 || id >= p.blocks) {
      if (lane == 0) report(p.status, NB_ST_BOUNDS, 10, a);
      continue;
    }
    const long long at = (((long long)id * p.hk + hk) * p.block + j % p.block) * D + lane * E;
    const float ks = p.scale[(long long)id * p.hk + hk], vs = p.scale[p.s_stride + (long long)id * p.hk + hk];
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < E; i += 2) {
      const float2 k = values_of(*reinterpret_cast<const uint16_t*>(p.codes + at + i));
      s += qv[i] * k.x + qv[i + 1] * k.y;
    }
    s = warp_sum(s) * ks;
    const float mn = fmaxf(m, s), w = exp2f(s - mn), r = exp2f(m - mn);
    m = mn;
    l = l * r + w;
#pragma unroll
    for (int i = 0; i < E; i += 2) {
      const float2 v = values_of(*reinterpret_cast<const uint16_t*>(p.codes + p.kv_stride + at + i));
      o[i] = o[i] * r + w * v.x * vs;
      o[i + 1] = o[i + 1] * r + w * v.y * vs;
    }
  }
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  __nv_bfloat16* out = (__nv_bfloat16*)p.out + t * p.o_token + h * p.o_head + lane * E;
#pragma unroll
  for (int i = 0; i < E; ++i) out[i] = __float2bfloat16(o[i] * inv);
}

}  // namespace

extern "C" int nb_kv_attention(const void* q, void* out, const void* codes, const float* scale, const int* tables, const int* starts,
                               const int* ends, int rows, int tokens, int max_new, int hq, int hk, int dim, int block, int blocks, int width,
                               long long q_token, long long q_head, long long o_token, long long o_head, long long kv_stride, long long s_stride,
                               float softmax_scale, float* work, long long work_floats, unsigned int* status, void* stream) {
  if (rows <= 0 || tokens < 0 || hk <= 0 || hq <= 0 || hq % hk || (dim != 64 && dim != 128) || block <= 0 || blocks <= 0 || width <= 0) return NB_ERR_BAD_ARG;
  if (tokens == 0) return NB_OK;
  KvAttn p{q, out, (const uint8_t*)codes, scale, tables, starts, ends, rows, tokens, hq, hk, block, blocks, width, q_token, q_head, o_token, o_head,
           kv_stride, s_stride, softmax_scale * 1.4426950408889634f, nullptr, nullptr, status};
  const dim3 grid(ceil_div(tokens, 4), hq);
  if (dim == 64) kv_attn_warp_kernel<64><<<grid, 128, 0, (cudaStream_t)stream>>>(p);
  else kv_attn_warp_kernel<128><<<grid, 128, 0, (cudaStream_t)stream>>>(p);
  NB_LAUNCH_CHECK();
  return NB_OK;
}
