// Paged key / value cache in 8 bits: block tables and slot maps, writing tokens, reordering for beam search.
//
// A layer of the cache is  codes e4m3 [2, N, H, bs, D]  (keys, values) with one fp32 scale per block and head [2, N, H];
// a value is code * scale.  Scales are powers of two: a block whose scale has to grow when a larger token arrives moves its
// codes by an exponent shift, which loses nothing but bits that fall below the smallest e4m3 value, and the relative
// precision of e4m3 does not depend on where the top of its range lies.
#include "common.cuh"
#include "kv_cache.h"

namespace {
using namespace nb;

constexpr float F8_TOP = 448.f;

// smallest 2^e >= 2^-118 with amax <= 448 * 2^e (448 = 1.75 * 2^8); amax finite and >= 0
__device__ __forceinline__ float scale_for(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  int e = (int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);   // biased exponent of the scale
  e = max(e, 127 - 118);
  return __uint_as_float((uint32_t)e << 23);
}
// exact reciprocal of a power of two in [2^-118, 2^120]
__device__ __forceinline__ float inv_pow2(float s) { return __uint_as_float((254u << 23) - __float_as_uint(s)); }

__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t code_of(float x) {   // e4m3 code of one value; infinities become NaN like NaN itself
  return fabsf(x) <= F8_TOP ? (e4m3x2(x, 0.f) & 0xffu) : 0x7fu;
}
__device__ __forceinline__ float value_of(uint32_t code) {
  uint32_t h2;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"((uint16_t)code));
  return __half2float(__ushort_as_half((unsigned short)(h2 & 0xffffu)));
}

// ------------------------------------------------------------------------------------------------ plan
// Inclusive sum over the block (256 threads); `sh` holds 8 values.
__device__ __forceinline__ long long block_scan(long long v, long long* sh, long long& total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  __syncthreads();
  if (lane == 31) sh[w] = v;
  __syncthreads();
  long long before = 0;
  total = 0;
  for (int i = 0; i < 8; ++i) {
    if (i < w) before += sh[i];
    total += sh[i];
  }
  return v + before;
}

__global__ void __launch_bounds__(256) kv_plan_kernel(KvPlan p) {
  extern __shared__ int sm[];
  int* s_start = sm;                 // [rows + 1]
  int* s_off = sm + p.rows + 1;      // [rows] first block of the row among the new ones, -1: refused
  __shared__ long long sh[8];
  const int tid = threadIdx.x, per = ceil_div(p.rows, 256);
  const int lo = min(p.rows, tid * per), hi = min(p.rows, lo + per);
  const int free_count = max(0, min(*p.free_count, p.free_size));
  long long sum = 0, total;
  for (int i = lo; i < hi; ++i) sum += max(0, p.new_lens[i]);
  long long at = block_scan(sum, sh, total) - sum;      // 64 bits: lengths are the caller's, their sum may be anything
  if (tid == 0) s_start[p.rows] = (int)min(total, 0x7fffffffLL);
  sum = 0;
  for (int i = lo; i < hi; ++i) {
    const int len = p.lengths[i], add = max(0, p.new_lens[i]);
    s_start[i] = (int)min(at, 0x7fffffffLL);
    at += add;
    const bool fits = len >= 0 && p.new_lens[i] >= 0 && (long long)len + add <= (long long)p.width * p.block && at <= p.tokens;
    s_off[i] = fits ? ceil_div(len + add, p.block) - ceil_div(len, p.block) : -1;
    sum += max(0, s_off[i]);
  }
  long long off = block_scan(sum, sh, total) - sum, taken = 0;
  for (int i = lo; i < hi; ++i) {
    const int need = s_off[i];
    if (need < 0 || (need > 0 && off + need > free_count)) {
      s_off[i] = -1;
      if (blockIdx.x == 0) report(p.status, NB_ST_CACHE_FULL, 1, i);
    } else {
      s_off[i] = (int)min(off, 0x7fffffffLL);           // with need = 0 any offset will do
      if (need > 0) taken = off + need;
    }
    if (need > 0) off += need;
    if (blockIdx.x == 0) p.ends[i] = p.lengths[i] + (s_off[i] < 0 ? 0 : p.new_lens[i]);
  }
  __syncthreads();
  if (blockIdx.x == 0) {
    for (int i = tid; i <= p.rows; i += 256) p.starts[i] = s_start[i];
    taken = (long long)__reduce_max_sync(0xffffffffu, (unsigned)taken);   // at most free_count
    if ((tid & 31) == 0) sh[tid >> 5] = taken;
    __syncthreads();
    if (tid == 0) {
      for (int i = 1; i < 8; ++i) taken = max(taken, sh[i]);
      *p.free_count_out = free_count - (int)taken;
    }
  }
  for (long long t = (long long)blockIdx.x * 256 + tid; t < p.tokens; t += (long long)gridDim.x * 256) {
    if (t >= s_start[p.rows]) {
      p.slots[t] = -1;
      p.positions[t] = 0;
      p.row_of[t] = -1;
      continue;
    }
    int a = 0, b = p.rows;             // last row with start <= t
    while (b - a > 1) {
      const int m = (a + b) >> 1;
      if (s_start[m] <= (int)t) a = m; else b = m;
    }
    const int len = p.lengths[a], pos = len + (int)t - s_start[a], pg = pos / p.block, in = pos - pg * p.block;
    int slot = -1;
    if (s_off[a] >= 0) {
      const int have = ceil_div(len, p.block);
      int id;
      if (pg < have) {
        id = p.tables[(long long)a * p.width + pg];
      } else {
        id = p.free_ids[free_count - 1 - (s_off[a] + pg - have)];
        if (in == 0) p.tables[(long long)a * p.width + pg] = id;
      }
      if (id >= 0) slot = id * p.block + in;
    }
    p.slots[t] = slot;
    p.positions[t] = pos;
    p.row_of[t] = a;
  }
}

// ------------------------------------------------------------------------------------------------ append
// Nearest token before / from `t` whose slot lies in the cache (-1 / tokens: none); all lanes take part.
__device__ __forceinline__ long long valid_before(const KvAppend& p, long long t) {
  const int lane = threadIdx.x & 31;
  for (long long e = t; e > 0; e -= 32) {
    const long long i = e - 1 - lane;
    const unsigned got = __ballot_sync(0xffffffffu, i >= 0 && (unsigned)p.slots[i] < (unsigned)p.limit);
    if (got) return e - __ffs(got);
  }
  return -1;
}
__device__ __forceinline__ long long valid_from(const KvAppend& p, long long t) {
  const int lane = threadIdx.x & 31;
  for (; t < p.tokens; t += 32) {
    const long long i = t + lane;
    const unsigned got = __ballot_sync(0xffffffffu, i < p.tokens && (unsigned)p.slots[i] < (unsigned)p.limit);
    if (got) return t + __ffs(got) - 1;
  }
  return p.tokens;
}

// One warp per (token, head, K or V).  A run is a stretch of neighbouring tokens and slots inside one block; the warp of a
// run's first token does the run, and what continues it in the same block behind skipped tokens.
__global__ void __launch_bounds__(128) kv_append_kernel(KvAppend p) {
  const int lane = threadIdx.x & 31;
  long long t0 = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (t0 >= p.tokens) return;
  const int h = blockIdx.y % p.heads, which = blockIdx.y / p.heads;
  int slot = p.slots[t0];
  if ((unsigned)slot >= (unsigned)p.limit) return;
  const int id = slot / p.block;
  int off = slot - id * p.block;
  if (off > 0) {
    const long long before = valid_before(p, t0);
    if (before >= 0 && p.slots[before] == slot - 1) return;
  }
  const long long step = which ? p.v_token : p.k_token;
  const long long bh = ((long long)which * p.blocks + id) * p.heads + h;
  uint8_t* codes = p.codes + (long long)which * p.kv_stride + ((long long)id * p.heads + h) * p.block * p.dim;
  float old = off > 0 ? p.scale[bh] : 0.f;
  for (;;) {
    const __nv_bfloat16* x = (const __nv_bfloat16*)(which ? p.v : p.k) + t0 * step + (long long)h * (which ? p.v_head : p.k_head);
    int n = 1;
    while (off + n < p.block && t0 + n < p.tokens && p.slots[t0 + n] == slot + n) ++n;
    float amax = 0.f;
    for (int i = 0; i < n; ++i)
      for (int d = lane; d < p.dim; d += 32) {
        const float v = fabsf(__bfloat162float(x[i * step + d]));
        if (v <= 3.4028235e38f) amax = fmaxf(amax, v);
      }
    amax = warp_max(amax);
    const float now = fmaxf(old, scale_for(amax));
    if (off > 0 && now != old) {
      const float r = old * inv_pow2(now);
      for (int i = lane; i < off * p.dim; i += 32) codes[i] = (uint8_t)code_of(value_of(codes[i]) * r);
    }
    const float inv = inv_pow2(now);
    for (int i = 0; i < n; ++i)
      for (int d = lane; d < p.dim; d += 32) codes[(off + i) * p.dim + d] = (uint8_t)code_of(__bfloat162float(x[i * step + d]) * inv);
    __syncwarp();
    old = now;
    off += n;
    slot += n;
    if (off == p.block) break;
    t0 = valid_from(p, t0 + n);
    if (t0 >= p.tokens || p.slots[t0] != slot) break;
  }
  if (lane == 0) p.scale[bh] = old;
}

// ------------------------------------------------------------------------------------------------ reorder
__global__ void __launch_bounds__(128) kv_reorder_kernel(KvReorder p) {
  const int j = blockIdx.x, g = j / p.beams * p.beams;
  int parent = p.parents[j];
  if (parent < 0 || parent >= p.beams) {
    if (threadIdx.x == 0 && blockIdx.y == 0) report(p.status, NB_ST_BOUNDS, 2, j);
    parent = j - g;
  }
  const int src = g + parent, len = max(0, min(p.lengths[src], p.width * p.block)), full = len / p.block, fill = len - full * p.block;
  bool move = src != j && fill > 0;
  const int from = move ? p.tables[(long long)src * p.width + full] : -1, to = p.spare[j];
  if (move && (from < 0 || from >= p.blocks || to < 0 || to >= p.blocks)) {
    if (threadIdx.x == 0 && blockIdx.y == 0) report(p.status, NB_ST_BOUNDS, 3, j);
    move = false;
  }
  if (blockIdx.y == 0) {
    const int pages = ceil_div(len, p.block);
    for (int i = threadIdx.x; i < p.width; i += blockDim.x) {
      int id = i < pages ? p.tables[(long long)src * p.width + i] : -1;
      if (move && i == full) id = to;
      p.tables_out[(long long)j * p.width + i] = id;
    }
    if (threadIdx.x == 0) {
      p.lengths_out[j] = p.lengths[src];
      int left = to;
      if (move) {
        const int mine = p.lengths[j];
        left = mine > 0 && mine % p.block && mine / p.block < p.width ? p.tables[(long long)j * p.width + mine / p.block] : -1;
      }
      p.spare_out[j] = left;
    }
  }
  if (!move) return;
  const long long page = (long long)p.heads * p.block * p.dim;
  uint8_t* base = p.codes + (long long)blockIdx.y * p.plane;
  const uint4* s = reinterpret_cast<const uint4*>(base + (long long)from * page);
  uint4* d = reinterpret_cast<uint4*>(base + (long long)to * page);
  const int head16 = p.block * p.dim / 16, fill16 = fill * p.dim / 16;
  for (int i = threadIdx.x; i < p.heads * fill16; i += blockDim.x) {
    const int h = i / fill16, o = h * head16 + i - h * fill16;
    d[o] = s[o];
  }
  float* sc = p.scale + (long long)blockIdx.y * p.blocks * p.heads;
  for (int i = threadIdx.x; i < p.heads; i += blockDim.x) sc[(long long)to * p.heads + i] = sc[(long long)from * p.heads + i];
}

}  // namespace

extern "C" {

// Block tables and slot maps.  rows <= 8192; `tables` int32 [rows, width] is completed in place, `free_count_out` may not be
// `free_count` (callers that keep one counter copy it back).
int nb_kv_plan(const int* lengths, const int* new_lens, int* tables, const int* free_ids, const int* free_count, int* free_count_out,
               int* starts, int* ends, int* row_of, int* positions, int* slots, int rows, int width, int block, int free_size,
               int tokens, unsigned int* status, void* stream) {
  if (rows <= 0 || rows > 8192 || width <= 0 || block <= 0 || tokens < 0 || free_size < 0) return NB_ERR_BAD_ARG;
  if (free_count == free_count_out || (long long)width * block > 0x7fffffffLL) return NB_ERR_BAD_ARG;
  KvPlan p{lengths, new_lens, tables, free_ids, free_count, free_count_out, starts, ends, row_of, positions, slots, rows, width, block, free_size, tokens, status};
  static bool configured[64] = {};
  int dev = 0;
  NB_CUDA(cudaGetDevice(&dev));
  if (dev >= 64) return NB_ERR_BAD_ARG;
  if (!configured[dev]) {
    NB_CUDA(cudaFuncSetAttribute(kv_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (2 * 8192 + 1) * 4));
    configured[dev] = true;
  }
  const int grid = max(1, min(296, ceil_div(tokens, 1024)));
  kv_plan_kernel<<<grid, 256, (2 * rows + 1) * 4, (cudaStream_t)stream>>>(p);
  NB_LAUNCH_CHECK();
  return NB_OK;
}

int nb_kv_append(const void* k, const void* v, void* codes, float* scale, const int* slots, int tokens, int heads, int dim, int block,
                 int blocks, long long k_token, long long k_head, long long v_token, long long v_head, long long kv_stride, void* stream) {
  if (tokens < 0 || heads <= 0 || (dim != 64 && dim != 128) || block <= 0 || blocks <= 0 || (long long)blocks * block > 0x7fffffffLL) return NB_ERR_BAD_ARG;
  if (tokens == 0) return NB_OK;
  KvAppend p{k, v, (uint8_t*)codes, scale, slots, tokens, heads, dim, block, blocks, blocks * block, k_token, k_head, v_token, v_head, kv_stride};
  kv_append_kernel<<<dim3(ceil_div(tokens, 4), 2 * heads), 128, 0, (cudaStream_t)stream>>>(p);
  NB_LAUNCH_CHECK();
  return NB_OK;
}

int nb_kv_reorder(void* codes, float* scale, const int* tables, const int* lengths, const int* parents, const int* spare, int* tables_out,
                  int* lengths_out, int* spare_out, int planes, int blocks, int heads, int block, int dim, int rows, int beams, int width,
                  unsigned int* status, void* stream) {
  if (planes <= 0 || planes > 65535 || blocks <= 0 || heads <= 0 || block <= 0 || dim % 16 || rows <= 0 || beams <= 0 || rows % beams || width <= 0) return NB_ERR_BAD_ARG;
  if (reinterpret_cast<uintptr_t>(codes) & 15) return NB_ERR_UNALIGNED;
  KvReorder p{(uint8_t*)codes, scale, tables, lengths, parents, spare, tables_out, lengths_out, spare_out, blocks, heads, block, dim, rows, beams, width,
              (long long)blocks * heads * block * dim, status};
  kv_reorder_kernel<<<dim3(rows, planes), 128, 0, (cudaStream_t)stream>>>(p);
  NB_LAUNCH_CHECK();
  return NB_OK;
}

}  // extern "C"
