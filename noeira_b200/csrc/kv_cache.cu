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
// Sums over the rows (tokens before a row, new blocks before a row), then a search for each token.  Every block does the sums for
// itself in shared memory: a kernel of its own for them would cost a launch, which is all that a decode step takes (64 rows of one
// token 3.3 us).  600k tokens of 2048 rows: 12.7 us; the bytes (7.6 MB written) would be 1.2, the sums take half of the rest and the
// eleven dependent reads of a search the other.
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

// Place of row i in shared memory: a thread's rows are neighbours, and without a gap every 32 the threads of a warp would meet in the
// same banks.
__host__ __device__ inline int spread(int i) { return i + (i >> 5); }

__global__ void __launch_bounds__(256) kv_plan_kernel(const KvPlan p) {
  extern __shared__ int sm[];
  int* s_start = sm;                 // [rows + 1]
  int* s_off = sm + spread(p.rows) + 1;   // [rows] first block of the row among the new ones, -1: refused
  int* s_len = s_off + spread(p.rows) + 1;   // [rows]
  __shared__ long long sh[8];
  const int tid = threadIdx.x, per = ceil_div(p.rows, 256);
  const int lo = min(p.rows, tid * per), hi = min(p.rows, lo + per);
  const int free_count = max(0, min(*p.free_count, p.free_size));
#pragma unroll 4
  for (int i = tid; i < p.rows; i += 256) {
    s_len[spread(i)] = p.lengths[i];
    s_off[spread(i)] = p.new_lens[i];
  }
  __syncthreads();
  long long sum = 0, total;
  for (int i = lo; i < hi; ++i) sum += max(0, s_off[spread(i)]);
  long long at = block_scan(sum, sh, total) - sum;      // 64 bits: lengths are the caller's, their sum may be anything
  if (tid == 0) s_start[spread(p.rows)] = (int)min(total, 0x7fffffffLL);
  sum = 0;
  for (int i = lo; i < hi; ++i) {
    const int len = s_len[spread(i)], given = s_off[spread(i)], add = max(0, given);
    s_start[spread(i)] = (int)min(at, 0x7fffffffLL);
    at += add;
    const bool fits = len >= 0 && given >= 0 && (long long)len + add <= p.limit && at <= p.tokens;
    s_off[spread(i)] = fits ? ((len + add + (1 << p.block_log) - 1) >> p.block_log) - ((len + (1 << p.block_log) - 1) >> p.block_log) : -1;
    sum += max(0, s_off[spread(i)]);
  }
  long long off = block_scan(sum, sh, total) - sum, taken = 0;
  for (int i = lo; i < hi; ++i) {
    const int need = s_off[spread(i)];
    if (need < 0 || (need > 0 && off + need > free_count)) {
      s_off[spread(i)] = -1;
      if (blockIdx.x == 0) report(p.status, NB_ST_CACHE_FULL, 1, i);
    } else {
      s_off[spread(i)] = (int)min(off, 0x7fffffffLL);           // with need = 0 any offset will do
      if (need > 0) taken = off + need;
    }
    if (need > 0) off += need;
  }
  __syncthreads();
  if (blockIdx.x == 0) {
    for (int i = tid; i <= p.rows; i += 256) {
      p.starts[i] = s_start[spread(i)];
      if (i < p.rows) p.ends[i] = s_len[spread(i)] + (s_off[spread(i)] < 0 ? 0 : s_start[spread(i + 1)] - s_start[spread(i)]);
    }
    taken = (long long)__reduce_max_sync(0xffffffffu, (unsigned)taken);   // at most free_count
    if ((tid & 31) == 0) sh[tid >> 5] = taken;
    __syncthreads();
    if (tid == 0) {
      for (int i = 1; i < 8; ++i) taken = max(taken, sh[i]);
      *p.free_count_out = free_count - (int)taken;
    }
  }
  // A token a thread: four neighbours to a thread, sharing a search and 16-byte stores, waited for their tables in turn and took
  // longer at every size (64 rows of one token 4.7 us instead of 3.4, 2000 rows of 30 tokens 7.7 instead of 7.2).
  for (long long t0 = (long long)blockIdx.x * 256 + tid; t0 < p.tokens; t0 += (long long)gridDim.x * 256) {
    const int t = (int)t0;
    int a = 0, b = p.rows;             // last row with start <= t
    while (b - a > 1) {
      const int m = (a + b) >> 1;
      if (s_start[spread(m)] <= t) a = m; else b = m;
    }
    const bool real = t < s_start[spread(p.rows)];
    const int len = s_len[spread(a)], off0 = s_off[spread(a)], pos = len + t - s_start[spread(a)];
    int slot = -1;
    if (real && off0 >= 0) {
      const int pg = pos >> p.block_log, in = pos - (pg << p.block_log), have = (int)(((long long)len + (1 << p.block_log) - 1) >> p.block_log);
      int id;
      if (pg < have) {
        id = p.tables[(long long)a * p.width + pg];
      } else {
        id = p.free_ids[free_count - 1 - (off0 + pg - have)];
        if ((unsigned)id >= (unsigned)p.blocks) id = -1;
        if (in == 0) p.tables[(long long)a * p.width + pg] = id;    // the first token of a block: the block is new
      }
      if ((unsigned)id < (unsigned)p.blocks) slot = (id << p.block_log) + in;
      else report(p.status, NB_ST_BOUNDS, 4, a);
    }
    p.slots[t0] = slot;
    p.positions[t0] = slot >= 0 ? pos : 0;   // a place that the row does not have is none to look up: it may lie anywhere
    p.row_of[t0] = real ? a : -1;
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

// Eight bf16 of a token, as raw words.
__device__ __forceinline__ uint4 eight(const __nv_bfloat16* x, int vec) {
  if (vec) return *reinterpret_cast<const uint4*>(x);
  const unsigned short* e = reinterpret_cast<const unsigned short*>(x);
  return make_uint4(e[0] | (uint32_t)e[1] << 16, e[2] | (uint32_t)e[3] << 16, e[4] | (uint32_t)e[5] << 16, e[6] | (uint32_t)e[7] << 16);
}
__device__ __forceinline__ uint32_t abs_max(uint32_t m, const uint4& w) {   // of bf16 pairs, by their bits
  constexpr uint32_t A = 0x7fff7fffu;
  return __vmaxu2(m, __vmaxu2(__vmaxu2(w.x & A, w.y & A), __vmaxu2(w.z & A, w.w & A)));
}
__device__ __forceinline__ uint32_t codes4(uint32_t a, uint32_t b, float inv) {
  return e4m3x2(__uint_as_float(a << 16) * inv, __uint_as_float(a & 0xffff0000u) * inv) |
         e4m3x2(__uint_as_float(b << 16) * inv, __uint_as_float(b & 0xffff0000u) * inv) << 16;
}
constexpr uint32_t BF16_INF = 0x7f80;

// Does slot `b` continue the block of slot `a`, which is one of the cache or none?
__device__ __forceinline__ bool follows(const KvAppend& p, int a, int b) {
  return (unsigned)a < (unsigned)p.limit && a >> p.block_log == b >> p.block_log && a < b;
}

// A run is a stretch of neighbouring tokens and slots inside one block.  A warp takes the runs that begin in a window of `window`
// tokens, for one head of K or V: D / 8 lanes a token, 16 bytes each, so that a run of up to 32 tokens is read once and stays in
// registers between the maximum and the codes (longer ones are read again, from the caches).  What continues a run in the same
// block, behind skipped tokens or skipped slots, is done by the same warp: the scale belongs to all of them.  One pass over the
// input at the copy rate is the bound; windows of eight tokens spread a decode step over the GPU, windows of 32 keep warps with
// nothing to do few.  26k tokens of 24 prompts, 8 heads of 128 (166 MB): 39 us, 4.3 TB/s; a warp has one run, whose loads, maximum
// and stores follow one another, and 16 warps fit an SM beside the 64 registers that hold a run.  64 single tokens, 5 heads of 64:
// 2.6 us.
template <int D>
__global__ void __launch_bounds__(128) kv_append_kernel(const KvAppend p) {
  constexpr int LANES = D / 8, TOKENS = 32 / LANES, HELD = 32 / TOKENS;
  const int lane = threadIdx.x & 31, sub = lane / LANES, d = lane % LANES * 8;
  const long long w0 = ((long long)blockIdx.x * 4 + (threadIdx.x >> 5)) * p.window;
  if (w0 >= p.tokens) return;
  const int h = blockIdx.y % p.heads, which = blockIdx.y / p.heads, vec = which ? p.v_vec : p.k_vec;
  const long long step = which ? p.v_token : p.k_token;
  const __nv_bfloat16* input = (const __nv_bfloat16*)(which ? p.v : p.k) + (long long)h * (which ? p.v_head : p.k_head) + d;
  // where runs begin
  const bool mine = lane < p.window && w0 + lane < p.tokens;
  const int my_slot = mine ? p.slots[w0 + lane] : -1;
  const bool valid = (unsigned)my_slot < (unsigned)p.limit;
  int prev = __shfl_up_sync(0xffffffffu, my_slot, 1);
  if (lane == 0) prev = w0 > 0 ? p.slots[w0 - 1] : -1;
  const bool inside = valid && (my_slot & ((1 << p.block_log) - 1)) != 0;
  bool start = valid && !(inside && follows(p, prev, my_slot));
  unsigned ask = __ballot_sync(0xffffffffu, start && inside && (unsigned)prev >= (unsigned)p.limit);
  while (ask) {                        // behind skipped tokens: does the last one that counts precede this one?
    const int j = __ffs(ask) - 1;
    ask &= ask - 1;
    const long long before = valid_before(p, w0 + j);
    const int last = before >= 0 ? p.slots[before] : -1;
    if (lane == j && follows(p, last, my_slot)) start = false;
  }
  unsigned runs = __ballot_sync(0xffffffffu, start);
  // Runs of one token, as in a decode step: several at a time, so that their loads go out together.  One that has to move earlier
  // codes or holds what is not finite is left to the loop below.
  int next = __shfl_down_sync(0xffffffffu, my_slot, 1);
  const long long behind = w0 + lane + 1;
  const bool more = behind < p.tokens;
  if (lane == 31 || lane + 1 >= p.window) next = more ? p.slots[behind] : -1;
  const bool room = ((my_slot + 1) & ((1 << p.block_log) - 1)) != 0;
  const unsigned single = __ballot_sync(0xffffffffu, start && !(room && more && (follows(p, my_slot, next) || (unsigned)next >= (unsigned)p.limit)));
  if (__popc(single) > 1) {
    constexpr int TURNS = 8 / TOKENS;
    for (int i0 = 0; i0 < p.window; i0 += 8) {
      uint4 x[TURNS];
      float old[TURNS];
      int slot[TURNS];
#pragma unroll
      for (int u = 0; u < TURNS; ++u) {
        const int j = i0 + u * TOKENS + sub;
        slot[u] = __shfl_sync(0xffffffffu, my_slot, j & 31);
        x[u] = make_uint4(0, 0, 0, 0);
        old[u] = 0.f;
        if (!((single >> (j & 31)) & 1u) || j >= p.window) {
          slot[u] = -1;
        } else {
          x[u] = eight(input + (w0 + j) * step, vec);
          if (slot[u] & ((1 << p.block_log) - 1)) old[u] = p.scale[((long long)which * p.blocks + (slot[u] >> p.block_log)) * p.heads + h];
        }
      }
#pragma unroll
      for (int u = 0; u < TURNS; ++u) {
        uint32_t top = abs_max(0, x[u]);
        top = max(top & 0xffffu, top >> 16);
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        const bool first = (slot[u] & ((1 << p.block_log) - 1)) == 0;
        const float now = fmaxf(old[u], scale_for(__uint_as_float(top << 16)));
        const bool done = slot[u] >= 0 && top < BF16_INF && (first || now == old[u]);
        if (done) {
          const long long bh = ((long long)which * p.blocks + (slot[u] >> p.block_log)) * p.heads + h;
          const float inv = inv_pow2(now);
          uint8_t* to = p.codes + (long long)which * p.kv_stride + ((((long long)(slot[u] >> p.block_log)) * p.heads + h) << p.block_log) * D +
                        (slot[u] & ((1 << p.block_log) - 1)) * D + d;
          *reinterpret_cast<uint2*>(to) = make_uint2(codes4(x[u].x, x[u].y, inv), codes4(x[u].z, x[u].w, inv));
          if (first && d == 0) p.scale[bh] = now;
        }
        // one lane of each token speaks for it
        const unsigned said = __ballot_sync(0xffffffffu, done && lane % LANES == 0);
#pragma unroll
        for (int k = 0; k < TOKENS; ++k)
          if ((said >> (k * LANES)) & 1u) runs &= ~(1u << ((i0 + u * TOKENS + k) & 31));
      }
    }
  }
  while (runs) {
    const int j = __ffs(runs) - 1;
    runs &= runs - 1;
    long long t0 = w0 + j;
    int slot = __shfl_sync(0xffffffffu, my_slot, j);
    const int id = slot >> p.block_log;
    int off = slot - (id << p.block_log);
    const long long bh = ((long long)which * p.blocks + id) * p.heads + h;
    uint8_t* codes = p.codes + (long long)which * p.kv_stride + (((long long)id * p.heads + h) << p.block_log) * D;
    float old = off > 0 ? p.scale[bh] : 0.f;
    for (;;) {
      int n = 0;
      for (;;) {                       // length
        const int i = n + lane;
        const bool on = off + i < (1 << p.block_log) && t0 + i < p.tokens && p.slots[t0 + i] == slot + i;
        const unsigned same = __ballot_sync(0xffffffffu, on);
        n += same == 0xffffffffu ? 32 : __ffs(~same) - 1;
        if (same != 0xffffffffu) break;
      }
      const __nv_bfloat16* x = input + t0 * step;
      uint4 held[HELD];
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < HELD; ++i) {
        const int tok = i * TOKENS + sub;
        held[i] = tok < n ? eight(x + tok * step, vec) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < HELD; ++i) top = abs_max(top, held[i]);
      for (int tok = 32 + sub; tok < n; tok += TOKENS) top = abs_max(top, eight(x + tok * step, vec));
      uint32_t most = __reduce_max_sync(0xffffffffu, max(top & 0xffffu, top >> 16));
      const bool odd = most >= BF16_INF;       // something is not finite: the maximum over what is, element by element
      if (odd) {
        most = 0;
        for (int tok = sub; tok < n; tok += TOKENS)
          for (int e = 0; e < 8; ++e) {
            const uint32_t v = reinterpret_cast<const unsigned short*>(x + tok * step)[e] & 0x7fffu;
            if (v < BF16_INF) most = max(most, v);
          }
        most = __reduce_max_sync(0xffffffffu, most);
      }
      const float now = fmaxf(old, scale_for(__uint_as_float(most << 16)));
      if (off > 0 && now != old) {     // the codes of earlier tokens go to the new scale
        const float r = old * inv_pow2(now);
        for (int i = lane; i < off * D / 4; i += 32) {
          const uint32_t c = reinterpret_cast<const uint32_t*>(codes)[i];
          uint32_t m = 0;
#pragma unroll
          for (int b = 0; b < 32; b += 8) m |= code_of(value_of((c >> b) & 0xffu) * r) << b;
          reinterpret_cast<uint32_t*>(codes)[i] = m;
        }
      }
      const float inv = inv_pow2(now);
      uint8_t* to = codes + off * D + d;
      if (odd) {
        for (int tok = sub; tok < n; tok += TOKENS)
          for (int e = 0; e < 8; ++e) to[tok * D + e] = (uint8_t)code_of(__bfloat162float(x[tok * step + e]) * inv);
      } else {
#pragma unroll
        for (int i = 0; i < HELD; ++i) {
          const int tok = i * TOKENS + sub;
          if (tok < n) *reinterpret_cast<uint2*>(to + tok * D) = make_uint2(codes4(held[i].x, held[i].y, inv), codes4(held[i].z, held[i].w, inv));
        }
        for (int tok = 32 + sub; tok < n; tok += TOKENS) {
          const uint4 w = eight(x + tok * step, vec);
          *reinterpret_cast<uint2*>(to + tok * D) = make_uint2(codes4(w.x, w.y, inv), codes4(w.z, w.w, inv));
        }
      }
      __syncwarp();
      old = now;
      slot += n - 1;                   // the run's last
      if (off + n == 1 << p.block_log) break;
      t0 = valid_from(p, t0 + n);
      if (t0 >= p.tokens || !follows(p, slot, p.slots[t0])) break;
      slot = p.slots[t0];
      off = slot - (id << p.block_log);
    }
    if (lane == 0) p.scale[bh] = old;
  }
}

// ------------------------------------------------------------------------------------------------ reorder
// A block per row and four planes (a plane: one layer's keys or values): what a row copies is found out once for them, and their
// loads go out together.  The table is the first plane's business.  384 rows with up to 63 tokens in their last block, 16 layers of 5
// heads of 64 (112 MB copied): 43 us, 5.1 TB/s read and written (one plane a block: 47); one search of 4 beams, 6 layers: 3.6 us.
constexpr int PLANES = 4;
__global__ void __launch_bounds__(128) kv_reorder_kernel(const KvReorder p) {
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
  // The copied places of a head lie together (fill * dim bytes); over the heads they are a head's whole size apart.
  const long long page = (long long)p.heads * p.block * p.dim;
  const int head16 = p.block * p.dim / 16, fill16 = fill * p.dim / 16, n = p.heads * fill16;
  const int last = min(p.planes, (int)(blockIdx.y + 1) * PLANES);
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int h = i / fill16;
    const long long o = (long long)h * head16 + (i - h * fill16);
    uint4 v[PLANES];
#pragma unroll
    for (int k = 0; k < PLANES; ++k) {
      const int plane = blockIdx.y * PLANES + k;
      if (plane < last) v[k] = __ldcs(reinterpret_cast<const uint4*>(p.codes + plane * p.plane + from * page) + o);
    }
#pragma unroll
    for (int k = 0; k < PLANES; ++k) {
      const int plane = blockIdx.y * PLANES + k;
      if (plane < last) __stcs(reinterpret_cast<uint4*>(p.codes + plane * p.plane + to * page) + o, v[k]);
    }
  }
  for (int i = threadIdx.x; i < p.heads * PLANES; i += blockDim.x) {
    const int plane = blockIdx.y * PLANES + i / p.heads, h = i % p.heads;
    if (plane < last) {
      float* sc = p.scale + (long long)plane * p.blocks * p.heads + h;
      sc[(long long)to * p.heads] = sc[(long long)from * p.heads];
    }
  }
}

}  // namespace

extern "C" {

// Block tables and slot maps.  rows <= 8192; `tables` int32 [rows, width] is completed in place; a row holds at most `limit` tokens,
// width * block at most; ids of `blocks` (blocks * block <= 2^31) and more get no slot and are reported; `free_count_out` may be
// `free_count`; `own`: one word of work space.
int nb_kv_plan(const int* lengths, const int* new_lens, int* tables, const int* free_ids, const int* free_count, int* free_count_out,
               int* starts, int* ends, int* row_of, int* positions, int* slots, int* own, int rows, int width, int block, int free_size,
               int tokens, int blocks, int limit, unsigned int* status, void* stream) {
  if (rows <= 0 || rows > 8192 || width <= 0 || block <= 0 || tokens < 0 || free_size < 0) return NB_ERR_BAD_ARG;
  if ((block & (block - 1)) || (long long)width * block > 0x7fffff00LL || tokens > 0x7fffff00 || limit < 0 || limit > (long long)width * block || blocks <= 0 || (long long)blocks * block > 1LL << 31) return NB_ERR_BAD_ARG;
  const int grid = max(1, min(148 * 4, ceil_div(tokens, 256)));
  // every block reads the count when it begins, so only a single block may write it back in place
  const bool later = grid > 1 && free_count == free_count_out;
  KvPlan p{lengths, new_lens, tables, free_ids, free_count, later ? own : free_count_out, starts, ends, row_of, positions, slots, rows, width, 0, free_size, tokens, blocks, limit, status};
  while ((1 << p.block_log) < block) ++p.block_log;
  static bool configured[64] = {};
  int dev = 0;
  NB_CUDA(cudaGetDevice(&dev));
  if (dev >= 64) return NB_ERR_BAD_ARG;
  if (!configured[dev]) {
    NB_CUDA(cudaFuncSetAttribute(kv_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 3 * (8192 + 256 + 1) * 4));
    configured[dev] = true;
  }
  kv_plan_kernel<<<grid, 256, 3 * (spread(rows) + 1) * 4, (cudaStream_t)stream>>>(p);
  NB_LAUNCH_CHECK();
  if (later) NB_CUDA(cudaMemcpyAsync(free_count_out, own, 4, cudaMemcpyDeviceToDevice, (cudaStream_t)stream));
  return NB_OK;
}

int nb_kv_append(const void* k, const void* v, void* codes, float* scale, const int* slots, int tokens, int heads, int dim, int block,
                 int blocks, long long k_token, long long k_head, long long v_token, long long v_head, long long kv_stride, void* stream) {
  if (tokens < 0 || heads <= 0 || heads > 32767 || (dim != 64 && dim != 128) || block < 16 || (block & (block - 1)) || blocks <= 0) return NB_ERR_BAD_ARG;
  if ((long long)blocks * block > 0x7fffffffLL) return NB_ERR_BAD_ARG;
  if ((reinterpret_cast<uintptr_t>(codes) & 15) || (kv_stride & 15)) return NB_ERR_UNALIGNED;
  if (tokens == 0) return NB_OK;
  KvAppend p{k, v, (uint8_t*)codes, scale, slots, tokens, heads, 0, blocks, blocks * block, 0, 0, 0, k_token, k_head, v_token, v_head, kv_stride};
  while ((1 << p.block_log) < block) ++p.block_log;
  p.k_vec = !((reinterpret_cast<uintptr_t>(k) & 15) || (k_token & 7) || (k_head & 7));
  p.v_vec = !((reinterpret_cast<uintptr_t>(v) & 15) || (v_token & 7) || (v_head & 7));
  p.window = tokens <= 1024 ? 8 : 32;   // 512 single tokens 3.6 us instead of 7.1; two prompts of 1024 6.5 instead of 8.0
  const dim3 grid(ceil_div(tokens, 4 * p.window), 2 * heads);
  if (dim == 64) kv_append_kernel<64><<<grid, 128, 0, (cudaStream_t)stream>>>(p);
  else kv_append_kernel<128><<<grid, 128, 0, (cudaStream_t)stream>>>(p);
  NB_LAUNCH_CHECK();
  return NB_OK;
}

int nb_kv_reorder(void* codes, float* scale, const int* tables, const int* lengths, const int* parents, const int* spare, int* tables_out,
                  int* lengths_out, int* spare_out, int planes, int blocks, int heads, int block, int dim, int rows, int beams, int width,
                  unsigned int* status, void* stream) {
  if (planes <= 0 || planes > 65535 || blocks <= 0 || heads <= 0 || block <= 0 || dim % 16 || rows <= 0 || beams <= 0 || rows % beams || width <= 0) return NB_ERR_BAD_ARG;
  if (reinterpret_cast<uintptr_t>(codes) & 15) return NB_ERR_UNALIGNED;
  KvReorder p{(uint8_t*)codes, scale, tables, lengths, parents, spare, tables_out, lengths_out, spare_out, blocks, heads, block, dim, rows, beams, width, planes,
              (long long)blocks * heads * block * dim, status};
  kv_reorder_kernel<<<dim3(rows, ceil_div(planes, PLANES)), 128, 0, (cudaStream_t)stream>>>(p);
  NB_LAUNCH_CHECK();
  return NB_OK;
}

}  // extern "C"
