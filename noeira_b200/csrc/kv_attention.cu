// Attention of new tokens over the paged 8-bit cache: o = softmax(c q K^T) V over the keys up to each token's own position.
//
// Few query rows per row of the batch (decode steps, short chunks).  The work is bound by the bytes of the cache: 2 D bytes per
// key and head at the copy rate, against 2 D operations per byte and query row.  So the cache is read once, straight from global
// memory into the registers of the matrix instructions, and nothing else is in the way:
//   * A tile has 16 query rows: all query heads of one cache head, of as many tokens as fit.  S = Q K^T and O += P V are
//     m16n8k16 products in f16 with fp32 sums.  e4m3 codes are exact in f16; q (bf16) is exact in f16 down to 2^-38 of the row's
//     largest element after a power-of-two scaling of the row; P keeps 11 bits.
//   * A lane's fragment of K is 16 consecutive bytes of a key (the order of the contraction is free as long as q has the same),
//     its fragment of V is D / 8 consecutive bytes of four keys (the order of the output columns is free).  No shared memory, no
//     transposition; every sector that is fetched is used.
//   * The key range of the whole batch is cut into equal pieces, one for each resident block (rows differ in length, so pieces
//     run over the ends of rows), and a second, small kernel joins rows that lie in several pieces.  The four warps of a block
//     take turns at steps of 4 KB and join in shared memory.
#include "common.cuh"
#include "kv_cache.h"

namespace {
using namespace nb;

constexpr int WARPS = 4, THREADS = 32 * WARPS;
constexpr int CHUNK = 32;              // steps of a piece when the batch does not fill the GPU: at most eight per warp, no joining up to 1024 (512) keys
constexpr float RAISE = 8.f;           // the running maximum is raised when it falls behind by more than 2^8 ...
constexpr float LIFT = 7.f;            // ... and weights are at most 2^(8 + 7), below f16's largest, so that small ones stay normal

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t f16_of_codes(uint32_t two) {   // two e4m3 codes (bits 0..15) as f16 pair
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)two));
  return r;
}
__device__ __forceinline__ uint32_t f16_pair(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// the largest of a row / the sum of a row over the four lanes that hold it
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}
__device__ __forceinline__ uint32_t nan_code(uint32_t w) {         // nonzero where one of four codes is NaN
  const uint32_t m = w & 0x7f7f7f7fu;
  return (m + 0x01010101u) & 0x80808080u;
}

// ---------------------------------------------------------------- how the batch is cut
// Row i costs q-tiles x heads x steps; `upto` (shared memory, rows + 1) are the exclusive sums.  `piece` is what a block takes.
struct Cut {
  long long total, piece;
  int pad;                             // steps of a (q-tile, head) are rounded up to a multiple of this
};
struct Job {
  int row, head, qt, steps;            // steps: rounded
  long long begin;                     // its first step
};

template <int KEYS>
__device__ __forceinline__ int row_steps(const KvAttn& p, int i) { return ceil_div(max(0, min(p.ends[i], p.width << p.block_log)), KEYS); }
__device__ __forceinline__ int row_tiles(const KvAttn& p, int i) {
  const int first = p.starts[i];
  const long long n = first < 0 ? 0 : (long long)min(p.starts[i + 1], p.tokens) - first;
  // rows with more query rows than `few` belong to the kernel of prompts
  return n <= 0 || n * p.group > p.few ? 0 : (int)((n * p.group + 15) / 16);
}
// A row without keys still gets its zeros written: one step.
template <int KEYS>
__device__ __forceinline__ Cut cut_batch(const KvAttn& p, long long* upto, long long* sh) {
  const int tid = threadIdx.x, per = ceil_div(p.rows, THREADS);
  const int lo = min(p.rows, tid * per), hi = min(p.rows, lo + per);
  long long a = 0, b = 0;
  for (int i = lo; i < hi; ++i) {
    const long long jobs = (long long)row_tiles(p, i) * p.hk;
    const int n = max(1, row_steps<KEYS>(p, i));
    a += jobs * n;
    b += jobs * ceil_div(n, CHUNK);
  }
  // sums over the block of both, and what lies before this thread
  long long ia = a, ib = b;
  const int lane = tid & 31, w = tid >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, ia, o), v = __shfl_up_sync(0xffffffffu, ib, o);
    if (lane >= o) { ia += u; ib += v; }
  }
  __syncthreads();
  if (lane == 31) { sh[w] = ia; sh[WARPS + w] = ib; }
  __syncthreads();
  long long ta = 0, tb = 0;
  for (int i = 0; i < WARPS; ++i) {
    if (i < w) { ia += sh[i]; ib += sh[WARPS + i]; }
    ta += sh[i];
    tb += sh[WARPS + i];
  }
  Cut c;
  const bool small = tb <= p.pieces;   // every (q-tile, head) in pieces of its own, none shared with the next
  c.pad = small ? CHUNK : 1;
  c.total = small ? tb * CHUNK : ta;
  c.piece = small ? CHUNK : max(1LL, (ta + p.pieces - 1) / p.pieces);
  long long at = small ? (ib - b) * CHUNK : ia - a;
  for (int i = lo; i < hi; ++i) {
    upto[i] = at;
    const int n = max(1, row_steps<KEYS>(p, i));
    at += (long long)row_tiles(p, i) * p.hk * (small ? ceil_div(n, CHUNK) * CHUNK : n);
  }
  if (tid == 0) upto[p.rows] = c.total;
  __syncthreads();
  return c;
}
template <int KEYS>
__device__ __forceinline__ Job job_at(const KvAttn& p, const Cut& c, const long long* upto, long long x) {
  int a = 0, b = p.rows;               // last row that begins at or before x (rows without work share their begin with the next)
  while (b - a > 1) {
    const int m = (a + b) >> 1;
    if (upto[m] <= x) a = m; else b = m;
  }
  Job j;
  j.row = a;
  j.steps = ceil_div(max(1, row_steps<KEYS>(p, a)), c.pad) * c.pad;
  const long long n = (x - upto[a]) / j.steps;
  j.head = (int)(n % p.hk);
  j.qt = (int)(n / p.hk);
  j.begin = upto[a] + n * j.steps;
  return j;
}

// ---------------------------------------------------------------- the step
template <int D>
struct Raw {                           // one step of a warp: 4 KB of codes
  static constexpr int SUB = 128 / D;  // sub-tiles of 16 keys
  static constexpr int KEYS = 16 * SUB;
  uint4 k[SUB][2][D / 64];             // [sub][n-block of 8 keys][64 dimensions]
  uint32_t v[SUB][4][D / 32];          // [sub][key 2c, 2c+1, 2c+8, 2c+9][bytes of dimensions (lane / 4) D / 8 ...]
  float ks[SUB], vs[SUB];
  bool has[SUB];                       // false: no keys there (past the end, or a bad block)
};

template <int D>
__device__ __forceinline__ void load_ids(const KvAttn& p, const int* table, int step, int limit, int (&id)[Raw<D>::SUB]) {
#pragma unroll
  for (int s = 0; s < Raw<D>::SUB; ++s) {
    const int k0 = step * Raw<D>::KEYS + s * 16;
    id[s] = k0 < limit ? table[k0 >> p.block_log] : -2;
  }
}
template <int D>
__device__ __forceinline__ void load_raw(const KvAttn& p, int row, int head, int step, const int (&id)[Raw<D>::SUB], Raw<D>& r) {
  const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
#pragma unroll
  for (int s = 0; s < Raw<D>::SUB; ++s) {
    r.ks[s] = 0.f;
    r.vs[s] = 0.f;
    r.has[s] = (unsigned)id[s] < (unsigned)p.blocks;
    if (!r.has[s]) {
      if (id[s] != -2 && lane == 0) report(p.status, NB_ST_BOUNDS, 10, row);
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int u = 0; u < D / 64; ++u) r.k[s][n][u] = make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int u = 0; u < D / 32; ++u) r.v[s][k][u] = 0;
      continue;
    }
    const long long page = (long long)id[s] * p.hk + head;
    const int in = (step * Raw<D>::KEYS + s * 16) & ((1 << p.block_log) - 1);
    const uint8_t* base = p.codes + ((page << p.block_log) + in) * D;
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int u = 0; u < D / 64; ++u) r.k[s][n][u] = __ldg(reinterpret_cast<const uint4*>(base + (n * 8 + g) * D + u * 64 + c * 16));
    const uint8_t* vb = base + p.kv_stride;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint8_t* a = vb + (2 * c + (k & 1) + (k >> 1) * 8) * D + g * (D / 8);
      if (D == 64) {
        const uint2 w = __ldg(reinterpret_cast<const uint2*>(a));
        r.v[s][k][0] = w.x;
        r.v[s][k][1] = w.y;
      } else {
        const uint4 w = __ldg(reinterpret_cast<const uint4*>(a));
        r.v[s][k][0] = w.x;
        r.v[s][k][1] = w.y;
        r.v[s][k][D / 32 - 2] = w.z;
        r.v[s][k][D / 32 - 1] = w.w;
      }
    }
    r.ks[s] = __ldg(p.scale + page);
    r.vs[s] = __ldg(p.scale + p.s_stride + page);
  }
}

template <int D>
struct Tile {                          // what a warp keeps of a tile of 16 query rows
  uint32_t q[D / 16][4];
  float o[D / 8][4];                   // in units of vref
  float m[2], l[2], f[2];              // rows g and g + 8: maximum (log2), this lane's sum, factor of a raw score
  int lim[2];                          // keys that the row sees
  float vref;
};

template <int D>
__device__ __forceinline__ void load_q(const KvAttn& p, int first, int count, int head, int end, int new_tokens, int qt, Tile<D>& t) {
  const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int idx = qt * 16 + r * 8 + g, tok = idx / p.group;
    const bool real = tok < count;
    t.lim[r] = real ? max(0, min(end, end - new_tokens + tok + 1)) : 0;
    t.m[r] = -INFINITY;
    t.l[r] = 0.f;
    float x[D / 4], top = 0.f;
    const __nv_bfloat16* q = (const __nv_bfloat16*)p.q + (long long)(first + tok) * p.q_token + (long long)(head * p.group + idx - tok * p.group) * p.q_head;
#pragma unroll
    for (int u = 0; u < D / 64; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint4 w = make_uint4(0, 0, 0, 0);
        const __nv_bfloat16* a = q + u * 64 + c * 16 + h * 8;
        if (real) {
          if (p.q_vec) {
            w = *reinterpret_cast<const uint4*>(a);
          } else {
            const unsigned short* b = reinterpret_cast<const unsigned short*>(a);
            w = make_uint4(b[0] | (uint32_t)b[1] << 16, b[2] | (uint32_t)b[3] << 16, b[4] | (uint32_t)b[5] << 16, b[6] | (uint32_t)b[7] << 16);
          }
        }
        const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[u * 16 + h * 8 + 2 * i] = __uint_as_float(ww[i] << 16);
          x[u * 16 + h * 8 + 2 * i + 1] = __uint_as_float(ww[i] & 0xffff0000u);
        }
      }
#pragma unroll
    for (int i = 0; i < D / 4; ++i) top = fmaxf(top, fabsf(x[i]));
    top = quad_max(top);
    // power of two that takes the largest element to [2^14, 2^15); the row's scores are scaled back by its inverse
    int e = (int)(__float_as_uint(top) >> 23) - 127;
    e = top > 0.f && e < 128 ? max(-100, min(112, e - 14)) : 0;
    const float s = __uint_as_float((uint32_t)(127 - e) << 23);
    t.f[r] = p.scale_log2 * __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
    for (int u = 0; u < D / 64; ++u)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        t.q[u * 4 + k][r] = f16_pair(x[u * 16 + k * 4] * s, x[u * 16 + k * 4 + 1] * s);
        t.q[u * 4 + k][2 + r] = f16_pair(x[u * 16 + k * 4 + 2] * s, x[u * 16 + k * 4 + 3] * s);
      }
  }
#pragma unroll
  for (int j = 0; j < D / 8; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) t.o[j][i] = 0.f;
  t.vref = 0.f;
}

// P V of one sub-tile: acc += P (16 x 16) V (16 x D)
template <int D>
__device__ __forceinline__ void times_v(float (&acc)[D / 8][4], const uint32_t (&pa)[4], const uint32_t (&v)[4][D / 32]) {
#pragma unroll
  for (int w = 0; w < D / 32; ++w) {
    // bytes of keys (2c, 2c + 1) and (2c + 8, 2c + 9) side by side: two dimensions per word
    const uint32_t a0 = __byte_perm(v[0][w], v[1][w], 0x5140), a1 = __byte_perm(v[0][w], v[1][w], 0x7362);
    const uint32_t b0 = __byte_perm(v[2][w], v[3][w], 0x5140), b1 = __byte_perm(v[2][w], v[3][w], 0x7362);
    mma(acc[w * 4 + 0], pa, f16_of_codes(a0), f16_of_codes(b0));
    mma(acc[w * 4 + 1], pa, f16_of_codes(a0 >> 16), f16_of_codes(b0 >> 16));
    mma(acc[w * 4 + 2], pa, f16_of_codes(a1), f16_of_codes(b1));
    mma(acc[w * 4 + 3], pa, f16_of_codes(a1 >> 16), f16_of_codes(b1 >> 16));
  }
}

// `seen`: the most keys that a row of the tile sees, `sure`: the fewest that a real row sees.
template <int D>
__device__ __forceinline__ void step_tile(const KvAttn& p, Tile<D>& t, Raw<D>& r, int step, int seen, int sure) {
  constexpr int SUB = Raw<D>::SUB;
  const int lane = threadIdx.x & 31, c = lane & 3;
  float s[SUB][2][4];
#pragma unroll
  for (int u = 0; u < SUB; ++u)
#pragma unroll
    for (int n = 0; n < 2; ++n) {
#pragma unroll
      for (int i = 0; i < 4; ++i) s[u][n][i] = 0.f;
#pragma unroll
      for (int d = 0; d < D / 64; ++d) {
        const uint32_t w[4] = {r.k[u][n][d].x, r.k[u][n][d].y, r.k[u][n][d].z, r.k[u][n][d].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) mma(s[u][n], t.q[d * 4 + k], f16_of_codes(w[k]), f16_of_codes(w[k] >> 16));
      }
    }
  // scores in log2 units, masked; a NaN score stays NaN (the comparisons below let it through)
  const int k0 = step * Raw<D>::KEYS;
  const bool whole = k0 + Raw<D>::KEYS <= sure;
  float top[2] = {-INFINITY, -INFINITY}, vtop = t.vref;
  bool lacks = false;
#pragma unroll
  for (int u = 0; u < SUB; ++u) lacks |= !r.has[u];
#pragma unroll
  for (int u = 0; u < SUB; ++u) {
    const float f0 = t.f[0] * r.ks[u], f1 = t.f[1] * r.ks[u];
    vtop = fmaxf(vtop, r.vs[u]);
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[u][n][i] *= i < 2 ? f0 : f1;
  }
  if (!whole || lacks) {
#pragma unroll
    for (int u = 0; u < SUB; ++u)
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (k0 + u * 16 + n * 8 + 2 * c + (i & 1) >= t.lim[i >> 1] || !r.has[u]) s[u][n][i] = -INFINITY;
    // values behind the last key that any row sees are not numbers to be multiplied by zero
#pragma unroll
    for (int u = 0; u < SUB; ++u)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (k0 + u * 16 + 2 * c + (k & 1) + (k >> 1) * 8 >= seen) {
#pragma unroll
          for (int w = 0; w < D / 32; ++w) r.v[u][k][w] = 0;
        }
  }
#pragma unroll
  for (int u = 0; u < SUB; ++u)
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      top[0] = fmaxf(top[0], fmaxf(s[u][n][0], s[u][n][1]));
      top[1] = fmaxf(top[1], fmaxf(s[u][n][2], s[u][n][3]));
    }
  top[0] = quad_max(top[0]);
  top[1] = quad_max(top[1]);
  const bool raise0 = top[0] > t.m[0] + RAISE || (t.m[0] == -INFINITY && top[0] > -INFINITY);
  const bool raise1 = top[1] > t.m[1] + RAISE || (t.m[1] == -INFINITY && top[1] > -INFINITY);
  if (__any_sync(0xffffffffu, raise0 || raise1) || vtop > t.vref) {
    const float v = t.vref > 0.f ? t.vref / vtop : 0.f;
    float a[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const bool raise = i ? raise1 : raise0;
      a[i] = raise ? ex2(t.m[i] - top[i]) : 1.f;
      if (raise) t.m[i] = top[i];
      t.l[i] *= a[i];
      a[i] *= v;
    }
    t.vref = vtop;
#pragma unroll
    for (int j = 0; j < D / 8; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) t.o[j][i] *= a[i >> 1];
  }
  const float b0 = (t.m[0] == -INFINITY ? 0.f : t.m[0]) - LIFT, b1 = (t.m[1] == -INFINITY ? 0.f : t.m[1]) - LIFT;
#pragma unroll
  for (int u = 0; u < SUB; ++u) {
    if (!r.has[u]) continue;
    // Weights relative to vref; a block whose values are less than 2^-24 of the largest block's would lose bits in f16, so
    // its product is taken by itself and added in fp32.
    const float ratio = t.vref > 0.f ? r.vs[u] / t.vref : 0.f;
    const bool apart = ratio < 5.9604645e-8f;
    uint32_t pa[4];
    float sum0 = 0.f, sum1 = 0.f;
    const float w = apart ? 1.f : ratio;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      float e0 = ex2(s[u][n][0] - b0), e1 = ex2(s[u][n][1] - b0), e2 = ex2(s[u][n][2] - b1), e3 = ex2(s[u][n][3] - b1);
      sum0 += e0 + e1;
      sum1 += e2 + e3;
      pa[2 * n] = f16_pair(e0 * w, e1 * w);
      pa[2 * n + 1] = f16_pair(e2 * w, e3 * w);
    }
    t.l[0] += sum0;
    t.l[1] += sum1;
    if (!whole) {
      // Rows that do not see a key that others see would multiply its value by zero; NaN there is taken out, and put into the
      // rows that do see it.
      uint32_t any = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int x = 0; x < D / 32; ++x) any |= nan_code(r.v[u][k][x]);
      if (__any_sync(0xffffffffu, any != 0)) {
        const int key = k0 + u * 16;
        for (int k = 0; k < 16 && key + k < seen; ++k)
          for (int x = 0; x < D / 32; ++x) {
            // lane (g = column group, c = keys) that holds key k: its word x carries dimensions g D / 8 + 4 x ..
            const int holder = (k & 7) >> 1, reg = (k & 1) + (k >> 3) * 2;
            uint32_t word = 0;
#pragma unroll
            for (int rr = 0; rr < 4; ++rr)
#pragma unroll
              for (int xx = 0; xx < D / 32; ++xx)
                if (rr == reg && xx == x) word = r.v[u][rr][xx];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              // this lane's output columns 2c + e of every n-block: dimensions (2c + e) D / 8 + j
              const uint32_t got = __shfl_sync(0xffffffffu, word, (2 * c + e) * 4 + holder);
#pragma unroll
              for (int j = 0; j < D / 8; ++j)
                if (j / 4 == x && ((got >> (8 * (j & 3))) & 0x7fu) == 0x7fu) {
                  if (key + k < t.lim[0]) t.o[j][e] = __int_as_float(0x7fffffff);
                  if (key + k < t.lim[1]) t.o[j][2 + e] = __int_as_float(0x7fffffff);
                }
            }
          }
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int x = 0; x < D / 32; ++x) {
            const uint32_t hit = nan_code(r.v[u][k][x]) >> 7;     // 1 in the byte of a NaN
            r.v[u][k][x] &= ~(hit * 0xffu);
          }
      }
    }
    if (!apart) {
      times_v<D>(t.o, pa, r.v[u]);
    } else {
      float acc[D / 8][4];
#pragma unroll
      for (int j = 0; j < D / 8; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[j][i] = 0.f;
      times_v<D>(acc, pa, r.v[u]);
#pragma unroll
      for (int j = 0; j < D / 8; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) t.o[j][i] += acc[j][i] * ratio;
    }
  }
}

template <int D>
__device__ __forceinline__ void store_out(const KvAttn& p, int first, int head, int idx, int d, float a, float b, float c, float e) {
  const int tok = idx / p.group;
  __nv_bfloat16* o = (__nv_bfloat16*)p.out + (long long)(first + tok) * p.o_token + (long long)(head * p.group + idx - tok * p.group) * p.o_head + d;
  const __nv_bfloat162 x = __floats2bfloat162_rn(a, b), y = __floats2bfloat162_rn(c, e);
  if (p.o_vec) {
    *reinterpret_cast<uint2*>(o) = make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
  } else {
    o[0] = x.x;
    o[1] = x.y;
    o[2] = y.x;
    o[3] = y.y;
  }
}

// Partial results of a block: slot 1 for the job that begins in its piece and runs on, slot 0 for the one that came from before.
template <int D>
__device__ __forceinline__ long long slot_at(long long piece, int slot) { return (piece * 2 + slot) * 16; }

template <int D>
__global__ void __launch_bounds__(THREADS, D == 64 ? 3 : 2) kv_attn_kernel(KvAttn p) {
  constexpr int KEYS = Raw<D>::KEYS;
  extern __shared__ __align__(16) uint8_t smem[];
  float* s_o = reinterpret_cast<float*>(smem);                    // [WARPS][16][D]
  float* s_m = s_o + WARPS * 16 * D;                              // [WARPS][16] maximum, then [WARPS][16] sum
  long long* sh = reinterpret_cast<long long*>(s_m + 2 * WARPS * 16);
  long long* upto = sh + 2 * WARPS;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const Cut cut = cut_batch<KEYS>(p, upto, sh);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  long long x = (long long)blockIdx.x * cut.piece;
  const long long x1 = min(cut.total, x + cut.piece);
  while (x < x1) {
    const Job j = job_at<KEYS>(p, cut, upto, x);
    const long long stop = min(x1, j.begin + j.steps);
    const int from = (int)(x - j.begin);
    const bool alone = from == 0 && stop == j.begin + j.steps;
    const int first = p.starts[j.row], new_tokens = p.starts[j.row + 1] - first, count = min(p.starts[j.row + 1], p.tokens) - first;
    const int end = max(0, min(p.ends[j.row], p.width << p.block_log));
    Tile<D> t;
    load_q<D>(p, first, count, j.head, end, new_tokens, j.qt, t);
    const int rows16 = min(16, count * p.group - j.qt * 16);       // real rows of the tile
    const int tok0 = j.qt * 16 / p.group, tok1 = (j.qt * 16 + rows16 - 1) / p.group;
    const int sure = max(0, min(end, end - new_tokens + tok0 + 1)), seen = max(0, min(end, end - new_tokens + tok1 + 1));
    const int last = min(from + (int)(stop - x), ceil_div(seen, KEYS));
    // three stages: block ids two steps ahead, codes one step ahead
    const int* table = p.tables + (long long)j.row * p.width;
    int id[Raw<D>::SUB];
    Raw<D> r[2];
    int st = from + warp;
    if (st < last) {
      load_ids<D>(p, table, st, seen, id);
      load_raw<D>(p, j.row, j.head, st, id, r[0]);
      if (st + WARPS < last) load_ids<D>(p, table, st + WARPS, seen, id);
    }
    while (st < last) {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        if (st >= last) break;
        if (st + WARPS < last) {
          load_raw<D>(p, j.row, j.head, st + WARPS, id, r[b ^ 1]);
          if (st + 2 * WARPS < last) load_ids<D>(p, table, st + 2 * WARPS, seen, id);
        }
        step_tile<D>(p, t, r[b], st, seen, sure);
        st += WARPS;
      }
    }
    // join the warps: sums relative to the largest maximum
    t.l[0] = quad_sum(t.l[0]);
    t.l[1] = quad_sum(t.l[1]);
    __syncthreads();
    if (c == 0) {
      s_m[warp * 16 + g] = t.m[0];
      s_m[warp * 16 + g + 8] = t.m[1];
      s_m[(WARPS + warp) * 16 + g] = t.l[0];
      s_m[(WARPS + warp) * 16 + g + 8] = t.l[1];
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = g + 8 * h;
      if (row >= rows16) continue;
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) top = fmaxf(top, s_m[w * 16 + row]);
      const float f = t.m[h] == -INFINITY ? (t.l[h] == 0.f ? 0.f : 1.f) * t.vref : ex2(t.m[h] - top) * t.vref;
      float* o = s_o + (warp * 16 + row) * D;
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int k = 0; k < D / 8; k += 4)
          *reinterpret_cast<float4*>(o + (2 * c + e) * (D / 8) + k) =
              make_float4(t.o[k][2 * h + e] * f, t.o[k + 1][2 * h + e] * f, t.o[k + 2][2 * h + e] * f, t.o[k + 3][2 * h + e] * f);
    }
    __syncthreads();
    const long long slot = slot_at<D>(blockIdx.x, from == 0 ? 1 : 0);
    for (int i = threadIdx.x; i < rows16 * (D / 4); i += THREADS) {
      const int row = i / (D / 4), d = i % (D / 4) * 4;
      float top = -INFINITY, l = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) top = fmaxf(top, s_m[w * 16 + row]);
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float m = s_m[w * 16 + row], lw = s_m[(WARPS + w) * 16 + row];
        l += m == -INFINITY ? lw : lw * ex2(m - top);              // without a maximum the sum is zero, or NaN
        const float4 v = *reinterpret_cast<const float4*>(s_o + (w * 16 + row) * D + d);
        o.x += v.x;
        o.y += v.y;
        o.z += v.z;
        o.w += v.w;
      }
      if (alone) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        store_out<D>(p, first, j.head, j.qt * 16 + row, d, o.x * inv, o.y * inv, o.z * inv, o.w * inv);
      } else {
        *reinterpret_cast<float4*>(p.part_o + (slot + row) * D + d) = o;
        if (d == 0) *reinterpret_cast<float2*>(p.part_ml + (slot + row) * 2) = make_float2(top, l);
      }
    }
    x = stop;
  }
}

// Joins the job that begins in piece blockIdx.x and runs past its end.
template <int D>
__global__ void __launch_bounds__(THREADS) kv_attn_join_kernel(KvAttn p) {
  constexpr int KEYS = Raw<D>::KEYS;
  extern __shared__ __align__(16) uint8_t smem[];
  long long* sh = reinterpret_cast<long long*>(smem);
  long long* upto = sh + 2 * WARPS;
  const Cut cut = cut_batch<KEYS>(p, upto, sh);
  const long long lo = (long long)blockIdx.x * cut.piece, hi = lo + cut.piece;
  // every block waits, also one with nothing to join: what follows in the stream may start when this kernel is done
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (hi >= cut.total) return;
  const Job j = job_at<KEYS>(p, cut, upto, hi - 1);
  if (j.begin < lo || j.begin + j.steps <= hi) return;
  const long long last = (j.begin + j.steps - 1) / cut.piece;
  const int first = p.starts[j.row], count = min(p.starts[j.row + 1], p.tokens) - first;
  const int rows16 = min(16, count * p.group - j.qt * 16);
  for (int i = threadIdx.x; i < rows16 * (D / 4); i += THREADS) {
    const int row = i / (D / 4), d = i % (D / 4) * 4;
    float top = -INFINITY;
    for (long long w = blockIdx.x; w <= last; ++w) top = fmaxf(top, p.part_ml[(slot_at<D>(w, w == blockIdx.x) + row) * 2]);
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (long long w = blockIdx.x; w <= last; ++w) {
      const long long s = slot_at<D>(w, w == blockIdx.x) + row;
      const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + s * 2);
      const float f = ml.x == -INFINITY ? 1.f : ex2(ml.x - top);   // without a maximum all is zero, or NaN
      const float4 v = *reinterpret_cast<const float4*>(p.part_o + s * D + d);
      l += ml.y * f;
      o.x += v.x * f;
      o.y += v.y * f;
      o.z += v.z * f;
      o.w += v.w * f;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    store_out<D>(p, first, j.head, j.qt * 16 + row, d, o.x * inv, o.y * inv, o.z * inv, o.w * inv);
  }
}

template <int D>
int launch_few(KvAttn p, cudaStream_t stream) {
  const int scan = (2 * WARPS + p.rows + 1) * 8, smem = (WARPS * 16 * D + 2 * WARPS * 16) * 4 + scan;
  static bool configured[64] = {};
  int dev = 0;
  NB_CUDA(cudaGetDevice(&dev));
  if (dev >= 64) return NB_ERR_BAD_ARG;
  if (!configured[dev]) {
    NB_CUDA(cudaFuncSetAttribute(kv_attn_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024));
    NB_CUDA(cudaFuncSetAttribute(kv_attn_join_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, 100 * 1024));
    configured[dev] = true;
  }
  kv_attn_kernel<D><<<p.pieces, THREADS, smem, stream>>>(p);
  NB_LAUNCH_CHECK();
  if (((long long)p.width << p.block_log) <= (long long)CHUNK * Raw<D>::KEYS && (long long)p.rows * p.hk * ceil_div(min(p.few, p.tokens * p.group), 16) <= p.pieces)
    return NB_OK;                      // no table is long enough for two pieces
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.pieces);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = scan;
  cfg.stream = stream;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;   // its blocks start while the first kernel's last ones run
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  NB_CUDA(cudaLaunchKernelEx(&cfg, kv_attn_join_kernel<D>, p));
  return NB_OK;
}

}  // namespace

extern "C" {

// Pieces that the batch is cut into, and floats of work space that nb_kv_attention needs.
int nb_kv_attention_pieces(int dim) { return 148 * (dim == 64 ? 3 : 2); }
long long nb_kv_attention_work(int dim) { return (long long)nb_kv_attention_pieces(dim) * 2 * 16 * (dim + 2); }

int nb_kv_attention(const void* q, void* out, const void* codes, const float* scale, const int* tables, const int* starts,
                    const int* ends, int rows, int tokens, int max_new, int hq, int hk, int dim, int block, int blocks, int width,
                    long long q_token, long long q_head, long long o_token, long long o_head, long long kv_stride, long long s_stride,
                    float softmax_scale, float* work, long long work_floats, unsigned int* status, void* stream) {
  if (rows <= 0 || rows > 8192 || tokens < 0 || hk <= 0 || hq <= 0 || hq % hk || (dim != 64 && dim != 128) || blocks <= 0 || width <= 0) return NB_ERR_BAD_ARG;
  if ((block & (block - 1)) || block < 16 || (long long)width * block > 0x7fffffffLL || (long long)blocks * block > 0x7fffffffLL) return NB_ERR_BAD_ARG;
  if ((long long)tokens * hq > 0x7fffffffLL) return NB_ERR_TOO_LARGE;
  if (tokens == 0) return NB_OK;
  if ((reinterpret_cast<uintptr_t>(codes) & 15) || (kv_stride & 15)) return NB_ERR_UNALIGNED;
  if (!work || work_floats < nb_kv_attention_work(dim) || (reinterpret_cast<uintptr_t>(work) & 15)) return NB_ERR_BAD_ARG;
  KvAttn p{};
  p.q = q; p.out = out; p.codes = (const uint8_t*)codes; p.scale = scale; p.tables = tables; p.starts = starts; p.ends = ends;
  p.rows = rows; p.tokens = tokens; p.hq = hq; p.hk = hk; p.group = hq / hk; p.blocks = blocks; p.width = width;
  while ((1 << p.block_log) < block) ++p.block_log;
  p.q_token = q_token; p.q_head = q_head; p.o_token = o_token; p.o_head = o_head; p.kv_stride = kv_stride; p.s_stride = s_stride;
  p.q_vec = !((reinterpret_cast<uintptr_t>(q) & 15) || (q_token & 7) || (q_head & 7));
  p.o_vec = !((reinterpret_cast<uintptr_t>(out) & 7) || (o_token & 3) || (o_head & 3));
  p.scale_log2 = softmax_scale * 1.4426950408889634f;
  p.pieces = nb_kv_attention_pieces(dim);
  p.part_o = work;
  p.part_ml = work + (long long)p.pieces * 2 * 16 * dim;
  p.few = 0x7fffffff;
  p.status = status;
  return dim == 64 ? launch_few<64>(p, (cudaStream_t)stream) : launch_few<128>(p, (cudaStream_t)stream);
}

}  // extern "C"
