// Attention of new tokens over the paged 8-bit cache: o = softmax(c q K^T) V over the keys up to each token's own position.
//
// Few query rows per row of the batch (decode steps, short chunks).  The work is bound by the bytes of the cache, 2 D per key and
// head at the copy rate, so the cache is read once, as it is, and nothing else is in the way:
//   * A tile has 8 or 16 query rows: all query heads of one cache head, of as many tokens as fit.  The products are transposed,
//     S^T = K Q^T and O^T += V^T P^T, as m16n8k16 in f16 with fp32 sums: the 16 rows of an instruction are keys or dimensions,
//     which there are enough of, and its 8 columns are query rows, which in a decode step there are not.  e4m3 codes are exact
//     in f16; q (bf16), after a power-of-two scaling of the row, is exact in f16 down to 2^-31 of the row's largest element, and
//     below that off by 2^-39 of it at most (f16's subnormals).  P keeps 11 bits (2^-11, an eighth of the bf16 output's own
//     rounding): more would need a second product for the lower bits.  P times the ratio of the values' scales is f16 as well: exact,
//     as ratios are powers of two, but below 2^-21 of the row's largest, where it is off by 2^-32 of that at most.
//   * A warp works by itself: TMA brings the codes into its own ring in shared memory, 4 KB a step (two boxes of 16 keys each for
//     keys and values at D = 64, one at 128; a block id that is none becomes a box outside the tensor, which arrives as zeros),
//     and from there they go as they are into the fragments.  The order of the contraction is free as long as q has the same,
//     so a lane's fragment of K is 16 consecutive bytes of a key; the order of the output rows is free, so its fragment of V is
//     D / 8 consecutive bytes of four keys.  The copies' swizzle keeps both reads at two bank conflicts or fewer.
//   * The steps of the whole batch are cut into equal pieces, one for each resident warp (rows differ in length, so pieces run
//     over the ends of rows, and the ring runs ahead into the next row); a second, small kernel joins rows that lie in several
//     pieces.
// Eight tokens over 275k keys, 32/8 heads of 128 (594 MB): 110 us, 5.4 TB/s; a warp spends about 1000 clocks on a step's 320
// instructions (a third of them turn codes into f16), twelve warps an SM.  96 tokens over 81k keys, 15/5 heads of 64 (53 MB): 28 us,
// of which the steps are 12: a warp has seven of them, and starting, the first look into the table and joining take the rest.  One
// token over 640 keys, 6 heads of 64: 10.5 us.
#include <cuda.h>

#include "common.cuh"
#include "kv_cache.h"

namespace {
using namespace nb;

constexpr int WARPS = 4, THREADS = 32 * WARPS;
constexpr int FEW = 64;                // query rows of a row of the batch and head, up to which this kernel does it in any case
constexpr int STAGES = 3;              // steps in flight: two ahead of the one in work
constexpr int LEAD = 2;                // steps that starting a tile costs, in the measure by which the batch is cut
constexpr int LEAST = 2;               // a piece has at least so many steps
constexpr float RAISE = 8.f;           // the running maximum is raised when it falls behind by more than 2^8 ...
constexpr float LIFT = 7.f;            // ... and weights are at most 2^(8 + 7), below f16's largest, so that small ones stay normal
constexpr float NONE = -3e38f;         // the running maximum of a row that has seen nothing
// Scores whose maximum (log2) lies beyond this are rounded before the maximum is taken off: a multiply-add would leave the product's
// rounding, up to 2^-24 of the score, in the exponent, and a weight of 2^(8 + 7) and that much more passes f16's largest.  Costs nothing
// where it is not needed, 110 -> 129 us for the eight tokens above where it is.
constexpr float FAR = 1048576.f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// four e4m3 codes as two f16 pairs
__device__ __forceinline__ void f16_of_codes(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n.reg .b16 a, b;\nmov.b32 {a, b}, %2;\ncvt.rn.f16x2.e4m3x2 %0, a;\ncvt.rn.f16x2.e4m3x2 %1, b;\n}" : "=r"(lo), "=r"(hi) : "r"(w));
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
// the largest of a row over the four lanes that hold it
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
// the same over the eight lanes that hold a column
__device__ __forceinline__ float column_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
}
__device__ __forceinline__ float column_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 4);
  v += __shfl_xor_sync(0xffffffffu, v, 8);
  return v + __shfl_xor_sync(0xffffffffu, v, 16);
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {       // 8 x 8 matrix of 16-bit elements
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t times(uint32_t a, uint32_t b) { // f16 pairs
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t nan_code(uint32_t w) {         // nonzero where one of four codes is NaN
  const uint32_t m = w & 0x7f7f7f7fu;
  return (m + 0x01010101u) & 0x80808080u;
}

// n / d for d >= 1 with m = 2^32 / d rounded up (0 for d = 1): exact below 2^16, a division beyond
__device__ __forceinline__ int quotient(int n, int d, unsigned m) {
  if ((unsigned)n < 65536u && d < 65536) return m ? (int)__umulhi((unsigned)n, m) : n;
  return n / d;
}

// ---------------------------------------------------------------- how the batch is cut
// A job is a tile of query rows and a cache head.  It costs LEAD + steps (one, where every job is one block's).  `upto`
// (shared memory, rows + 1): exclusive sums over the rows; `piece`: what a warp takes.  I: what counts the steps of a batch, 32 bits
// where they are enough for tables that are filled to their ends (most_steps), else 64.
template <class I>
struct Cut {
  I total, piece;
};
template <class I>
struct Job {
  int row, head, qt, cost;
  I begin;
};
template <class I>
__host__ __device__ constexpr long long most_steps() {
  return sizeof(I) == 4 ? 0x7fffffffLL - 4096 : 1LL << 49;   // 4096: a rounding up to pieces
}

template <int KEYS>
__device__ __forceinline__ int job_cost(const KvAttn& p, int end) {
  return p.team ? 1 : LEAD + ceil_div(max(1, min(end, p.width << p.block_log)), KEYS);
}
template <int KEYS>
__device__ __forceinline__ long long row_cost(const KvAttn& p, int few, int i) {
  const int first = __ldg(p.starts + i), next = __ldg(p.starts + i + 1), end = __ldg(p.ends + i);
  const long long n = first < 0 ? 0 : (long long)min(next, p.tokens) - first;
  // rows with more query rows than `few` belong to the kernel of prompts
  const long long tiles = n <= 0 || n * p.group > few ? 0 : (n * p.group + p.tile - 1) >> (p.tile == 8 ? 3 : 4);
  return tiles * p.hk * job_cost<KEYS>(p, end);
}
// Only first tokens that are none (`starts` not ascending) make more steps than the sizes allow: reported, and nothing is done.
template <int KEYS, class I>
__device__ __forceinline__ Cut<I> cut_batch(const KvAttn& p, I* upto, I* sh) {
  constexpr long long MOST = most_steps<I>();
  const int tid = threadIdx.x, per = ceil_div(p.rows, THREADS);
  const int lo = min(p.rows, tid * per), hi = min(p.rows, lo + per);
  int few = p.few;
  if (p.far_size) {                    // the kernel of prompts was here before: did it meet scores that are this one's?
    int far = 0;
#pragma unroll 4
    for (int i = tid; i < p.far_size; i += THREADS) far |= p.far[i];
    if (__syncthreads_or(far)) few = 0x7fffffff;
  }
  long long sum = 0;
  for (int i = lo; i < hi; ++i) sum += row_cost<KEYS>(p, few, i);
  const bool large = sum > MOST;
  const I mine = large ? 0 : (I)sum;
  auto add = [](I a, I b) { return sizeof(I) == 4 ? (I)min((unsigned)a + (unsigned)b, (unsigned)MOST + 1) : a + b; };   // 128 of 2^49 fit in 64 bits
  I at = mine;
  const int lane = tid & 31, w = tid >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const I u = __shfl_up_sync(0xffffffffu, at, o);
    if (lane >= o) at = add(at, u);
  }
  if (lane == 31) sh[w] = at;
  bool refused = __syncthreads_or(large);
  Cut<I> c;
  c.total = 0;
#pragma unroll
  for (int i = 0; i < WARPS; ++i) {
    if (i < w) at = add(at, sh[i]);
    c.total = add(c.total, sh[i]);
  }
  refused |= c.total > MOST;
  if (refused) {
    if (tid == 0 && blockIdx.x == 0) report(p.status, NB_ST_BOUNDS, 11, 0);
    c.total = 0;
  }
  c.piece = p.team ? 1 : max((I)LEAST, (c.total + p.pieces - 1) / p.pieces);
  I begin = at - mine;
  for (int i = lo; i < hi; ++i) {
    upto[i] = begin;
    if (per > 1) begin += (I)row_cost<KEYS>(p, few, i);
  }
  if (tid == 0) upto[p.rows] = c.total;
  __syncthreads();
  return c;
}
template <int KEYS, class I>
__device__ __forceinline__ Job<I> job_at(const KvAttn& p, const I* upto, I x) {
  int a = 0, b = p.rows;               // last row that begins at or before x (rows without work share their begin with the next)
  while (b - a > 1) {
    const int m = (a + b) >> 1;
    if (upto[m] <= x) a = m; else b = m;
  }
  Job<I> j;
  j.row = a;
  j.cost = job_cost<KEYS>(p, __ldg(p.ends + a));
  const int n = (int)((x - upto[a]) / j.cost);
  j.qt = quotient(n, p.hk, p.hk_mul);
  j.head = n - j.qt * p.hk;
  j.begin = upto[a] + (I)n * j.cost;
  return j;
}

// The part of a job that lies in a piece: steps [from, last), none of them behind the last key that a row of the tile sees.
template <int KEYS, class I>
struct Part {
  Job<I> j;
  I stop;                              // where it ends, in the measure of the cut
  int first, count, real, end, new_tokens, sure, seen, from, last;
  // `skip`: the first of the job's steps that is this warp's (a team's warps take every fourth)
  __device__ __forceinline__ void set(const KvAttn& p, const I* upto, I x, I x1, int skip) {
    j = job_at<KEYS, I>(p, upto, x);
    stop = min(x1, j.begin + j.cost);
    first = __ldg(p.starts + j.row);
    const int next = __ldg(p.starts + j.row + 1);
    new_tokens = next - first;
    count = min(next, p.tokens) - first;
    end = max(0, min(__ldg(p.ends + j.row), p.width << p.block_log));
    real = min(p.tile, count * p.group - j.qt * p.tile);          // real rows of the tile
    const int tok0 = quotient(j.qt * p.tile, p.group, p.group_mul), tok1 = quotient(j.qt * p.tile + real - 1, p.group, p.group_mul);
    sure = max(0, min(end, end - new_tokens + tok0 + 1));         // the fewest keys that a real row sees
    seen = max(0, min(end, end - new_tokens + tok1 + 1));         // the most
    const int all = ceil_div(seen, KEYS);
    from = p.team ? skip : max(0, (int)(x - j.begin) - LEAD);
    last = p.team ? all : min(all, max(0, (int)(stop - j.begin) - LEAD));
  }
};

// ---------------------------------------------------------------- the ring
constexpr int STAGE = 4096;            // half of it keys, half values
template <int D>
struct Shape {
  static constexpr int SUB = STAGE / 32 / D;   // sub-tiles of 16 keys in a step
  static constexpr int KEYS = 16 * SUB;
};
struct Head {                          // of a stage
  float ks[STAGE / 2048], vs[STAGE / 2048];   // scales of the sub-tiles; a scale below zero: no keys there
};

// Byte of 16-byte chunk `ch` of row `r` (0..15) of a sub-tile, as the copy's swizzle leaves it.
template <int D>
__device__ __forceinline__ int chunk_at(int r, int ch) {
  return D == 64 ? r * 64 + ((ch ^ ((r >> 1) & 3)) << 4) : r * 128 + ((ch ^ (r & 7)) << 4);
}

template <int D, class I>
struct Feed {                          // runs over the steps of a warp's piece, ahead of the work
  Part<Shape<D>::KEYS, I> part;
  I x, x1;
  int stride, skip, hop;               // skip, hop: this warp's first step of a job, and how far it is to the next
  int step, page0, base;               // lane l: first row of page page0 + l among the tensor's rows, none: behind the last
  __device__ __forceinline__ void begin(I at, I end, int by, int first, int every) {
    x = at;
    x1 = end;
    stride = by;
    skip = first;
    hop = every;
    step = part.last = 0;
  }
  __device__ __forceinline__ void turn(const KvAttn& p, int page) {                  // the next 32 pages
    page0 = page;
    const int pg = page + (int)(threadIdx.x & 31);
    base = p.kv_rows;
    if ((long long)pg << p.block_log < part.seen) {
      const int b = __ldg(p.tables + (long long)part.j.row * p.width + pg);
      if ((unsigned)b < (unsigned)p.blocks) base = (b * p.hk + part.j.head) << p.block_log;
      else report(p.status, NB_ST_BOUNDS, 10, part.j.row);
    }
  }
  // The barrier of a stage completes with the bytes of the boxes and with the copies of the scales.
  __device__ __forceinline__ void next(const KvAttn& p, const CUtensorMap& map, const I* upto, uint32_t stage, Head* head, uint32_t bar) {
    constexpr int SUB = Shape<D>::SUB, KEYS = Shape<D>::KEYS;
    while (step >= part.last) {        // the next part that has steps
      if (x >= x1) return;
      part.set(p, upto, x, x1, skip);
      x = stride ? x + stride : part.stop;
      step = part.from;
      page0 = -64;
    }
    int row[SUB];
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      const int k0 = step * KEYS + s * 16, pg = k0 >> p.block_log;
      if (pg - page0 >= 32) turn(p, pg);
      row[s] = __shfl_sync(0xffffffffu, base, pg - page0);
    }
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
      for (int s = 0; s < SUB; ++s) {
        if (row[s] < p.kv_rows) {
          const float* from = p.scale + (row[s] >> p.block_log);
          copy4(smem_u32(&head->ks[s]), from);
          copy4(smem_u32(&head->vs[s]), from + p.s_stride);
        } else {
          head->ks[s] = head->vs[s] = -1.f;
        }
      }
      mbar_expect_tx_at(bar, STAGE);
#pragma unroll
      for (int s = 0; s < SUB; ++s) {
        const int y = row[s] + ((step * KEYS + s * 16) & ((1 << p.block_log) - 1));
        copy_box(stage + s * 16 * D, map, bar, y, 0);
        copy_box(stage + STAGE / 2 + s * 16 * D, map, bar, y, 1);
      }
      asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
    }
    step += hop;
  }
  static __device__ __forceinline__ void copy4(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
  }
  static __device__ __forceinline__ void mbar_expect_tx_at(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
  }
  static __device__ __forceinline__ void copy_box(uint32_t dst, const CUtensorMap& map, uint32_t bar, int row, int which) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
                 "l"(reinterpret_cast<uint64_t>(&map)), "r"(bar), "r"(0), "r"(row), "r"(which)
                 : "memory");
  }
};

template <int D, int NB>
struct Tile {                          // what a warp keeps of a tile of 8 NB query rows
  uint32_t q[NB][D / 16][2];           // row g of each 8
  float o[NB][D / 16][4];              // dimensions g D / 8 + 2 b, + 1 of rows 2c, 2c + 1; in units of vref
  float m[NB][2], l[NB][2], f[NB][2];  // rows 2c, 2c + 1: maximum (log2), this lane's sum, factor of a raw score
  int lim[NB][2];                      // keys that the row sees
  float vref, vinv;                    // the largest scale of the values so far, and its inverse
  float kick;                          // +inf where some row's maximum lies beyond FAR, else -inf
};

// The query rows of a tile as they are in memory: 16 dimensions of each 64, of row g of each 8.
template <int D, int NB, class I>
__device__ __forceinline__ void fetch_q(const KvAttn& p, const Part<Shape<D>::KEYS, I>& w, uint32_t (&raw)[NB][D / 8]) {
  const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const int idx = w.j.qt * p.tile + b * 8 + g, tok = quotient(idx, p.group, p.group_mul);
    const __nv_bfloat16* q = (const __nv_bfloat16*)p.q + (long long)(w.first + tok) * p.q_token + (long long)(w.j.head * p.group + idx - tok * p.group) * p.q_head + c * 16;
    uint32_t (&x)[D / 8] = raw[b];
#pragma unroll
    for (int i = 0; i < D / 8; ++i) x[i] = 0;
    if (tok < w.count) {
#pragma unroll
      for (int u = 0; u < D / 32; ++u) {
        const __nv_bfloat16* a = q + (u >> 1) * 64 + (u & 1) * 8;
        if (p.q_vec) {
          const uint4 r = *reinterpret_cast<const uint4*>(a);
          x[4 * u] = r.x;
          x[4 * u + 1] = r.y;
          x[4 * u + 2] = r.z;
          x[4 * u + 3] = r.w;
        } else {
          const unsigned short* e = reinterpret_cast<const unsigned short*>(a);
#pragma unroll
          for (int i = 0; i < 4; ++i) x[4 * u + i] = e[2 * i] | (uint32_t)e[2 * i + 1] << 16;
        }
      }
    }
  }
}
template <int D, int NB, class I>
__device__ __forceinline__ void open_tile(const KvAttn& p, const Part<Shape<D>::KEYS, I>& w, const uint32_t (&raw)[NB][D / 8], Tile<D, NB>& t) {
  const int c = threadIdx.x & 3;
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const uint32_t (&x)[D / 8] = raw[b];
    // power of two that takes the row's largest element to [2^14, 2^15); the row's scores are scaled back by its inverse
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < D / 8; ++i) top = fmaxf(top, fmaxf(fabsf(__uint_as_float(x[i] << 16)), fabsf(__uint_as_float(x[i] & 0xffff0000u))));
    top = quad_max(top);
    int e = (int)(__float_as_uint(top) >> 23) - 127;
    e = top > 0.f && e < 128 ? max(-100, min(112, e - 14)) : 0;
    const float s = __uint_as_float((uint32_t)(127 - e) << 23);
    const float back = p.scale_log2 * __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
    for (int k = 0; k < D / 16; ++k)
#pragma unroll
      for (int h = 0; h < 2; ++h) t.q[b][k][h] = f16_pair(__uint_as_float(x[2 * k + h] << 16) * s, __uint_as_float(x[2 * k + h] & 0xffff0000u) * s);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = b * 8 + 2 * c + h;
      t.f[b][h] = __shfl_sync(0xffffffffu, back, (2 * c + h) * 4);
      t.lim[b][h] = row < w.real ? max(0, min(w.end, w.end - w.new_tokens + quotient(w.j.qt * p.tile + row, p.group, p.group_mul) + 1)) : 0;
      t.m[b][h] = NONE;
      t.l[b][h] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < D / 16; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) t.o[b][j][i] = 0.f;
  }
  t.vref = t.vinv = 0.f;
  t.kick = -INFINITY;
}

// V^T P^T of one sub-tile: acc += V^T (D x 16 keys) P^T (16 keys x 8 rows)
template <int D, int NB>
__device__ __forceinline__ void times_v(float (&acc)[NB][D / 16][4], const uint32_t (&pt)[NB][2], const uint32_t (&v)[4][D / 32]) {
#pragma unroll
  for (int w = 0; w < D / 32; ++w) {
    // bytes of two keys side by side: two dimensions per word
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t a[4];
      f16_of_codes(__byte_perm(v[0][w], v[1][w], h ? 0x7362 : 0x5140), a[0], a[1]);
      f16_of_codes(__byte_perm(v[2][w], v[3][w], h ? 0x7362 : 0x5140), a[2], a[3]);
#pragma unroll
      for (int b = 0; b < NB; ++b) mma(acc[b][w * 2 + h], a, pt[b][0], pt[b][1]);
    }
  }
}

// One step of a tile.  Row g + 8 h of the transposed scores is that key of its sub-tile.  `seen`: the most keys that a row of the tile sees, `sure`: the fewest that a real row sees.
template <int D, int NB>
__device__ __forceinline__ void step_tile(const KvAttn& p, Tile<D, NB>& t, const uint8_t* st, const Head* head, int step, int seen, int sure) {
  constexpr int SUB = Shape<D>::SUB, KEYS = Shape<D>::KEYS;
  const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int k0 = step * KEYS;
  const bool whole = k0 + KEYS <= sure;
  float s[SUB][NB][4];                 // keys g and g + 8 of rows 2c, 2c + 1
#pragma unroll
  for (int u = 0; u < SUB; ++u) {
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[u][b][i] = 0.f;
#pragma unroll
    for (int d = 0; d < D / 64; ++d) {
      const uint4 x = *reinterpret_cast<const uint4*>(st + u * 16 * D + chunk_at<D>(g, d * 4 + c));
      const uint4 y = *reinterpret_cast<const uint4*>(st + u * 16 * D + chunk_at<D>(g + 8, d * 4 + c));
      const uint32_t xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t a[4];
        f16_of_codes(xw[k], a[0], a[2]);
        f16_of_codes(yw[k], a[1], a[3]);
#pragma unroll
        for (int b = 0; b < NB; ++b) mma(s[u][b], a, t.q[b][d * 4 + k][0], t.q[b][d * 4 + k][1]);
      }
    }
  }
  float f[SUB][NB][2], vs[SUB], vtop = t.vref;
  bool has[SUB], lacks = false;
#pragma unroll
  for (int u = 0; u < SUB; ++u) {
    const float ks = head->ks[u];
    vs[u] = head->vs[u];
    has[u] = ks >= 0.f;
    lacks |= !has[u];
    vtop = fmaxf(vtop, vs[u]);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      f[u][b][0] = fmaxf(t.f[b][0] * ks, 1.2e-38f);   // not zero, which would make a masked -inf a NaN
      f[u][b][1] = fmaxf(t.f[b][1] * ks, 1.2e-38f);
    }
  }
  if (!whole || lacks) {
#pragma unroll
    for (int u = 0; u < SUB; ++u)
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        if (!has[u]) f[u][b][0] = f[u][b][1] = 1.f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (k0 + u * 16 + g + (i >> 1) * 8 >= t.lim[b][i & 1] || !has[u]) s[u][b][i] = -INFINITY;
      }
  }
  // exponents; where one is too large for f16 the maxima are raised first.  A NaN lets itself through.
  float big = t.kick, base[NB][2];     // base: what is added to a score
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    base[b][0] = LIFT - t.m[b][0];
    base[b][1] = LIFT - t.m[b][1];
  }
#pragma unroll
  for (int u = 0; u < SUB; ++u)
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i) big = fmaxf(big, fmaf(s[u][b][i], f[u][b][i & 1], -t.m[b][i & 1]));
  if (__any_sync(0xffffffffu, big > RAISE) || vtop > t.vref) {
    bool far = false;
    const float over = t.kick > 0.f ? 0.f : RAISE;
    const float v = t.vref > 0.f ? t.vref / vtop : 0.f;
    t.vref = vtop;
    t.vinv = vtop > 0.f ? 1.f / vtop : 0.f;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      float a[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float top = -INFINITY;
#pragma unroll
        for (int u = 0; u < SUB; ++u) top = fmaxf(top, fmaxf(s[u][b][i], s[u][b][2 + i]) * f[u][b][i]);
        top = column_max(top);
        const bool raise = top > t.m[b][i] + over;
        a[i] = raise ? ex2(t.m[b][i] - top) : 1.f;
        if (raise) t.m[b][i] = top;
        far |= fabsf(t.m[b][i]) > FAR && t.m[b][i] != NONE;
        base[b][i] = LIFT - t.m[b][i];
        t.l[b][i] *= a[i];
        a[i] *= v;
      }
#pragma unroll
      for (int j = 0; j < D / 16; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) t.o[b][j][i] *= a[i & 1];
    }
    if (__any_sync(0xffffffffu, far)) {
      t.kick = INFINITY;
#pragma unroll
      for (int b = 0; b < NB; ++b) {
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
#pragma unroll
          for (int i = 0; i < 4; ++i) s[u][b][i] = __fsub_rn(__fmul_rn(s[u][b][i], f[u][b][i & 1]), t.m[b][i & 1]);
          f[u][b][0] = f[u][b][1] = 1.f;
        }
        base[b][0] = base[b][1] = LIFT;
      }
    } else {
      t.kick = -INFINITY;
    }
  }
#pragma unroll
  for (int u = 0; u < SUB; ++u) {
    uint32_t v[4][D / 32];             // [keys 2c, 2c + 1, 2c + 8, 2c + 9][bytes of dimensions g D / 8 ...]
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (D == 64) {
        const uint2 x = *reinterpret_cast<const uint2*>(st + STAGE / 2 + u * 16 * D + chunk_at<D>(2 * c + (k & 1) + (k >> 1) * 8, g >> 1) + (g & 1) * 8);
        v[k][0] = x.x;
        v[k][1] = x.y;
      } else {
        const uint4 x = *reinterpret_cast<const uint4*>(st + STAGE / 2 + u * 16 * D + chunk_at<D>(2 * c + (k & 1) + (k >> 1) * 8, g));
        v[k][0] = x.x;
        v[k][1] = x.y;
        v[k][D / 32 - 2] = x.z;
        v[k][D / 32 - 1] = x.w;
      }
    }
    if (!has[u]) continue;
    // Weights relative to vref; a block whose values are less than 2^-14 of the largest block's would lose bits in f16, so its
    // product is taken by itself and added in fp32.
    const float ratio = vs[u] * t.vinv;
    const bool apart = ratio < 6.1035156e-5f;
    const uint32_t w2 = f16_pair(apart ? 1.f : ratio, apart ? 1.f : ratio);
    uint32_t pt[NB][2];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      float e[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        e[i] = ex2(fmaf(s[u][b][i], f[u][b][i & 1], base[b][i & 1]));
        t.l[b][i & 1] += e[i];
      }
      pt[b][0] = times(transposed(f16_pair(e[0], e[1])), w2);
      pt[b][1] = times(transposed(f16_pair(e[2], e[3])), w2);
    }
    if (!whole) {
      // values behind the last key that any row sees are not numbers to be multiplied by zero
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (k0 + u * 16 + 2 * c + (k & 1) + (k >> 1) * 8 >= seen) {
#pragma unroll
          for (int x = 0; x < D / 32; ++x) v[k][x] = 0;
        }
      // Rows that do not see a key that others see would multiply its value by zero; NaN there is taken out, and put into the
      // rows that do see it.
      uint32_t any = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int x = 0; x < D / 32; ++x) any |= nan_code(v[k][x]);
      if (__any_sync(0xffffffffu, any != 0)) {
        for (int k = 0; k < 16; ++k) {
          // key k lies with the lanes c = (k & 7) / 2, in register (k & 1) + k / 8 * 2; word x carries dimensions g D / 8 + 4 x ..
          const int reg = (k & 1) + (k >> 3) * 2;
#pragma unroll
          for (int x = 0; x < D / 32; ++x) {
            const uint32_t mine = reg == 0 ? v[0][x] : reg == 1 ? v[1][x] : reg == 2 ? v[2][x] : v[3][x];
            const uint32_t got = __shfl_sync(0xffffffffu, mine, g * 4 + ((k & 7) >> 1));
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (((got >> (8 * j)) & 0x7fu) == 0x7fu)
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                  for (int i = 0; i < 2; ++i)
                    if (k0 + u * 16 + k < t.lim[b][i]) t.o[b][x * 2 + (j >> 1)][(j & 1) * 2 + i] = __int_as_float(0x7fffffff);
          }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int x = 0; x < D / 32; ++x) v[k][x] &= ~((nan_code(v[k][x]) >> 7) * 0xffu);
      }
    }
    if (!apart) {
      times_v<D, NB>(t.o, pt, v);
    } else {
      float acc[NB][D / 16][4];
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int j = 0; j < D / 16; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[b][j][i] = 0.f;
      times_v<D, NB>(acc, pt, v);
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int j = 0; j < D / 16; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) t.o[b][j][i] += acc[b][j][i] * ratio;
    }
  }
}

template <int D>
__device__ __forceinline__ void store_out(const KvAttn& p, int first, int head, int idx, int d, float a, float b, float c, float e) {
  const int tok = quotient(idx, p.group, p.group_mul);
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

// Joins what the warps of a block have of a tile, relative to the largest maximum of each row.
template <int D, int NB, class I>
__device__ __forceinline__ void join_team(const KvAttn& p, const Part<Shape<D>::KEYS, I>& w, const Tile<D, NB>& t, float* team_o, float2* team_ml) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = b * 8 + 2 * c + h;
      const float l = column_sum(t.l[b][h]);
      if (row >= w.real) continue;
      float* o = team_o + (warp * 8 * NB + row) * D + g * (D / 8);
#pragma unroll
      for (int k = 0; k < D / 16; k += 2)
        *reinterpret_cast<float4*>(o + 2 * k) = make_float4(t.o[b][k][h] * t.vref, t.o[b][k][2 + h] * t.vref, t.o[b][k + 1][h] * t.vref, t.o[b][k + 1][2 + h] * t.vref);
      if (g == 0) team_ml[warp * 8 * NB + row] = make_float2(t.m[b][h], l);
    }
  __syncthreads();
  for (int i = threadIdx.x; i < w.real * (D / 4); i += THREADS) {
    const int row = i / (D / 4), d = i % (D / 4) * 4;
    float top = NONE, l = 0.f;
#pragma unroll
    for (int k = 0; k < WARPS; ++k) top = fmaxf(top, team_ml[k * 8 * NB + row].x);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < WARPS; ++k) {
      const float2 ml = team_ml[k * 8 * NB + row];
      const float f = ml.x == NONE ? 1.f : ex2(ml.x - top);          // without a maximum all is zero, or NaN
      const float4 v = *reinterpret_cast<const float4*>(team_o + (k * 8 * NB + row) * D + d);
      l += ml.y * f;
      o.x += v.x * f;
      o.y += v.y * f;
      o.z += v.z * f;
      o.w += v.w * f;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    store_out<D>(p, w.first, w.j.head, w.j.qt * p.tile + row, d, o.x * inv, o.y * inv, o.z * inv, o.w * inv);
  }
  __syncthreads();                     // before the next tile's
}

// Partial results of a warp: slot 1 for the job that begins in its piece and runs on, slot 0 for the one that came from before.
__device__ __forceinline__ long long slot_at(long long piece, int slot) { return (piece * 2 + slot) * 16; }

template <int D, int NB, class I>
__global__ void __launch_bounds__(THREADS, 3) kv_attn_kernel(const __grid_constant__ CUtensorMap map, const KvAttn p) {
  constexpr int KEYS = Shape<D>::KEYS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const uint8_t* ring = smem + warp * STAGES * STAGE;
  Head* heads = reinterpret_cast<Head*>(smem + WARPS * STAGES * STAGE) + warp * STAGES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + WARPS * STAGES * (STAGE + sizeof(Head))) + warp * STAGES;
  I* sh = reinterpret_cast<I*>(smem + WARPS * STAGES * (STAGE + sizeof(Head) + 8));
  float* team_o = reinterpret_cast<float*>(sh + WARPS);           // [WARPS][8 NB][D], a team's only
  float2* team_ml = reinterpret_cast<float2*>(team_o + (p.team ? WARPS * 8 * NB * D : 0));
  I* upto = reinterpret_cast<I*>(team_ml + (p.team ? WARPS * 8 * NB : 0));
  if (lane == 0) {
    prefetch_tensormap(&map);
    for (int i = 0; i < STAGES; ++i) mbar_init(&bars[i], 2);
    fence_barrier_init();
  }
  const Cut<I> cut = cut_batch<KEYS, I>(p, upto, sh);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int piece = blockIdx.x * WARPS + warp, hop = p.team ? WARPS : 1;
  I x = p.team ? (I)blockIdx.x : (I)min((long long)cut.total, (long long)piece * cut.piece);
  const I x1 = p.team ? cut.total : (I)min((long long)cut.total, (long long)x + cut.piece);
  const int stride = p.team ? gridDim.x : 0;
  if (!p.team && lane == 0) p.part_job[piece].w = 0;
  const uint32_t ring_a = smem_u32(ring), bars_a = smem_u32(bars);
  Feed<D, I> feed;
  feed.begin(x, x1, stride, p.team ? warp : 0, hop);
  int at = 0;                          // stage of the next step
  uint32_t phase = 0;
  bool ok = true, primed = false;
  while (x < x1) {
    Part<KEYS, I> w;
    w.set(p, upto, x, x1, p.team ? warp : 0);
    uint32_t raw[NB][D / 8];
    fetch_q<D, NB>(p, w, raw);
    if (!primed) {                     // the first copies go out while the queries are on their way
#pragma unroll 1
      for (int i = 0; i < STAGES - 1; ++i) feed.next(p, map, upto, ring_a + i * STAGE, heads + i, bars_a + 8 * i);
      primed = true;
    }
    Tile<D, NB> t;
    open_tile<D, NB>(p, w, raw, t);
#pragma unroll 1
    for (int st = w.from; st < w.last && ok; st += hop) {
      __syncwarp();                    // all lanes are done with the step before, whose stage is filled anew
      const int ahead = (at + STAGES - 1) % STAGES;
      feed.next(p, map, upto, ring_a + ahead * STAGE, heads + ahead, bars_a + 8 * ahead);
      ok = __all_sync(0xffffffffu, mbar_wait(&bars[at], phase, p.status, 401));
      if (!ok) {
        // Copies that do not come: give the others in flight their time, so that none writes into memory that is no longer this
        // block's, and do nothing more but take part in the block's barriers.
        for (int i = 1; i < STAGES; ++i) {
          const int b = (at + i) % STAGES;
          mbar_wait(&bars[b], phase ^ (b < at ? 1u : 0u), p.status, 402);
        }
        break;
      }
      step_tile<D, NB>(p, t, ring + at * STAGE, heads + at, st, w.seen, w.sure);
      at = (at + 1) % STAGES;
      phase ^= at == 0 ? 1u : 0u;
    }
    if (p.team) {
      join_team<D, NB>(p, w, t, team_o, team_ml);
      x += stride;
      continue;
    }
    if (!ok) return;
    const bool alone = x == w.j.begin && w.stop == w.j.begin + w.j.cost;
    const long long slot = slot_at(piece, x == w.j.begin);
    if (!alone && x == w.j.begin && lane == 0)   // this piece's warp of the join kernel does this job, of so many pieces
      p.part_job[piece] = make_int4(w.first, w.j.head, w.j.qt, (int)((w.j.begin + w.j.cost - 1) / cut.piece - piece + 1) | w.real << 16);
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = b * 8 + 2 * c + h;
        const float l = column_sum(t.l[b][h]);
        if (row >= w.real) continue;
        const float f = alone ? (l == 0.f ? 0.f : t.vref / l) : t.vref;
#pragma unroll
        for (int k = 0; k < D / 16; k += 2) {
          const int d = g * (D / 8) + 2 * k;
          const float4 o = make_float4(t.o[b][k][h] * f, t.o[b][k][2 + h] * f, t.o[b][k + 1][h] * f, t.o[b][k + 1][2 + h] * f);
          if (alone) store_out<D>(p, w.first, w.j.head, w.j.qt * p.tile + row, d, o.x, o.y, o.z, o.w);
          else *reinterpret_cast<float4*>(p.part_o + (slot + row) * D + d) = o;
        }
        if (!alone && g == 0) *reinterpret_cast<float2*>(p.part_ml + (slot + row) * 2) = make_float2(t.m[b][h], l);
      }
    x = w.stop;
  }
}

// Joins the jobs that begin in one piece and run past its end, as the warps of the first kernel noted them: a block for four
// pieces, a warp per row, lanes over the columns (and at D = 64 over halves of the pieces).
template <int D>
__global__ void __launch_bounds__(THREADS) kv_attn_join_kernel(const KvAttn p) {
  constexpr int COLS = D / 4, SHARES = 32 / COLS;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, col = lane % COLS, share = lane / COLS;
  // every block waits, also one with nothing to join: what follows in the stream may start when this kernel is done
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 all = p.part_job[blockIdx.x * WARPS + (lane & (WARPS - 1))];
#pragma unroll 1
  for (int i = 0; i < WARPS; ++i) {
    const int piece = blockIdx.x * WARPS + i, size = __shfl_sync(0xffffffffu, all.w, i);
    const int first = __shfl_sync(0xffffffffu, all.x, i), head = __shfl_sync(0xffffffffu, all.y, i), qt = __shfl_sync(0xffffffffu, all.z, i);
    const int n = size & 0xffff, real = size >> 16;
    if (n == 0) continue;
#pragma unroll 1
    for (int row = warp; row < real; row += WARPS) {
      float top = NONE;
      for (int w = lane; w < n; w += 32) top = fmaxf(top, p.part_ml[(slot_at(piece + w, w == 0) + row) * 2]);
      top = warp_max(top);
      float l = 0.f;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
      for (int w = share; w < n; w += SHARES) {
        const long long s = slot_at(piece + w, w == 0) + row;
        const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + s * 2);
        const float f = ml.x == NONE ? 1.f : ex2(ml.x - top);      // without a maximum all is zero, or NaN
        const float4 v = *reinterpret_cast<const float4*>(p.part_o + s * D + col * 4);
        l += ml.y * f;
        o.x += v.x * f;
        o.y += v.y * f;
        o.z += v.z * f;
        o.w += v.w * f;
      }
      if (SHARES == 2) {
        o.x += __shfl_xor_sync(0xffffffffu, o.x, 16);
        o.y += __shfl_xor_sync(0xffffffffu, o.y, 16);
        o.z += __shfl_xor_sync(0xffffffffu, o.z, 16);
        o.w += __shfl_xor_sync(0xffffffffu, o.w, 16);
        l += __shfl_xor_sync(0xffffffffu, l, 16);
      }
      const float inv = l == 0.f ? 0.f : 1.f / l;
      if (share == 0) store_out<D>(p, first, head, qt * p.tile + row, col * 4, o.x * inv, o.y * inv, o.z * inv, o.w * inv);
    }
  }
}

template <int D, int NB, class I>
int launch_few(KvAttn p, cudaStream_t stream) {
  constexpr int fixed = 1024 + WARPS * STAGES * (STAGE + (int)sizeof(Head) + 8);
  const int scan = (WARPS + p.rows + 1) * (int)sizeof(I) + (p.team ? WARPS * 8 * NB * (D * 4 + 8) : 0);
  static bool configured[64] = {};
  int dev = 0;
  NB_CUDA(cudaGetDevice(&dev));
  if (dev >= 64) return NB_ERR_BAD_ARG;
  if (!configured[dev]) {
    NB_CUDA(cudaFuncSetAttribute(kv_attn_kernel<D, NB, I>, cudaFuncAttributeMaxDynamicSharedMemorySize, fixed + (WARPS + 8193) * (int)sizeof(I) + WARPS * 8 * NB * (D * 4 + 8)));
    configured[dev] = true;
  }
  CUtensorMap map;
  const int rc = kv_code_map(&map, p, D, 1);
  if (rc) return rc;
  kv_attn_kernel<D, NB, I><<<p.pieces / WARPS, THREADS, fixed + scan, stream>>>(map, p);
  NB_LAUNCH_CHECK();
  if (p.team) return NB_OK;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.pieces / WARPS);
  cfg.blockDim = dim3(THREADS);
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

typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                             CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static EncodeFn encode_fn() {
  static EncodeFn fn = nullptr;
  if (!fn) {
    void* sym = nullptr;
    cudaDriverEntryPointQueryResult res;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &res) == cudaSuccess && res == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeFn>(sym);
  }
  return fn;
}
int kv_code_map(CUtensorMap* m, const KvAttn& p, int dim, int swizzled) {
  EncodeFn enc = encode_fn();
  if (!enc) return NB_ERR_NO_DRIVER_SYMBOL;
  cuuint64_t dims[3] = {(cuuint64_t)dim, (cuuint64_t)p.kv_rows, 2}, strides[2] = {(cuuint64_t)dim, (cuuint64_t)p.kv_stride};
  cuuint32_t box[3] = {(cuuint32_t)dim, 16, 1}, one[3] = {1, 1, 1};
  const CUtensorMapSwizzle sw = !swizzled ? CU_TENSOR_MAP_SWIZZLE_NONE : dim == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B;
  const CUresult r = enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<uint8_t*>(p.codes), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, sw,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? NB_OK : NB_ERR_TENSORMAP;
}

extern "C" {

// Selects the kernel of rows with many query rows (tests compare the two): 0 by the rule below, 1 the one that reads codes into
// the fragments, 2 the tensor cores' one.  Returns the previous setting.
static int g_mode = 0;
int nb_kv_attention_mode(int mode) {
  const int old = g_mode;
  if (mode >= 0 && mode <= 2) g_mode = mode;
  return old;
}

}  // extern "C"

static constexpr int PIECES = 148 * WARPS * 3;                    // the warps that are resident together

// What a call is done by, from its sizes alone.
struct Plan {
  bool tiles;                          // rows with more than `few` query rows on the tensor cores
  int few, units;
  bool one, team;                      // tiles of 8 query rows, not 16; a block to a tile, not pieces of equal length
  bool wide;                           // steps are counted in 64 bits
};
static Plan plan_for(int dim, int rows, int tokens, int max_new, int hq, int hk, long long keys) {
  Plan r{false, 0x7fffffff, 0, false, false, false};
  const int group = hq / hk;
  const long long most = max(1, min(max_new, tokens));
  // Rows with many query rows go to the tensor cores when there are tiles enough: a tile of 256 query rows walks its keys alone,
  // while the other kernel spreads the keys of few tiles over all SMs.  Measured, other kernel / tiles, 2000 keys behind: one row of
  // 256 query rows 34 / 52 us, of 512 47 / 56, of 1024 90 / 64 (12 heads of 64: 12, 24, 48 tiles); 256 x 8 heads of 128 44 / 60,
  // 1024 x 8 (32 tiles) 90 / 62.  Below 64 query rows a row fills a quarter of its tile: 64 rows of 64 100 / 114, of 68 144 / 107.
  const long long units = (long long)tokens * group / 256 + min(rows, tokens);
  if (g_mode != 1 && most * group > FEW && (g_mode == 2 || (long long)tokens * group / 256 * hk >= 32) && units * hk <= 0x7fffffffLL) {
    r.tiles = true;
    r.few = FEW;
    r.units = (int)units;
  }
  // Tiles of 16 query rows share every conversion of a code; tiles of 8 are twice as many and spread little work better.  Measured,
  // 8 / 16 rows: one row of 64 tokens over 2000 keys, 12 heads of 64 (48 tiles of 16) 18 / 28 us, of 256 (192 tiles) 34 / 34, 16 rows
  // of 32 over 500 (384 tiles) 22 / 16; 32 rows of one token, 16 heads to one (32 tiles), up to 9000 keys 42 / 80; 256 tokens x 32/8
  // heads of 128 (512 tiles) 107 / 90.
  r.one = min(most * group, (long long)r.few) <= 8 || (long long)tokens * group / 16 * hk < 256;
  // Short tables: a block to a tile, its warps taking turns at the steps and joining in shared memory, which saves the second
  // kernel; where there are many such tiles, pieces spread them better.  Measured, block / pieces: one row of 300 keys 7.8 / 10.5
  // us, of 640 11.2 / 11.9, of 1200 15.4 / 11.3 (D = 64); 128 rows of 300 keys 15.3 / 18.7, 1024 rows 98 / 64.  Tiles of 16 rows
  // come several to a row and share its keys: 4 rows of 64 tokens over 560 keys (D = 128) 37 / 53, 64 rows of 17 over 520 50 / 68.
  const long long steps = (keys * dim + STAGE / 2 - 1) / (STAGE / 2);
  const long long jobs = ((long long)tokens * group / (r.one ? 8 : 16) + min(rows, tokens)) * hk;
  r.team = r.one ? steps <= 24 && jobs <= 1024 : steps <= 40 && jobs <= 4096;
  // The sizes bound the steps of the batch, with the tables full to their ends; lengths are the device's.  Counting in
  // 64 bits costs registers and divisions: 8 tokens over 275k keys (D = 128) 109.1 us in 32 bits, 110.8 in 64.
  r.wide = !r.team && jobs * (steps + LEAD) > most_steps<int>();
  return r;
}

extern "C" {

static long long part_floats(const Plan& plan, int dim) { return plan.team ? 0 : (long long)PIECES * (2 * 16 * (dim + 2) + 4); }

// Floats of work space that nb_kv_attention needs for these sizes: partial results, where rows are cut into pieces, and a byte per
// block of the kernel of prompts.
long long nb_kv_attention_work(int dim, int rows, int tokens, int max_new, int hq, int hk, int block, int width) {
  if (hk <= 0 || hq < hk || tokens <= 0) return 0;
  const Plan plan = plan_for(dim, rows, tokens, max_new, hq, hk, (long long)width * block);
  return part_floats(plan, dim) + (plan.tiles ? ((long long)plan.units * hk + 3) / 4 : 0);
}

int nb_kv_attention(const void* q, void* out, const void* codes, const float* scale, const int* tables, const int* starts,
                    const int* ends, int rows, int tokens, int max_new, int hq, int hk, int dim, int block, int blocks, int width,
                    long long q_token, long long q_head, long long o_token, long long o_head, long long kv_stride, long long s_stride,
                    float softmax_scale, float* work, long long work_floats, unsigned int* status, void* stream) {
  if (rows <= 0 || rows > 8192 || tokens < 0 || hk <= 0 || hq <= 0 || hq % hk || (dim != 64 && dim != 128) || blocks <= 0 || width <= 0) return NB_ERR_BAD_ARG;
  if ((block & (block - 1)) || block < 16 || (long long)width * block > 0x7fffffffLL || (long long)blocks * block > 0x7fffffffLL) return NB_ERR_BAD_ARG;
  if (!(softmax_scale > 0.f)) return NB_ERR_BAD_ARG;
  if ((long long)tokens * hq > 0x7fffffffLL) return NB_ERR_TOO_LARGE;
  if ((long long)blocks * hk * block > 0x7fffffffLL - 256) return NB_ERR_TOO_LARGE;   // rows of the copies' tensor
  if (tokens == 0) return NB_OK;
  if ((reinterpret_cast<uintptr_t>(codes) & 15) || (kv_stride & 15)) return NB_ERR_UNALIGNED;
  const long long floats = nb_kv_attention_work(dim, rows, tokens, max_new, hq, hk, block, width);
  if (floats > 0 && (!work || work_floats < floats || (reinterpret_cast<uintptr_t>(work) & 15))) return NB_ERR_BAD_ARG;
  KvAttn p{};
  p.q = q; p.out = out; p.codes = (const uint8_t*)codes; p.scale = scale; p.tables = tables; p.starts = starts; p.ends = ends;
  p.rows = rows; p.tokens = tokens; p.hq = hq; p.hk = hk; p.group = hq / hk; p.blocks = blocks; p.width = width; p.kv_rows = blocks * hk * block;
  while ((1 << p.block_log) < block) ++p.block_log;
  p.group_mul = p.group > 1 ? (unsigned)((0x100000000ULL + p.group - 1) / p.group) : 0;
  p.hk_mul = hk > 1 ? (unsigned)((0x100000000ULL + hk - 1) / hk) : 0;
  p.q_token = q_token; p.q_head = q_head; p.o_token = o_token; p.o_head = o_head; p.kv_stride = kv_stride; p.s_stride = s_stride;
  p.q_vec = !((reinterpret_cast<uintptr_t>(q) & 15) || (q_token & 7) || (q_head & 7));
  p.o_vec = !((reinterpret_cast<uintptr_t>(out) & 7) || (o_token & 3) || (o_head & 3));
  p.o_vec16 = !((reinterpret_cast<uintptr_t>(out) & 15) || (o_token & 7) || (o_head & 7));
  p.scale_log2 = softmax_scale * 1.4426950408889634f;
  p.pieces = PIECES;
  p.part_o = work;
  p.part_ml = work + (long long)p.pieces * 2 * 16 * dim;
  p.part_job = (int4*)(p.part_ml + (long long)p.pieces * 2 * 16 * 2);
  p.status = status;
  const Plan plan = plan_for(dim, rows, tokens, max_new, hq, hk, (long long)width * block);
  const cudaStream_t s = (cudaStream_t)stream;
  p.few = plan.few;
  p.tile = plan.one ? 8 : 16;
  p.team = plan.team;
  if (plan.tiles) {
    p.far = (uint8_t*)(work + part_floats(plan, dim));
    p.far_size = plan.units * hk;
    const int rc = kv_launch_prompts(p, dim, plan.units, s);
    if (rc) return rc;
  }
  if (plan.wide) {
    if (dim == 64) return plan.one ? launch_few<64, 1, long long>(p, s) : launch_few<64, 2, long long>(p, s);
    return plan.one ? launch_few<128, 1, long long>(p, s) : launch_few<128, 2, long long>(p, s);
  }
  if (dim == 64) return plan.one ? launch_few<64, 1, int>(p, s) : launch_few<64, 2, int>(p, s);
  return plan.one ? launch_few<128, 1, int>(p, s) : launch_few<128, 2, int>(p, s);
}

}  // extern "C"
