// Attention over the paged 8-bit cache for prompts: many new tokens of a row, o = softmax(c Q K^T) V, causal.
//
// Bound by the matrix products (4 D operations per query row and key), so they run on the tcgen05 tensor cores.  A CTA owns
// 256 query rows of one cache head as two 128-row tiles; the query heads that share a cache head are neighbours among the rows
// (row = token * group + head), so that with grouped heads a tile still fills up, and one K / V tile serves all of them.
// A code is exact in f16, and turning one into f16 is one instruction for two, so a key block is turned into f16 once per CTA
// without its scales:
//   * keys: the scale of each 16 keys multiplies their scores, which the exponent's multiply-add does at no cost;
//   * queries: after a power-of-two scaling of the row bf16 is exact in f16 down to 2^-31 of the row's largest element, and below
//     that off by 2^-39 of it at most;
//   * values: the weights P carry the scale relative to the largest that the CTA sees, 2^lr, as an addition to the exponent, and
//     the sum of the weights takes it out again, 16 keys at a time.  f16 weights have 11 bits,
//     an eighth of the bf16 output's own rounding, and lose some below 2^-14; where scales differ by more than 2^20 the CTA takes
//     values times their scale and P in bf16, which has the exponents but 8 bits: a weight's rounding is then as large as the
//     output's.  What a CTA sees decides, so rows of one call can differ in that.
//
// The exponent's multiply-add leaves the rounding of the maximum, up to 2^-24 of it, in the weights.  A CTA that may have scores
// (log2) beyond 2^22, by its largest query element and the largest scale of its keys, says so, and prompts are done over by the other
// kernel, which rounds such scores before the maximum is taken off (the prompts below: 1756 us instead of 228); in here, in whatever
// form, it cost all prompts 4 to 7 %.
//
//   warp 0       MMA issuer: S_t = Q_t K^T, O_t += P_t V, P from tensor memory (the schedule of attention_fwd2_tcgen05.cu)
//   warp 1       TMA producer: looks up the blocks of 128 keys a step ahead and brings their codes, 16 rows a copy, into one buffer
//                for keys and one for values, with the scale of each 16 rows; a block that is none arrives as zeros
//   warps 2, 3   turn codes into operand tiles (two stages each), 16 codes a thread and turn; values behind the last key that any
//                row sees become zeros.  A NaN value would reach rows that do not see it (0 * NaN), so in blocks that some row sees
//                in part it becomes zero too, and the first key with a NaN is noted per dimension: a row sees a prefix of the keys,
//                so its output is NaN where that key is in its prefix
//   warps 4-11   copy Q into the swizzled operand layout, then softmax: a thread per query row, 128 scores in registers, running
//                maximum and sum
// Four prompts of 700 to 2048 tokens over up to 4000 earlier keys, 32/8 heads of 128 (135 GFLOP): 229 us, 590 TFLOP/s.  A key block
// takes a CTA about 5500 clocks, of which the products are 2800: the exponentials of its two tiles share the special-function
// units (2048), and the chain of one tile, scores to weights to product, is not covered whole by the other's.  Measured on the
// way: four warps that turn codes cost the softmax warps registers (282 -> 320 us); bf16 operands with the scales multiplied in
// kept the two turning warps busy for 6000 clocks a block (387 us); a copy of the softmax per kind of mask and of P did not stay
// in the instruction cache (358 us).
#include <cuda.h>

#include "attention_common.cuh"
#include "kv_cache.h"

namespace {
using namespace nb;
using nbattn::add2;
using nbattn::exp2_fast;
using nbattn::fma2;
using nbattn::max3;
using nbattn::mbar_arrive_a;
using nbattn::mbar_expect_tx_a;
using nbattn::mbar_wait_a;
using nbattn::pack2;
using nbattn::umma_commit_a;
using nbattn::unpack2;

constexpr int BQ = 128, BKV = 128, KS = 2, THREADS = 384, CONV = 64;   // CONV: threads that turn codes
// The registers of the launch, moved between the warpgroups; an increase waits until the block's own share has them.
static_assert(128 * 88 + 256 * 208 <= THREADS * 168, "register split");

// P = 2^(s f_c - m + lr_c) of half a row, f_c and lr_c of the 16 keys of group c, packed into tensor memory; returns the half's sum
// of 2^(s f_c - m).
template <int HALF, bool BF>
__device__ __forceinline__ float exp_store(const float (&s)[128], const float (&f)[8], float m_use, const float4* group, uint32_t s_addr) {
  float total = 0.f;
  const float4 lr4 = group[2 + HALF], back4 = group[4 + HALF];
  const float lrs[4] = {lr4.x, lr4.y, lr4.z, lr4.w}, backs[4] = {back4.x, back4.y, back4.z, back4.w};
#pragma unroll
  for (int c = HALF * 4; c < HALF * 4 + 4; ++c) {
    const float add1 = (BF ? 0.f : lrs[c % 4]) - m_use;
    const uint64_t mult2 = pack2(f[c], f[c]), add = pack2(add1, add1);
    uint64_t sum = pack2(0.f, 0.f);
    float e[16];
    uint32_t pk[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      unpack2(fma2(pack2(s[c * 16 + 2 * u], s[c * 16 + 2 * u + 1]), mult2, add), e[2 * u], e[2 * u + 1]);
      e[2 * u] = exp2_fast(e[2 * u]);
      e[2 * u + 1] = exp2_fast(e[2 * u + 1]);
      sum = add2(sum, pack2(e[2 * u], e[2 * u + 1]));
    }
    if (BF) {
#pragma unroll
      for (int u = 0; u < 8; ++u) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(pk[u]) : "f"(e[2 * u + 1]), "f"(e[2 * u]));
    } else {
#pragma unroll
      for (int u = 0; u < 8; ++u) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(pk[u]) : "f"(e[2 * u + 1]), "f"(e[2 * u]));
    }
    float a, b;
    unpack2(sum, a, b);
    total = BF ? total + (a + b) : fmaf(a + b, backs[c % 4], total);
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(s_addr + c * 8), "r"(pk[0]), "r"(pk[1]), "r"(pk[2]),
                 "r"(pk[3]), "r"(pk[4]), "r"(pk[5]), "r"(pk[6]), "r"(pk[7])
                 : "memory");
  }
  return total;
}

// four codes as two f16 pairs
__device__ __forceinline__ void f16_of_codes(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n.reg .b16 a, b;\nmov.b32 {a, b}, %2;\ncvt.rn.f16x2.e4m3x2 %0, a;\ncvt.rn.f16x2.e4m3x2 %1, b;\n}" : "=r"(lo), "=r"(hi) : "r"(w));
}
// two codes (bits 0..15) times a scale, as bf16 pair
__device__ __forceinline__ uint32_t bf16_of_codes(uint32_t two, float scale) {
  uint32_t h2;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"((uint16_t)two));
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h2));
  const __nv_bfloat162 b = __floats2bfloat162_rn(f.x * scale, f.y * scale);
  return *reinterpret_cast<const uint32_t*>(&b);
}
__device__ __forceinline__ uint32_t nan_code(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

__device__ __forceinline__ void copy_box(uint32_t dst, const CUtensorMap& map, uint32_t bar, int row, int which) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
               "l"(reinterpret_cast<uint64_t>(&map)), "r"(bar), "r"(0), "r"(row), "r"(which)
               : "memory");
}

template <int HD>
struct Smem {
  static constexpr int Q = BQ * HD * 2, KV = BKV * HD * 2, RAW = BKV * HD;
  static constexpr int OFF_K = 2 * Q, OFF_V = OFF_K + KS * KV, OFF_RAW = OFF_V + KS * KV, OFF_SC = OFF_RAW + 2 * RAW;
  static constexpr int OFF_QF = OFF_SC + 4 * 32 * 4, OFF_NAN = OFF_QF + 2 * BQ, OFF_BAR = OFF_NAN + HD * 4, BARS = 1 + 4 + 4 * KS + 8, OFF_MISC = OFF_BAR + BARS * 8;
  static constexpr int TOTAL = OFF_MISC + 160 + 1024;
  static_assert(TOTAL <= 232448, "shared memory");
};

template <int HD>
__global__ void __launch_bounds__(THREADS, 1) kv_attn_prompt_kernel(const __grid_constant__ CUtensorMap map, const KvAttn p) {
  using S = Smem<HD>;
  constexpr float RESCALE_THRESHOLD = 4.f, LIFT = 11.f;   // weights are at most 2^15, below f16's largest
  constexpr float FAR = 4194304.f;     // up to here roundings add a quarter each: of the maximum, of what is added, of the threshold
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  // of the last four key blocks, for each 16 keys: scale of the keys [8], lr [8], 2^-lr [8], scale of the values [8]
  float* s_group = reinterpret_cast<float*>(smem + S::OFF_SC);
  signed char* s_qe = reinterpret_cast<signed char*>(smem + S::OFF_QF);   // [2 BQ] exponent by which a query row was scaled down
  int* s_nan = reinterpret_cast<int*>(smem + S::OFF_NAN);           // [HD] first key with a NaN value
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::OFF_BAR);
  int* misc = reinterpret_cast<int*>(smem + S::OFF_MISC);           // [0] tensor memory, [1] abort, [2] any NaN, [3..5] the CTA's tile, [8..23] sums
  volatile int* abort_flag = misc + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // ---------------------------------------------------------------- which rows: long ones first, and of a row the tiles that see most
  auto tiles_of = [&](int i) {
    const int first = p.starts[i];
    const long long n = first < 0 ? 0 : (long long)min(p.starts[i + 1], p.tokens) - first;
    return n * p.group <= p.few ? 0 : (int)((n * p.group + 2 * BQ - 1) / (2 * BQ));
  };
  const int unit = blockIdx.x / p.hk, head = blockIdx.x % p.hk;
  if (threadIdx.x == 0) {
    misc[1] = misc[2] = 0;
    misc[3] = -1;
    misc[6] = 0;                       // largest scale of the values (its bits), smallest that is not zero
    misc[7] = 0x7f800000;
    misc[24] = 0;                      // largest scale of the keys (its bits)
    misc[25] = 0;                      // scores may lie beyond FAR
  }
  if (threadIdx.x < HD) s_nan[threadIdx.x] = 0x7fffffff;
  if (p.rows <= THREADS) {
    // a thread per row: the tiles of all rows with more keys come before its own
    int2* all = reinterpret_cast<int2*>(smem);                      // Q is not there yet
    const int i = threadIdx.x;
    int2 me = make_int2(0, 0);
    if (i < p.rows) all[i] = me = make_int2(p.ends[i], tiles_of(i));
    __syncthreads();
    int before = 0;
    for (int k = 0; k < p.rows; ++k) {
      const int2 o = all[k];
      if (o.x > me.x || (o.x == me.x && k < i)) before += o.y;
    }
    if (i < p.rows && unit >= before && unit < before + me.y) {
      misc[3] = i;
      misc[4] = before + me.y - 1 - unit;
    }
  } else {
    // more rows than threads: in their order, from the last
    int mine = 0;
    const int per = ceil_div(p.rows, THREADS), lo = min(p.rows, (int)threadIdx.x * per), hi = min(p.rows, lo + per);
    for (int i = lo; i < hi; ++i) mine += tiles_of(i);
    int upto = mine, total = 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += u;
    }
    if (lane == 31) misc[8 + warp] = upto;
    __syncthreads();
    for (int w = 0; w < THREADS / 32; ++w) {
      if (w < warp) upto += misc[8 + w];
      total += misc[8 + w];
    }
    const int want = total - 1 - unit;
    int at = upto - mine;
    for (int i = lo; i < hi && want >= at; ++i) {
      const int n = tiles_of(i);
      if (want < at + n) {
        misc[3] = i;
        misc[4] = want - at;
      }
      at += n;
    }
  }
  __syncthreads();
  if (misc[3] < 0) {                   // the grid is an upper bound
    if (threadIdx.x == 0) p.far[blockIdx.x] = 0;
    return;
  }
  const uint32_t aS = smem_u32(smem), aB = smem_u32(bars);
  auto q_full = aB;
  auto raw_full = [&](int w) { return aB + 8u * (1 + w); };
  auto raw_empty = [&](int w) { return aB + 8u * (3 + w); };
  auto k_full = [&](int i) { return aB + 8u * (5 + i); };
  auto k_empty = [&](int i) { return aB + 8u * (5 + KS + i); };
  auto v_full = [&](int i) { return aB + 8u * (5 + 2 * KS + i); };
  auto v_empty = [&](int i) { return aB + 8u * (5 + 3 * KS + i); };
  auto s_full = [&](int t) { return aB + 8u * (5 + 4 * KS + t); };
  auto p_lo = [&](int t) { return aB + 8u * (7 + 4 * KS + t); };
  auto p_full = [&](int t) { return aB + 8u * (9 + 4 * KS + t); };
  auto o_done = [&](int t) { return aB + 8u * (11 + 4 * KS + t); };
  if (threadIdx.x == 0) {
    mbar_init(&bars[0], 8);
    for (int w = 0; w < 2; ++w) {
      mbar_init(&bars[1 + w], 1);
      mbar_init(&bars[3 + w], CONV / 32);
    }
    for (int i = 0; i < KS; ++i) {
      mbar_init(&bars[5 + i], CONV / 32);
      mbar_init(&bars[5 + KS + i], 1);
      mbar_init(&bars[5 + 2 * KS + i], CONV / 32);
      mbar_init(&bars[5 + 3 * KS + i], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&bars[5 + 4 * KS + t], 1);
      mbar_init(&bars[7 + 4 * KS + t], 4);
      mbar_init(&bars[9 + 4 * KS + t], 4);
      mbar_init(&bars[11 + 4 * KS + t], 1);
    }
    fence_barrier_init();
    prefetch_tensormap(&map);
  }
  if (warp == 0) {
    tmem_alloc(reinterpret_cast<uint32_t*>(misc), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(misc);
  const int row = misc[3], tile0 = misc[4] * 2 * BQ;                // first query row among the row's token * group
  const int first = p.starts[row], new_tokens = p.starts[row + 1] - first, count = min(p.starts[row + 1], p.tokens) - first;
  const int end = max(0, min(p.ends[row], p.width << p.block_log));
  const int qrows = count * p.group;
  // keys that query row r sees
  auto sees = [&](int r) { return max(0, min(end, end - new_tokens + r / p.group + 1)); };
  int nkb[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) nkb[t] = tile0 + t * BQ < qrows ? ceil_div(sees(min(tile0 + (t + 1) * BQ, qrows) - 1), BKV) : 0;
  const int nmax = max(nkb[0], nkb[1]);
  const int seen = sees(min(tile0 + 2 * BQ, qrows) - 1), sure = sees(tile0);   // the most that a row of this CTA sees, and the fewest

  // scales of the keys and values that this CTA will see
  for (int pg = threadIdx.x; (long long)pg << p.block_log < seen; pg += THREADS) {
    const int b = p.tables[(long long)row * p.width + pg];
    const bool is = (unsigned)b < (unsigned)p.blocks;
    const float v = is ? p.scale[p.s_stride + b * p.hk + head] : 0.f, k = is ? p.scale[b * p.hk + head] : 0.f;
    if (k > 0.f) atomicMax(&misc[24], __float_as_int(k));
    if (v > 0.f) {
      atomicMax(&misc[6], __float_as_int(v));
      atomicMin(&misc[7], __float_as_int(v));
    }
  }
  __syncthreads();
  const float vref = __int_as_float(misc[6]) > 0.f ? __int_as_float(misc[6]) : 1.f;
  const bool bf = __int_as_float(misc[7]) * 1048576.f < vref;

  if (warp == 0) {
    // ---------------------------------------------------------------- MMA issuer
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (elect_one()) {
      const uint32_t idesc_s = make_idesc(0u, BQ, BKV, 0u, 0u), idesc_o = make_idesc(bf ? 1u : 0u, BQ, HD, 0u, 1u);
      bool ok = nmax == 0 || mbar_wait_a(q_full, 0u, p.status, 410);
      auto issue_s = [&](int t, int j) -> bool {
        const int st = j % KS;
        const bool opens = t == 0 || !(j < nkb[0]), closes = t == 1 || !(j < nkb[1]);
        if (opens && (*abort_flag || !mbar_wait_a(k_full(st), (uint32_t)(j / KS) & 1u, p.status, 411))) return false;
        tc_fence_after();
        const uint64_t a0 = make_smem_desc(aS + t * S::Q, 16, 1024, 2), b0 = make_smem_desc(aS + S::OFF_K + st * S::KV, 16, 1024, 2);
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
          const uint32_t off = ((k / 4) * (BQ * 128) + (k % 4) * 32) >> 4;
          umma_f16(tmem + t * 128, a0 + off, b0 + off, idesc_s, k != 0 ? 1u : 0u);
        }
        umma_commit_a(s_full(t));
        if (closes) umma_commit_a(k_empty(st));
        return true;
      };
      auto issue_pv = [&](int t, int j) -> bool {
        const int st = j % KS;
        const bool opens = t == 0 || !(j < nkb[0]), closes = t == 1 || !(j < nkb[1]);
        if (*abort_flag || !mbar_wait_a(p_lo(t), (uint32_t)j & 1u, p.status, 412)) return false;
        if (opens && !mbar_wait_a(v_full(st), (uint32_t)(j / KS) & 1u, p.status, 413)) return false;
        tc_fence_after();
        const uint64_t b0 = make_smem_desc(aS + S::OFF_V + st * S::KV, BKV * 128, 1024, 2);
#pragma unroll
        for (int k = 0; k < BKV / 16; ++k) {
          if (k == BKV / 32) {
            if (!mbar_wait_a(p_full(t), (uint32_t)j & 1u, p.status, 414)) return false;
            tc_fence_after();
          }
          umma_f16_ts(tmem + 256 + t * 128, tmem + t * 128 + k * 8, b0 + ((k * 16 * 128) >> 4), idesc_o, (j | k) != 0 ? 1u : 0u);
        }
        if (closes) umma_commit_a(v_empty(st));
        if (j == nkb[t] - 1) umma_commit_a(o_done(t));
        return true;
      };
      for (int t = 0; t < 2 && ok; ++t)
        if (nkb[t] > 0) ok = issue_s(t, 0);
      for (int j = 0; j < nmax && ok; ++j)
        for (int t = 0; t < 2 && ok; ++t) {
          if (j >= nkb[t]) continue;
          ok = issue_pv(t, j);
          if (ok && j + 1 < nkb[t]) ok = issue_s(t, j + 1);
        }
      if (!ok) *abort_flag = 1;
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- codes: lane l < 8 brings key rows 16 l .. of each step
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    const int* table = p.tables + (long long)row * p.width;
    int src = p.kv_rows;
    float ks = 0.f, vs = 0.f;
    auto look = [&](int j) {
      const int key = j * BKV + lane * 16;
      src = p.kv_rows;                 // behind the tensor: zeros
      ks = vs = 0.f;
      if (lane < 8 && key < seen) {
        const int b = table[key >> p.block_log];
        if ((unsigned)b < (unsigned)p.blocks) {
          const int ph = b * p.hk + head;
          src = (ph << p.block_log) + (key & ((1 << p.block_log) - 1));
          ks = p.scale[ph];
          vs = p.scale[p.s_stride + ph];
        } else {
          report(p.status, NB_ST_BOUNDS, 12, row);
        }
      }
    };
    int issued[2] = {0, 0};
    if (nmax > 0) look(0);
    for (int j = 0; j < nmax; ++j) {
      const int s = src;
      const float sc[2] = {ks, vs};
      if (j + 1 < nmax) look(j + 1);
      bool ok = true;
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        ok = ok && __all_sync(0xffffffffu, !*abort_flag && mbar_wait_a(raw_empty(w), ((uint32_t)j & 1u) ^ 1u, p.status, 420 + w));
        if (!ok) break;
        if (w == 0 && lane < 8) {      // block j - 4 is done: its successor's keys wait for its softmax
          float* g = s_group + (j & 3) * 32 + lane;
          const float lr = sc[1] > 0.f ? fmaxf(log2f(sc[1] / vref), -40.f) : -40.f;
          g[0] = sc[0];
          g[8] = lr;
          g[16] = exp2f(-lr);
          g[24] = sc[1];
        }
        __syncwarp();
        if (lane == 0) mbar_expect_tx_a(raw_full(w), S::RAW);
        __syncwarp();
        if (lane < 8) copy_box(aS + S::OFF_RAW + w * S::RAW + lane * 16 * HD, map, raw_full(w), s, w);
        issued[w] = j + 1;
      }
      if (!ok) {
        *abort_flag = 1;
        break;
      }
    }
    // no copy may be in flight when the block ends
    for (int w = 0; w < 2; ++w)
      if (issued[w] > 0) mbar_wait_a(raw_full(w), (uint32_t)(issued[w] - 1) & 1u, p.status, 422);
  } else if (warp < 4) {
    // ---------------------------------------------------------------- operands
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    const int tid = threadIdx.x - 64;
    constexpr int CH = HD / 16;        // 16-code chunks of a key row
    for (int j = 0; j < nmax; ++j) {
      const int st = j % KS;
      bool ok = true;
#pragma unroll 1
      for (int w = 0; w < 2; ++w) {
        ok = ok && __all_sync(0xffffffffu, !*abort_flag && mbar_wait_a(raw_full(w), (uint32_t)j & 1u, p.status, 430 + w) &&
                                               mbar_wait_a(w ? v_empty(st) : k_empty(st), ((uint32_t)(j / KS) & 1u) ^ 1u, p.status, 432 + w));
        if (!ok) break;
        const uint8_t* raw = smem + S::OFF_RAW + w * S::RAW;
        uint8_t* to = smem + (w ? S::OFF_V : S::OFF_K) + st * S::KV;
        const bool part = w == 1 && (j + 1) * BKV > sure;           // some row sees only some of the keys
        // 32 bytes of a chunk as two; the halves of a 128-wide row in opposite order, so that eight lanes write eight different places
        auto put = [&](int r, int c, const uint32_t (&o)[8]) {
          uint8_t* line = to + (c / 4) * (BKV * 128) + r * 128;
          const int ch = (c & 3) * 2, flip = c / 4;
          const uint4 lo4 = make_uint4(o[0], o[1], o[2], o[3]), hi4 = make_uint4(o[4], o[5], o[6], o[7]);
          *reinterpret_cast<uint4*>(line + (((ch + flip) ^ (r & 7)) << 4)) = flip ? hi4 : lo4;
          *reinterpret_cast<uint4*>(line + (((ch + (flip ^ 1)) ^ (r & 7)) << 4)) = flip ? lo4 : hi4;
        };
        if (!part && !(w == 1 && bf)) {
          // rows of this thread are CONV / CH apart, its chunk is always the same
#pragma unroll 1
          for (int i0 = 0; i0 < BKV * CH / CONV; i0 += 4) {
            uint4 x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = *reinterpret_cast<const uint4*>(raw + ((i0 + e) * CONV + tid) * 16);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              uint32_t o[8];
              f16_of_codes(x[e].x, o[0], o[1]);
              f16_of_codes(x[e].y, o[2], o[3]);
              f16_of_codes(x[e].z, o[4], o[5]);
              f16_of_codes(x[e].w, o[6], o[7]);
              put((i0 + e) * (CONV / CH) + tid / CH, tid % CH, o);
            }
          }
        } else {
#pragma unroll 1
          for (int i = tid; i < BKV * CH; i += CONV) {
            const int r = i / CH, c = i % CH;
            const uint4 x = *reinterpret_cast<const uint4*>(raw + i * 16);
            uint32_t cw[4] = {x.x, x.y, x.z, x.w}, o[8];
            if (part) {
              if (j * BKV + r >= seen) cw[0] = cw[1] = cw[2] = cw[3] = 0;
              if (nan_code(cw[0]) | nan_code(cw[1]) | nan_code(cw[2]) | nan_code(cw[3])) {
                misc[2] = 1;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const uint32_t bad = nan_code(cw[e]) >> 7;
#pragma unroll
                  for (int b = 0; b < 4; ++b)
                    if ((bad >> (8 * b)) & 1u) atomicMin(&s_nan[c * 16 + e * 4 + b], j * BKV + r);
                  cw[e] &= ~(bad * 0xffu);
                }
              }
            }
            const float sc = s_group[(j & 3) * 32 + 24 + (r >> 4)];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if (w == 1 && bf) {
                o[2 * e] = bf16_of_codes(cw[e] & 0xffffu, sc);
                o[2 * e + 1] = bf16_of_codes(cw[e] >> 16, sc);
              } else {
                f16_of_codes(cw[e], o[2 * e], o[2 * e + 1]);
              }
            }
            put(r, c, o);
          }
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive_a(w ? v_full(st) : k_full(st));
          mbar_arrive_a(raw_empty(w));
        }
      }
      if (!ok) {
        *abort_flag = 1;
        break;
      }
    }
  } else {
    // ---------------------------------------------------------------- softmax and output: one thread per query row
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int t = (warp - 4) >> 2, quarter = warp & 3, r = quarter * 32 + lane;
    {
      constexpr int LANES = HD / 8, STEP = 128 / LANES, BATCH = 8;   // lanes of a query row, rows of a turn, turns whose loads go out together
      const int tid = threadIdx.x - 128 - t * 128, ch = tid % LANES;
      float most = 0.f;                // largest element
#pragma unroll 1
      for (int r0 = tid / LANES; r0 < BQ; r0 += STEP * BATCH) {
        uint4 w[BATCH];
#pragma unroll
        for (int u = 0; u < BATCH; ++u) {
          const int q = tile0 + t * BQ + r0 + u * STEP, tok = q / p.group;
          const __nv_bfloat16* a = (const __nv_bfloat16*)p.q + (long long)(first + tok) * p.q_token + (long long)(head * p.group + q - tok * p.group) * p.q_head + ch * 8;
          w[u] = make_uint4(0, 0, 0, 0);
          if (q < qrows && p.q_vec) w[u] = *reinterpret_cast<const uint4*>(a);
          if (q < qrows && !p.q_vec) {
            const unsigned short* e = reinterpret_cast<const unsigned short*>(a);
            w[u] = make_uint4(e[0] | (uint32_t)e[1] << 16, e[2] | (uint32_t)e[3] << 16, e[4] | (uint32_t)e[5] << 16, e[6] | (uint32_t)e[7] << 16);
          }
        }
#pragma unroll
        for (int u = 0; u < BATCH; ++u) {
          // power of two that takes the row's largest element to [2^14, 2^15)
          const int qr = r0 + u * STEP;
          uint32_t x[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
          float top = 0.f;
#pragma unroll
          for (int e = 0; e < 4; ++e) top = fmaxf(top, fmaxf(fabsf(__uint_as_float(x[e] << 16)), fabsf(__uint_as_float(x[e] & 0xffff0000u))));
#pragma unroll
          for (int o = LANES / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          most = fmaxf(most, top);
          int e2 = (int)(__float_as_uint(top) >> 23) - 127;
          e2 = top > 0.f && e2 < 128 ? max(-100, min(112, e2 - 14)) : 0;
          const float by = __uint_as_float((uint32_t)(127 - e2) << 23);
          if (ch == 0) s_qe[t * BQ + qr] = (signed char)e2;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float a = __uint_as_float(x[e] << 16) * by, b = __uint_as_float(x[e] & 0xffff0000u) * by;
            asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(x[e]) : "f"(b), "f"(a));
          }
          *reinterpret_cast<uint4*>(smem + t * S::Q + (ch / 8) * (BQ * 128) + qr * 128 + (((ch & 7) ^ (qr & 7)) << 4)) = make_uint4(x[0], x[1], x[2], x[3]);
        }
      }
      if (p.scale_log2 * most * (448.f * HD * __int_as_float(misc[24])) > FAR) misc[25] = 1;
    }
    fence_proxy_async();
    __syncwarp();
    if (lane == 0) mbar_arrive_a(q_full);
    const int q = tile0 + t * BQ + r, n = nkb[t];
    const int lim = q < qrows ? sees(q) : 0;
    const uint32_t s_addr = tmem + ((uint32_t)(quarter * 32) << 16) + t * 128, o_addr = s_addr - t * 128 + 256 + t * 128;
    float m_ref = -INFINITY, l = 0.f;
    bool ok = true;
    float qf = 0.f;
    // One key block, in one place: a variant per kind of mask or of P would not fit the instruction cache beside the others.
    auto block = [&](int j, bool whole) -> bool {
      if (!__all_sync(0xffffffffu, !*abort_flag && mbar_wait_a(s_full(t), (uint32_t)j & 1u, p.status, 440))) return false;
      tc_fence_after();
      float s[128];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld_32x32b_x32_nowait(s_addr + c * 32, reinterpret_cast<uint32_t*>(s) + c * 32);
      tmem_ld_wait();
      if (!whole) {                    // a row sees a prefix of the block
        const int see = lim - j * BKV;
#pragma unroll
        for (int i = 0; i < 128; ++i) s[i] = i < see ? s[i] : -INFINITY;
      }
      const float4* group = reinterpret_cast<const float4*>(s_group + (j & 3) * 32);
      const float4 ks0 = group[0], ks1 = group[1];
      float f[8] = {ks0.x, ks0.y, ks0.z, ks0.w, ks1.x, ks1.y, ks1.z, ks1.w};
      float mx = -INFINITY;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        float m0 = max3(s[c * 16], s[c * 16 + 1], s[c * 16 + 2]), m1 = max3(s[c * 16 + 3], s[c * 16 + 4], s[c * 16 + 5]);
        m0 = max3(m0, s[c * 16 + 6], s[c * 16 + 7]);
        m1 = max3(m1, s[c * 16 + 8], s[c * 16 + 9]);
        m0 = max3(m0, s[c * 16 + 10], s[c * 16 + 11]);
        m1 = max3(m1, s[c * 16 + 12], s[c * 16 + 13]);
        m0 = max3(m0, s[c * 16 + 14], s[c * 16 + 15]);
        f[c] = fmaxf(qf * f[c], 1.2e-38f);                          // not zero, which would make a masked -inf a NaN
        mx = fmaxf(mx, fmaxf(m0, m1) * f[c]);
      }
      float alpha = 1.f;
      const bool grow = mx > m_ref + RESCALE_THRESHOLD || (m_ref == -INFINITY && mx > -INFINITY);
      if (grow) {
        alpha = exp2_fast(m_ref - mx);
        m_ref = mx;
      }
      const float m_use = (m_ref == -INFINITY ? 0.f : m_ref) - LIFT;
      if (j > 0 && __any_sync(0xffffffffu, grow)) {
#pragma unroll 1
        for (int c = 0; c < HD; c += 32) {
          uint32_t o[32];
          tmem_ld_32x32b_x32(o_addr + c, o);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
          tmem_st_32x32b_x32(o_addr + c, o);
        }
      }
      float sum = bf ? exp_store<0, true>(s, f, m_use, group, s_addr) : exp_store<0, false>(s, f, m_use, group, s_addr);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_a(p_lo(t));
      sum += bf ? exp_store<1, true>(s, f, m_use, group, s_addr) : exp_store<1, false>(s, f, m_use, group, s_addr);
      l = l * alpha + sum;
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_a(p_full(t));
      return true;
    };
    const int whole = n > 0 ? min(n, sees(tile0 + t * BQ) / BKV) : 0;
    if (n > 0) {
      ok = __all_sync(0xffffffffu, mbar_wait_a(q_full, 0u, p.status, 442));
      qf = p.scale_log2 * __uint_as_float((uint32_t)(127 + s_qe[t * BQ + r]) << 23);   // what a raw score is multiplied by
    }
#pragma unroll 1
    for (int j = 0; j < n && ok; ++j) ok = block(j, j < whole);
    if (ok && n > 0) ok = __all_sync(0xffffffffu, mbar_wait_a(o_done(t), 0u, p.status, 441));
    if (!ok) *abort_flag = 1;
    if (ok && tile0 + t * BQ < qrows) {
      tc_fence_after();
      const float inv = l == 0.f ? 0.f : (bf ? 1.f : vref) / l;      // NaN stays NaN
      const bool any_nan = misc[2] != 0;
      const int qc = min(q, qrows - 1), tok = qc / p.group;
      __nv_bfloat16* orow = (__nv_bfloat16*)p.out + (long long)(first + tok) * p.o_token + (long long)(head * p.group + qc - tok * p.group) * p.o_head;
#pragma unroll 1
      for (int c = 0; c < HD; c += 32) {
        uint32_t o[32];
        if (n > 0) {
          tmem_ld_32x32b_x32(o_addr + c, o);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0u;
        }
        if (q < qrows) {
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            uint32_t pk[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float a = __uint_as_float(o[i + 2 * e]) * inv, b = __uint_as_float(o[i + 2 * e + 1]) * inv;
              if (any_nan) {
                if (s_nan[c + i + 2 * e] < lim) a = __int_as_float(0x7fffffff);
                if (s_nan[c + i + 2 * e + 1] < lim) b = __int_as_float(0x7fffffff);
              }
              const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
              pk[e] = *reinterpret_cast<const uint32_t*>(&h);
            }
            if (p.o_vec16) {
              *reinterpret_cast<uint4*>(orow + c + i) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const __nv_bfloat162 h = *reinterpret_cast<const __nv_bfloat162*>(&pk[e]);
                orow[c + i + 2 * e] = h.x;
                orow[c + i + 2 * e + 1] = h.y;
              }
            }
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
    if (lane == 0) p.far[blockIdx.x] = (uint8_t)misc[25];
  }
}

template <int HD>
int launch(const KvAttn& p, int units, cudaStream_t s) {
  static bool configured[64] = {};
  int dev = 0;
  NB_CUDA(cudaGetDevice(&dev));
  if (dev >= 64) return NB_ERR_BAD_ARG;
  if (!configured[dev]) {
    NB_CUDA(cudaFuncSetAttribute(kv_attn_prompt_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<HD>::TOTAL));
    configured[dev] = true;
  }
  CUtensorMap map;
  const int rc = kv_code_map(&map, p, HD, 0);
  if (rc) return rc;
  kv_attn_prompt_kernel<HD><<<units * p.hk, THREADS, Smem<HD>::TOTAL, s>>>(map, p);
  NB_LAUNCH_CHECK();
  return NB_OK;
}

}  // namespace

// `units`: an upper bound of the 256-row tiles of the rows with more than `few` query rows.
int kv_launch_prompts(const KvAttn& p, int dim, int units, cudaStream_t s) { return dim == 64 ? launch<64>(p, units, s) : launch<128>(p, units, s); }
