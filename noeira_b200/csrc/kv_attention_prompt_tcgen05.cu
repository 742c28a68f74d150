// Attention over the paged 8-bit cache for prompts: many new tokens of a row, o = softmax(c Q K^T) V, causal.
//
// Bound by the matrix products (4 D operations per query row and key), so they run on the tcgen05 tensor cores in bf16.  A CTA owns
// 256 query rows of one cache head as two 128-row tiles; the query heads that share a cache head are neighbours among the rows
// (row = token * group + head), so that with grouped heads a tile still fills up, and one K / V tile serves all of them.
// e4m3 codes times a power-of-two scale are exact in bf16, so a key block is turned into bf16 once per CTA:
//
//   warp 0       MMA issuer: S_t = Q_t K^T, O_t += P_t V, P from tensor memory (the schedule of attention_fwd2_tcgen05.cu)
//   warp 1       TMA producer: looks up the blocks of 128 keys a step ahead and brings their codes, 16 rows a copy, into one buffer
//                for keys and one for values, with the scale of each 16 rows; a block that is none arrives as zeros
//   warps 4-7    copy Q into the swizzled operand layout, then turn codes into bf16 operand tiles (two stages each), 16 codes a
//                thread and turn; values behind the last key that any row sees become zeros.  A NaN value would reach rows that do
//                not see it (0 * NaN), so it becomes zero too, and the first key with a NaN is noted per dimension: a row sees a
//                prefix of the keys, so its output is NaN exactly where that key is in its prefix
//   warps 8-15   softmax, a thread per query row, 128 scores in registers, running maximum and sum
#include <cuda.h>

#include <type_traits>

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

constexpr int BQ = 128, BKV = 128, KS = 2, THREADS = 512;
// The registers of the launch, moved between the warpgroups; an increase waits until the block's own share has them.
static_assert(128 * 56 + 128 * 72 + 256 * 192 <= THREADS * 128, "register split");

// P = 2^(s * mult - m) of half a row as packed bf16 into tensor memory; returns the half's sum.
template <int HALF>
__device__ __forceinline__ float exp_store(const float (&s)[128], float mult, float m_use, uint32_t s_addr) {
  uint64_t sum = pack2(0.f, 0.f);
  const uint64_t mult2 = pack2(mult, mult), negm2 = pack2(-m_use, -m_use);
#pragma unroll
  for (int c = HALF * 4; c < HALF * 4 + 4; ++c) {
    uint32_t pk[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      float e0, e1;
      unpack2(fma2(pack2(s[c * 16 + 2 * u], s[c * 16 + 2 * u + 1]), mult2, negm2), e0, e1);
      e0 = exp2_fast(e0);
      e1 = exp2_fast(e1);
      sum = add2(sum, pack2(e0, e1));
      const __nv_bfloat162 h = __floats2bfloat162_rn(e0, e1);
      pk[u] = *reinterpret_cast<const uint32_t*>(&h);
    }
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(s_addr + c * 8), "r"(pk[0]), "r"(pk[1]), "r"(pk[2]),
                 "r"(pk[3]), "r"(pk[4]), "r"(pk[5]), "r"(pk[6]), "r"(pk[7])
                 : "memory");
  }
  float a, b;
  unpack2(sum, a, b);
  return a + b;
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
  static constexpr int OFF_NAN = OFF_SC + 64, OFF_BAR = OFF_NAN + HD * 4, BARS = 1 + 4 + 4 * KS + 8, OFF_MISC = OFF_BAR + BARS * 8;
  static constexpr int TOTAL = OFF_MISC + 160 + 1024;
  static_assert(TOTAL <= 232448, "shared memory");
};

template <int HD>
__global__ void __launch_bounds__(THREADS, 1) kv_attn_prompt_kernel(const __grid_constant__ CUtensorMap map, const KvAttn p) {
  using S = Smem<HD>;
  constexpr int NSUB = HD / 64;
  constexpr float RESCALE_THRESHOLD = 8.f;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* s_scale = reinterpret_cast<float*>(smem + S::OFF_SC);      // [2][8] of 16 key rows each
  int* s_nan = reinterpret_cast<int*>(smem + S::OFF_NAN);           // [HD] first key with a NaN value
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::OFF_BAR);
  int* misc = reinterpret_cast<int*>(smem + S::OFF_MISC);           // [0] tensor memory, [1] abort, [2] any NaN, [3..5] the CTA's tile, [8..23] sums
  volatile int* abort_flag = misc + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // ---------------------------------------------------------------- which rows: the batch's tiles in reverse, the long ones of a row first
  int tiles_mine = 0;
  const int per = ceil_div(p.rows, THREADS), lo = min(p.rows, (int)threadIdx.x * per), hi = min(p.rows, lo + per);
  auto tiles_of = [&](int i) {
    const int first = p.starts[i];
    const long long n = first < 0 ? 0 : (long long)min(p.starts[i + 1], p.tokens) - first;
    return n * p.group <= p.few ? 0 : (int)((n * p.group + 2 * BQ - 1) / (2 * BQ));
  };
  for (int i = lo; i < hi; ++i) tiles_mine += tiles_of(i);
  int upto = tiles_mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += u;
  }
  if (lane == 31) misc[8 + warp] = upto;
  if (threadIdx.x == 0) {
    misc[1] = misc[2] = 0;
    misc[3] = -1;
  }
  if (threadIdx.x < HD) s_nan[threadIdx.x] = 0x7fffffff;
  __syncthreads();
  int total = 0;
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) upto += misc[8 + w];
    total += misc[8 + w];
  }
  const int want = total - 1 - (int)(blockIdx.x / p.hk), head = blockIdx.x % p.hk;
  if (want < 0) return;                // the grid is an upper bound
  if (want >= upto - tiles_mine && want < upto) {
    int at = upto - tiles_mine;
    for (int i = lo; i < hi; ++i) {
      const int n = tiles_of(i);
      if (want < at + n) {
        misc[3] = i;
        misc[4] = want - at;
        break;
      }
      at += n;
    }
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
    mbar_init(&bars[0], 4);
    for (int w = 0; w < 2; ++w) {
      mbar_init(&bars[1 + w], 1);
      mbar_init(&bars[3 + w], 4);
    }
    for (int i = 0; i < KS; ++i) {
      mbar_init(&bars[5 + i], 4);
      mbar_init(&bars[5 + KS + i], 1);
      mbar_init(&bars[5 + 2 * KS + i], 4);
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
  const int seen = sees(min(tile0 + 2 * BQ, qrows) - 1);            // the most that a row of this CTA sees

  if (warp == 0) {
    // ---------------------------------------------------------------- MMA issuer
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (elect_one()) {
      const uint32_t idesc_s = make_idesc(1u, BQ, BKV, 0u, 0u), idesc_o = make_idesc(1u, BQ, HD, 0u, 1u);
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
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
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
        if (lane < 8) s_scale[w * 8 + lane] = sc[w];
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
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
  } else if (warp < 8) {
    // ---------------------------------------------------------------- operands
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    const int tid = threadIdx.x - 128;
    for (int i = tid; i < 2 * BQ * (HD / 8); i += 128) {
      const int r = i / (HD / 8), ch = i % (HD / 8), q = tile0 + r;
      uint4 w = make_uint4(0, 0, 0, 0);
      if (q < qrows) {
        const int tok = q / p.group;
        const __nv_bfloat16* a = (const __nv_bfloat16*)p.q + (long long)(first + tok) * p.q_token + (long long)(head * p.group + q - tok * p.group) * p.q_head + ch * 8;
        if (p.q_vec) {
          w = *reinterpret_cast<const uint4*>(a);
        } else {
          const unsigned short* e = reinterpret_cast<const unsigned short*>(a);
          w = make_uint4(e[0] | (uint32_t)e[1] << 16, e[2] | (uint32_t)e[3] << 16, e[4] | (uint32_t)e[5] << 16, e[6] | (uint32_t)e[7] << 16);
        }
      }
      *reinterpret_cast<uint4*>(smem + (r / BQ) * S::Q + (ch / 8) * (BQ * 128) + (r % BQ) * 128 + (((ch & 7) ^ (r & 7)) << 4)) = w;
    }
    fence_proxy_async();
    __syncwarp();
    if (lane == 0) mbar_arrive_a(q_full);
    constexpr int CH = HD / 16;        // 16-code chunks of a key row
    for (int j = 0; j < nmax; ++j) {
      const int st = j % KS;
      bool ok = true;
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        ok = ok && __all_sync(0xffffffffu, !*abort_flag && mbar_wait_a(raw_full(w), (uint32_t)j & 1u, p.status, 430 + w) &&
                                               mbar_wait_a(w ? v_empty(st) : k_empty(st), ((uint32_t)(j / KS) & 1u) ^ 1u, p.status, 432 + w));
        if (!ok) break;
        const uint8_t* raw = smem + S::OFF_RAW + w * S::RAW;
        uint8_t* to = smem + (w ? S::OFF_V : S::OFF_K) + st * S::KV;
#pragma unroll 2
        for (int i = tid; i < BKV * CH; i += 128) {
          const int r = i / CH, c = i % CH;
          const uint4 x = *reinterpret_cast<const uint4*>(raw + i * 16);
          uint32_t cw[4] = {x.x, x.y, x.z, x.w};
          if (w == 1) {
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
          const float sc = s_scale[w * 8 + (r >> 4)];
          uint32_t o[8];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            o[2 * e] = bf16_of_codes(cw[e] & 0xffffu, sc);
            o[2 * e + 1] = bf16_of_codes(cw[e] >> 16, sc);
          }
          // 32 bytes as two chunks; the halves of a 128-wide row in opposite order, so that eight lanes write eight different chunks
          uint8_t* line = to + (c / 4) * (BKV * 128) + r * 128;
          const int ch = (c & 3) * 2, flip = c / 4;
          const uint4 lo4 = make_uint4(o[0], o[1], o[2], o[3]), hi4 = make_uint4(o[4], o[5], o[6], o[7]);
          *reinterpret_cast<uint4*>(line + (((ch + flip) ^ (r & 7)) << 4)) = flip ? hi4 : lo4;
          *reinterpret_cast<uint4*>(line + (((ch + (flip ^ 1)) ^ (r & 7)) << 4)) = flip ? lo4 : hi4;
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
    asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
    const int t = (warp - 8) >> 2, quarter = warp & 3, r = quarter * 32 + lane;
    const int q = tile0 + t * BQ + r, n = nkb[t];
    const int lim = q < qrows ? sees(q) : 0;
    const uint32_t s_addr = tmem + ((uint32_t)(quarter * 32) << 16) + t * 128, o_addr = s_addr - t * 128 + 256 + t * 128;
    float m_ref = -INFINITY, l = 0.f;
    bool ok = true;
    // MODE 0: every real row of the tile sees the whole block; MODE 1: a row sees a prefix of it
    auto block = [&](int j, auto mode_tag) -> bool {
      constexpr int MODE = decltype(mode_tag)::value;
      if (!__all_sync(0xffffffffu, !*abort_flag && mbar_wait_a(s_full(t), (uint32_t)j & 1u, p.status, 440))) return false;
      tc_fence_after();
      float s[128];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld_32x32b_x32_nowait(s_addr + c * 32, reinterpret_cast<uint32_t*>(s) + c * 32);
      tmem_ld_wait();
      if (MODE == 1) {
        const int see = lim - j * BKV;
#pragma unroll
        for (int i = 0; i < 128; ++i) s[i] = i < see ? s[i] : -INFINITY;
      }
      float m0 = s[0], m1 = s[1], m2 = s[2], m3 = s[3];
#pragma unroll
      for (int i = 4; i < 124; i += 8) {
        m0 = max3(m0, s[i], s[i + 1]);
        m1 = max3(m1, s[i + 2], s[i + 3]);
        m2 = max3(m2, s[i + 4], s[i + 5]);
        m3 = max3(m3, s[i + 6], s[i + 7]);
      }
      m0 = max3(m0, s[124], s[125]);
      m1 = max3(m1, s[126], s[127]);
      const float mx = fmaxf(fmaxf(m0, m1), fmaxf(m2, m3)) * p.scale_log2;
      float alpha = 1.f;
      const bool grow = mx > m_ref + RESCALE_THRESHOLD || (m_ref == -INFINITY && mx > -INFINITY);
      if (grow) {
        alpha = exp2_fast(m_ref - mx);
        m_ref = mx;
      }
      const float m_use = m_ref == -INFINITY ? 0.f : m_ref;
      if (j > 0 && __any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int c = 0; c < HD; c += 32) {
          uint32_t o[32];
          tmem_ld_32x32b_x32(o_addr + c, o);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
          tmem_st_32x32b_x32(o_addr + c, o);
        }
      }
      float sum = exp_store<0>(s, p.scale_log2, m_use, s_addr);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_a(p_lo(t));
      sum += exp_store<1>(s, p.scale_log2, m_use, s_addr);
      l = l * alpha + sum;
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_a(p_full(t));
      return true;
    };
    const int whole = n > 0 ? min(n, sees(tile0 + t * BQ) / BKV) : 0;
    int j = 0;
#pragma unroll 1
    for (; j < whole && ok; ++j) ok = block(j, std::integral_constant<int, 0>{});
#pragma unroll 1
    for (; j < n && ok; ++j) ok = block(j, std::integral_constant<int, 1>{});
    if (ok && n > 0) ok = __all_sync(0xffffffffu, mbar_wait_a(o_done(t), 0u, p.status, 441));
    if (!ok) *abort_flag = 1;
    if (ok && tile0 + t * BQ < qrows) {
      tc_fence_after();
      const float inv = l == 0.f ? 0.f : 1.f / l;                    // NaN stays NaN
      const bool any_nan = misc[2] != 0;
      const int qc = min(q, qrows - 1), tok = qc / p.group;
      __nv_bfloat16* orow = (__nv_bfloat16*)p.out + (long long)(first + tok) * p.o_token + (long long)(head * p.group + qc - tok * p.group) * p.o_head;
#pragma unroll
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
