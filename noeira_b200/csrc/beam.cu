// Beam search: the best continuations over beams and vocabulary.
//
// value(b, v) = score_b + x_bv - log sum_u exp x_bu, in 64 bits.  It never falls while x rises, so the candidates of a beam are
// found by its logits alone; only the winners of the beams are compared by value.  Ties go to the lowest b * vocab + v.  Where
// different logits round to one value (beside an infinite one, next to zero, at a score of 1e20) the last candidate's value is
// looked for from the row's begin; a beam that does not exist (-inf) offers its first tokens.  NaN counts as -inf, +inf as the
// largest finite number.
//
// One pass over the logits, which is all that there is to read (R * beams * vocab elements at the copy rate), split over blocks of
// one part of one beam's row each, the elements in registers.  The maximum and sum of each warp come first; then the K = beams best
// of the block's elements: the K-th largest of a warp's lane maxima is a lower bound of the block's K-th element, and the largest of these
// bounds over the warps leaves few elements above it (about 2 K of 8192 in random order, and never more than K lanes' shares per
// warp), which are ranked by counting.  A second kernel, a block per request, joins the parts of each beam and ranks the beams.
// 48 x 8 beams over 32003 fp32 logits (49 MB): 24 us, the pass about 18 of them: 15 instructions a logit and 300 a warp for the
// maximum, bound and sum of a part, then the join's chain of reads and ranks.  1 x 4 over 49152 bf16 logits: 7 us, two launches.
#include "common.cuh"

namespace {
using namespace nb;

constexpr int THREADS = 256;
constexpr float TOP = 3.4028235e38f;
constexpr int MOST_TOKENS = 0x7fff0000;    // a part's last index, up to 8191 behind the last token, is still one of 32 bits
typedef unsigned long long Key;              // order of the value above, inverse index below: larger is better, all distinct

struct BeamSel {
  const void* logits;
  const float* scores;
  const unsigned char* finished;   // [R, beams] or null
  float* scores_out;
  int *parents, *tokens;
  unsigned char* done;
  int requests, beams, vocab, eos, parts, fp32;
  long long pitch;                 // elements between beams' rows
  float2* part_ms;                 // [R * beams, parts] maximum, sum of exponentials
  Key* part_key;                   // [R * beams, parts, beams] best first
};

__device__ __forceinline__ Key key_of(float x, int v) {
  uint32_t u = __float_as_uint(x + 0.f);             // -0 and 0 are the same value
  u ^= (uint32_t)((int)u >> 31) | 0x80000000u;
  return (Key)u << 32 | (uint32_t)~v;
}
__device__ __forceinline__ float value_of(Key k) {
  uint32_t u = (uint32_t)(k >> 32);
  u ^= (u >> 31) ? 0x80000000u : 0xffffffffu;
  return __uint_as_float(u);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Largest of the warp's keys; all lanes get it.
__device__ __forceinline__ Key warp_best(Key k) {
  const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(k >> 32));
  const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(k >> 32) == hi ? (uint32_t)k : 0u);
  return (Key)hi << 32 | lo;
}

template <bool FP32, int EACH, bool WIDE>
__global__ void __launch_bounds__(THREADS) beam_part_kernel(const BeamSel p) {
  constexpr int VEC = WIDE ? (FP32 ? 4 : 8) : 1, SIZE = FP32 ? 4 : 2;   // neighbouring elements of a thread, bytes of an element
  __shared__ float2 sum_sh[THREADS / 32];            // maximum, sum of exponentials of each warp
  __shared__ Key bound_sh[THREADS / 32];
  __shared__ int found;
  extern __shared__ Key cand[];                      // the elements above the bound
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, K = p.beams;
  const long long row = blockIdx.x / p.parts;
  const int part = blockIdx.x - (int)row * p.parts;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (p.finished && p.finished[row]) return;         // its one continuation is known
  // Where every row begins on a 16-byte boundary a thread reads 16 bytes at a time, else neighbouring threads read neighbouring
  // elements.  One or the other for all rows of a call: beams with equal logits then have equal sums, and their ties are ties.
  const char* base = (const char*)p.logits + row * p.pitch * SIZE;
  const int first = part * THREADS * EACH + tid * VEC;
  float x[EACH];
  if ((part + 1) * THREADS * EACH <= p.vocab) {      // all loads at once, none behind a condition
#pragma unroll
    for (int i = 0; i < EACH / VEC; ++i) {
      const int v = first + i * THREADS * VEC;
      if (WIDE) {
        const uint4 w = __ldcs(reinterpret_cast<const uint4*>(base + (long long)v * SIZE));
        const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (FP32) {
            x[i * VEC + e % VEC] = __uint_as_float(ww[e]);
          } else {
            x[i * VEC + (2 * e) % VEC] = __uint_as_float(ww[e] << 16);
            x[i * VEC + (2 * e + 1) % VEC] = __uint_as_float(ww[e] & 0xffff0000u);
          }
        }
      } else {
        x[i] = FP32 ? __ldcs((const float*)base + v) : __bfloat162float(__ldcs((const __nv_bfloat16*)base + v));
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int v = first + (i / VEC) * THREADS * VEC + i % VEC, at = min(v, p.vocab - 1);
      x[i] = FP32 ? ((const float*)base)[at] : __bfloat162float(((const __nv_bfloat16*)base)[at]);
      if (v >= p.vocab) x[i] = -INFINITY;
    }
  }
  float m = -INFINITY;
  int best = 0;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    x[i] = fminf(fmaxf(x[i], -INFINITY), TOP);       // the maximum of NaN and -inf is -inf
    if (x[i] > m) {
      m = x[i];
      best = i;
    }
  }
  const int at_best = first + (best / VEC) * THREADS * VEC + best % VEC;
  const Key mine = at_best < p.vocab ? key_of(m, at_best) : 0;   // this thread's best; 0: it has no element
  if (tid == 0) found = 0;
  // a warp's sum is relative to its own maximum: nothing waits for the block's
  const float top = warp_max(m), from = top == -INFINITY ? 0.f : top;
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const float d = x[i] - from;
    s += ex2(fmaf(d, 1.44269502f, d * 1.92596303e-8f));     // log2(e) in two parts: the first alone is off by 2^-26, always the same way
  }
  s = warp_sum(s);
  Key left = mine, bound = 0;
  for (int k = 0; k < K; ++k) {
    bound = warp_best(left);
    if (left == bound) left = 0;
  }
  if (lane == 0) {
    bound_sh[warp] = bound;
    sum_sh[warp] = make_float2(top, s);
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) bound = max(bound, bound_sh[w]);
  if (mine >= bound && mine != 0) {
    const float least = bound ? value_of(bound) : -INFINITY;   // 0: a block of fewer elements than K
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      if (x[i] >= least) {
        const int v = first + (i / VEC) * THREADS * VEC + i % VEC;
        const Key k = key_of(x[i], v);
        if (k >= bound && v < p.vocab) cand[atomicAdd(&found, 1)] = k;
      }
    }
  }
  __syncthreads();
  const long long at = row * p.parts + part;
  if (tid == 0) {
    float2 all = sum_sh[0];
#pragma unroll
    for (int w = 1; w < THREADS / 32; ++w) all.x = fmaxf(all.x, sum_sh[w].x);
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) sum += sum_sh[w].x == -INFINITY ? 0.f : sum_sh[w].y * expf(sum_sh[w].x - all.x);
    p.part_ms[at] = make_float2(all.x, sum);
  }
  const int n = found;
  for (int i = tid; i < n; i += THREADS) {
    const Key k = cand[i];
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) rank += cand[j] > k;
    if (rank < K) p.part_key[at * K + rank] = k;
  }
  for (int i = n + tid; i < K; i += THREADS) p.part_key[at * K + i] = 0;   // a part of fewer elements
}

// Joins the parts of a request: the K best and the log-sum-exp of each beam, a warp per beam; then the ranks of beams x K.
__global__ void __launch_bounds__(THREADS) beam_join_kernel(const BeamSel p) {
  __shared__ unsigned long long val[32 * 32];        // order of the value as an unsigned number; 0: no candidate
  __shared__ long long idx[32 * 32];                 // b * vocab + v
  __shared__ Key key_sh[THREADS / 32][64];
  const int r = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, K = p.beams;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  for (int b = warp; b < K; b += THREADS / 32) {
    const long long row = (long long)r * K + b;
    const float s0 = p.scores[row];
    const double score = s0 != s0 ? -INFINITY : (double)s0;
    long long at = 0x7fffffffffffffffLL;
    double v = -INFINITY;
    if (score == -INFINITY) {
      if (lane < p.vocab) at = (long long)b * p.vocab + lane;      // all alike: the first ones
    } else if (p.finished && p.finished[row]) {
      // eos at the beam's score; behind it, in order, what it does not continue with
      const int t = lane == 0 ? p.eos : lane - 1 + (lane - 1 >= p.eos);
      if (t < p.vocab) at = (long long)b * p.vocab + t;
      if (lane == 0) v = score;
    } else {
      float top = -INFINITY;
      for (int i = lane; i < p.parts; i += 32) top = fmaxf(top, p.part_ms[row * p.parts + i].x);
      top = warp_max(top);
      const float from = top == -INFINITY ? 0.f : top;
      double s = 0.0;
      for (int i = lane; i < p.parts; i += 32) {
        const float2 ms = p.part_ms[row * p.parts + i];
        if (ms.x > -INFINITY) s += (double)ms.y * (double)expf(ms.x - from);   // of weight one at the largest
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      const double lsum = log(s);
      const int m = p.parts * K;
      const Key* keys = p.part_key + row * m;
      Key mine = 0;                                  // the lane-th best
      if (m <= 64) {
        // few: the rank of each among all
        const Key k0 = lane < m ? keys[lane] : 0, k1 = lane + 32 < m ? keys[lane + 32] : 0;
        Key* all = key_sh[warp];
        all[lane] = k0;
        all[lane + 32] = k1;
        __syncwarp();
        int r0 = 0, r1 = 0;
#pragma unroll 8
        for (int j = 0; j < m; ++j) {
          const Key y = all[j];
          r0 += y > k0;
          r1 += y > k1;
        }
        __syncwarp();
        all[lane] = 0;
        __syncwarp();
        if (k0 && r0 < K) all[r0] = k0;
        if (k1 && r1 < K) all[r1] = k1;
        __syncwarp();
        mine = all[lane];
        __syncwarp();
      } else {
        // K rounds of the largest key below the last one; each lane looks through its own
        constexpr int HELD = 8;                      // in registers, more are read again
        Key held[HELD];
#pragma unroll
        for (int i = 0; i < HELD; ++i) held[i] = lane + 32 * i < m ? keys[lane + 32 * i] : 0;
        Key last = ~0ULL;
        for (int k = 0; k < K && last; ++k) {        // zero: fewer tokens than beams
          Key best = 0;
#pragma unroll
          for (int i = 0; i < HELD; ++i) best = held[i] < last && held[i] > best ? held[i] : best;
          for (int i = lane + 32 * HELD; i < m; i += 32) {
            const Key y = keys[i];
            best = y < last && y > best ? y : best;
          }
          last = warp_best(best);
          if (lane == k) mine = last;
        }
      }
      auto value = [&](float x) { return x > -INFINITY ? score + ((double)x - (double)from - lsum) : (double)-INFINITY; };
      if (mine && lane < K) {
        at = (long long)b * p.vocab + (int)~(uint32_t)mine;
        v = value(value_of(mine));
      }
      // Does the next smaller logit have the last candidate's value too?  Then the row may hold more of that value, ahead of those
      // found.
      const Key least = __shfl_sync(0xffffffffu, mine, K - 1);
      const double floor_v = __shfl_sync(0xffffffffu, v, K - 1);
      if (K < p.vocab && value_of(least) > -INFINITY && value(value_of(least - (1ULL << 32))) == floor_v) {
        const int above = __popc(__ballot_sync(0xffffffffu, lane < K && v > floor_v));
        const char* logits = (const char*)p.logits + row * p.pitch * (p.fp32 ? 4 : 2);
        int found = above;
        for (int i0 = 0; found < K && i0 < p.vocab; i0 += 32) {
          const int i = min(i0 + lane, p.vocab - 1);
          float x = p.fp32 ? ((const float*)logits)[i] : __bfloat162float(((const __nv_bfloat16*)logits)[i]);
          x = fminf(fmaxf(x, -INFINITY), TOP);
          const unsigned hit = __ballot_sync(0xffffffffu, i0 + lane < p.vocab && value(x) == floor_v);
          const int nth = lane - found;                // the hit of this lane, which holds the lane-th candidate
          if (nth >= 0 && nth < __popc(hit)) {
            at = (long long)b * p.vocab + i0 + (int)__fns(hit, 0, nth + 1);
            v = floor_v;
          }
          found += __popc(hit);
        }
      }
    }
    if (lane < K) {
      unsigned long long u = __double_as_longlong(v + 0.0);
      u ^= (unsigned long long)((long long)u >> 63) | 0x8000000000000000ULL;
      val[b * K + lane] = at == 0x7fffffffffffffffLL ? 0 : u;
      idx[b * K + lane] = at;
    }
  }
  __syncthreads();
  const int n = K * K;
  for (int i = tid; i < n; i += THREADS) {
    const unsigned long long u = val[i];
    const long long at = idx[i];
    if (u == 0) continue;
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < n; ++j) rank += val[j] > u || (val[j] == u && idx[j] < at);
    if (rank < K) {
      const long long o = (long long)r * K + rank;
      const int b = (int)(at / p.vocab), v = (int)(at - (long long)b * p.vocab);
      p.scores_out[o] = (float)__longlong_as_double((long long)(u ^ ((u >> 63) ? 0x8000000000000000ULL : ~0ULL)));
      p.parents[o] = b;
      p.tokens[o] = v;
      p.done[o] = p.eos >= 0 && ((p.finished && p.finished[(long long)r * K + b]) || v == p.eos);
    }
  }
}

template <bool FP32, int EACH, bool WIDE>
int launch_parts(const BeamSel& p, cudaStream_t s) {
  const int smem = THREADS / 32 * p.beams * EACH * 8;
  if (smem > 47 * 1024) {              // 48 KB hold the kernel's own arrays too
    static bool configured[64] = {};
    int dev = 0;
    NB_CUDA(cudaGetDevice(&dev));
    if (dev >= 64) return NB_ERR_BAD_ARG;
    if (!configured[dev]) {
      NB_CUDA(cudaFuncSetAttribute(beam_part_kernel<FP32, EACH, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, THREADS * EACH * 8));
      configured[dev] = true;
    }
  }
  beam_part_kernel<FP32, EACH, WIDE><<<(unsigned)(p.requests * p.beams * p.parts), THREADS, smem, s>>>(p);
  NB_LAUNCH_CHECK();
  return NB_OK;
}

// Elements of a thread: long parts read with more loads in flight and leave less to join; short ones spread few rows over the GPU.
// Measured, 8 / 32 (4 beams, vocabulary 49152, bf16): 4 rows 7.1 / 7.4 us, 16 rows 8.8 / 8.2, 32 rows 10.5 / 9.1, 64 rows 13.3 / 10.2.
int elements_each(long long rows, int vocab) { return rows * ceil_div(vocab, THREADS * 32) >= 148 ? 32 : 8; }

}  // namespace

extern "C" {

// Bytes of work space that nb_beam_select needs.
long long nb_beam_select_work(int requests, int beams, int vocab) {
  const long long rows = (long long)requests * beams, parts = ceil_div(vocab, THREADS * elements_each(rows, vocab));
  return rows * parts * (8 + 8LL * beams);
}

int nb_beam_select(const void* logits, const float* scores, const unsigned char* finished, float* scores_out, int* parents, int* tokens,
                   unsigned char* done, int requests, int beams, int vocab, int eos, int fp32, long long pitch, void* work, long long work_bytes, void* stream) {
  if (requests <= 0 || beams <= 0 || beams > 32 || vocab <= 0 || vocab > MOST_TOKENS || eos >= vocab || pitch < vocab || (finished && eos < 0)) return NB_ERR_BAD_ARG;
  if (reinterpret_cast<uintptr_t>(logits) & (fp32 ? 3 : 1)) return NB_ERR_UNALIGNED;
  const long long rows = (long long)requests * beams;
  if (!work || work_bytes < nb_beam_select_work(requests, beams, vocab) || (reinterpret_cast<uintptr_t>(work) & 15)) return NB_ERR_BAD_ARG;
  const int each = elements_each(rows, vocab), parts = ceil_div(vocab, THREADS * each);
  if (rows * parts > 0x7fffffffLL) return NB_ERR_TOO_LARGE;
  BeamSel p{logits, scores, finished, scores_out, parents, tokens, done, requests, beams, vocab, eos, parts, fp32, pitch, nullptr, nullptr};
  p.part_key = (Key*)work;
  p.part_ms = (float2*)(p.part_key + rows * parts * beams);
  const cudaStream_t s = (cudaStream_t)stream;
  int rc;
  const bool wide = !(reinterpret_cast<uintptr_t>(logits) & 15) && (rows == 1 || !(pitch & (fp32 ? 3 : 7)));
  if (fp32 && wide) rc = each == 32 ? launch_parts<true, 32, true>(p, s) : launch_parts<true, 8, true>(p, s);
  else if (fp32) rc = each == 32 ? launch_parts<true, 32, false>(p, s) : launch_parts<true, 8, false>(p, s);
  else if (wide) rc = each == 32 ? launch_parts<false, 32, true>(p, s) : launch_parts<false, 8, true>(p, s);
  else rc = each == 32 ? launch_parts<false, 32, false>(p, s) : launch_parts<false, 8, false>(p, s);
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(requests);
  cfg.blockDim = dim3(THREADS);
  cfg.stream = s;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;   // its blocks start while the first kernel's last ones run
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  NB_CUDA(cudaLaunchKernelEx(&cfg, beam_join_kernel, p));
  return NB_OK;
}

}  // extern "C"
