// Beam search: the best continuations over beams and vocabulary.
//
// value(b, v) = score_b + x_bv - log sum_u exp x_bu.  Within a beam the order of the values is the order of the logits, so
// the candidates of a beam are found by its logits alone, exactly; only the winners of the beams are compared by value, in
// 64 bits.  Ties go to the lowest b * vocab + v.  NaN counts as -inf, +inf as the largest finite number.
#include "common.cuh"

namespace {
using namespace nb;

struct BeamSel {
  const void* logits;
  const float* scores;
  const unsigned char* finished;   // [R, beams] or null
  float* scores_out;
  int *parents, *tokens;
  unsigned char* done;
  int requests, beams, vocab, eos, fp32;
  long long pitch;                 // elements between beams' rows
};

__device__ __forceinline__ float logit(const BeamSel& p, long long row, int v) {
  float x = p.fp32 ? ((const float*)p.logits)[row * p.pitch + v] : __bfloat162float(((const __nv_bfloat16*)p.logits)[row * p.pitch + v]);
  return x != x ? -INFINITY : fminf(x, 3.4028235e38f);
}

// One block per request: log-sum-exp of each beam, then `beams` rounds of a maximum over what has not been taken.
__global__ void __launch_bounds__(1024) beam_select_kernel(BeamSel p) {
  __shared__ float sh[32];
  __shared__ double top[32], lsum[32];   // maximum and log of the sum of each beam; together they would lose the sum beside a huge maximum
  __shared__ double bv[32];
  __shared__ long long bi[32];
  __shared__ double last_v;
  __shared__ long long last_i;
  const int r = blockIdx.x, tid = threadIdx.x;
  for (int b = 0; b < p.beams; ++b) {
    const long long row = (long long)r * p.beams + b;
    float m = -INFINITY;
    for (int v = tid; v < p.vocab; v += 1024) m = fmaxf(m, logit(p, row, v));
    m = block_max(m, sh);
    if (m == -INFINITY) m = 0.f;
    float s = 0.f;
    for (int v = tid; v < p.vocab; v += 1024) s += expf(logit(p, row, v) - m);
    s = block_sum(s, sh);
    if (tid == 0) {
      top[b] = (double)m;
      lsum[b] = log((double)s);
    }
  }
  if (tid == 0) { last_v = INFINITY; last_i = -1; }
  __syncthreads();
  for (int k = 0; k < p.beams; ++k) {
    double best = -INFINITY;
    long long at = 0x7fffffffffffffffLL;
    const double lv = last_v;
    const long long li = last_i;
    for (int b = 0; b < p.beams; ++b) {
      const long long row = (long long)r * p.beams + b;
      const bool fin = p.finished && p.finished[row];
      const float s0 = p.scores[row];
      const double sc = s0 != s0 ? -INFINITY : (double)s0;
      for (int v = tid; v < p.vocab; v += 1024) {
        const long long i = (long long)b * p.vocab + v;
        double val = -INFINITY;
        if (fin) {
          if (v == p.eos) val = sc;
        } else {
          const float x = logit(p, row, v);
          if (x > -INFINITY && sc > -INFINITY) val = sc + ((double)x - top[b] - lsum[b]);
        }
        if ((val < lv || (val == lv && i > li)) && (val > best || (val == best && i < at))) { best = val; at = i; }
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const double ov = __shfl_xor_sync(0xffffffffu, best, o);
      const long long oi = __shfl_xor_sync(0xffffffffu, at, o);
      if (ov > best || (ov == best && oi < at)) { best = ov; at = oi; }
    }
    if ((tid & 31) == 0) { bv[tid >> 5] = best; bi[tid >> 5] = at; }
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < 32; ++w)
        if (bv[w] > best || (bv[w] == best && bi[w] < at)) { best = bv[w]; at = bi[w]; }
      last_v = best;
      last_i = at;
      const long long o = (long long)r * p.beams + k;
      const int b = (int)(at / p.vocab), v = (int)(at % p.vocab);
      p.scores_out[o] = (float)best;
      p.parents[o] = b;
      p.tokens[o] = v;
      p.done[o] = p.eos >= 0 && ((p.finished && p.finished[(long long)r * p.beams + b]) || v == p.eos);
    }
    __syncthreads();
  }
}

}  // namespace

extern "C" int nb_beam_select(const void* logits, const float* scores, const unsigned char* finished, float* scores_out, int* parents, int* tokens,
                              unsigned char* done, int requests, int beams, int vocab, int eos, int fp32, long long pitch, void* stream) {
  if (requests <= 0 || beams <= 0 || beams > 32 || vocab <= 0 || eos >= vocab || pitch < vocab || (finished && eos < 0)) return NB_ERR_BAD_ARG;
  BeamSel p{logits, scores, finished, scores_out, parents, tokens, done, requests, beams, vocab, eos, fp32, pitch};
  beam_select_kernel<<<requests, 1024, 0, (cudaStream_t)stream>>>(p);
  NB_LAUNCH_CHECK();
  return NB_OK;
}
