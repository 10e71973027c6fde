// Beam search's selection: of a group's beams and the vocabulary, the best continuations.
//
//   score(b, v) = scores[b] + x[b, v] - log sum_u exp(x[b, u])
//   out: the `count` largest scores of a group's beams x vocabulary, largest first; equal scores by (beam, token).
//
// Stage 1, one workgroup per row: maximum, sum of exponentials (in 64 bits: candidates of different beams lie closer to
// one another than a 32-bit score can tell apart) and the row's own `count` best.  Stage 2, one workgroup per group:
// the best of the rows' lists.
#include "common.h"

#define BEAM_THREADS 1024
#define BEAM_MAX_COUNT 64
#define BEAM_MAX_BEAMS 64

struct Cand {
  double v;
  int64_t i;
};

__device__ __forceinline__ Cand better(Cand a, Cand b) { return (b.v > a.v || (b.v == a.v && b.i < a.i)) ? b : a; }
__device__ __forceinline__ bool after(Cand a, Cand last) { return a.v < last.v || (a.v == last.v && a.i > last.i); }

template <int N>
__device__ __forceinline__ Cand block_best(Cand a, Cand* scratch) {
#pragma unroll
  for (int o = MI_WAVE / 2; o > 0; o >>= 1) a = better(a, Cand{__shfl_xor(a.v, o, MI_WAVE), __shfl_xor(a.i, o, MI_WAVE)});
  __syncthreads();
  if ((threadIdx.x & (MI_WAVE - 1)) == 0) scratch[threadIdx.x / MI_WAVE] = a;
  __syncthreads();
  Cand r = scratch[0];
  for (int w = 1; w < N / MI_WAVE; ++w) r = better(r, scratch[w]);
  return r;
}

// a logit that is not a number counts as minus infinity
__device__ __forceinline__ float logit_of(float x) { return x == x ? x : -INFINITY; }

__global__ __launch_bounds__(BEAM_THREADS) void beam_rows_kernel(const float* __restrict__ logits, int64_t row_stride,
                                                                 int V, const float* __restrict__ scores, int count,
                                                                 double* __restrict__ row_v, int* __restrict__ row_i) {
  __shared__ Cand scratch[BEAM_THREADS / MI_WAVE];
  __shared__ double sums[BEAM_THREADS / MI_WAVE];
  const int r = blockIdx.x;
  const float* row = logits + (int64_t)r * row_stride;
  const float start = scores[r];
  Cand best = {-INFINITY, V};
  for (int v = threadIdx.x; v < V; v += BEAM_THREADS) best = better(best, Cand{(double)logit_of(row[v]), v});
  best = block_best<BEAM_THREADS>(best, scratch);
  const double m = best.v;
  // a dead beam, or a row that leaves nothing, has no candidate better than another
  const bool dead = !(start > -INFINITY) || m == -INFINITY;
  double s = 0.0;
  for (int v = threadIdx.x; v < V; v += BEAM_THREADS) {
    const double x = logit_of(row[v]);
    s += x == m ? 1.0 : exp(x - m);
  }
#pragma unroll
  for (int o = MI_WAVE / 2; o > 0; o >>= 1) s += __shfl_xor(s, o, MI_WAVE);
  if ((threadIdx.x & (MI_WAVE - 1)) == 0) sums[threadIdx.x / MI_WAVE] = s;
  __syncthreads();
  s = 0.0;
  for (int w = 0; w < BEAM_THREADS / MI_WAVE; ++w) s += sums[w];
  const double log_s = log(s);
  Cand last = {INFINITY, -1};
  for (int n = 0; n < count; ++n) {
    Cand c = {-INFINITY, (int64_t)V + threadIdx.x};
    for (int v = threadIdx.x; v < V; v += BEAM_THREADS) {
      const float l = logit_of(row[v]);
      // (beside an infinite logit a finite one has no mass)
      const Cand x = {dead || (m == INFINITY && l < INFINITY) ? (double)-INFINITY : (double)l, v};
      if (after(x, last)) c = better(c, x);
    }
    last = block_best<BEAM_THREADS>(c, scratch);
    if (threadIdx.x == 0) {
      const bool real = last.i < V;
      row_v[(int64_t)r * count + n] = dead || !real ? -INFINITY : (last.v == m ? 0.0 : last.v - m) - log_s + (double)start;
      row_i[(int64_t)r * count + n] = real ? (int)last.i : -1;
    }
  }
}

__global__ __launch_bounds__(256) void beam_pick_kernel(const double* __restrict__ row_v, const int* __restrict__ row_i,
                                                        int beams, int count, int V, float* __restrict__ out_scores,
                                                        int* __restrict__ out_beams, int* __restrict__ out_tokens) {
  __shared__ Cand scratch[256 / MI_WAVE];
  const int64_t g = blockIdx.x;
  const int n = beams * count;
  Cand last = {INFINITY, -1};
  for (int o = 0; o < count; ++o) {
    Cand c = {-INFINITY, INT64_MAX};
    for (int j = threadIdx.x; j < n; j += 256) {
      const int token = row_i[g * n + j];
      const Cand x = {row_v[g * n + j], (int64_t)(j / count) * V + token};
      if (token >= 0 && after(x, last)) c = better(c, x);
    }
    last = block_best<256>(c, scratch);
    if (threadIdx.x == 0) {
      out_scores[g * count + o] = (float)last.v;
      out_beams[g * count + o] = (int)(last.i / V);
      out_tokens[g * count + o] = (int)(last.i % V);
    }
  }
}

// Scratch of mi_beam_select, in 8-byte words.
MI_EXPORT int mi_beam_scratch(int groups, int beams, int V, int count, int64_t* words) {
  *words = (int64_t)groups * beams * count * 2;
  return 0;
}

MI_EXPORT int mi_beam_select(const float* logits, int64_t row_stride, const float* scores, int groups, int beams, int V,
                             int count, double* scratch, float* out_scores, int* out_beams, int* out_tokens,
                             hipStream_t stream) {
  MI_REQUIRE(groups >= 0 && beams >= 1 && V >= 1 && row_stride >= V, "beam_select: bad sizes groups=%d beams=%d V=%d stride=%lld",
             groups, beams, V, (long long)row_stride);
  MI_REQUIRE(count >= 1 && count <= BEAM_MAX_COUNT && count <= (int64_t)beams * V,
             "beam_select: %d candidates of %d beams x %d tokens (at most %d)", count, beams, V, BEAM_MAX_COUNT);
  MI_REQUIRE(beams <= BEAM_MAX_BEAMS, "beam_select: %d beams, at most %d", beams, BEAM_MAX_BEAMS);
  if (groups == 0) return 0;
  double* row_v = scratch;
  int* row_i = (int*)(scratch + (int64_t)groups * beams * count);
  beam_rows_kernel<<<groups * beams, BEAM_THREADS, 0, stream>>>(logits, row_stride, V, scores, count, row_v, row_i);
  MI_CHECK_LAUNCH("beam rows");
  beam_pick_kernel<<<groups, 256, 0, stream>>>(row_v, row_i, beams, count, V, out_scores, out_beams, out_tokens);
  MI_CHECK_LAUNCH("beam pick");
  return 0;
}
