// Beam search's selection: of a group's beams and the vocabulary, the best continuations.
//
//   score(b, v) = scores[b] + x[b, v] - log sum_u exp(x[b, u])
//   out: the `count` largest scores of a group's beams x vocabulary, largest first; equal scores by (beam, token).
//
// One pass over the logits, which is what the operator cannot do without: a workgroup takes a part of a row and leaves
// its maximum, its sum of exponentials and its `count` best (value, token), in order; within a row the order of the
// logits is the order of the scores.  A second kernel, one workgroup to a group, joins the parts' sums to the rows'
// logarithms and picks the best of the lists.
//
// Candidates of different beams lie closer to one another than a 32-bit score can tell apart (32 bits of a score of
// -40 are steps of 4e-6, and a hundred thousand candidates share a few units), so exponentials, sums and compared scores
// are 64-bit; the exponential is a polynomial good to 1e-11, half of the arithmetic of the pass, and hides behind the
// loads.
#include "common.h"

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef f32x4 f32x4_any __attribute__((aligned(4)));      // 16 bytes from any element on

#define BEAM_MAX_COUNT 64
#define BEAM_MAX_BEAMS 64
#define BEAM_WAVES 4
#define BEAM_THREADS (BEAM_WAVES * MI_WAVE)
#define BEAM_TILE 1024                 // logits that a wave holds at once, 16 to a lane

// The order of candidates.  An empty place is (-inf, INT_MAX): every real candidate comes before it.
template <typename X>
__device__ __forceinline__ bool before(X ax, int ai, X bx, int bi) { return ax > bx || (ax == bx && ai < bi); }

__device__ __forceinline__ float lane_value(float x, int lane) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), lane)); }
__device__ __forceinline__ double lane_value(double x, int lane) {
  return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(x), lane), __builtin_amdgcn_readlane(__double2loint(x), lane));
}
// the value one lane below (wave_shr:1); lane 0 keeps its own
__device__ __forceinline__ int lane_below(int x) { return __builtin_amdgcn_update_dpp(x, x, 0x138, 0xf, 0xf, false); }
__device__ __forceinline__ float lane_below(float x) { return __int_as_float(lane_below(__float_as_int(x))); }
__device__ __forceinline__ double lane_below(double x) {
  return __hiloint2double(lane_below(__double2hiint(x)), lane_below(__double2loint(x)));
}

// A wave's best candidates in order: lane l holds the l-th.
template <typename X>
struct Best {
  X x;
  int i;
  int count;
  X last_x;          // the last of the `count` that are wanted: what a newcomer has to come before
  int last_i;
  __device__ __forceinline__ explicit Best(int n) : x(-INFINITY), i(INT32_MAX), count(n), last_i(INT32_MAX) {
    // (the compiler loads a 64-bit -inf into a scalar register pair as zero, so that it must not know this value)
    asm volatile("" : "+v"(x));
    last_x = lane_value(x, 0);
  }
  // one candidate of every lane
  __device__ __forceinline__ void take(X nx, int ni, int lane) {
    uint64_t mask = __ballot(before(nx, ni, last_x, last_i));
    while (mask) {
      const int from = __builtin_ctzll(mask);
      const X cx = lane_value(nx, from);
      const int ci = __builtin_amdgcn_readlane(ni, from);
      const int place = __builtin_popcountll(__ballot(before(x, i, cx, ci)));
      const X bx = lane_below(x);
      const int bi = lane_below(i);
      x = lane < place ? x : lane == place ? cx : bx;
      i = lane < place ? i : lane == place ? ci : bi;
      last_x = lane_value(x, count - 1);
      last_i = __builtin_amdgcn_readlane(i, count - 1);
      mask &= mask - 1;
      mask &= __ballot(before(nx, ni, last_x, last_i));
    }
  }
};

// What at least `count` of the lanes' values reach: the count-th largest of them.
template <typename X>
__device__ __forceinline__ X reached_by(X x, int count) {
  int above = 0;
  for (int l = 0; l < MI_WAVE; ++l) {
    const X y = lane_value(x, l);
    above += (y > x || (y == x && l < (int)(threadIdx.x & (MI_WAVE - 1)))) ? 1 : 0;
  }
  const uint64_t mask = __ballot(above == count - 1);
  return lane_value(x, mask ? __builtin_ctzll(mask) : 0);
}

// The places of the waves' sorted lists (in LDS, `count` entries each) in the list of all of them: own place plus how many
// of every other list come before.
template <typename X>
__device__ __forceinline__ int joined_place(const X* xs, const int* is, int waves, int count, int list, int at) {
  const X x = xs[list * count + at];
  const int i = is[list * count + at];
  int place = at;
  for (int w = 0; w < waves; ++w) {
    if (w == list) continue;
    int lo = 0, hi = count;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      const X y = xs[w * count + mid];
      const int j = is[w * count + mid];
      // (empty places are equal: the list's number decides)
      if (before(y, j, x, i) || (y == x && j == i && w < list)) lo = mid + 1;
      else hi = mid;
    }
    place += lo;
  }
  return place;
}

// e^d for d <= 0, to 1e-11 of its value: 2^n e^r, |r| <= ln 2 / 2, by the series of e^r up to r^9.
__device__ __forceinline__ double exp_of(double d) {
  const double t = fmax(d * 1.4426950408889634, -1100.0);       // (2^-1100 is 0)
  const double n = __builtin_rint(t);
  const double r = (t - n) * 0.6931471805599453;
  double p = 1.0 / 362880;
  p = fma(p, r, 1.0 / 40320);
  p = fma(p, r, 1.0 / 5040);
  p = fma(p, r, 1.0 / 720);
  p = fma(p, r, 1.0 / 120);
  p = fma(p, r, 1.0 / 24);
  p = fma(p, r, 1.0 / 6);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  return __builtin_ldexp(p, (int)n);
}

struct BeamParts {
  double* sum;             // [rows][parts]: of exp(x - max)
  float* max;              // [rows][parts]
  float* x;                // [rows][parts][count], in order
  int* token;
};

// Block (part, row): `tiles` tiles to a wave.
__global__ __launch_bounds__(BEAM_THREADS) void beam_rows_kernel(const float* __restrict__ logits, int64_t row_stride, int V,
                                                                 int count, int parts, int tiles, BeamParts out) {
  __shared__ float xs[BEAM_WAVES * BEAM_MAX_COUNT];
  __shared__ int is[BEAM_WAVES * BEAM_MAX_COUNT];
  __shared__ float maxima[BEAM_WAVES];
  __shared__ double sums[BEAM_WAVES];
  const int lane = threadIdx.x & (MI_WAVE - 1), wave = threadIdx.x / MI_WAVE;
  const int64_t r = blockIdx.x / parts;
  const int part = blockIdx.x % parts;
  const float* row = logits + r * row_stride;
  Best<float> best(count);
  float m = -INFINITY;
  double s = 0.0;
  // the part's tiles go round the waves
  const int64_t first = ((int64_t)part * tiles * BEAM_WAVES + wave) * BEAM_TILE;
  for (int t = 0; t < tiles; ++t) {
    const int64_t at = first + (int64_t)t * BEAM_WAVES * BEAM_TILE;
    if (at >= V) break;
    f32x4 x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      // (which lane adds up a logit follows from its index alone: equal rows have equal sums wherever they lie)
      const int64_t e = at + (j * MI_WAVE + lane) * 4;
      if (e + 4 <= V) {
        x[j] = *reinterpret_cast<const f32x4_any*>(row + e);
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) x[j][c] = e + c < V ? row[e + c] : -INFINITY;
      }
    }
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        x[j][c] = x[j][c] == x[j][c] ? x[j][c] : -INFINITY;
        top = fmaxf(top, x[j][c]);
      }
    const float tile_top = wave_max(top);
    if (tile_top > m) {
      s *= exp_of((double)m - (double)tile_top);
      m = tile_top;
    }
    if (m == INFINITY) {                 // (only such logits have a share)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) s += x[j][c] == INFINITY ? 1.0 : 0.0;
    } else if (m > -INFINITY) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) s += exp_of((double)x[j][c] - (double)m);
    }
    // the candidates: at first those that `count` lanes reach, then those that come before the last of the list
    if (tile_top < best.last_x) continue;
    const float floor_x = t == 0 ? reached_by(top, count) : -INFINITY;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int64_t e = at + (j * MI_WAVE + lane) * 4 + c;
        const bool real = e < V && x[j][c] >= floor_x;
        best.take(real ? x[j][c] : -INFINITY, real ? (int)e : INT32_MAX, lane);
      }
  }
  if (lane < count) {
    xs[wave * count + lane] = best.x;
    is[wave * count + lane] = best.i;
  }
#pragma unroll
  for (int o = MI_WAVE / 2; o > 0; o >>= 1) s += __shfl_xor(s, o, MI_WAVE);
  if (lane == 0) {
    maxima[wave] = m;
    sums[wave] = s;
  }
  __syncthreads();
  const int64_t to = r * parts + part;
  for (int i = threadIdx.x; i < BEAM_WAVES * count; i += BEAM_THREADS) {
    const int place = joined_place(xs, is, BEAM_WAVES, count, i / count, i % count);
    if (place < count) {
      out.x[to * count + place] = xs[i];
      out.token[to * count + place] = is[i];
    }
  }
  if (threadIdx.x == 0) {
    float all = maxima[0];
    for (int w = 1; w < BEAM_WAVES; ++w) all = fmaxf(all, maxima[w]);
    double sum = 0.0;
    for (int w = 0; w < BEAM_WAVES; ++w)
      sum += maxima[w] == all ? sums[w] : sums[w] * exp_of((double)maxima[w] - (double)all);
    out.max[to] = all;
    out.sum[to] = sum;
  }
}

// Block: a group.
__global__ __launch_bounds__(BEAM_THREADS) void beam_pick_kernel(const float* __restrict__ logits, int64_t row_stride,
                                                                 const float* __restrict__ scores, BeamParts in, int beams,
                                                                 int count, int parts, int V, float* __restrict__ out_scores,
                                                                 int* __restrict__ out_beams, int* __restrict__ out_tokens) {
  __shared__ float row_max[BEAM_MAX_BEAMS];
  __shared__ double row_base[BEAM_MAX_BEAMS];      // scores[b] - log of the row's sum; NaN: no candidate above -inf
  __shared__ int special;                          // rows whose lists do not say it all
  __shared__ double xs[BEAM_WAVES * BEAM_MAX_COUNT];
  __shared__ int is[BEAM_WAVES * BEAM_MAX_COUNT];
  const int lane = threadIdx.x & (MI_WAVE - 1), wave = threadIdx.x / MI_WAVE;
  const int64_t r0 = (int64_t)blockIdx.x * beams;
  if (threadIdx.x == 0) special = 0;
  __syncthreads();
  for (int b = wave; b < beams; b += BEAM_WAVES) {
    float m = -INFINITY;
    for (int p = lane; p < parts; p += MI_WAVE) m = fmaxf(m, in.max[(r0 + b) * parts + p]);
    m = wave_max(m);
    double s = 0.0;
    for (int p = lane; p < parts; p += MI_WAVE) {
      const float pm = in.max[(r0 + b) * parts + p];
      s += pm == m ? in.sum[(r0 + b) * parts + p] : in.sum[(r0 + b) * parts + p] * exp_of((double)pm - (double)m);
    }
#pragma unroll
    for (int o = MI_WAVE / 2; o > 0; o >>= 1) s += __shfl_xor(s, o, MI_WAVE);
    if (lane == 0) {
      const float start = scores[r0 + b];
      const bool dead = !(fabsf(start) < INFINITY) || m == -INFINITY;
      row_max[b] = m;
      row_base[b] = dead ? NAN : (double)start - log(s);
      if (dead || m == INFINITY) special = 1;
    }
  }
  __syncthreads();
  Best<double> best(count);
  const int lists = parts * count, n = beams * lists;
  for (int c0 = wave * MI_WAVE; c0 < n; c0 += BEAM_THREADS) {
    const int c = c0 + lane, b = min(c / lists, beams - 1);
    const double base = row_base[b];
    const float m = row_max[b];
    float x = -INFINITY;
    int token = INT32_MAX;
    if (c < n) {
      x = in.x[r0 * lists + c];
      token = in.token[r0 * lists + c];
    }
    const bool real = token != INT32_MAX && base == base && (m < INFINITY || x == INFINITY);
    best.take(real ? (x == m ? base : (double)x - (double)m + base) : -INFINITY, real ? b * V + token : INT32_MAX, lane);
  }
  if (special) {
    // A row without a candidate above -inf: its first tokens, as far as they can be wanted.  A row with infinite logits:
    // the first of its other tokens, whose score is -inf (at most `count` of the infinite ones come before them).
    const int reach = min(2 * count, V);
    for (int c0 = wave * MI_WAVE; c0 < beams * reach; c0 += BEAM_THREADS) {
      const int c = c0 + lane, b = min(c / reach, beams - 1), token = c % reach;
      bool real = c < beams * reach;
      if (real && row_base[b] == row_base[b]) real = row_max[b] == INFINITY && logits[(r0 + b) * row_stride + token] != INFINITY;
      best.take(-INFINITY, real ? b * V + token : INT32_MAX, lane);
    }
  }
  if (lane < count) {
    xs[wave * count + lane] = best.x;
    is[wave * count + lane] = best.i;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < BEAM_WAVES * count; i += BEAM_THREADS) {
    const int place = joined_place(xs, is, BEAM_WAVES, count, i / count, i % count);
    if (place < count) {
      const int64_t to = (int64_t)blockIdx.x * count + place;
      out_scores[to] = (float)xs[i];
      out_beams[to] = is[i] / V;
      out_tokens[to] = is[i] % V;
    }
  }
}

// Tiles to a wave: one while that leaves waves for every compute unit's sixteen, else as many as make that many.
static int tiles_of(int64_t rows, int V, int units) {
  const int64_t tiles = ((int64_t)V + BEAM_TILE - 1) / BEAM_TILE;
  const int64_t n = (rows * tiles + 16 * (int64_t)units - 1) / (16 * (int64_t)units);
  return (int)(n < 1 ? 1 : n);
}

static int parts_of(int V, int tiles) {
  const int64_t all = ((int64_t)V + BEAM_TILE - 1) / BEAM_TILE;
  return (int)((all + (int64_t)tiles * BEAM_WAVES - 1) / ((int64_t)tiles * BEAM_WAVES));
}

// Scratch of mi_beam_select, in 8-byte words.
MI_EXPORT int64_t mi_beam_scratch(int groups, int beams, int V, int count, int units) {
  const int64_t rows = (int64_t)groups * beams, parts = parts_of(V, tiles_of(rows, V, units));
  return rows * parts * (2 + count);
}

MI_EXPORT int mi_beam_select(const float* logits, int64_t row_stride, const float* scores, int groups, int beams, int V,
                             int count, int units, double* scratch, float* out_scores, int* out_beams, int* out_tokens,
                             hipStream_t stream) {
  MI_REQUIRE(groups >= 0 && beams >= 1 && V >= 1 && row_stride >= V && units >= 1, "beam_select: bad sizes groups=%d beams=%d V=%d stride=%lld",
             groups, beams, V, (long long)row_stride);
  MI_REQUIRE(beams <= BEAM_MAX_BEAMS && (int64_t)beams * V < INT32_MAX, "beam_select: %d beams x %d tokens, at most %d beams and 2^31 together",
             beams, V, BEAM_MAX_BEAMS);
  MI_REQUIRE(count >= 1 && count <= BEAM_MAX_COUNT && count <= (int64_t)beams * V,
             "beam_select: %d candidates of %d beams x %d tokens (at most %d)", count, beams, V, BEAM_MAX_COUNT);
  if (groups == 0) return 0;
  const int64_t rows = (int64_t)groups * beams;
  const int tiles = tiles_of(rows, V, units), parts = parts_of(V, tiles);
  MI_REQUIRE(rows * parts <= 0x7fffffff && (int64_t)beams * parts * count <= 0x7fffffff, "beam_select: too many rows (%lld) for one launch", (long long)rows);
  BeamParts p;
  p.sum = scratch;
  p.max = (float*)(scratch + rows * parts);
  p.x = (float*)(scratch + 2 * rows * parts);
  p.token = (int*)(p.x + rows * parts * count);
  beam_rows_kernel<<<(uint32_t)(rows * parts), BEAM_THREADS, 0, stream>>>(logits, row_stride, V, count, parts, tiles, p);
  MI_CHECK_LAUNCH("beam rows");
  beam_pick_kernel<<<groups, BEAM_THREADS, 0, stream>>>(logits, row_stride, scores, p, beams, count, parts, V, out_scores,
                                                        out_beams, out_tokens);
  MI_CHECK_LAUNCH("beam pick");
  return 0;
}
