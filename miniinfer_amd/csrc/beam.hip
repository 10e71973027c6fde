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
// are 64-bit; the exponential is a polynomial good to 3e-12, half of the arithmetic of the pass, and hides behind the
// loads.  The running scores come and go in 32 or 64 bits: a search that keeps them in 64 keeps that order from step to step.
#include "common.h"

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef f32x4 f32x4_any __attribute__((aligned(4)));      // 16 bytes from any element on

#define BEAM_MAX_COUNT 64
#define BEAM_MAX_BEAMS 64
#define BEAM_WAVES 4
#define BEAM_THREADS (BEAM_WAVES * MI_WAVE)
#define BEAM_FEW 1024                  // up to so many candidates of a group, four waves pick
#define BEAM_TILE 1024                 // logits that a wave holds at once, 16 to a lane

// The order of candidates.  An empty place is (-inf, INT_MAX): every real candidate comes before it.
template <typename X>
__device__ __forceinline__ bool before(X ax, int ai, X bx, int bi) { return (ax > bx) | ((ax == bx) & (ai < bi)); }

__device__ __forceinline__ float lane_value(float x, int lane) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), lane)); }
__device__ __forceinline__ double lane_value(double x, int lane) {
  return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(x), lane), __builtin_amdgcn_readlane(__double2loint(x), lane));
}
// The value of lane l ^ step, without a way through LDS: permutations within 4, 8 and 16 lanes, swaps of rows of 16 and of
// halves of the wave.  `step`: a power of two, a constant where this is inlined.
__device__ __forceinline__ int xor_lane(int x, int step, int lane) {
#define PERMUTED(X, CTRL) __builtin_amdgcn_update_dpp(X, X, CTRL, 0xf, 0xf, false)
  switch (step) {
    case 1: return PERMUTED(x, 0xB1);                           // quad_perm [1, 0, 3, 2]
    case 2: return PERMUTED(x, 0x4E);                           // quad_perm [2, 3, 0, 1]
    case 4: {
      const int y = PERMUTED(x, 0x141);                         // row_half_mirror: l ^ 7, then l ^ 3
      return PERMUTED(y, 0x1B);                                 // quad_perm [3, 2, 1, 0]
    }
    case 8: return PERMUTED(x, 0x128);                          // row_ror:8
    case 16: {
      const auto r = __builtin_amdgcn_permlane16_swap((uint32_t)x, (uint32_t)x, false, false);
      return (lane & 16) ? (int)r[0] : (int)r[1];
    }
    default: {
      const auto r = __builtin_amdgcn_permlane32_swap((uint32_t)x, (uint32_t)x, false, false);
      return (lane & 32) ? (int)r[0] : (int)r[1];
    }
  }
}
__device__ __forceinline__ float xor_lane(float x, int step, int lane) { return __int_as_float(xor_lane(__float_as_int(x), step, lane)); }
__device__ __forceinline__ double xor_lane(double x, int step, int lane) {
  return __hiloint2double(xor_lane(__double2hiint(x), step, lane), xor_lane(__double2loint(x), step, lane));
}
__device__ __forceinline__ uint64_t xor_lane(uint64_t x, int step, int lane) {
  return (uint64_t)(uint32_t)xor_lane((int)(x >> 32), step, lane) << 32 | (uint32_t)xor_lane((int)x, step, lane);
}
// The value of lane 63 - l.
__device__ __forceinline__ int mirrored(int x, int lane) {
  return xor_lane(xor_lane(PERMUTED(x, 0x140), 16, lane), 32, lane);       // row_mirror
}
__device__ __forceinline__ double mirrored(double x, int lane) {
  return __hiloint2double(mirrored(__double2hiint(x), lane), mirrored(__double2loint(x), lane));
}
__device__ __forceinline__ uint64_t mirrored(uint64_t x, int lane) {
  return (uint64_t)(uint32_t)mirrored((int)(x >> 32), lane) << 32 | (uint32_t)mirrored((int)x, lane);
}
#undef PERMUTED
__device__ __forceinline__ double sum_of_lanes(double x, int lane) {
#pragma unroll
  for (int step = 1; step < MI_WAVE; step <<= 1) x += xor_lane(x, step, lane);
  return x;
}
// The largest value of the wave, in a scalar register.
__device__ __forceinline__ float wave_top(float x, int lane) {
#pragma unroll
  for (int step = 1; step < MI_WAVE; step <<= 1) x = fmaxf(x, xor_lane(x, step, lane));
  return lane_value(x, 0);
}
// What at least `count` of the lanes' values reach: the count-th largest of them (the lanes sorted, largest first, by a
// bitonic network).
__device__ __forceinline__ float reached_by(float x, int count, int lane) {
#pragma unroll
  for (int k = 2; k <= MI_WAVE; k <<= 1)
#pragma unroll
    for (int step = k >> 1; step > 0; step >>= 1) {
      const float o = xor_lane(x, step, lane);
      x = ((lane & k) == 0) == ((lane & step) == 0) ? fmaxf(x, o) : fminf(x, o);
    }
  return lane_value(x, count - 1);
}

// A wave's best candidates: lane l holds the l-th in order.  Newcomers that come before the last of the `count` that are
// wanted gather in LDS and join 64 at a time: sorted (a bitonic network over the lanes), then merged.  One by one they
// would cost a tenth of a microsecond each, and a wave meets `count` * (1 + ln(logits / count)) of them.
template <typename X>
struct Best {
  X x;
  int i;
  int count, waiting;
  X last_x;          // the last of the `count`: what a newcomer has to come before
  int last_i;
  X* wait_x;         // room for 63 that wait and what is taken until the next `join`
  int* wait_i;
  __device__ __forceinline__ Best(int n, X* wx, int* wi)
      : x(-INFINITY), i(INT32_MAX), count(n), waiting(0), last_i(INT32_MAX), wait_x(wx), wait_i(wi) {
    // (the compiler loads a 64-bit -inf into a scalar register pair as zero, so that it must not know this value)
    asm volatile("" : "+v"(x));
    last_x = lane_value(x, 0);
  }
  // A candidate as one number that compares as candidates do, where it fits: the float's bits made to order as whole
  // numbers do, then the index, lower ones first.
  static __device__ __forceinline__ uint64_t key_of(float x, int i) {
    const uint32_t u = __float_as_uint(x + 0.f);       // (-0 and 0 are equal)
    return (uint64_t)((u & 0x80000000u) ? ~u : (u | 0x80000000u)) << 32 | (uint32_t)~i;
  }
  // the wave's candidates and those of the lanes `step` away: the better one to the lanes where `up`
  static __device__ __forceinline__ void exchange(uint64_t& k, int step, bool up, int lane) {
    const uint64_t o = xor_lane(k, step, lane);
    k = (o > k) == up ? o : k;
  }
  static __device__ __forceinline__ void exchange(double& x, int& i, int step, bool up, int lane) {
    const double ox = xor_lane(x, step, lane);
    const int oi = xor_lane(i, step, lane);
    const bool take = before(ox, oi, x, i) == up;
    x = take ? ox : x;
    i = take ? oi : i;
  }
  // The better of the list's and the newcomers' candidates, best first.  The newcomers are sorted; of the list, and of
  // the newcomers in rising order, the better one lane by lane are the best 64, falling, then rising; merged.
  static __device__ __forceinline__ void merge(float& x, int& i, float nx, int ni, int lane) {
    uint64_t n = key_of(nx, ni), own = key_of(x, i);
#pragma unroll
    for (int k = 2; k <= MI_WAVE; k <<= 1)
#pragma unroll
      for (int step = k >> 1; step > 0; step >>= 1) exchange(n, step, ((lane & k) == 0) == ((lane & step) == 0), lane);
    const uint64_t r = mirrored(n, lane);
    own = r > own ? r : own;
#pragma unroll
    for (int step = MI_WAVE / 2; step > 0; step >>= 1) exchange(own, step, (lane & step) == 0, lane);
    const uint32_t u = (uint32_t)(own >> 32);
    x = __uint_as_float((u & 0x80000000u) ? u & 0x7fffffffu : ~u);
    i = ~(int)own;
  }
  static __device__ __forceinline__ void merge(double& x, int& i, double nx, int ni, int lane) {
#pragma unroll
    for (int k = 2; k <= MI_WAVE; k <<= 1)
#pragma unroll
      for (int step = k >> 1; step > 0; step >>= 1) exchange(nx, ni, step, ((lane & k) == 0) == ((lane & step) == 0), lane);
    const double rx = mirrored(nx, lane);
    const int ri = mirrored(ni, lane);
    const bool newer = before(rx, ri, x, i);
    x = newer ? rx : x;
    i = newer ? ri : i;
#pragma unroll
    for (int step = MI_WAVE / 2; step > 0; step >>= 1) exchange(x, i, step, (lane & step) == 0, lane);
  }
  // one candidate of every lane (`real` of them)
  __device__ __forceinline__ void take(X nx, int ni, bool real, int lane) {
    const uint64_t mask = __ballot(real & before(nx, ni, last_x, last_i));
    if ((mask >> lane) & 1) {
      const int at = waiting + __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
      wait_x[at] = nx;
      wait_i[at] = ni;
    }
    waiting += __builtin_popcountll(mask);
  }
  // those that wait, as far as they are whole 64s or, with `all`, to the last
  __device__ __forceinline__ void join(int lane, bool all) {
    int from = 0;
    for (; waiting - from >= MI_WAVE || (all && waiting > from); from += MI_WAVE) {
      X nx = -INFINITY;
      int ni = INT32_MAX;
      if (from + lane < waiting) {
        nx = wait_x[from + lane];
        ni = wait_i[from + lane];
      }
      merge(x, i, nx, ni, lane);
      last_x = lane_value(x, count - 1);
      last_i = __builtin_amdgcn_readlane(i, count - 1);
    }
    if (from) {                        // the rest, fewer than 64, moves to the front
      waiting = max(waiting - from, 0);
      if (lane < waiting) {
        const X rx = wait_x[from + lane];
        const int ri = wait_i[from + lane];
        wait_x[lane] = rx;
        wait_i[lane] = ri;
      }
    }
  }
};

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

// e^d for d <= 0, to 3e-12 of its value: with t = d / ln 2, n the whole number next to it and f = t - n, 2^n 2^f;
// 2^f = 1 + f q(f), where q interpolates at the eight Chebyshev points of [-1/2, 1/2], so e^0 is 1.  The coefficients sit
// in scalar registers, which the multiply-adds take as they are (constants are copied into vector registers before each).
struct Exponential {
  double c[8];
  __device__ __forceinline__ Exponential()
      : c{0.6931471805568324, 0.2402265069588842, 0.05550410906325485, 0.009618129135261179, 0.0013333478474028277,
          0.0001540347517242934, 1.5303700625385598e-05, 1.3250807607943917e-06} {
#pragma unroll
    for (int i = 0; i < 8; ++i) asm volatile("" : "+s"(c[i]));
  }
  __device__ __forceinline__ double operator()(double d) const {
    const double t = fmax(d * 1.4426950408889634, -1100.0);       // (2^-1100 is 0)
    const double n = __builtin_rint(t), f = t - n;
    double p = fma(c[7], f, c[6]);
#pragma unroll
    for (int i = 5; i >= 0; --i) p = fma(p, f, c[i]);
    return __builtin_ldexp(fma(p, f, 1.0), (int)n);
  }
  // Four at once, the steps of one between those of the others: sums[j] += e^(x[j] - m).  PLAIN: no x is 700 or more below
  // m, and |m| is so small that x / ln 2 - m / ln 2 is as good as (x - m) / ln 2.
  template <bool PLAIN>
  __device__ __forceinline__ void add(double (&sums)[4], f32x4 x, double m) const {
    double f[4], p[4];
    int n[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const double t = PLAIN ? fma((double)x[j], 1.4426950408889634, m * -1.4426950408889634)
                             : fmax(((double)x[j] - m) * 1.4426950408889634, -1100.0);
      const double r = __builtin_rint(t);
      f[j] = t - r;
      n[j] = (int)r;
      p[j] = fma(c[7], f[j], c[6]);
    }
#pragma unroll
    for (int i = 5; i >= 0; --i)
#pragma unroll
      for (int j = 0; j < 4; ++j) p[j] = fma(p[j], f[j], c[i]);
#pragma unroll
    for (int j = 0; j < 4; ++j) sums[j] += __builtin_ldexp(fma(p[j], f[j], 1.0), n[j]);
  }
};

// The 16 logits of a lane in the tile at `at`: pieces of 4 side by side, -inf past the row's end.
__device__ __forceinline__ void load_tile(const float* __restrict__ row, int64_t at, int V, int lane, f32x4 (&x)[4]) {
  if (at + BEAM_TILE <= V) {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = *reinterpret_cast<const f32x4_any*>(row + at + (j * MI_WAVE + lane) * 4);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int64_t e = at + (j * MI_WAVE + lane) * 4 + c;
        x[j][c] = e < V ? row[e] : -INFINITY;
      }
  }
}

struct BeamParts {
  double* sum;             // [rows][parts]: of exp(x - max)
  float* max;              // [rows][parts]
  float* x;                // [rows][parts][count], in order
  int* token;
};

// Block (part, row): `tiles` tiles to a wave.
// (four workgroups to a compute unit, as many as the launch has for each)
__global__ __launch_bounds__(BEAM_THREADS, 4) void beam_rows_kernel(const float* __restrict__ logits, int64_t row_stride, int V,
                                                                 int count, int parts, int tiles, BeamParts out) {
  __shared__ float xs[BEAM_WAVES * BEAM_MAX_COUNT];
  __shared__ int is[BEAM_WAVES * BEAM_MAX_COUNT];
  __shared__ float wait_x[BEAM_WAVES][BEAM_TILE + MI_WAVE];
  __shared__ int wait_i[BEAM_WAVES][BEAM_TILE + MI_WAVE];
  __shared__ float maxima[BEAM_WAVES];
  __shared__ double sums[BEAM_WAVES];
  const int lane = threadIdx.x & (MI_WAVE - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / MI_WAVE);
  const int64_t r = blockIdx.x / parts;
  const int part = blockIdx.x % parts;
  const float* row = logits + r * row_stride;
  const Exponential exp_of;
  Best<float> best(count, wait_x[wave], wait_i[wave]);
  float m = -INFINITY;
  double sum[4] = {0.0, 0.0, 0.0, 0.0};
  // The part's tiles go round the waves.  Which lane adds up a logit follows from its index alone: equal rows have equal
  // sums wherever they lie.
  const int64_t first = ((int64_t)part * tiles * BEAM_WAVES + wave) * BEAM_TILE;
  constexpr int64_t step = BEAM_WAVES * BEAM_TILE;
  f32x4 next[4];
  if (first < V) load_tile(row, first, V, lane, next);
  for (int t = 0; t < tiles; ++t) {
    const int64_t at = first + t * step;
    if (at >= V) break;
    f32x4 x[4];
    float top = -INFINITY;
    float tops[4];                         // of a lane's pieces
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[j] = next[j];
      tops[j] = fmaxf(fmaxf(fmaxf(x[j][0], x[j][1]), fmaxf(x[j][2], x[j][3])), -INFINITY);   // (of a NaN and another value the other)
      top = fmaxf(top, tops[j]);
    }
    if (t + 1 < tiles && at + step < V) load_tile(row, at + step, V, lane, next);
    const float tile_top = wave_top(top, lane);
    if (tile_top > m) {
      const double less = exp_of((double)m - (double)tile_top);
#pragma unroll
      for (int c = 0; c < 4; ++c) sum[c] *= less;
      m = tile_top;
    }
    // (mask values, infinities, NaN, far outliers)
    bool odd = !(fabsf(m) < 1e4f);
    const float low = m - 700.f;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) odd |= !(x[j][c] >= low);
    if (__ballot(odd) == 0) {
#pragma unroll
      for (int j = 0; j < 4; ++j) exp_of.add<true>(sum, x[j], (double)m);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          x[j][c] = x[j][c] == x[j][c] ? x[j][c] : -INFINITY;         // a NaN counts as -inf
          if (m == INFINITY) sum[c] += x[j][c] == INFINITY ? 1.0 : 0.0;         // (only such logits have a share)
        }
      if (m > -INFINITY && m < INFINITY) {
#pragma unroll
        for (int j = 0; j < 4; ++j) exp_of.add<false>(sum, x[j], (double)m);
      }
    }
    // the candidates
    const float bar = t == 0 ? reached_by(top, count, lane) : best.last_x;
    if (tile_top >= bar) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (__ballot(tops[j] >= bar) == 0) continue;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          if (__ballot(x[j][c] >= bar) == 0) continue;
          const int e = (int)at + (j * MI_WAVE + lane) * 4 + c;
          best.take(x[j][c], e, (e < V) & (x[j][c] >= bar), lane);
        }
      }
    }
    best.join(lane, t == 0 || t + 1 == tiles || at + step >= V);
  }
  if (lane < count) {
    xs[wave * count + lane] = best.x;
    is[wave * count + lane] = best.i;
  }
  const double s = sum_of_lanes((sum[0] + sum[1]) + (sum[2] + sum[3]), lane);
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
    double total = 0.0;
    for (int w = 0; w < BEAM_WAVES; ++w)
      total += maxima[w] == all ? sums[w] : sums[w] * exp_of((double)maxima[w] - (double)all);
    out.max[to] = all;
    out.sum[to] = total;
  }
}

// Block: a group.  S: the type of the running scores.
template <int WAVES, typename S>
__global__ __launch_bounds__(WAVES * MI_WAVE) void beam_pick_kernel(const float* __restrict__ logits, int64_t row_stride,
                                                                 const S* __restrict__ scores, BeamParts in, int beams,
                                                                 int count, int parts, int V, S* __restrict__ out_scores,
                                                                 int* __restrict__ out_beams, int* __restrict__ out_tokens) {
  __shared__ float row_max[BEAM_MAX_BEAMS];
  __shared__ double row_base[BEAM_MAX_BEAMS];      // scores[b] - log of the row's sum; NaN: no candidate above -inf
  __shared__ int special;                          // rows whose lists do not say it all
  __shared__ double wait_x[WAVES][2 * MI_WAVE];
  __shared__ int wait_i[WAVES][2 * MI_WAVE];
  __shared__ double xs[WAVES * BEAM_MAX_COUNT];
  __shared__ int is[WAVES * BEAM_MAX_COUNT];
  const int lane = threadIdx.x & (MI_WAVE - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / MI_WAVE);
  const int64_t r0 = (int64_t)blockIdx.x * beams;
  const Exponential exp_of;
  if (threadIdx.x == 0) special = 0;
  __syncthreads();
  // 16 lanes to a row: what its parts say, all rows of a wave's lanes at once
  for (int b0 = 0; b0 < beams; b0 += WAVES * 4) {
    const int b = b0 + wave * 4 + lane / 16, l = lane & 15;
    float m = -INFINITY;
    if (b < beams)
      for (int p = l; p < parts; p += 16) m = fmaxf(m, in.max[(r0 + b) * parts + p]);
#pragma unroll
    for (int step = 1; step < 16; step <<= 1) m = fmaxf(m, xor_lane(m, step, lane));
    double s = 0.0;
    if (b < beams)
      for (int p = l; p < parts; p += 16) {
        const float pm = in.max[(r0 + b) * parts + p];
        const double ps = in.sum[(r0 + b) * parts + p];
        s += pm == m ? ps : ps * exp_of((double)pm - (double)m);
      }
#pragma unroll
    for (int step = 1; step < 16; step <<= 1) s += xor_lane(s, step, lane);
    if (b < beams && l == 0) {
      const double start = (double)scores[r0 + b];
      const bool dead = !(fabs(start) < INFINITY) || m == -INFINITY;
      row_max[b] = m;
      row_base[b] = dead ? NAN : start - log(s);
      if (dead || m == INFINITY) special = 1;
    }
  }
  __syncthreads();
  Best<double> best(count, wait_x[wave], wait_i[wave]);
  const int lists = parts * count, n = beams * lists;
  // ...the lists, then, where one of the rows is special: of a row without a candidate above -inf its first tokens, as far
  // as they can be wanted; of a row with infinite logits the first of its other tokens, whose score is -inf (at most
  // `count` of the infinite ones come before them)
  const int reach = min(2 * count, V), all = n + (special ? beams * reach : 0);
  const int rounds = (all + WAVES * MI_WAVE - 1) / (WAVES * MI_WAVE);
  for (int round = 0; round < rounds; ++round) {
    const int c = (round * WAVES + wave) * MI_WAVE + lane;
    const bool listed = c < n;
    const int b = min(listed ? c / lists : (c - n) / reach, beams - 1);
    const double base = row_base[b];
    const float m = row_max[b];
    float x = -INFINITY;
    int token = listed ? in.token[r0 * lists + c] : (c - n) % reach;
    if (listed) x = in.x[r0 * lists + c];
    bool real;
    if (listed) real = token != INT32_MAX && base == base && (m < INFINITY || x == INFINITY);
    else real = c < all && (base != base || (m == INFINITY && logits[(r0 + b) * row_stride + token] != INFINITY));
    best.take(!listed ? -INFINITY : x == m ? base : (double)x - (double)m + base, real ? b * V + token : INT32_MAX, real, lane);
    best.join(lane, round + 1 == rounds);
  }
  if (lane < count) {
    xs[wave * count + lane] = best.x;
    is[wave * count + lane] = best.i;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < WAVES * count; i += WAVES * MI_WAVE) {
    const int place = joined_place(xs, is, WAVES, count, i / count, i % count);
    if (place < count) {
      const int64_t to = (int64_t)blockIdx.x * count + place;
      out_scores[to] = (S)xs[i];
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

// wide: scores and out_scores are double, else float.
MI_EXPORT int mi_beam_select(const float* logits, int64_t row_stride, const void* scores, int groups, int beams, int V,
                             int count, int units, int wide, double* scratch, void* out_scores, int* out_beams, int* out_tokens,
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
  const bool many = beams * parts * count > BEAM_FEW;
#define PICK(WAVES, S)                                                                                                  \
  beam_pick_kernel<WAVES, S><<<groups, WAVES * MI_WAVE, 0, stream>>>(logits, row_stride, (const S*)scores, p, beams, count, parts, V, \
                                                                     (S*)out_scores, out_beams, out_tokens)
  if (many && wide) PICK(16, double);
  else if (many) PICK(16, float);
  else if (wide) PICK(4, double);
  else PICK(4, float);
#undef PICK
  MI_CHECK_LAUNCH("beam pick");
  return 0;
}
