// Linear attention with a decay for each head, over fixed-size states.
//
//   S_t = a S_{t-1} + k_t v_t^T        S [d, d] float32 per request and kv head, a = exp(log_decay[kv head])
//   o_t = scale * q_t S_t              for each of the kv head's query heads
//
// The recurrent form: a workgroup owns 32 columns of one request's and kv head's state in registers and takes the
// tokens one after the other.  It is the whole operator for single tokens, which are bound by the state's bytes (read
// and written once).
#include "common.h"

#include <atomic>

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

#define LA_THREADS 256
#define LA_COLS 32                        // columns of the state to a workgroup: whole 128-byte lines
#define LA_ROW_GROUPS (LA_THREADS / (LA_COLS / 4))
#define LA_MAX_D 256
#define LA_MAX_ROWS (LA_MAX_D / LA_ROW_GROUPS)

__device__ __forceinline__ float decay_power(float log_decay, int n) {   // a^n; a^0 = 1 for a decay of zero too
  return n == 0 ? 1.f : (float)exp((double)log_decay * n);
}

// cu == nullptr: request b's only token is token b.
template <typename T, int NR>   // NR: rows of the state that a thread holds
__global__ __launch_bounds__(LA_THREADS) void la_recurrent_kernel(
    const T* __restrict__ q, int64_t q_stride, const T* __restrict__ k, int64_t k_stride, const T* __restrict__ v,
    int64_t v_stride, T* __restrict__ out, int64_t out_stride, float* __restrict__ state, int64_t state_stride,
    int num_rows, const int* __restrict__ rows, const int* __restrict__ cu, int num_tokens, int nkv, int rep, int d,
    const float* __restrict__ log_decay, float scale) {
  __shared__ float part[2][LA_THREADS / MI_WAVE][LA_COLS];
  const int h = blockIdx.x % nkv, slice = blockIdx.x / nkv, b = blockIdx.y;
  const int lo = cu ? min(max(cu[b], 0), num_tokens) : b;
  const int hi = cu ? min(max(cu[b + 1], 0), num_tokens) : b + 1;
  if (lo >= hi) return;
  const int tx = threadIdx.x % (LA_COLS / 4), ty = threadIdx.x / (LA_COLS / 4);
  const int lane = threadIdx.x & (MI_WAVE - 1), wave = threadIdx.x / MI_WAVE;
  const int c0 = slice * LA_COLS + tx * 4;
  const bool live = c0 < d;
  const int row = rows[b];
  const int q0 = h * rep;
  if (row < 0 || row >= num_rows) {       // no such state: rows of NaN
    for (int t = lo; t < hi; ++t)
      for (int i = threadIdx.x; i < rep * LA_COLS; i += LA_THREADS)
        if (slice * LA_COLS + i % LA_COLS < d)
          out[(int64_t)t * out_stride + (int64_t)(q0 + i / LA_COLS) * d + slice * LA_COLS + i % LA_COLS] = from_float<T>(NAN);
    return;
  }
  float* s_at = state + (int64_t)row * state_stride + (int64_t)h * d * d + c0;
  f32x4 s[NR];
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    const int i = ty + r * LA_ROW_GROUPS;
    s[r] = live && i < d ? *reinterpret_cast<const f32x4*>(s_at + (int64_t)i * d) : f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const float a = decay_power(log_decay[h], 1);
  int turn = 0;
  for (int t = lo; t < hi; ++t) {
    const T* kt = k + (int64_t)t * k_stride + (int64_t)h * d;
    const T* vt = v + (int64_t)t * v_stride + (int64_t)h * d + c0;
    f32x4 vv = {0.f, 0.f, 0.f, 0.f};
    if (live) vv = f32x4{to_float(vt[0]), to_float(vt[1]), to_float(vt[2]), to_float(vt[3])};
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const int i = ty + r * LA_ROW_GROUPS;
      if (i < d) {
        const float kk = to_float(kt[i]);
#pragma unroll
        for (int c = 0; c < 4; ++c) s[r][c] = fmaf(kk, vv[c], a * s[r][c]);
      }
    }
    for (int g = 0; g < rep; ++g) {
      const T* qt = q + (int64_t)t * q_stride + (int64_t)(q0 + g) * d;
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        const int i = ty + r * LA_ROW_GROUPS;
        if (i < d) {
          const float qq = to_float(qt[i]);
#pragma unroll
          for (int c = 0; c < 4; ++c) o[c] = fmaf(qq, s[r][c], o[c]);
        }
      }
#pragma unroll
      for (int x = LA_COLS / 4; x < MI_WAVE; x <<= 1)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[c] += __shfl_xor(o[c], x, MI_WAVE);
      if (lane < LA_COLS / 4)
#pragma unroll
        for (int c = 0; c < 4; ++c) part[turn][wave][tx * 4 + c] = o[c];
      __syncthreads();        // (the other half of `part` is written next: one barrier a round is enough)
      const int c = threadIdx.x;
      if (c < LA_COLS && slice * LA_COLS + c < d) {
        float sum = 0.f;
        for (int w = 0; w < LA_THREADS / MI_WAVE; ++w) sum += part[turn][w][c];
        out[(int64_t)t * out_stride + (int64_t)(q0 + g) * d + slice * LA_COLS + c] = from_float<T>(sum * scale);
      }
      turn ^= 1;
    }
  }
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    const int i = ty + r * LA_ROW_GROUPS;
    if (live && i < d) *reinterpret_cast<f32x4*>(s_at + (int64_t)i * d) = s[r];
  }
}

template <typename T>
static void launch_recurrent(const void* q, int64_t q_stride, const void* k, int64_t k_stride, const void* v,
                             int64_t v_stride, void* out, int64_t out_stride, float* state, int64_t state_stride,
                             int num_rows, const int* rows, const int* cu, int num_tokens, int num_requests, int nq,
                             int nkv, int d, const float* log_decay, float scale, hipStream_t stream) {
  const dim3 grid(nkv * ((d + LA_COLS - 1) / LA_COLS), num_requests);
  const int nr = (d + LA_ROW_GROUPS - 1) / LA_ROW_GROUPS;
#define LAUNCH(N)                                                                                                     \
  la_recurrent_kernel<T, N><<<grid, LA_THREADS, 0, stream>>>((const T*)q, q_stride, (const T*)k, k_stride, (const T*)v, \
                                                             v_stride, (T*)out, out_stride, state, state_stride, num_rows, rows, \
                                                             cu, num_tokens, nkv, nq / nkv, d, log_decay, scale)
  if (nr <= 2) LAUNCH(2);
  else if (nr <= 4) LAUNCH(4);
  else LAUNCH(8);
#undef LAUNCH
}

#define LA_ARGS                                                                                                       \
  int dtype, const void *q, int64_t q_stride, const void *k, int64_t k_stride, const void *v, int64_t v_stride, void *out, \
      int64_t out_stride, float *state, int64_t state_stride, int num_rows, const int *rows, const int *cu, int num_tokens, \
      int num_requests, int nq, int nkv, int d, const float *log_decay, float scale

static int check_sizes(int nq, int nkv, int d, int num_requests, int64_t state_stride) {
  MI_REQUIRE(d >= 8 && d <= LA_MAX_D && d % 8 == 0, "linear attention: head size %d is no multiple of 8 up to %d", d, LA_MAX_D);
  MI_REQUIRE(nkv >= 1 && nq >= nkv && nq % nkv == 0, "linear attention: %d query heads are no multiple of %d kv heads", nq, nkv);
  MI_REQUIRE(num_requests >= 0 && num_requests <= 65535, "linear attention: %d requests, at most 65535 in a launch", num_requests);
  MI_REQUIRE(state_stride % 4 == 0, "linear attention: rows of states must be a multiple of 16 bytes apart");
  return 0;
}

MI_EXPORT int mi_linear_attention_recurrent(LA_ARGS, hipStream_t stream) {
  if (check_sizes(nq, nkv, d, num_requests, state_stride)) return 1;
  if (num_requests == 0 || num_tokens == 0) return 0;
  if (dtype == MI_DTYPE_BF16)
    launch_recurrent<bf16>(q, q_stride, k, k_stride, v, v_stride, out, out_stride, state, state_stride, num_rows, rows, cu,
                           num_tokens, num_requests, nq, nkv, d, log_decay, scale, stream);
  else if (dtype == MI_DTYPE_F32)
    launch_recurrent<float>(q, q_stride, k, k_stride, v, v_stride, out, out_stride, state, state_stride, num_rows, rows, cu,
                            num_tokens, num_requests, nq, nkv, d, log_decay, scale, stream);
  else
    MI_FAIL("linear attention: dtype %d", dtype);
  MI_CHECK_LAUNCH("linear attention");
  return 0;
}

// ---------------------------------------------------------------- prompts: chunks of C tokens on the matrix cores
//
// With S the state before a chunk, i and j tokens of it, n how many it has (the rest of its C rows are zeros):
//
//   O[i]  = scale * ( a^(i+1) q_i S  +  sum_{j <= i} a^(i-j) (q_i . k_j) v_j )
//   S'    = a^n S + sum_j a^(n-1-j) k_j v_j^T
//
// Every power has an exponent of 0 or more, so nothing overflows however fast a head forgets.  A workgroup owns VS
// columns of one request's (or segment's) and kv head's state and walks over the chunks; a wave owns 16 NT of the
// columns and keeps them, [DP, 16 NT] in 32 bits, in registers as the accumulators of the last product.  Products:
//
//   P^T = K Q^T        by blocks of 16 queries, one to a wave; weighted, masked, through LDS to every wave
//   O^T = S^T Q^T      S from the accumulators' registers: an accumulator's lanes sit where an operand's do
//   O^T += V^T P^T     V^T by the LDS's transposing reads
//   S  += K^T (w V)    K^T likewise
//
// An operand of the matrix cores is 4 consecutive elements along the axis that is summed, from 16 rows and 4 groups of
// lanes (a "half"): bfloat16 takes two halves to a product (16x16x32), 32-bit one half to four (16x16x4).
// Roundings of the bfloat16 form: what is 32-bit (S, the weighted P and w V) is split into bfloat16 parts that are
// multiplied one after the other into the same accumulators: two parts (what is left out is 2^-17 of a term) for what
// ends in a bfloat16 output, three (2^-25) for the state, which is 32-bit whatever the inputs are.

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

#define LA_LDS(T) __attribute__((address_space(3))) T

template <typename T>
struct Half;      // 4 elements of an operand
template <>
struct Half<bf16> {
  typedef s16x4 type;
};
template <>
struct Half<float> {
  typedef f32x4 type;
};

__device__ __forceinline__ bf16x8 join(s16x4 a, s16x4 b) {
  return __builtin_bit_cast(bf16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}
// acc += A B over two 16-element pieces of the summed axis
__device__ __forceinline__ void mma(f32x4& acc, s16x4 a0, s16x4 a1, s16x4 b0, s16x4 b1) {
  acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(join(a0, a1), join(b0, b1), acc, 0, 0, 0);
}
__device__ __forceinline__ void mma(f32x4& acc, f32x4 a0, f32x4 a1, f32x4 b0, f32x4 b1) {
#pragma unroll
  for (int i = 0; i < 4; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a0[i], b0[i], acc, 0, 0, 0);
#pragma unroll
  for (int i = 0; i < 4; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a1[i], b1[i], acc, 0, 0, 0);
}
__device__ __forceinline__ s16x4 to_half(f32x4 x) { return __builtin_bit_cast(s16x4, __builtin_convertvector(x, bf16x4)); }
__device__ __forceinline__ f32x4 widen(s16x4 h) {
  const mi_u32x2 u = __builtin_bit_cast(mi_u32x2, h);
  return f32x4{__uint_as_float(u[0] << 16), __uint_as_float(u[0] & 0xffff0000u), __uint_as_float(u[1] << 16),
               __uint_as_float(u[1] & 0xffff0000u)};
}
__device__ __forceinline__ f32x4 widen(f32x4 h) { return h; }

// A 32-bit value as a sum of parts that the matrix cores take.
template <typename T, int PARTS>
struct Split;
template <int PARTS>
struct Split<bf16, PARTS> {
  s16x4 part[PARTS];
  __device__ __forceinline__ explicit Split(f32x4 x) {
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
      part[p] = to_half(x);
      if (p + 1 < PARTS) x -= widen(part[p]);
    }
  }
  static constexpr int parts = PARTS;
};
template <int PARTS>
struct Split<float, PARTS> {
  f32x4 part[1];
  __device__ __forceinline__ explicit Split(f32x4 x) : part{x} {}
  static constexpr int parts = 1;
};

// Tiles in LDS are rows of tokens.  A bfloat16 row is padded by 32 bytes and rows 8 .. 15 of every 16 are shifted by
// another 16: the 8-byte reads of a half (16 rows, 4 groups) and the transposing reads (4 rows of 32 bytes to 16 lanes)
// then meet every bank once.  32-bit rows are padded by 16 bytes.
template <typename T, int COLS>
struct Tile {
  static constexpr int stride = COLS * (int)sizeof(T) + (sizeof(T) == 2 ? 32 : 16);
  static constexpr int shift = sizeof(T) == 2 ? 16 : 0;
  static __device__ __forceinline__ int at(int row, int col) {
    return row * stride + ((row >> 3) & 1) * shift + col * (int)sizeof(T);
  }
  static constexpr int bytes(int rows) { return rows * stride + 16; }
};

template <typename T>
__device__ __forceinline__ typename Half<T>::type half_at(const char* p) {
  return *reinterpret_cast<const typename Half<T>::type*>(p);
}

// Elements [row 4 g .. 4 g + 3] of column l % 16 of a 16 x 16 piece whose first element is at (row0, col0): the lane's
// half along the rows.
template <int COLS>
__device__ __forceinline__ s16x4 half_down(const char* tile, int row0, int col0, int lane, bf16*) {
  const char* p = tile + Tile<bf16, COLS>::at(row0 + lane / 16 * 4 + lane % 16 / 4, col0 + lane % 4 * 4);
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((LA_LDS(s16x4)*)(LA_LDS(char)*)p);
}
template <int COLS>
__device__ __forceinline__ f32x4 half_down(const char* tile, int row0, int col0, int lane, float*) {
  f32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = *reinterpret_cast<const float*>(tile + Tile<float, COLS>::at(row0 + lane / 16 * 4 + i, col0 + lane % 16));
  return r;
}

// 16 bytes of a row of `d` columns from column c on (zeros past its end); `wide`: the row is 16-byte aligned
template <typename T>
__device__ __forceinline__ u32x4 piece_at(const T* row, int c, int d, bool wide) {
  u32x4 r = {0, 0, 0, 0};
  if (c < d) {
    if (wide) {
      r = *reinterpret_cast<const u32x4*>(row + c);
    } else {
      T tmp[16 / sizeof(T)];
#pragma unroll
      for (int i = 0; i < (int)(16 / sizeof(T)); ++i) tmp[i] = row[c + i];
      r = *reinterpret_cast<const u32x4*>(tmp);
    }
  }
  return r;
}
__device__ __forceinline__ bool all_finite(u32x4 x, bf16*) {
  bool ok = true;
#pragma unroll
  for (int i = 0; i < 4; ++i) ok = ok && (x[i] & 0x7f80u) != 0x7f80u && (x[i] & 0x7f800000u) != 0x7f800000u;
  return ok;
}
__device__ __forceinline__ bool all_finite(u32x4 x, float*) {
  bool ok = true;
#pragma unroll
  for (int i = 0; i < 4; ++i) ok = ok && (x[i] & 0x7f800000u) != 0x7f800000u;
  return ok;
}

struct LinearAttention {
  const void *q, *k, *v;
  void* out;
  float* state;
  const int *rows, *cu;
  const float* log_decay;
  float* work;                       // states at the segments' starts, [unit][nkv][d][d]
  int64_t q_stride, k_stride, v_stride, out_stride, state_stride;
  int num_rows, num_tokens, num_requests, nkv, rep, d;
  int segment;                       // tokens of a segment; 0: every request is one
  float scale;
  bool wide_q, wide_k, wide_v, wide_out;
};

// A request's segments are consecutive units from first_unit on: ceil(length / segment) of them fit before the next
// request's first one, and all units are fewer than num_tokens / segment + num_requests.
__device__ __forceinline__ void bounds_of(const LinearAttention& a, int b, int& lo, int& hi) {
  lo = min(max(a.cu[b], 0), a.num_tokens);
  hi = max(lo, min(a.cu[b + 1], a.num_tokens));
}
__device__ __forceinline__ int first_unit(const LinearAttention& a, int b) {
  return min(max(a.cu[b], 0), a.num_tokens) / a.segment + b;
}

template <typename T, int DP, int NT, int C>
struct ChunkShape {
  static constexpr int waves = 4, threads = 256;
  static constexpr int VS = 16 * NT * waves;
  static constexpr int kt = DP / 16, ct = C / 16;
  static constexpr int q_bytes = (Tile<T, DP>::bytes(C) + 15) / 16 * 16;
  static constexpr int v_bytes = (Tile<T, VS>::bytes(C) + 15) / 16 * 16;
  static constexpr int p_bytes = (Tile<T, C>::bytes(C) + 15) / 16 * 16;
  static constexpr int parts = sizeof(T) == 2 ? 2 : 1;
  static constexpr int lds(bool states) { return q_bytes + v_bytes + (states ? 0 : q_bytes + parts * p_bytes); }
};

// STATES: only what a segment adds to its request's state (from zero), left in `work`; the last segment's is not needed.
template <typename T, int DP, int NT, int C, bool STATES>
__global__ __launch_bounds__(256) void la_chunk_kernel(LinearAttention a) {
  typedef ChunkShape<T, DP, NT, C> Shape;
  typedef typename Half<T>::type half;
  typedef Tile<T, DP> QTile;
  typedef Tile<T, Shape::VS> VTile;
  typedef Tile<T, C> PTile;
  constexpr int KT = Shape::kt, CT = Shape::ct, VS = Shape::VS, PE = 16 / sizeof(T);
  extern __shared__ __attribute__((aligned(16))) char lds[];
  __shared__ float power[C + 1];
  __shared__ int found, not_finite;
  char* const k_lds = lds;
  char* const v_lds = k_lds + Shape::q_bytes;
  char* const q_lds = v_lds + Shape::v_bytes;
  char* const p_lds = q_lds + Shape::q_bytes;

  const int tid = threadIdx.x, lane = tid & (MI_WAVE - 1), wave = tid / MI_WAVE, l16 = lane & 15, g4 = lane / 16 * 4;
  const int slices = (a.d + VS - 1) / VS;
  const int h = blockIdx.x % a.nkv, slice = blockIdx.x / a.nkv % slices, unit = blockIdx.x / (a.nkv * slices);
  const int d = a.d;

  int b = unit, lo, hi, segment = 0, segments = 1;
  if (a.segment) {
    if (tid == 0) found = 0;
    __syncthreads();
    int n = 0;
    for (int i = tid; i < a.num_requests; i += Shape::threads) n += first_unit(a, i) <= unit;
    if (n) atomicAdd(&found, n);
    __syncthreads();
    b = found - 1;
    if (b < 0) return;
    bounds_of(a, b, lo, hi);
    segment = unit - first_unit(a, b);
    segments = (hi - lo + a.segment - 1) / a.segment;
    if (segment < 0 || segment >= segments) return;
    if (STATES && segment == segments - 1) return;
    lo += segment * a.segment;
    hi = min(hi, lo + a.segment);
  } else {
    bounds_of(a, b, lo, hi);
  }
  if (lo >= hi) return;

  const int n0 = slice * VS + wave * 16 * NT;            // first column of the wave
  const int row = a.rows[b];
  T* const out = (T*)a.out;
  if (row < 0 || row >= a.num_rows) {                    // no such state: rows of NaN
    if (!STATES)
      for (int t = lo; t < hi; ++t)
        for (int i = tid; i < a.rep * VS; i += Shape::threads)
          if (slice * VS + i % VS < d)
            out[(int64_t)t * a.out_stride + (int64_t)(h * a.rep + i / VS) * d + slice * VS + i % VS] = from_float<T>(NAN);
    return;
  }
  for (int i = tid; i <= C; i += Shape::threads) power[i] = decay_power(a.log_decay[h], i);
  if (tid == 0) not_finite = 0;

  // the wave's columns of the state, accumulator (nt, t): rows 16 t + g4 + i, column n0 + 16 nt + l16
  f32x4 s[NT][KT];
  float* const s_row = a.state + (int64_t)row * a.state_stride + (int64_t)h * d * d;
  float* const s_work = a.segment ? a.work + ((int64_t)unit * a.nkv + h) * d * d : nullptr;
  const float* const s_from = segments > 1 ? s_work : s_row;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 16 * t + g4 + i, c = n0 + 16 * nt + l16;
        s[nt][t][i] = !STATES && r < d && c < d ? s_from[(int64_t)r * d + c] : 0.f;
      }

  const T* const kp = (const T*)a.k + (int64_t)h * d;
  const T* const vp = (const T*)a.v + (int64_t)h * d;
  const T* const qp = (const T*)a.q + (int64_t)h * a.rep * d;

  // staging: a thread's pieces of a tile
  constexpr int KP = C * DP / PE / Shape::threads, VP = C * VS / PE / Shape::threads;
  static_assert(KP >= 1 && VP >= 1, "a tile has a piece for every thread");
  u32x4 kr[KP], vr[VP], qr[KP];
  auto load_k = [&](int t, int n) {
#pragma unroll
    for (int i = 0; i < KP; ++i) {
      const int p = tid + i * Shape::threads, r = p / (DP / PE), c = p % (DP / PE) * PE;
      kr[i] = r < n ? piece_at(kp + (int64_t)(t + r) * a.k_stride, c, d, a.wide_k) : u32x4{0, 0, 0, 0};
    }
#pragma unroll
    for (int i = 0; i < VP; ++i) {
      const int p = tid + i * Shape::threads, r = p / (VS / PE), c = p % (VS / PE) * PE + slice * VS;
      vr[i] = r < n ? piece_at(vp + (int64_t)(t + r) * a.v_stride, c, d, a.wide_v) : u32x4{0, 0, 0, 0};
    }
  };
  auto load_q = [&](int t, int n, int g) {
#pragma unroll
    for (int i = 0; i < KP; ++i) {
      const int p = tid + i * Shape::threads, r = p / (DP / PE), c = p % (DP / PE) * PE;
      qr[i] = r < n ? piece_at(qp + (int64_t)(t + r) * a.q_stride + (int64_t)g * d, c, d, a.wide_q) : u32x4{0, 0, 0, 0};
    }
  };
  auto store_q = [&]() {
#pragma unroll
    for (int i = 0; i < KP; ++i) {
      const int p = tid + i * Shape::threads;
      *reinterpret_cast<u32x4*>(q_lds + QTile::at(p / (DP / PE), p % (DP / PE) * PE)) = qr[i];
    }
  };
  auto store_k = [&]() -> bool {      // whether a value is not finite
    bool ok = true;
#pragma unroll
    for (int i = 0; i < KP; ++i) {
      const int p = tid + i * Shape::threads;
      *reinterpret_cast<u32x4*>(k_lds + QTile::at(p / (DP / PE), p % (DP / PE) * PE)) = kr[i];
    }
#pragma unroll
    for (int i = 0; i < VP; ++i) {
      const int p = tid + i * Shape::threads;
      *reinterpret_cast<u32x4*>(v_lds + VTile::at(p / (VS / PE), p % (VS / PE) * PE)) = vr[i];
      ok = ok && all_finite(vr[i], (T*)nullptr);
    }
    return !ok;
  };

  const int lane_q = QTile::at(l16, g4), lane_p = PTile::at(l16, g4);
  int t = lo, n = min(C, hi - lo);
  // Tokens before `careful` go one to a chunk: a masked weight of zero times a value that is not finite would reach
  // the tokens before it.
  int careful = lo;
  load_k(t, n);
  if (!STATES) load_q(t, n, 0);
  int weighted = -1;                 // the number of tokens that `w` is for
  f32x4 w[CT];                       // a^(n-1-j) of tokens j = 16 jt + g4 + i
  for (;;) {
    // K, V (and the first Q) to LDS
    if (store_k() && !STATES) not_finite = 1;
    if (!STATES) store_q();
    __syncthreads();
    if (!STATES && not_finite) {
      __syncthreads();
      if (tid == 0) not_finite = 0;
      if (n > 1) {
        careful = t + n;
        n = 1;
        load_k(t, n);
        load_q(t, n, 0);
        store_k();
        store_q();
      }
      __syncthreads();
    }
    const int t_next = t + n;
    const int n_next = t_next < careful ? 1 : min(C, hi - t_next);
    if (n != weighted) {
      weighted = n;
#pragma unroll
      for (int jt = 0; jt < CT; ++jt)
#pragma unroll
        for (int i = 0; i < 4; ++i) w[jt][i] = power[max(0, n - 1 - (16 * jt + g4 + i))];
    }
    if (STATES || a.rep == 1) {
      if (t_next < hi) load_k(t_next, n_next);
    }
    half vt[NT][CT];                 // V^T: 16 columns, tokens 16 jt + g4 + i
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int jt = 0; jt < CT; ++jt) vt[nt][jt] = half_down<VS>(v_lds, 16 * jt, wave * 16 * NT + 16 * nt, lane, (T*)nullptr);

    if constexpr (!STATES) {
      for (int g = 0; g < a.rep; ++g) {
        const bool last = g + 1 == a.rep;
        if (!last) load_q(t, n, g + 1);
        else if (t_next < hi) load_q(t_next, n_next, 0);
        if (a.rep > 1 && last && t_next < hi) load_k(t_next, n_next);
        // ---- P^T of 16 queries
        for (int ib = wave; ib < CT; ib += Shape::waves) {
          half qf[KT];
#pragma unroll
          for (int kt = 0; kt < KT; ++kt) qf[kt] = half_at<T>(q_lds + lane_q + 16 * ib * QTile::stride + 16 * kt * (int)sizeof(T));
          for (int jt = 0; jt <= (ib | 1); ++jt) {
            f32x4 acc = {0.f, 0.f, 0.f, 0.f};
            if (jt <= ib) {
#pragma unroll
              for (int kt = 0; kt < KT; kt += 2) {
                const char* kf = k_lds + lane_q + 16 * jt * QTile::stride + 16 * kt * (int)sizeof(T);
                mma(acc, half_at<T>(kf), half_at<T>(kf + 16 * sizeof(T)), qf[kt], qf[kt + 1]);
              }
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int e = 16 * ib + l16 - (16 * jt + g4 + i);
                acc[i] = e >= 0 ? acc[i] * power[max(e, 0)] : 0.f;
              }
            }
            const Split<T, 2> p(acc);
#pragma unroll
            for (int x = 0; x < Split<T, 2>::parts; ++x)
              *reinterpret_cast<half*>(p_lds + x * Shape::p_bytes + lane_p + 16 * ib * PTile::stride + 16 * jt * (int)sizeof(T)) = p.part[x];
          }
        }
        // ---- what the state gives
        f32x4 o[NT][CT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int ib = 0; ib < CT; ++ib) o[nt][ib] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kt = 0; kt < KT; kt += 2) {
          half q0[CT], q1[CT];
#pragma unroll
          for (int ib = 0; ib < CT; ++ib) {
            const char* qf = q_lds + lane_q + 16 * ib * QTile::stride + 16 * kt * (int)sizeof(T);
            q0[ib] = half_at<T>(qf);
            q1[ib] = half_at<T>(qf + 16 * sizeof(T));
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const Split<T, 2> s0(s[nt][kt]), s1(s[nt][kt + 1]);
#pragma unroll
            for (int x = 0; x < Split<T, 2>::parts; ++x)
#pragma unroll
              for (int ib = 0; ib < CT; ++ib) mma(o[nt][ib], s0.part[x], s1.part[x], q0[ib], q1[ib]);
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int ib = 0; ib < CT; ++ib) o[nt][ib] *= power[16 * ib + l16 + 1];
        __syncthreads();             // P is whole; nobody reads Q any more
        if (!last) store_q();
        // ---- what the chunk's own tokens give
#pragma unroll
        for (int ib = 0; ib < CT; ++ib)
#pragma unroll
          for (int jt = 0; jt <= ib; jt += 2)
#pragma unroll
            for (int x = 0; x < Split<T, 2>::parts; ++x) {
              const char* pf = p_lds + x * Shape::p_bytes + lane_p + 16 * ib * PTile::stride + 16 * jt * (int)sizeof(T);
              const half p0 = half_at<T>(pf), p1 = half_at<T>(pf + 16 * sizeof(T));
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma(o[nt][ib], vt[nt][jt], vt[nt][jt + 1], p0, p1);
            }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const int c = n0 + 16 * nt + g4;
#pragma unroll
          for (int ib = 0; ib < CT; ++ib) {
            const int i = 16 * ib + l16;
            if (i < n && c < d) {
              T* at = out + (int64_t)(t + i) * a.out_stride + (int64_t)(h * a.rep + g) * d + c;
              const float r[4] = {o[nt][ib][0] * a.scale, o[nt][ib][1] * a.scale, o[nt][ib][2] * a.scale, o[nt][ib][3] * a.scale};
              if (a.wide_out) {
                store4(at, r);
              } else {
#pragma unroll
                for (int x = 0; x < 4; ++x) at[x] = from_float<T>(r[x]);
              }
            }
          }
        }
        if (!last) __syncthreads();  // the next Q is there, P is free
      }
    }
    // ---- the state after the chunk
    const float an = power[n];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) s[nt][kt] *= an;
#pragma unroll
      for (int jt = 0; jt < CT; jt += 2) {
        const Split<T, 3> v0(widen(vt[nt][jt]) * w[jt]), v1(widen(vt[nt][jt + 1]) * w[jt + 1]);
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
          const half k0 = half_down<DP>(k_lds, 16 * jt, 16 * kt, lane, (T*)nullptr);
          const half k1 = half_down<DP>(k_lds, 16 * jt + 16, 16 * kt, lane, (T*)nullptr);
#pragma unroll
          for (int x = 0; x < Split<T, 3>::parts; ++x) mma(s[nt][kt], k0, k1, v0.part[x], v1.part[x]);
        }
      }
    }
    t = t_next;
    n = n_next;
    if (t >= hi) break;
    __syncthreads();                 // nobody reads K and V any more
  }

  float* const s_to = STATES ? s_work : segment == segments - 1 ? s_row : nullptr;
  if (s_to) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = 16 * kt + g4 + i, c = n0 + 16 * nt + l16;
          if (r < d && c < d) s_to[(int64_t)r * d + c] = s[nt][kt][i];
        }
  }
}

// What the segments add becomes the states at their starts, in place: one thread to 4 elements of a request's state.
__global__ __launch_bounds__(256) void la_scan_kernel(LinearAttention a) {
  const int per_head = a.d * a.d / 4;
  const int b = blockIdx.y, i = blockIdx.x * 256 + threadIdx.x;
  int lo, hi;
  bounds_of(a, b, lo, hi);
  const int segments = (hi - lo + a.segment - 1) / a.segment;
  const int row = a.rows[b];
  if (segments <= 1 || i >= a.nkv * per_head || row < 0 || row >= a.num_rows) return;
  const int h = i / per_head;
  const float an = decay_power(a.log_decay[h], a.segment);
  f32x4 s = *reinterpret_cast<const f32x4*>(a.state + (int64_t)row * a.state_stride + (int64_t)i * 4);
  const int64_t unit = (int64_t)a.nkv * a.d * a.d;
  float* w = a.work + (int64_t)first_unit(a, b) * unit + (int64_t)i * 4;
  for (int x = 0; x < segments; ++x, w += unit) {
    f32x4 added = {0.f, 0.f, 0.f, 0.f};
    if (x + 1 < segments) added = *reinterpret_cast<const f32x4*>(w);
    *reinterpret_cast<f32x4*>(w) = s;
#pragma unroll
    for (int c = 0; c < 4; ++c) s[c] = fmaf(an, s[c], added[c]);
  }
}

template <typename T, int DP, int NT, int C, bool STATES>
static int launch_chunks(const LinearAttention& a, int64_t units, hipStream_t stream) {
  typedef ChunkShape<T, DP, NT, C> Shape;
  static std::atomic<uint64_t> ready{0};           // devices on which the kernel may use this much LDS
  constexpr int bytes = Shape::lds(STATES);
  int device = 0;
  (void)hipGetDevice(&device);
  if (!((ready.load(std::memory_order_relaxed) >> (device & 63)) & 1)) {
    hipError_t e = hipFuncSetAttribute((const void*)la_chunk_kernel<T, DP, NT, C, STATES>, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    MI_REQUIRE(e == hipSuccess, "linear attention: %d bytes of LDS: %s", bytes, hipGetErrorString(e));
    ready.fetch_or(1ull << (device & 63), std::memory_order_relaxed);
  }
  const int64_t blocks = units * a.nkv * ((a.d + Shape::VS - 1) / Shape::VS);
  MI_REQUIRE(blocks <= 0x7fffffff, "linear attention: %lld workgroups are too many for one launch", (long long)blocks);
  la_chunk_kernel<T, DP, NT, C, STATES><<<(uint32_t)blocks, Shape::threads, bytes, stream>>>(a);
  MI_CHECK_LAUNCH("linear attention, chunks");
  return 0;
}

template <typename T, int DP, int NT, int C>
static int launch_prompt(const LinearAttention& a, hipStream_t stream) {
  if (!a.segment) return launch_chunks<T, DP, NT, C, false>(a, a.num_requests, stream);
  const int64_t units = a.num_tokens / a.segment + a.num_requests;
  if (launch_chunks<T, DP, NT, C, true>(a, units, stream)) return 1;
  la_scan_kernel<<<dim3((a.nkv * a.d * a.d / 4 + 255) / 256, a.num_requests), 256, 0, stream>>>(a);
  MI_CHECK_LAUNCH("linear attention, scan");
  return launch_chunks<T, DP, NT, C, false>(a, units, stream);
}

// segment: tokens of a segment (a multiple of 64), or 0 for one workgroup's walk over each whole request; work: then
// (num_tokens / segment + num_requests) * nkv * d * d floats.
MI_EXPORT int mi_linear_attention(LA_ARGS, int segment, float* work, hipStream_t stream) {
  if (check_sizes(nq, nkv, d, num_requests, state_stride)) return 1;
  MI_REQUIRE(segment >= 0 && segment % 64 == 0 && (segment == 0 || work), "linear attention: segments of %d tokens", segment);
  if (num_requests == 0 || num_tokens == 0) return 0;
  const int size = dtype == MI_DTYPE_BF16 ? 2 : 4;
  auto wide = [&](const void* p, int64_t stride, int bytes) { return ((uint64_t)p | (uint64_t)(stride * size)) % bytes == 0; };
  LinearAttention a = {q, k, v, out, state, rows, cu, log_decay, work, q_stride, k_stride, v_stride, out_stride, state_stride,
                       num_rows, num_tokens, num_requests, nkv, nq / nkv, d, segment, scale, wide(q, q_stride, 16),
                       wide(k, k_stride, 16), wide(v, v_stride, 16), wide(out, out_stride, 4 * size)};
  if (dtype == MI_DTYPE_BF16) {
    if (d <= 64) return launch_prompt<bf16, 64, 1, 64>(a, stream);
    if (d <= 128) return launch_prompt<bf16, 128, 1, 64>(a, stream);
    return launch_prompt<bf16, 256, 1, 64>(a, stream);
  }
  if (dtype == MI_DTYPE_F32) {
    if (d <= 64) return launch_prompt<float, 64, 1, 64>(a, stream);
    if (d <= 128) return launch_prompt<float, 128, 1, 64>(a, stream);
    return launch_prompt<float, 256, 1, 32>(a, stream);
  }
  MI_FAIL("linear attention: dtype %d", dtype);
}
