// Linear attention with a decay for each head, over fixed-size states.
//
//   S_t = a S_{t-1} + k_t v_t^T        S [d, d] float32 per request and kv head, a = exp(log_decay[kv head])
//   o_t = scale * q_t S_t              for each of the kv head's query heads
//
// Prompts go by chunks of tokens on the matrix cores, single tokens by the formula as it stands: those are bound by the
// state's bytes, read and written once.
#include "common.h"

#include <atomic>

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

#define LA_MAX_D 256

__device__ __forceinline__ float decay_power(float log_decay, int n) {   // a^n; a^0 = 1 for a decay of zero too
  return n == 0 ? 1.f : (float)exp((double)log_decay * n);
}

// ---------------------------------------------------------------- single tokens
//
// A workgroup takes 32 columns (whole 128-byte lines) of one request's and kv head's state: a thread 4 columns of every
// 32nd row.  Everything that is read is asked for at once: the token's q, k, v (through LDS, since every thread needs
// all rows of k and q) and the state; the query heads' sums over rows meet in LDS, STEP_HEADS heads at a time.
#define STEP_THREADS 256
#define STEP_COLS 32
#define STEP_ROW_GROUPS (STEP_THREADS / (STEP_COLS / 4))
#define STEP_HEADS 4

// States of a launch of this many bytes and more are read with nontemporal loads: they are read once and push out what
// could stay (256 requests of 8 heads of 128, 134 MB: 54.5 us against 61; 64 requests, 34 MB: 17.8 against 17.4).
#define STEP_STREAM_BYTES (64ll << 20)

template <typename T, int NR, bool STREAM>   // NR: rows of the state that a thread holds
__global__ __launch_bounds__(STEP_THREADS) void la_step_kernel(
    const T* __restrict__ q, int64_t q_stride, const T* __restrict__ k, int64_t k_stride, const T* __restrict__ v,
    int64_t v_stride, T* __restrict__ out, int64_t out_stride, float* __restrict__ state, int64_t state_stride,
    int num_rows, int idle_row, const int* __restrict__ rows, int nkv, int rep, int d, const float* __restrict__ log_decay,
    float scale) {
  constexpr int ROWS = NR * STEP_ROW_GROUPS;
  __shared__ float k_lds[ROWS], q_lds[STEP_HEADS][ROWS], v_lds[STEP_COLS], a_lds;
  __shared__ float part[STEP_THREADS / MI_WAVE][STEP_HEADS][STEP_COLS];
  const int h = blockIdx.x % nkv, slice = blockIdx.x / nkv;
  const int64_t b = blockIdx.y;
  const int tid = threadIdx.x, tx = tid % (STEP_COLS / 4), ty = tid / (STEP_COLS / 4);
  const int lane = tid & (MI_WAVE - 1), wave = tid / MI_WAVE;
  const int c0 = slice * STEP_COLS + tx * 4;
  const int row = rows[b];
  const bool known = row >= 0 && row < num_rows, kept = known && row != idle_row, live = kept && c0 < d;
  float* s_at = state + (kept ? row : 0) * state_stride + (int64_t)h * d * d + c0;
  f32x4 s[NR];
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    const int i = ty + r * STEP_ROW_GROUPS;
    s[r] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (live && i < d) {
      const f32x4* from = reinterpret_cast<const f32x4*>(s_at + (int64_t)i * d);
      s[r] = STREAM ? __builtin_nontemporal_load(from) : *from;
    }
  }
  for (int i = tid; i < ROWS; i += STEP_THREADS) k_lds[i] = i < d ? to_float(k[b * k_stride + (int64_t)h * d + i]) : 0.f;
  if (tid < STEP_COLS) {
    const int c = slice * STEP_COLS + tid;
    v_lds[tid] = c < d ? to_float(v[b * v_stride + (int64_t)h * d + c]) : 0.f;
  }
  if (tid == STEP_THREADS - 1) a_lds = decay_power(log_decay[h], 1);
  for (int g0 = 0; g0 < rep; g0 += STEP_HEADS) {
    for (int i = tid; i < STEP_HEADS * ROWS; i += STEP_THREADS) {
      const int g = g0 + i / ROWS, c = i % ROWS;
      q_lds[i / ROWS][c] = g < rep && c < d ? to_float(q[b * q_stride + (int64_t)(h * rep + g) * d + c]) : 0.f;
    }
    __syncthreads();
    if (g0 == 0) {
      const float a = a_lds;
      const f32x4 vv = *reinterpret_cast<const f32x4*>(v_lds + tx * 4);
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        const int i = ty + r * STEP_ROW_GROUPS;
        const float kk = k_lds[i];
#pragma unroll
        for (int c = 0; c < 4; ++c) s[r][c] = fmaf(kk, vv[c], a * s[r][c]);
        if (live && i < d) *reinterpret_cast<f32x4*>(s_at + (int64_t)i * d) = s[r];
      }
    }
#pragma unroll
    for (int g = 0; g < STEP_HEADS; ++g) {
      if (g0 + g >= rep) break;
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        const int i = ty + r * STEP_ROW_GROUPS;
        const float qq = q_lds[g][i];
        if (i < d)
#pragma unroll
          for (int c = 0; c < 4; ++c) o[c] = fmaf(qq, s[r][c], o[c]);
      }
#pragma unroll
      for (int x = STEP_COLS / 4; x < MI_WAVE; x <<= 1)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[c] += __shfl_xor(o[c], x, MI_WAVE);
      if (lane < STEP_COLS / 4) *reinterpret_cast<f32x4*>(&part[wave][g][tx * 4]) = o;
    }
    __syncthreads();
    for (int i = tid; i < STEP_HEADS * STEP_COLS; i += STEP_THREADS) {
      const int g = i / STEP_COLS, c = slice * STEP_COLS + i % STEP_COLS;
      if (g0 + g >= rep || c >= d) continue;
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < STEP_THREADS / MI_WAVE; ++w) sum += part[w][g][i % STEP_COLS];
      out[b * out_stride + (int64_t)(h * rep + g0 + g) * d + c] = from_float<T>(known ? sum * scale : NAN);
    }
    if (g0 + STEP_HEADS < rep) __syncthreads();
  }
}

template <typename T, bool STREAM>
static void launch_step(const void* q, int64_t q_stride, const void* k, int64_t k_stride, const void* v, int64_t v_stride,
                        void* out, int64_t out_stride, float* state, int64_t state_stride, int num_rows, int idle_row,
                        const int* rows, int num_requests, int nq, int nkv, int d, const float* log_decay, float scale,
                        hipStream_t stream) {
  const dim3 grid(nkv * ((d + STEP_COLS - 1) / STEP_COLS), num_requests);
  const int nr = (d + STEP_ROW_GROUPS - 1) / STEP_ROW_GROUPS;
#define LAUNCH(N)                                                                                                      \
  la_step_kernel<T, N, STREAM><<<grid, STEP_THREADS, 0, stream>>>((const T*)q, q_stride, (const T*)k, k_stride, (const T*)v,    \
                                                          v_stride, (T*)out, out_stride, state, state_stride, num_rows, \
                                                          idle_row, rows, nkv, nq / nkv, d, log_decay, scale)
  if (nr <= 1) LAUNCH(1);
  else if (nr <= 2) LAUNCH(2);
  else if (nr <= 3) LAUNCH(3);
  else if (nr <= 4) LAUNCH(4);
  else LAUNCH(8);
#undef LAUNCH
}

#define LA_ARGS                                                                                                       \
  int dtype, const void *q, int64_t q_stride, const void *k, int64_t k_stride, const void *v, int64_t v_stride, void *out, \
      int64_t out_stride, float *state, int64_t state_stride, int num_rows, int idle_row, const int *rows, const int *cu, int num_tokens, \
      int num_requests, int nq, int nkv, int d, const float *log_decay, float scale

static int check_sizes(int nq, int nkv, int d, int num_requests, int64_t state_stride) {
  MI_REQUIRE(d >= 8 && d <= LA_MAX_D && d % 8 == 0, "linear attention: head size %d is no multiple of 8 up to %d", d, LA_MAX_D);
  MI_REQUIRE(nkv >= 1 && nq >= nkv && nq % nkv == 0, "linear attention: %d query heads are no multiple of %d kv heads", nq, nkv);
  MI_REQUIRE(num_requests >= 0 && num_requests <= 65535, "linear attention: %d requests, at most 65535 in a launch", num_requests);
  MI_REQUIRE(state_stride % 4 == 0, "linear attention: rows of states must be a multiple of 16 bytes apart");
  return 0;
}

// One token for each request: num_tokens == num_requests, cu is not read.
MI_EXPORT int mi_linear_attention_step(LA_ARGS, hipStream_t stream) {
  if (check_sizes(nq, nkv, d, num_requests, state_stride)) return 1;
  MI_REQUIRE(num_tokens == num_requests, "linear attention: %d tokens of %d requests in a step", num_tokens, num_requests);
  if (num_requests == 0) return 0;
  const bool stream_states = 4ll * num_requests * nkv * d * d >= STEP_STREAM_BYTES;
#define STEP(T, STREAM)                                                                                                   \
  launch_step<T, STREAM>(q, q_stride, k, k_stride, v, v_stride, out, out_stride, state, state_stride, num_rows, idle_row, \
                         rows, num_requests, nq, nkv, d, log_decay, scale, stream)
  if (dtype == MI_DTYPE_BF16) {
    if (stream_states) STEP(bf16, true);
    else STEP(bf16, false);
  } else if (dtype == MI_DTYPE_F32) {
    if (stream_states) STEP(float, true);
    else STEP(float, false);
  }
#undef STEP
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
// columns of one request's (or segment's) and kv head's state and walks over the chunks; a wave owns 16 of the
// columns and keeps them, [DP, 16] in 32 bits, in registers as the accumulators of the last product.  Products:
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
typedef float f32x8 __attribute__((ext_vector_type(8)));

#ifndef LA_C64
#define LA_C64 64
#endif
#ifndef LA_PBUF64
#define LA_PBUF64 2
#endif
#define LA_LDS(T) __attribute__((address_space(3))) T

template <typename T>
struct Half;      // 4 elements of an operand, and the two halves of 32 elements of the summed axis
template <>
struct Half<bf16> {
  typedef s16x4 type;
  typedef s16x8 pair;
};
template <>
struct Half<float> {
  typedef f32x4 type;
  typedef f32x8 pair;
};

__device__ __forceinline__ s16x8 join(s16x4 a, s16x4 b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }
__device__ __forceinline__ f32x8 join(f32x4 a, f32x4 b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }
// acc += A B over 32 elements of the summed axis
__device__ __forceinline__ void mma(f32x4& acc, s16x8 a, s16x8 b) {
  acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), acc, 0, 0, 0);
}
__device__ __forceinline__ void mma(f32x4& acc, f32x8 a, f32x8 b) {
#pragma unroll
  for (int i = 0; i < 8; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], acc, 0, 0, 0);
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

// Tiles in LDS are rows of tokens.  The two halves that a lane takes to a bfloat16 product, columns 4 g .. and
// 16 + 4 g .. of every 32, lie side by side (column 16 x + 4 g + i of a block at place 8 g + 4 x + i), so that an
// operand is one 16-byte read; 32-bit columns keep their order.  Rows are padded by 32 bytes: an operand read, which
// takes 16 bytes to a lane from 16 rows and 4 neighbouring pieces, is served 4 rows x 2 pieces at a time, and these then
// lie in different banks.
template <typename T, int COLS>
struct Tile {
  static constexpr int stride = COLS * (int)sizeof(T) + 32;
  // of the 4 columns from col on (a multiple of 4)
  static __device__ __forceinline__ int at(int row, int col) {
    if (sizeof(T) == 2) return row * stride + (col & ~31) * 2 + (col & 12) * 4 + (col & 16) / 2;
    return row * stride + col * 4;
  }
  static constexpr int bytes(int rows) { return rows * stride; }
};

// The halves of columns col .. col + 31 of the lane's row; `p`: where Tile::at puts (row, 4 g).
__device__ __forceinline__ s16x8 halves_at(const char* p, int col, bf16*) { return *reinterpret_cast<const s16x8*>(p + col * 2); }
__device__ __forceinline__ f32x8 halves_at(const char* p, int col, float*) {
  return join(*reinterpret_cast<const f32x4*>(p + col * 4), *reinterpret_cast<const f32x4*>(p + col * 4 + 64));
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
  for (int i = 0; i < 4; ++i) r[i] = *reinterpret_cast<const float*>(tile + (row0 + lane / 16 * 4 + i) * Tile<float, COLS>::stride + (col0 + lane % 16) * 4);
  return r;
}

// 16 bytes from p on, element by element
template <typename T>
__device__ __forceinline__ u32x4 piece_of_elements(const T* p) {
  T tmp[16 / sizeof(T)];
#pragma unroll
  for (int i = 0; i < (int)(16 / sizeof(T)); ++i) tmp[i] = p[i];
  return __builtin_bit_cast(u32x4, tmp);
}

// A thread's pieces (16 bytes) of a tile of C rows: rows r0, r0 + step, ... at column c0.
template <typename T, int COLS, int C, int THREADS>
struct Pieces {
  static constexpr int to_row = COLS * (int)sizeof(T) / 16, step = THREADS / to_row, count = C / step;
  static_assert(THREADS % to_row == 0 && C % step == 0, "whole rows to a round");
  int r0, c0;
  uint32_t offset;                   // of the first piece, in bytes, from the tile's first element in memory
  int lds;
  bool live;
  u32x4 held[count];
  __device__ __forceinline__ Pieces(int tid, int64_t stride, int columns) {
    r0 = tid / to_row;
    c0 = tid % to_row * (16 / (int)sizeof(T));
    live = c0 < columns;
    offset = (uint32_t)((r0 * stride + c0) * (int)sizeof(T));
    lds = Tile<T, COLS>::at(r0, c0);
  }
  // n rows from `from` on; the rest, and columns past the end, are zeros
  template <bool ALIGNED>
  __device__ __forceinline__ void load(const T* from, int64_t stride, int n) {
    if (ALIGNED && n == C) {
#pragma unroll
      for (int i = 0; i < count; ++i) {
        held[i] = u32x4{0, 0, 0, 0};
        if (live) held[i] = *reinterpret_cast<const u32x4*>((const char*)(from + i * step * stride) + offset);
      }
    } else {
#pragma unroll
      for (int i = 0; i < count; ++i) {
        held[i] = u32x4{0, 0, 0, 0};
        if (live && r0 + i * step < n) {
          const T* at = from + (r0 + i * step) * stride + c0;
          held[i] = ALIGNED ? *reinterpret_cast<const u32x4*>(at) : piece_of_elements(at);
        }
      }
    }
  }
  __device__ __forceinline__ void store(char* tile) const {
#pragma unroll
    for (int i = 0; i < count; ++i) {
      char* at = tile + lds + i * step * Tile<T, COLS>::stride;
      if (sizeof(T) == 2) {              // columns c0 .. c0 + 3 and the next 4
        *reinterpret_cast<mi_u32x2*>(at) = mi_u32x2{held[i][0], held[i][1]};
        *reinterpret_cast<mi_u32x2*>(at + 16) = mi_u32x2{held[i][2], held[i][3]};
      } else {
        *reinterpret_cast<u32x4*>(at) = held[i];
      }
    }
  }
};

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
  int num_rows, idle_row, num_tokens, num_requests, nkv, rep, d;
  int segment;                       // tokens of a segment; 0: every request is one
  float scale;
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

template <typename T, int DP, int WAVES, int C, int PBUF>
struct ChunkShape {
  static constexpr int waves = WAVES, threads = 64 * WAVES;
  static constexpr int VS = 16 * waves;
  static constexpr int kt = DP / 16, ct = C / 16;
  static constexpr int q_bytes = (Tile<T, DP>::bytes(C) + 15) / 16 * 16;
  static constexpr int v_bytes = (Tile<T, VS>::bytes(C) + 15) / 16 * 16;
  static constexpr int part_bytes = (Tile<T, C>::bytes(C) + 15) / 16 * 16;
  static constexpr int p_bytes = (sizeof(T) == 2 ? 2 : 1) * part_bytes;
  static constexpr int lds(bool states) { return 2 * (q_bytes + v_bytes) + (states ? 0 : 2 * q_bytes + PBUF * p_bytes); }
};

// STATES: only what a segment adds to its request's state (from zero), left in `work`; the last segment's is not needed.
// ALIGNED: rows of q, k and v start at multiples of 16 bytes, of out at multiples of 4 elements, and a chunk of a tensor
// spans less than 2^31 bytes.
template <typename T, int DP, int WAVES, int C, int PBUF, bool STATES, bool ALIGNED, int PER_SIMD>
__global__ __launch_bounds__(64 * WAVES, PER_SIMD) void la_chunk_kernel(LinearAttention a) {
  typedef ChunkShape<T, DP, WAVES, C, PBUF> Shape;
  typedef typename Half<T>::type half;
  typedef typename Half<T>::pair pair;
  constexpr int PARTS = Split<T, 2>::parts;
  typedef Tile<T, DP> QTile;
  typedef Tile<T, Shape::VS> VTile;
  typedef Tile<T, C> PTile;
  constexpr int KT = Shape::kt, CT = Shape::ct, VS = Shape::VS;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  __shared__ float power[C + 1];     // a^i
  __shared__ float left[2 * C];      // a^(C-1-i), zeros from C on
  __shared__ int found, not_finite[2];
  char* const k_lds = lds;
  char* const v_lds = k_lds + 2 * Shape::q_bytes;
  char* const q_lds = v_lds + 2 * Shape::v_bytes;
  char* const p_lds = q_lds + 2 * Shape::q_bytes;

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

  const int n0 = slice * VS + wave * 16;                 // first column of the wave
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
  for (int i = tid; i < 2 * C; i += Shape::threads) left[i] = i < C ? decay_power(a.log_decay[h], C - 1 - i) : 0.f;
  if (tid < 2) not_finite[tid] = 0;
  __syncthreads();

  // the wave's columns of the state, accumulator t: rows 16 t + g4 + i, column n0 + l16
  f32x4 s[KT];
  float* const s_row = a.state + (int64_t)row * a.state_stride + (int64_t)h * d * d;
  float* const s_work = a.segment ? a.work + ((int64_t)unit * a.nkv + h) * d * d : nullptr;
  const float* const s_from = segments > 1 ? s_work : row == a.idle_row ? nullptr : s_row;
#pragma unroll
  for (int t = 0; t < KT; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 16 * t + g4 + i, c = n0 + l16;
      s[t][i] = !STATES && s_from && r < d && c < d ? s_from[(int64_t)r * d + c] : 0.f;
    }

  const T* const kp = (const T*)a.k + (int64_t)h * d;
  const T* const vp = (const T*)a.v + (int64_t)h * d + slice * VS;
  const T* const qp = (const T*)a.q + (int64_t)h * a.rep * d;

  Pieces<T, DP, C, Shape::threads> kr(tid, a.k_stride, d), qr(tid, a.q_stride, d);
  Pieces<T, VS, C, Shape::threads> vr(tid, a.v_stride, d - slice * VS);
  auto load_k = [&](int t, int n) {
    kr.template load<ALIGNED>(kp + t * a.k_stride, a.k_stride, n);
    vr.template load<ALIGNED>(vp + t * a.v_stride, a.v_stride, n);
  };
  auto load_q = [&](int t, int n, int g) { qr.template load<ALIGNED>(qp + t * a.q_stride + g * d, a.q_stride, n); };
  auto store_k = [&](int buf) -> bool {      // whether a value is not finite
    kr.store(k_lds + buf * Shape::q_bytes);
    vr.store(v_lds + buf * Shape::v_bytes);
    bool ok = true;
#pragma unroll
    for (int i = 0; i < vr.count; ++i) ok = ok && all_finite(vr.held[i], (T*)nullptr);
    return !ok;
  };
  half vt[CT];                       // V^T of the chunk: the wave's 16 columns, tokens 16 jt + g4 + i
  T* const typed = nullptr;          // (picks an overload)
  auto read_v = [&](int buf) {
#pragma unroll
    for (int jt = 0; jt < CT; ++jt) vt[jt] = half_down<VS>(v_lds + buf * Shape::v_bytes, 16 * jt, wave * 16, lane, typed);
  };
  auto update = [&](int buf, int n) {        // the state after a chunk of n tokens
    const char* const kb = k_lds + buf * Shape::q_bytes;
    const float an = power[n];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) s[kt] *= an;
#pragma unroll
    for (int jt = 0; jt < CT; jt += 2) {
      pair kp[KT];
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
        kp[kt] = join(half_down<DP>(kb, 16 * jt, 16 * kt, lane, typed), half_down<DP>(kb, 16 * jt + 16, 16 * kt, lane, typed));
      f32x4 w0, w1;                  // a^(n-1-j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        w0[i] = left[C - n + 16 * jt + g4 + i];
        w1[i] = left[C - n + 16 * jt + 16 + g4 + i];
      }
      __builtin_amdgcn_sched_barrier(0);     // (the reads are on their way together)
      const Split<T, 3> v0(widen(vt[jt]) * w0), v1(widen(vt[jt + 1]) * w1);
#pragma unroll
      for (int z = 0; z < Split<T, 3>::parts; ++z)
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) mma(s[kt], kp[kt], join(v0.part[z], v1.part[z]));
    }
  };

  // The chunk at hand has the n tokens from t on.  Tiles are double-buffered: while one chunk (K, V) or query head (Q) is
  // worked on, the next one's pieces are on their way in registers; they are stored to the other buffer before the one
  // barrier of each step, and the loads after them are issued at once.
  int t = lo, n = min(C, hi - lo), kv = 0;
  if constexpr (STATES) {
    load_k(t, n);
    store_k(0);
    if (t + n < hi) load_k(t + n, min(C, hi - t - n));
    __syncthreads();
    for (;;) {
      read_v(kv);
      update(kv, n);
      t += n;
      if (t >= hi) break;
      n = min(C, hi - t);
      kv ^= 1;
      store_k(kv);
      if (t + n < hi) load_k(t + n, min(C, hi - t - n));
      __syncthreads();
    }
  } else {
    const uint32_t out_offset = (uint32_t)((l16 * a.out_stride + n0 + g4) * (int)sizeof(T));
    const int lane_q = QTile::at(l16, g4), lane_p = PTile::at(l16, g4);
    // the weights a^(i-j) of the P that the wave makes, and a^(i+1) of its tokens, both with the scale
    constexpr int PW = (CT * CT / 2 + WAVES - 1) / WAVES;
    int reach[PW];                   // i - j of a lane's first element: those of the next ones are less
    f32x4 weight[PW][2];
    float reached[CT];
#pragma unroll
    for (int y = 0; y < PW; ++y) {
      const int x = wave + y * WAVES;
      reach[y] = 16 * (x % CT) + l16 - (x / CT * 32 + g4);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        weight[y][0][i] = power[min(max(reach[y] - i, 0), C)] * a.scale;
        weight[y][1][i] = power[min(max(reach[y] - 16 - i, 0), C)] * a.scale;
      }
    }
#pragma unroll
    for (int ib = 0; ib < CT; ++ib) reached[ib] = power[16 * ib + l16 + 1] * a.scale;
    // the state's parts, held for all query heads of a chunk where there are registers for them
    constexpr bool HELD = DP <= 128;
    pair sp[HELD ? KT / 2 : 1][PARTS];
    // Tokens before `careful` go one to a chunk: a masked weight of zero times a value that is not finite would reach
    // the tokens before it.
    int careful = lo;
    auto tokens_at = [&](int t) { return t < careful ? 1 : min(C, hi - t); };
    // the query head whose Q is on its way: of tokens nt .. nt + nn - 1
    int nt = t, nn = n, ng = 0;
    auto fetch_next_q = [&]() {
      if (++ng == a.rep) {
        ng = 0;
        nt += nn;
        nn = tokens_at(nt);
      }
      if (nt < hi) load_q(nt, nn, ng);
    };
    load_k(t, n);
    load_q(t, n, 0);
    if (store_k(0)) not_finite[0] = 1;
    qr.store(q_lds);
    fetch_next_q();
    if (t + n < hi) load_k(t + n, tokens_at(t + n));
    __syncthreads();
    int g = 0, qb = 0, pb = 0;
    for (;;) {
      if (g == 0) {
        if (not_finite[kv]) {          // the first of this chunk's tokens alone
          __syncthreads();
          if (tid == 0) not_finite[kv] = 0;
          if (n > 1) {
            careful = t + n;
            n = 1;
            load_k(t, n);
            load_q(t, n, 0);
            store_k(kv);
            qr.store(q_lds + qb * Shape::q_bytes);
            nt = t, nn = n, ng = 0;
            fetch_next_q();
            if (t + n < hi) load_k(t + n, tokens_at(t + n));
          }
          __syncthreads();
        }
        read_v(kv);
        if (HELD) {
#pragma unroll
          for (int kt = 0; kt < KT / 2; ++kt) {
            const Split<T, 2> s0(s[2 * kt]), s1(s[2 * kt + 1]);
#pragma unroll
            for (int z = 0; z < PARTS; ++z) sp[kt][z] = join(s0.part[z], s1.part[z]);
          }
        }
      }
      const char* const qt = q_lds + qb * Shape::q_bytes + lane_q;
      const char* const kt_lds = k_lds + kv * Shape::q_bytes + lane_q;
      char* const pt = p_lds + pb * Shape::p_bytes + lane_p;
      // ---- P^T: to a wave 16 queries and 32 tokens, or that again for the next waves' worth of them
#pragma unroll
      for (int y = 0; y < PW; ++y) {
        const int x = wave + y * WAVES, ib = x % CT, jt = x / CT * 2;
        if (x >= CT * CT / 2 || jt > ib) continue;             // (no product below reads these)
        pair qf[KT / 2], k0[KT / 2], k1[KT / 2];
#pragma unroll
        for (int kt = 0; kt < KT / 2; ++kt) {
          qf[kt] = halves_at(qt + 16 * ib * QTile::stride, 32 * kt, typed);
          k0[kt] = halves_at(kt_lds + 16 * jt * QTile::stride, 32 * kt, typed);
          k1[kt] = halves_at(kt_lds + (16 * jt + 16) * QTile::stride, 32 * kt, typed);
        }
        __builtin_amdgcn_sched_barrier(0);
        f32x4 p0 = {0.f, 0.f, 0.f, 0.f}, p1 = p0;
#pragma unroll
        for (int kt = 0; kt < KT / 2; ++kt) {
          mma(p0, k0[kt], qf[kt]);
          mma(p1, k1[kt], qf[kt]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          p0[i] = reach[y] >= i ? p0[i] * weight[y][0][i] : 0.f;
          p1[i] = reach[y] >= 16 + i ? p1[i] * weight[y][1][i] : 0.f;
        }
        const Split<T, 2> s0(p0), s1(p1);
#pragma unroll
        for (int z = 0; z < PARTS; ++z) {
          char* at = pt + z * Shape::part_bytes + 16 * ib * PTile::stride;
          *reinterpret_cast<half*>(at + PTile::at(0, 16 * jt)) = s0.part[z];
          *reinterpret_cast<half*>(at + PTile::at(0, 16 * jt + 16)) = s1.part[z];
        }
      }
      // ---- what the state gives
      f32x4 o[CT];
#pragma unroll
      for (int ib = 0; ib < CT; ++ib) o[ib] = f32x4{0.f, 0.f, 0.f, 0.f};
      pair qf[2][CT];
#pragma unroll
      for (int ib = 0; ib < CT; ++ib) qf[0][ib] = halves_at(qt + 16 * ib * QTile::stride, 0, typed);
#pragma unroll
      for (int kt = 0; kt < KT / 2; ++kt) {
        if (kt + 1 < KT / 2) {
#pragma unroll
          for (int ib = 0; ib < CT; ++ib) qf[(kt + 1) & 1][ib] = halves_at(qt + 16 * ib * QTile::stride, 32 * (kt + 1), typed);
        }
        __builtin_amdgcn_sched_barrier(0);
        if (!HELD) {
          const Split<T, 2> s0(s[2 * kt]), s1(s[2 * kt + 1]);
#pragma unroll
          for (int z = 0; z < PARTS; ++z) sp[0][z] = join(s0.part[z], s1.part[z]);
        }
#pragma unroll
        for (int z = 0; z < PARTS; ++z)
#pragma unroll
          for (int ib = 0; ib < CT; ++ib) mma(o[ib], sp[HELD ? kt : 0][z], qf[kt & 1][ib]);
      }
#pragma unroll
      for (int ib = 0; ib < CT; ++ib) o[ib] *= reached[ib];
      const bool last = g + 1 == a.rep, more = t + n < hi;
      if (last) update(kv, n);
      if (!last || more) qr.store(q_lds + (qb ^ 1) * Shape::q_bytes);
      if (last && more) {
        if (store_k(kv ^ 1)) not_finite[kv ^ 1] = 1;
        const int after = t + n + tokens_at(t + n);
        if (after < hi) load_k(after, tokens_at(after));
      }
      fetch_next_q();
      __syncthreads();
      // ---- what the chunk's own tokens give
      pair pf[CT][(CT + 1) / 2][PARTS];
#pragma unroll
      for (int ib = 0; ib < CT; ++ib)
#pragma unroll
        for (int jt = 0; jt <= ib; jt += 2)
#pragma unroll
          for (int z = 0; z < PARTS; ++z) pf[ib][jt / 2][z] = halves_at(pt + z * Shape::part_bytes + 16 * ib * PTile::stride, 16 * jt, typed);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int jt = 0; jt < CT; jt += 2)
#pragma unroll
        for (int z = 0; z < PARTS; ++z)
#pragma unroll
          for (int ib = jt; ib < CT; ++ib) mma(o[ib], join(vt[jt], vt[jt + 1]), pf[ib][jt / 2][z]);
      const int c = n0 + g4;
      T* const o_at = out + t * a.out_stride + (int64_t)(h * a.rep + g) * d;
#pragma unroll
      for (int ib = 0; ib < CT; ++ib) {
        const int i = 16 * ib + l16;
        if (i < n && c < d) {
          const float r[4] = {o[ib][0], o[ib][1], o[ib][2], o[ib][3]};
          if (ALIGNED) {
            store4((T*)((char*)(o_at + 16 * ib * a.out_stride) + out_offset), r);
          } else {
#pragma unroll
            for (int x = 0; x < 4; ++x) o_at[i * a.out_stride + c + x] = from_float<T>(r[x]);
          }
        }
      }
      if (PBUF == 1) __syncthreads();              // P is free
      else pb ^= 1;
      qb ^= 1;
      if (last) {
        t += n;
        if (t >= hi) break;
        n = tokens_at(t);
        kv ^= 1;
        g = 0;
      } else {
        ++g;
      }
    }
  }

  float* const s_to = STATES ? s_work : segment == segments - 1 && row != a.idle_row ? s_row : nullptr;
  if (s_to) {
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 16 * kt + g4 + i, c = n0 + l16;
        if (r < d && c < d) s_to[(int64_t)r * d + c] = s[kt][i];
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
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  if (row != a.idle_row) s = *reinterpret_cast<const f32x4*>(a.state + (int64_t)row * a.state_stride + (int64_t)i * 4);
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

template <typename T, int DP, int WAVES, int C, int PBUF, bool STATES, bool ALIGNED, int PER_SIMD>
static int launch_chunks(const LinearAttention& a, int64_t units, hipStream_t stream) {
  typedef ChunkShape<T, DP, WAVES, C, PBUF> Shape;
  static std::atomic<uint64_t> ready{0};           // devices on which the kernel may use this much LDS
  constexpr int bytes = Shape::lds(STATES);
  int device = 0;
  (void)hipGetDevice(&device);
  if (!((ready.load(std::memory_order_relaxed) >> (device & 63)) & 1)) {
    hipError_t e = hipFuncSetAttribute((const void*)la_chunk_kernel<T, DP, WAVES, C, PBUF, STATES, ALIGNED, PER_SIMD>, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    MI_REQUIRE(e == hipSuccess, "linear attention: %d bytes of LDS: %s", bytes, hipGetErrorString(e));
    ready.fetch_or(1ull << (device & 63), std::memory_order_relaxed);
  }
  const int64_t blocks = units * a.nkv * ((a.d + Shape::VS - 1) / Shape::VS);
  MI_REQUIRE(blocks <= 0x7fffffff, "linear attention: %lld workgroups are too many for one launch", (long long)blocks);
  la_chunk_kernel<T, DP, WAVES, C, PBUF, STATES, ALIGNED, PER_SIMD><<<(uint32_t)blocks, Shape::threads, bytes, stream>>>(a);
  MI_CHECK_LAUNCH("linear attention, chunks");
  return 0;
}

template <typename T, int DP, int WAVES, int C, int PBUF, bool ALIGNED, int PER_SIMD>
static int launch_aligned(const LinearAttention& a, hipStream_t stream) {
  if (!a.segment) return launch_chunks<T, DP, WAVES, C, PBUF, false, ALIGNED, PER_SIMD>(a, a.num_requests, stream);
  const int64_t units = a.num_tokens / a.segment + a.num_requests;
  if (launch_chunks<T, DP, WAVES, C, PBUF, true, ALIGNED, PER_SIMD>(a, units, stream)) return 1;
  la_scan_kernel<<<dim3((a.nkv * a.d * a.d / 4 + 255) / 256, a.num_requests), 256, 0, stream>>>(a);
  MI_CHECK_LAUNCH("linear attention, scan");
  return launch_chunks<T, DP, WAVES, C, PBUF, false, ALIGNED, PER_SIMD>(a, units, stream);
}

template <typename T, int DP, int WAVES, int C, int PBUF, int PER_SIMD>
static int launch_prompt(const LinearAttention& a, hipStream_t stream) {
  auto fits = [](const void* p, int64_t stride, int bytes) {
    return ((uint64_t)p | (uint64_t)(stride * (int64_t)sizeof(T))) % bytes == 0 && stride * C * (int64_t)sizeof(T) < (1ll << 31);
  };
  const bool aligned = fits(a.q, a.q_stride, 16) && fits(a.k, a.k_stride, 16) && fits(a.v, a.v_stride, 16) &&
                       fits(a.out, a.out_stride, 4 * sizeof(T));
  return aligned ? launch_aligned<T, DP, WAVES, C, PBUF, true, PER_SIMD>(a, stream)
                 : launch_aligned<T, DP, WAVES, C, PBUF, false, 1>(a, stream);
}

// segment: tokens of a segment (a multiple of 64), or 0 for one workgroup's walk over each whole request; work: then
// (num_tokens / segment + num_requests) * nkv * d * d floats.
MI_EXPORT int mi_linear_attention(LA_ARGS, int segment, float* work, hipStream_t stream) {
  if (check_sizes(nq, nkv, d, num_requests, state_stride)) return 1;
  MI_REQUIRE(segment >= 0 && segment % 64 == 0 && (segment == 0 || work), "linear attention: segments of %d tokens", segment);
  if (num_requests == 0 || num_tokens == 0) return 0;
  LinearAttention a = {q, k, v, out, state, rows, cu, log_decay, work, q_stride, k_stride, v_stride, out_stride, state_stride,
                       num_rows, idle_row, num_tokens, num_requests, nkv, nq / nkv, d, segment, scale};
  if (dtype == MI_DTYPE_BF16) {
    if (d <= 64) return launch_prompt<bf16, 64, 4, LA_C64, LA_PBUF64, 2>(a, stream);
    if (d <= 128) return launch_prompt<bf16, 128, 8, 64, 2, 2>(a, stream);
    return launch_prompt<bf16, 256, 8, 32, 2, 2>(a, stream);
  }
  if (dtype == MI_DTYPE_F32) {
    if (d <= 64) return launch_prompt<float, 64, 4, 32, 2, 2>(a, stream);
    if (d <= 128) return launch_prompt<float, 128, 8, 32, 2, 2>(a, stream);
    return launch_prompt<float, 256, 4, 32, 1, 1>(a, stream);
  }
  MI_FAIL("linear attention: dtype %d", dtype);
}
