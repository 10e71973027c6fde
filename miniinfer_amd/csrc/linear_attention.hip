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

// a^n; a^0 = 1 for a decay of zero too.  (The product's rounding puts an error of |n log a| 2^-24 on the power, at most
// 0.4 * 2^-24 of the weight 1 for a decay.)  Only a decay of zero has powers of zero, the others end at the
// smallest number: an infinity in a state or a value does not become NaN by a power that has left the range.
__device__ __forceinline__ float decay_power(float log_decay, int n) {
  const float least = 1.4e-45f, power = n == 0 ? 1.f : expf(log_decay * n);
  return power < least && log_decay > -INFINITY ? least : power;          // (of NaN NaN)
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
// With S the state before a chunk, i and j tokens of it, n how many it has (the rest of its C rows weigh nothing):
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
// The bfloat16 form multiplies what is 32-bit (S, the weighted P and w V) as it is: split into three bfloat16 parts whose sum
// it is to the last bit, one after the other into the same accumulators.  (Two parts for S and P leave out 2^-17 of a term,
// which an output keeps where its terms cancel.  They were 4 to 13% quicker: 2,048 tokens 31 us against 32, 24 ragged
// requests 68 against 78, 32,768 tokens 233 against 260.)  The one rounding to fewer bits is the output's.
//
// Operands: lane l of an operand has row l % 16 and, of 32 elements of the summed axis, with g = l / 16: in bfloat16
// (16x16x32) the 8 from 8 g on, in 32 bits (eight products 16x16x4) the 4 from 4 g on and the 4 from 16 + 4 g on.  Its
// first and last 4 are a "half".  An accumulator's lane has column l % 16 and rows 4 g .. 4 g + 3, so that two
// accumulators are the two halves of an operand: for S, whose rows are given out accordingly (`dim_of`).
//
// Q, K and V go straight from memory to LDS (lane i's 16 bytes land at base + 16 i), in tiles of whole rows, two of each:
// one is worked on while the other one is filled (three made no difference); the waits are written out by count.  The
// piece of 16 bytes that a lane asks for is chosen such that piece p of row r lies at place p ^ swap(r): then the
// operands' reads, 16 pieces at a time (lanes 0-3, 12-15 and 20-27, ...), and the transposing reads, 16 times 8 bytes of
// 4 rows, meet no bank twice (with p ^ 2 (r mod 4), as good for the former alone, the LDS was busy twice as long, and
// 32,768 tokens of 32 heads on 8 of 128 took 209 us instead of 198, without the kernels for segments, with S and P in two
// parts).

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));

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
// ...over the first half of them, as far as that is less work
__device__ __forceinline__ void mma_first(f32x4& acc, s16x8 a, s16x8 b) { mma(acc, a, b); }
__device__ __forceinline__ void mma_first(f32x4& acc, f32x8 a, f32x8 b) {
#pragma unroll
  for (int i = 0; i < 4; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], acc, 0, 0, 0);
}
__device__ __forceinline__ s16x4 to_half(f32x4 x) { return __builtin_bit_cast(s16x4, __builtin_convertvector(x, bf16x4)); }
__device__ __forceinline__ f32x4 widen(s16x4 h) {
  const mi_u32x2 u = __builtin_bit_cast(mi_u32x2, h);
  return f32x4{__uint_as_float(u[0] << 16), __uint_as_float(u[0] & 0xffff0000u), __uint_as_float(u[1] << 16),
               __uint_as_float(u[1] & 0xffff0000u)};
}
__device__ __forceinline__ f32x4 widen(f32x4 h) { return h; }

// A 32-bit value as a sum of parts that the matrix cores take, exactly: a part is what is left cut off after 8 bits, and
// 24 bits are three times 8.  (Bits below bfloat16's smallest number, 2^-133, are lost.)
template <typename T>
struct Split;
template <>
struct Split<bf16> {
  static constexpr int parts = 3;
  s16x4 part[parts];
  static __device__ __forceinline__ s16x4 first(f32x4 x) {
    auto two = [&](int i) { return __builtin_amdgcn_perm(__float_as_uint(x[i + 1]), __float_as_uint(x[i]), 0x07060302); };
    return __builtin_bit_cast(s16x4, mi_u32x2{two(0), two(2)});
  }
  __device__ __forceinline__ explicit Split(f32x4 x) {
#pragma unroll
    for (int p = 0; p < parts; ++p) {
      part[p] = first(x);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] -= __uint_as_float(__float_as_uint(x[i]) & 0xffff0000u);
    }
  }
  // Infinities of x are their first parts; else nothing is left to change.  (For every split a tenth of a call's time.)
  __device__ __forceinline__ void keep_infinities(f32x4 x) {
#pragma unroll
    for (int p = 1; p < parts; ++p)
#pragma unroll
      for (int i = 0; i < 4; ++i) part[p][i] = fabsf(x[i]) == INFINITY ? 0 : part[p][i];
  }
};
template <>
struct Split<float> {
  static constexpr int parts = 1;
  f32x4 part[1];
  static __device__ __forceinline__ f32x4 first(f32x4 x) { return x; }
  __device__ __forceinline__ explicit Split(f32x4 x) : part{x} {}
  __device__ __forceinline__ void keep_infinities(f32x4) {}
};

// A tile of whole rows in LDS: piece p of row r lies at place p ^ swap(r) of it.
template <typename T, int COLS>
struct Tile {
  static constexpr int stride = COLS * (int)sizeof(T);
  static constexpr int pieces = stride / 16;
  static constexpr int block = stride < 256 ? stride : 256;      // of a row; swaps stay inside
  static __device__ __forceinline__ int swap(int r) {
    if (sizeof(T) == 4 && stride >= 256) return 4 * (r >> 2 & 3) ^ (r & 3);
    return (r >> 2 & 1) * 2 ^ (stride >= 256 ? (r & 3) * 4 : stride >= 128 ? (r >> 1 & 1) * 4 : 0);
  }
  static __device__ __forceinline__ int at(int row, int col) {
    const int byte = col * (int)sizeof(T);
    return row * stride + (((byte >> 4) ^ swap(row)) << 4) + (byte & 15);
  }
  // from a place in the first 64 bytes of a row to that in 64 bytes number x
  static __device__ __forceinline__ int on(int place, int x) { return (place ^ (64 * x) % block) + 64 * x / block * block; }
};

// Where a lane finds its pieces of operands of 16 rows in a tile
template <typename T, int COLS>
struct OperandAt {
  int first;
  __device__ __forceinline__ explicit OperandAt(int lane) : first(Tile<T, COLS>::at(lane & 15, lane / 16 * (16 / (int)sizeof(T)))) {}
  // 16 rows from `row0` on (a multiple of 16), 64 bytes number x of each
  __device__ __forceinline__ int operator()(int row0, int x) const { return row0 * Tile<T, COLS>::stride + Tile<T, COLS>::on(first, x); }
};
// An operand: 32 elements, number kt, of 16 rows.
template <int COLS>
__device__ __forceinline__ s16x8 operand(const char* tile, const OperandAt<bf16, COLS>& at, int row0, int kt) {
  return *reinterpret_cast<const s16x8*>(tile + at(row0, kt));
}
template <int COLS>
__device__ __forceinline__ f32x8 operand(const char* tile, const OperandAt<float, COLS>& at, int row0, int kt) {
  return join(*reinterpret_cast<const f32x4*>(tile + at(row0, 2 * kt)), *reinterpret_cast<const f32x4*>(tile + at(row0, 2 * kt + 1)));
}

// Element i of half h of the lane's 32 elements number x, along a summed axis.
template <typename T>
__device__ __forceinline__ int summed(int x, int h, int g, int i) {
  return sizeof(T) == 2 ? 32 * x + 8 * g + 4 * h + i : 32 * x + 16 * h + 4 * g + i;
}
// Row m of half h of the pair of accumulators number x, such that the pair is an operand.
template <typename T>
__device__ __forceinline__ int dim_of(int x, int h, int m) {
  return sizeof(T) == 2 ? 32 * x + 8 * (m / 4) + 4 * h + m % 4 : 32 * x + 16 * h + m;
}

// Operands along the rows of a tile.  In bfloat16 by the LDS's transposing reads: of 16 lanes, lane 4 j + c brings 4
// columns of row j and gets column l % 16 of the 4 rows.  (Not by the builtin, before which the compiler waits for
// everything that is on its way to LDS.)
template <typename T, int COLS>
struct DownAt {
  int v, k;                          // the first of 16 columns from col0 on; of those that are rows of accumulators
  __device__ __forceinline__ DownAt(int lane, int col0) {
    const int g = lane / 16, j = lane % 16 / 4, c = lane % 4;
    if (sizeof(T) == 2) {
      v = Tile<T, COLS>::at(8 * g + j, col0 + 4 * c);
      k = Tile<T, COLS>::at(8 * g + j, dim_of<T>(0, 0, 4 * c));
    } else {
      v = Tile<T, COLS>::at(4 * g, col0 + lane % 16);
      k = Tile<T, COLS>::at(4 * g, lane % 16);
    }
  }
};
__device__ __forceinline__ uint32_t lds_address(const char* p) { return (uint32_t)(uintptr_t)(LA_LDS(char)*)p; }

// Rows 32 x .. 32 x + 31, 16 columns
template <int COLS>
__device__ __forceinline__ s16x8 columns_down(const char* tile, const DownAt<bf16, COLS>& at, int x) {
  const uint32_t from = lds_address(tile) + 32 * x * Tile<bf16, COLS>::stride;
  s16x4 lo, hi;                      // (rows 4 on are swapped by 2 pieces more)
  asm volatile("ds_read_b64_tr_b16 %0, %2\n\t"
               "ds_read_b64_tr_b16 %1, %3 offset:%4\n\t"
               "s_waitcnt lgkmcnt(0)"
               : "=&v"(lo), "=&v"(hi)
               : "v"(from + at.v), "v"(from + (at.v ^ 32)), "n"(4 * Tile<bf16, COLS>::stride)
               : "memory");
  return join(lo, hi);
}
template <int COLS>
__device__ __forceinline__ f32x8 columns_down(const char* tile, const DownAt<float, COLS>& at, int x) {
  f32x8 r;
#pragma unroll
  for (int i = 0; i < 8; ++i)        // (row 4 g + i: swapped by i more)
    r[i] = *reinterpret_cast<const float*>(tile + (at.v ^ 16 * (i % 4)) + summed<float>(x, i / 4, 0, i % 4) * Tile<float, COLS>::stride);
  return r;
}
// Rows 32 x .. 32 x + 31 of the columns that are the rows of the accumulators (kt, 0), (kt, 1), (kt + 1, 0), (kt + 1, 1);
// kt is even
template <int COLS>
__device__ __forceinline__ void dims_down(s16x8 (&r)[2][2], const char* tile, const DownAt<bf16, COLS>& at, int x, int kt) {
  const uint32_t from = lds_address(tile) + 32 * x * Tile<bf16, COLS>::stride;
  const uint32_t k0 = from + Tile<bf16, COLS>::on(at.k, kt), k1 = from + Tile<bf16, COLS>::on(at.k, kt + 1);
  s16x4 p[8];
  asm volatile("ds_read_b64_tr_b16 %0, %8\n\t"
               "ds_read_b64_tr_b16 %1, %9 offset:%12\n\t"
               "ds_read_b64_tr_b16 %2, %8 offset:8\n\t"
               "ds_read_b64_tr_b16 %3, %9 offset:%13\n\t"
               "ds_read_b64_tr_b16 %4, %10\n\t"
               "ds_read_b64_tr_b16 %5, %11 offset:%12\n\t"
               "ds_read_b64_tr_b16 %6, %10 offset:8\n\t"
               "ds_read_b64_tr_b16 %7, %11 offset:%13\n\t"
               "s_waitcnt lgkmcnt(0)"
               : "=&v"(p[0]), "=&v"(p[1]), "=&v"(p[2]), "=&v"(p[3]), "=&v"(p[4]), "=&v"(p[5]), "=&v"(p[6]), "=&v"(p[7])
               : "v"(k0), "v"(k0 ^ 32), "v"(k1), "v"(k1 ^ 32), "n"(4 * Tile<bf16, COLS>::stride),
                 "n"(4 * Tile<bf16, COLS>::stride + 8)
               : "memory");
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i / 2][i % 2] = join(p[2 * i], p[2 * i + 1]);
}
template <int COLS>
__device__ __forceinline__ void dims_down(f32x8 (&r)[2][2], const char* tile, const DownAt<float, COLS>& at, int x, int kt) {
#pragma unroll
  for (int y = 0; y < 4; ++y)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      r[y / 2][y % 2][i] = *reinterpret_cast<const float*>(tile + Tile<float, COLS>::on(at.k ^ 16 * (i % 4), 2 * kt + y) +
                                                           summed<float>(x, i / 4, 0, i % 4) * Tile<float, COLS>::stride);
}

// 16 bytes from p on, element by element
template <typename T>
__device__ __forceinline__ u32x4 piece_of_elements(const T* p) {
  T tmp[16 / sizeof(T)];
#pragma unroll
  for (int i = 0; i < (int)(16 / sizeof(T)); ++i) tmp[i] = p[i];
  return __builtin_bit_cast(u32x4, tmp);
}

// A wave's share of the way of a tile of C rows from memory to LDS: `count` requests of 1 KB.  Columns past the end are
// never written (they are zeros from the start); rows past the last token are that token's again: the weights of such
// tokens are zeros.  Not ALIGNED: the elements one by one through registers.
template <typename T, int COLS, int C, int WAVES>
struct Loader {
  typedef Tile<T, COLS> Shape;
  static constexpr int rows = MI_WAVE / Shape::pieces, count = C / rows / WAVES;
  static_assert(MI_WAVE % Shape::pieces == 0 && C % (rows * WAVES) == 0, "whole rows to a request");
  int row0, column[count];             // column: of the lane's piece; -1: past the end
  uint32_t offset[count];              // bytes from the tile's first element
  __device__ __forceinline__ Loader(int wave, int lane, int64_t stride, int columns) {
    row0 = wave * count * rows + lane / Shape::pieces;
#pragma unroll
    for (int i = 0; i < count; ++i) {
      const int row = row0 + i * rows;
      column[i] = ((lane % Shape::pieces) ^ Shape::swap(row)) * (16 / (int)sizeof(T));
      if (column[i] >= columns) column[i] = -1;
      offset[i] = (uint32_t)((row * stride + column[i]) * (int)sizeof(T));
    }
  }
  template <bool ALIGNED>
  __device__ __forceinline__ void load(const T* from, int64_t stride, int n, char* tile, int wave, int lane) const {
    char* to = tile + wave * count * 1024;
    if (ALIGNED && n == C) {
#pragma unroll
      for (int i = 0; i < count; ++i)
        if (column[i] >= 0) request((const char*)from + offset[i], to + i * 1024);
    } else {
#pragma unroll
      for (int i = 0; i < count; ++i) {
        if (column[i] < 0) continue;
        const T* at = from + min(row0 + i * rows, n - 1) * stride + column[i];
        if (ALIGNED)
          request(at, to + i * 1024);
        else
          *reinterpret_cast<u32x4*>(to + i * 1024 + lane * 16) = piece_of_elements(at);
      }
    }
  }
  static __device__ __forceinline__ void request(const void* from, char* to) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from, (LA_LDS(void)*)to, 16, 0, 0);
  }
};

// 16 bytes of a row from the accumulators of O^T.  In bfloat16 the lanes of two neighbouring groups of 16 change halves
// between two accumulators, 4 columns of 16 rows each: one has then 8 columns of a row of the first, the other of the second.
template <int CT>
__device__ __forceinline__ u32x4 rows_of_out(int x, const f32x4 (&o)[CT], float) { return __builtin_bit_cast(u32x4, o[x]); }
template <int CT>
__device__ __forceinline__ u32x4 rows_of_out(int x, const f32x4 (&o)[CT], bf16) {
  const mi_u32x2 p = __builtin_bit_cast(mi_u32x2, to_half(o[2 * x])), q = __builtin_bit_cast(mi_u32x2, to_half(o[2 * x + 1]));
  const auto lo = __builtin_amdgcn_permlane16_swap(p[0], q[0], false, false);
  const auto hi = __builtin_amdgcn_permlane16_swap(p[1], q[1], false, false);
  return u32x4{(uint32_t)lo[0], (uint32_t)hi[0], (uint32_t)lo[1], (uint32_t)hi[1]};
}

// All but the last `N` requests to memory of the wave are done, and every wave's LDS accesses; the waves meet.
template <int N>
__device__ __forceinline__ void arrive() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

__device__ __forceinline__ bool all_finite(s16x8 x) {
  bool ok = true;
#pragma unroll
  for (int i = 0; i < 8; ++i) ok &= (x[i] & 0x7f80) != 0x7f80;
  return ok;
}
__device__ __forceinline__ bool all_finite(f32x8 x) {
  bool ok = true;
#pragma unroll
  for (int i = 0; i < 8; ++i) ok &= fabsf(x[i]) < INFINITY;
  return ok;
}
__device__ __forceinline__ f32x4 half_of(s16x8 x, int h) { return h ? widen(__builtin_shufflevector(x, x, 4, 5, 6, 7)) : widen(__builtin_shufflevector(x, x, 0, 1, 2, 3)); }
__device__ __forceinline__ f32x4 half_of(f32x8 x, int h) { return h ? __builtin_shufflevector(x, x, 4, 5, 6, 7) : __builtin_shufflevector(x, x, 0, 1, 2, 3); }

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

// PBUF: buffers of P.
template <typename T, int DP, int WAVES, int C, int PBUF>
struct ChunkShape {
  static constexpr int waves = WAVES, threads = 64 * WAVES;
  static constexpr int VS = 16 * waves;
  static constexpr int parts = Split<T>::parts;
  static constexpr int q_bytes = C * Tile<T, DP>::stride, v_bytes = C * Tile<T, VS>::stride;
  static constexpr int part_bytes = C * Tile<T, C>::stride, p_bytes = parts * part_bytes;
  static constexpr int lds(bool states) {
    return 2 * (q_bytes + v_bytes) + (states ? 0 : 2 * q_bytes + PBUF * p_bytes);
  }
};

// What bounds it (that workload, 214 us at 3.1 TB/s): the matrix cores are busy for 38% of the time, the vector ALUs and the
// LDS for about as long, memory for half of it.  With 8 waves on a compute unit, all that the registers (256) and the LDS
// (144 KB) allow, the waits between a head's products are not covered: with S and P in two parts it took 186 us, 142 of
// them without loads and stores, 25 less without stores, 0 to 17 less without any one of the products.  Chunks of 32 tokens
// are slower with heads of 128 (273 us for the whole call, 260 with 64; 8 requests of 8,192 tokens together 75, 70) and
// were quicker with heads up to 64, where several workgroups share a compute unit (8,192 tokens, 32 heads: 76 us, 114 with
// 64).
//
// STATES: only what a segment adds to its request's state (from zero), left in `work`; the last segment's is not needed.
// ALIGNED: rows of q, k, v and out start at multiples of 16 bytes, and a chunk of a tensor spans less than 2^31 bytes.
template <typename T, int DP, int WAVES, int C, int PBUF, bool STATES, bool ALIGNED, int PER_SIMD>
__global__ __launch_bounds__(64 * WAVES, PER_SIMD) void la_chunk_kernel(LinearAttention a) {
  typedef ChunkShape<T, DP, WAVES, C, PBUF> Shape;
  typedef typename Half<T>::type half;
  typedef typename Half<T>::pair pair;
  constexpr int PARTS = Shape::parts, KX = DP / 32, KB = KX < 4 ? KX : 4, CX = C / 32, CT = C / 16, VS = Shape::VS;
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  __shared__ float power[C + 1];     // a^i
  __shared__ float scaled[C + 1];    // scale a^i, as far as it ends too
  __shared__ float left[2 * C];      // a^(C-1-i), zeros from C on
  __shared__ int found;
  char* const k_lds = lds;
  char* const v_lds = k_lds + 2 * Shape::q_bytes;
  char* const q_lds = v_lds + 2 * Shape::v_bytes;
  char* const p_lds = q_lds + 2 * Shape::q_bytes;

  const int tid = threadIdx.x, lane = tid & (MI_WAVE - 1), l16 = lane & 15, g = lane / 16, g4 = 4 * g;
  const int wave = __builtin_amdgcn_readfirstlane(tid / MI_WAVE);
  const int slices = (a.d + VS - 1) / VS;
  const int h = blockIdx.x % a.nkv, slice = blockIdx.x / a.nkv % slices, unit = blockIdx.x / (a.nkv * slices);
  const int d = a.d;

  int b = unit, lo, hi, segment = 0, segments = 1;
  if (a.segment) {
    if (a.num_requests == 1) {
      b = 0;
    } else {
      if (tid == 0) found = 0;
      __syncthreads();
      int n = 0;
      for (int i = tid; i < a.num_requests; i += Shape::threads) n += first_unit(a, i) <= unit;
      if (n) atomicAdd(&found, n);
      __syncthreads();
      b = found - 1;
      if (b < 0) return;
    }
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
  const bool columns = n0 < d;                           // whether it has any: else it helps with loads and P only
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
  if (d < DP || d < (slice + 1) * VS) {                  // columns past the end
    for (int i = tid; i < Shape::lds(STATES) / 16; i += Shape::threads) reinterpret_cast<u32x4*>(lds)[i] = u32x4{0, 0, 0, 0};
    __syncthreads();
  }
  auto tables = [&]() {              // (after the first requests to memory: the exponentials take a while)
    if (tid <= C) {
      const float p = decay_power(a.log_decay[h], tid);
      power[tid] = p;
      const float ps = p * a.scale;
      scaled[tid] = ps == 0.f && p != 0.f && a.scale != 0.f ? copysignf(1.4e-45f, a.scale) : ps;
      if (tid < C) left[C - 1 - tid] = p;
    }
    for (int i = C + tid; i < 2 * C; i += Shape::threads) left[i] = 0.f;
    if (!STATES && CX == 1)          // (of chunks of 32 tokens nobody makes P's block that is all behind its queries)
      for (int i = tid; i < PBUF * Shape::p_bytes / 16; i += Shape::threads) reinterpret_cast<u32x4*>(p_lds)[i] = u32x4{0, 0, 0, 0};
    __syncthreads();
  };

  // the wave's columns of the state, accumulators (x, y): row dim_of(x, y, g4 + i), column n0 + l16
  f32x4 s[KX][2];
  float* const s_row = a.state + (int64_t)row * a.state_stride + (int64_t)h * d * d;
  float* const s_work = a.segment ? a.work + ((int64_t)unit * a.nkv + h) * d * d : nullptr;
  float* const s_to = STATES ? s_work : segment == segments - 1 && row != a.idle_row ? s_row : nullptr;
  const float* const s_from = segments > 1 ? s_work : row == a.idle_row ? nullptr : s_row;

  const T* const kp = (const T*)a.k + (int64_t)h * d;
  const T* const vp = (const T*)a.v + (int64_t)h * d + slice * VS;
  const T* const qp = (const T*)a.q + (int64_t)h * a.rep * d;
  const Loader<T, DP, C, WAVES> k_way(wave, lane, a.k_stride, d), q_way(wave, lane, a.q_stride, d);
  const Loader<T, VS, C, WAVES> v_way(wave, lane, a.v_stride, d - slice * VS);
  auto load_kv = [&](int t, int n, int buf) {
    k_way.template load<ALIGNED>(kp + t * a.k_stride, a.k_stride, n, k_lds + buf * Shape::q_bytes, wave, lane);
    v_way.template load<ALIGNED>(vp + t * a.v_stride, a.v_stride, n, v_lds + buf * Shape::v_bytes, wave, lane);
  };
  // f(element of the wave's columns of the state, its place)
  auto each_of_state = [&](auto f) {
    auto walk = [&](int cols) {
#pragma unroll
      for (int x = 0; x < KX; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = dim_of<T>(x, y, i) + dim_of<T>(0, 0, g4);
            if (r < cols) s[x][y][i] = f(s[x][y][i], (dim_of<T>(0, 0, g4) * cols + n0 + l16) + dim_of<T>(x, y, i) * cols);
          }
    };
    if (d == DP) walk(DP);           // (the usual sizes: no checks, constant strides)
    else if (n0 + l16 < d) walk(d);
  };
  auto load_state = [&]() {
#pragma unroll
    for (int x = 0; x < KX; ++x)
#pragma unroll
      for (int y = 0; y < 2; ++y) s[x][y] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (!STATES && s_from) each_of_state([&](float, int at) { return s_from[at]; });
  };

  const DownAt<T, DP> k_down(lane, 0);
  const DownAt<T, VS> v_down(lane, wave * 16);
  pair vt[CX];                       // V^T of the chunk: the wave's 16 columns
  auto read_v = [&](int buf, int n) {
#pragma unroll
    for (int x = 0; x < CX; ++x) {
      vt[x] = columns_down(v_lds + buf * Shape::v_bytes, v_down, x);
      if (n < C) {                   // (a weight of zero times what is not finite is not zero)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (summed<T>(x, i / 4, g, i % 4) >= n) vt[x][i] = 0;
      }
    }
  };
  auto update = [&](int buf, int n, bool infinities) {       // the state after a chunk of n tokens; infinities: V may hold some
    const char* const kb = k_lds + buf * Shape::q_bytes;
    const float an = power[n];
#pragma unroll
    for (int x = 0; x < KX; ++x)
#pragma unroll
      for (int y = 0; y < 2; ++y) s[x][y] *= an;
#pragma unroll
    for (int j = 0; j < CX; ++j) {
      f32x4 w[2];                    // a^(n-1-token)
#pragma unroll
      for (int y = 0; y < 2; ++y)
#pragma unroll
        for (int i = 0; i < 4; ++i) w[y][i] = left[C - n + summed<T>(j, y, g, i)];
      const f32x4 wv[2] = {half_of(vt[j], 0) * w[0], half_of(vt[j], 1) * w[1]};
      Split<T> v0(wv[0]), v1(wv[1]);
      if (infinities) {
        v0.keep_infinities(wv[0]);
        v1.keep_infinities(wv[1]);
      }
#pragma unroll
      for (int x0 = 0; x0 < KX; x0 += 2) {
        pair kd[2][2];
        dims_down(kd, kb, k_down, j, x0);
#pragma unroll
        for (int z = 0; z < Split<T>::parts; ++z)
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int y = 0; y < 2; ++y) mma(s[x0 + x][y], kd[x][y], join(v0.part[z], v1.part[z]));
      }
    }
  };

  // The chunk at hand has the n tokens from t on.
  int t = lo, n = min(C, hi - lo), kv = 0;
  if constexpr (STATES) {
    load_state();                    // (zeros)
    load_kv(t, n, 0);
    tables();
    arrive<0>();
    for (;;) {
      const bool more = t + n < hi;
      if (more) load_kv(t + n, min(C, hi - t - n), kv ^ 1);
      if (columns) {
        read_v(kv, n);
        update(kv, n, true);
      }
      if (!more) break;
      arrive<0>();
      t += n;
      n = min(C, hi - t);
      kv ^= 1;
    }
  } else {
    // the 16 bytes of a row of out that a lane writes (see rows_of_out)
    constexpr int OUT_STEP = 4 / (int)sizeof(T), STORES = CT / OUT_STEP;
    const int out_row = sizeof(T) == 2 ? 16 * (g & 1) + l16 : l16, out_col = n0 + (sizeof(T) == 2 ? 8 * (g >> 1) : g4);
    const uint32_t out_offset = (uint32_t)((out_row * a.out_stride + out_col) * (int)sizeof(T));
    const OperandAt<T, DP> q_at(lane);
    const OperandAt<T, C> p_at(lane);
    // the query head whose Q is fetched next: head fg of tokens ft .. ft + fn - 1
    int ft = t, fn = n, fg = 0, slot = 0;
    auto fetch_q = [&]() {
      if (ft >= hi) return;
      q_way.template load<ALIGNED>(qp + ft * a.q_stride + fg * d, a.q_stride, fn, q_lds + slot * Shape::q_bytes, wave, lane);
      slot ^= 1;
      if (++fg == a.rep) {
        fg = 0;
        ft += fn;
        fn = min(C, hi - ft);
      }
    };
    auto fetch_kv = [&](int from, int buf) {
      if (from < hi) load_kv(from, min(C, hi - from), buf);
    };
    load_kv(t, n, 0);
    fetch_q();
    load_state();
    fetch_kv(t + C, 1);
    fetch_q();
    tables();
    // The wave's block of P, of those that some product reads: 16 queries and 16 tokens in chunks of 32 (three blocks), else
    // 16 and 32 (six).  Waves without columns take one first.
    constexpr int P_WIDE = CX == 1 ? 1 : 2, BLOCKS = CX == 1 ? 3 : 2 * CT - 2;
    static_assert(CX <= 2 && BLOCKS <= WAVES, "a block to a wave");
    const int idle = max(0, WAVES - (d - slice * VS + 15) / 16), block = columns ? idle + wave : wave - (WAVES - idle);
    const int p_row = CX == 1 ? 16 * min(block, 1) : 16 * (block < CT ? block : block - CT + 2);
    const int p_col = CX == 1 ? 16 * (block / 2) : block < CT ? 0 : 32;
    // its weights a^(i-j) and the a^(i+1) of the wave's queries, both with the scale
    const int reach = p_row + l16 - (p_col + g4);          // i - j of a lane's first element: those of the next ones are less
    f32x4 weight[P_WIDE];
#pragma unroll
    for (int w = 0; w < P_WIDE; ++w)
#pragma unroll
      for (int i = 0; i < 4; ++i) weight[w][i] = scaled[min(max(reach - 16 * w - i, 0), C)];
    // the state's parts but the first, which is the state's upper halves: held for all query heads of a chunk where there
    // are registers for them
    constexpr bool HELD = DP <= 128 && PARTS > 1;
    pair sp[HELD ? KX : 1][PARTS];
    bool odd = false;                // whether one of the wave's values is not finite
    bool infinite = false;           // whether its state holds infinities
    auto split_state = [&](int to, int x) {
      Split<T> s0(s[x][0]), s1(s[x][1]);
      if (infinite) {
        s0.keep_infinities(s[x][0]);
        s1.keep_infinities(s[x][1]);
      }
#pragma unroll
      for (int z = 1; z < PARTS; ++z) sp[to][z] = join(s0.part[z], s1.part[z]);
    };
    bool stored = false;             // whether the last head's rows of out are known to be STORES stores of the wave
    arrive<0>();
    // (the state is here: else the compiler would wait for it, and for all that came after it, in every turn)
#pragma unroll
    for (int x = 0; x < KX; ++x)
#pragma unroll
      for (int y = 0; y < 2; ++y) asm volatile("" : "+v"(s[x][y]));
    int head = 0, qb = 0, pb = 0;
    for (;;) {
      const bool last = head + 1 == a.rep;
      if (head == 0 && columns) {
        read_v(kv, n);
        odd = false;
#pragma unroll
        for (int x = 0; x < CX; ++x) odd |= !all_finite(vt[x]);
        odd = __ballot(odd) != 0;
        if (PARTS > 1) {
          float top = 0.f;
#pragma unroll
          for (int x = 0; x < KX; ++x)
#pragma unroll
            for (int y = 0; y < 2; ++y)
#pragma unroll
              for (int i = 0; i < 4; ++i) top = fmaxf(top, fabsf(s[x][y][i]));
          infinite = __ballot(top == INFINITY) != 0;
        }
        if (HELD) {
#pragma unroll
          for (int x = 0; x < KX; ++x) split_state(HELD ? x : 0, x);
        }
      }
      const char* const qt = q_lds + qb * Shape::q_bytes;
      const char* const kt = k_lds + kv * Shape::q_bytes;
      char* const pt = p_lds + pb * Shape::p_bytes;
      // ---- P^T.  All waves wait for it, so it goes before the other wave's products (32,768 tokens 262 us, without that 264;
      // 24 requests of 9,001 tokens together, 32 heads on 8, 164, 166)
      __builtin_amdgcn_s_setprio(1);
      if (block < BLOCKS) {
        f32x4 p[P_WIDE];
#pragma unroll
        for (int w = 0; w < P_WIDE; ++w) p[w] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x0 = 0; x0 < KX; x0 += KB) {
          pair qf[KB], kf[P_WIDE][KB];
#pragma unroll
          for (int kx = 0; kx < KB; ++kx) {
            qf[kx] = operand(qt, q_at, p_row, x0 + kx);
#pragma unroll
            for (int w = 0; w < P_WIDE; ++w) kf[w][kx] = operand(kt, q_at, p_col + 16 * w, x0 + kx);
          }
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int kx = 0; kx < KB; ++kx)
#pragma unroll
            for (int w = 0; w < P_WIDE; ++w) mma(p[w], kf[w][kx], qf[kx]);
        }
#pragma unroll
        for (int w = 0; w < P_WIDE; ++w) {
#pragma unroll
          for (int i = 0; i < 4; ++i) p[w][i] = reach >= 16 * w + i ? p[w][i] * weight[w][i] : 0.f;   // (0 * inf is not 0)
          const Split<T> parts(p[w]);
#pragma unroll
          for (int z = 0; z < PARTS; ++z)
            *reinterpret_cast<half*>(pt + z * Shape::part_bytes + Tile<T, C>::at(p_row + l16, p_col + 16 * w + g4)) = parts.part[z];
        }
      }
      __builtin_amdgcn_s_setprio(0);
      // ---- what the state gives
      f32x4 o[CT];
#pragma unroll
      for (int ib = 0; ib < CT; ++ib) o[ib] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (columns) {
        pair qf[2][CT];
#pragma unroll
        for (int ib = 0; ib < CT; ++ib) qf[0][ib] = operand(qt, q_at, 16 * ib, 0);
#pragma unroll
        for (int x = 0; x < KX; ++x) {
          if (x + 1 < KX) {
#pragma unroll
            for (int ib = 0; ib < CT; ++ib) qf[(x + 1) & 1][ib] = operand(qt, q_at, 16 * ib, x + 1);
          }
          __builtin_amdgcn_sched_barrier(0);
          if (!HELD) split_state(0, x);
          sp[HELD ? x : 0][0] = join(Split<T>::first(s[x][0]), Split<T>::first(s[x][1]));
#pragma unroll
          for (int z = 0; z < PARTS; ++z)
#pragma unroll
            for (int ib = 0; ib < CT; ++ib) mma(o[ib], sp[HELD ? x : 0][z], qf[x & 1][ib]);
        }
#pragma unroll
        for (int ib = 0; ib < CT; ++ib) o[ib] *= scaled[16 * ib + l16 + 1];
        if (last && (t + n < hi || s_to)) update(kv, n, odd);
      }
      // P is whole; the next head's Q and, after the last head, the next chunk's K and V are here: all that was asked for
      // but the last head's rows of out, which went off after it.  This head's Q and, after the last head, the chunk's K
      // and V are read for the last time, so that their places take the Q of the head after next and the chunk after next.
      if (stored) arrive<STORES>();
      else arrive<0>();
      if (last) fetch_kv(t + n + C, kv);
      fetch_q();
      auto store = [&]() {
        T* const o_at = out + t * a.out_stride + (int64_t)(h * a.rep + head) * d;
        if (ALIGNED) {
#pragma unroll
          for (int x = 0; x < STORES; ++x) {
            const u32x4 r = rows_of_out(x, o, T{});
            const int i = out_row + 16 * OUT_STEP * x;
            if (i < n && out_col < d) *reinterpret_cast<u32x4*>((char*)(o_at + 16 * OUT_STEP * x * a.out_stride) + out_offset) = r;
          }
        } else {
#pragma unroll
          for (int ib = 0; ib < CT; ++ib) {
            const int i = 16 * ib + l16;
            if (i < n && n0 + g4 < d)
#pragma unroll
              for (int x = 0; x < 4; ++x) o_at[i * a.out_stride + n0 + g4 + x] = from_float<T>(o[ib][x]);
          }
        }
      };
      // ---- what the chunk's own tokens give
      if (!columns) {
      } else if (!odd) {
        pair pf[2][CT][CX];            // of a part of P; the next part's reads go before this one's products
        auto read_p = [&](int z) {
#pragma unroll
          for (int ib = 0; ib < CT; ++ib)
#pragma unroll
            for (int jx = 0; 2 * jx <= ib; ++jx) pf[z & 1][ib][jx] = operand(pt + z * Shape::part_bytes, p_at, 16 * ib, jx);
        };
        read_p(0);
#pragma unroll
        for (int z = 0; z < PARTS; ++z) {
          if (z + 1 < PARTS) read_p(z + 1);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int jx = 0; jx < CX; ++jx)
#pragma unroll
            for (int ib = 2 * jx; ib < CT; ++ib) {
              if (ib == 2 * jx) mma_first(o[ib], vt[jx], pf[z & 1][ib][jx]);     // (the other half is behind the queries)
              else mma(o[ib], vt[jx], pf[z & 1][ib][jx]);
            }
        }
        store();
      } else {
        // a masked weight of zero times a value that is not finite would reach the tokens before it: only what a token
        // sees is added, one by one
#pragma unroll 1
        for (int at = 0; at < C; ++at) {
          const int j = summed<T>(at / 32, at / 16 % 2, at % 4, at / 4 % 4);
          float mine = 0.f;
#pragma unroll
          for (int x = 0; x < 8 * CX; ++x) mine = x == at / 4 ? half_of(vt[x / 8], x / 4 % 2)[x % 4] : mine;
          f32x4 v;
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] = __shfl(mine, 16 * (at % 4) + g4 + i);
#pragma unroll
          for (int ib = 0; ib < CT; ++ib) {
            const int i = 16 * ib + l16;
            float p = 0.f;
#pragma unroll
            for (int z = 0; z < PARTS; ++z) p += to_float(*reinterpret_cast<const T*>(pt + z * Shape::part_bytes + Tile<T, C>::at(i, j)));
#pragma unroll
            for (int x = 0; x < 4; ++x) o[ib][x] = j <= i ? fmaf(p, v[x], o[ib][x]) : o[ib][x];
          }
        }
        store();
      }
      stored = ALIGNED && n == C && columns;
      if (PBUF == 1) arrive<63>();                 // P is free
      else pb ^= 1;
      qb ^= 1;
      if (last) {
        t += n;
        if (t >= hi) break;
        n = min(C, hi - t);
        kv ^= 1;
        head = 0;
      } else {
        ++head;
      }
    }
  }

  if (s_to) each_of_state([&](float e, int at) { return s_to[at] = e; });
}

#define SCAN_AHEAD 16

// What the segments add becomes the states at their starts, in place: one thread to 4 elements of a request's state.
__global__ __launch_bounds__(64) void la_scan_kernel(LinearAttention a) {
  const int per_head = a.d * a.d / 4;
  const int b = blockIdx.y, i = blockIdx.x * 64 + threadIdx.x;
  int lo, hi;
  bounds_of(a, b, lo, hi);
  const int segments = (hi - lo + a.segment - 1) / a.segment;
  const int row = a.rows[b];
  if (segments <= 1 || i >= a.nkv * per_head || row < 0 || row >= a.num_rows) return;
  const int h = i / per_head;
  const float log_decay = a.log_decay[h];
  f32x4 s = *reinterpret_cast<const f32x4*>(a.state + (int64_t)row * a.state_stride + (int64_t)i * 4);
  const int64_t unit = (int64_t)a.nkv * a.d * a.d;
  float* w = a.work + (int64_t)first_unit(a, b) * unit + (int64_t)i * 4;
  // SCAN_AHEAD at a time: their loads are on their way together (the last segment adds nothing that is needed)
  float an = 0.f;
  for (int x0 = 0; x0 < segments; x0 += SCAN_AHEAD) {
    f32x4 added[SCAN_AHEAD];
#pragma unroll
    for (int x = 0; x < SCAN_AHEAD; ++x) added[x] = *reinterpret_cast<const f32x4*>(w + min(x0 + x, segments - 2) * unit);
    if (x0 == 0) {
      an = decay_power(log_decay, a.segment);
      if (row == a.idle_row) s = f32x4{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int x = 0; x < SCAN_AHEAD; ++x) {
      if (x0 + x < segments) *reinterpret_cast<f32x4*>(w + (x0 + x) * unit) = s;
#pragma unroll
      for (int c = 0; c < 4; ++c) s[c] = fmaf(an, s[c], added[x][c]);
    }
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
  la_scan_kernel<<<dim3((a.nkv * a.d * a.d / 4 + 63) / 64, a.num_requests), 64, 0, stream>>>(a);
  MI_CHECK_LAUNCH("linear attention, scan");
  return launch_chunks<T, DP, WAVES, C, PBUF, false, ALIGNED, PER_SIMD>(a, units, stream);
}

template <typename T, int DP, int WAVES, int C, int PBUF, int PER_SIMD>
static int launch_prompt(const LinearAttention& a, hipStream_t stream) {
  auto fits = [](const void* p, int64_t stride, int bytes) {
    return ((uint64_t)p | (uint64_t)(stride * (int64_t)sizeof(T))) % bytes == 0 && stride * C * (int64_t)sizeof(T) < (1ll << 31);
  };
  const bool aligned = fits(a.q, a.q_stride, 16) && fits(a.k, a.k_stride, 16) && fits(a.v, a.v_stride, 16) &&
                       fits(a.out, a.out_stride, 16);
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
    if (d <= 64) return launch_prompt<bf16, 64, 4, 32, 2, 2>(a, stream);
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
