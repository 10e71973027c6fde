// Linear attention with a decay for each head, over fixed-size states.
//
//   S_t = a S_{t-1} + k_t v_t^T        S [d, d] float32 per request and kv head, a = exp(log_decay[kv head])
//   o_t = scale * q_t S_t              for each of the kv head's query heads
//
// The recurrent form: a workgroup owns 32 columns of one request's and kv head's state in registers and takes the
// tokens one after the other.  It is the whole operator for single tokens, which are bound by the state's bytes (read
// and written once).
#include "common.h"

typedef float f32x4 __attribute__((ext_vector_type(4)));

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
