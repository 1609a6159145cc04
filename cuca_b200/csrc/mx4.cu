// Rows to microscaled 4-bit floating point and back (layout and codes: mx4.cuh).
//
// With a = max |x| of a block of 32 values:
//
//   e = max(floor(log2 a) - 2, -127),   code = x 2^-e to the nearest of 0, 1/2, 1, 3/2, 2, 3, 4, 6 and their negatives,
//
// ties to the even code, at most 6 (a 2^-e lies in [4, 8)). floor(log2 a) is a's exponent field, so nothing here is approximate and
// equal rows make equal bytes whatever their type, alignment or place. A block of zeros has byte 0. A block that is not finite has
// byte 255 and codes 0 and reads back as NaN whole: codes have no infinity and no NaN of their own.
//
// Both kernels do a few operations per byte: bound by memory, by the launch where rows are few. A thread takes eight values, four
// threads a block, and sixteen write the four bytes of their step's scales as one word.
#include "mx4.cuh"

namespace {

constexpr int THREADS = 256;
constexpr int RUN = 8;  // values of a thread

struct RowsParams {
  const void* x;
  void* out;
  uint8_t* codes;
  uint8_t* scales;
  int64_t ldx, first, rows;  // rows of this launch start at `first`
  int cols, steps;
  bool wide;  // rows start on 16 bytes
};

template <typename T> struct Eight { float v[RUN]; uint32_t most; };  // eight values and the bits of the largest magnitude

__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

template <typename T>
__device__ __forceinline__ Eight<T> load8(const RowsParams& p, int64_t row, int c) {
  Eight<T> e;
  const T* src = (const T*)p.x + row * p.ldx + c;
  if (p.wide && c + RUN <= p.cols) {
    if constexpr (sizeof(T) == 2) {
      const uint4 q = __ldcg(reinterpret_cast<const uint4*>(src));
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        e.v[2 * i] = __uint_as_float(w[i] << 16);
        e.v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    } else {
      const float4 a = __ldcg(reinterpret_cast<const float4*>(src)), b = __ldcg(reinterpret_cast<const float4*>(src) + 1);
      e.v[0] = a.x; e.v[1] = a.y; e.v[2] = a.z; e.v[3] = a.w;
      e.v[4] = b.x; e.v[5] = b.y; e.v[6] = b.z; e.v[7] = b.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < RUN; ++i) e.v[i] = c + i < p.cols ? to_f32(src[i]) : 0.f;
  }
  e.most = 0;
#pragma unroll
  for (int i = 0; i < RUN; ++i) e.most = max(e.most, magnitude(e.v[i]));
  return e;
}

template <typename T>
__global__ void __launch_bounds__(THREADS) mx4_quantise_kernel(const RowsParams p) {
  pdl_trigger();
  pdl_wait();
  const int runs = p.steps * (MX4_STEP / RUN);  // of a row, a multiple of 16
  const int64_t i = (int64_t)blockIdx.x * THREADS + threadIdx.x;
  // (32 bits: a launch has at most 2^31 runs)
  const int64_t in = (uint32_t)i / (uint32_t)runs;
  const int run = (int)((uint32_t)i - (uint32_t)in * (uint32_t)runs);
  const bool live = in < p.rows;  // the sixteen threads of a step alike
  const int64_t row = p.first + (live ? in : 0);
  Eight<T> e;
  e.most = 0;
#pragma unroll
  for (int j = 0; j < RUN; ++j) e.v[j] = 0.f;
  if (live) e = load8<T>(p, row, run * RUN);
  uint32_t most = e.most;
  most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
  most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
  const bool finite = most < 0x7f800000u;
  const uint32_t field = most >> 23;
  const uint32_t byte = finite ? (field > 2 ? field - 2 : 0) : 255u;
  const float inv = __uint_as_float((254u - min(byte, 252u)) << 23);  // 2^-e
  uint32_t word = 0;
  if (finite) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = mx4_first_of(j);
      word |= mx4_code_pair(e.v[i] * inv, e.v[i + 2] * inv) << (8 * j);
    }
  }
  // the four blocks' bytes, lowest first, by the step's first thread
  const uint32_t s1 = __shfl_down_sync(0xffffffffu, byte, 4), s2 = __shfl_down_sync(0xffffffffu, byte, 8),
                 s3 = __shfl_down_sync(0xffffffffu, byte, 12);
  if (!live) return;
  *reinterpret_cast<uint32_t*>(p.codes + row * (p.steps * 64ll) + run * 4) = word;
  if ((run & 15) == 0)
    *reinterpret_cast<uint32_t*>(p.scales + mx4_scale_at(row, run >> 4, p.steps)) = byte | s1 << 8 | s2 << 16 | s3 << 24;
}

// Rows of 16 or 32 bits as eight rows in 4 bits each, whose values add up to theirs: digits of three bits (mx4_digit). After eight what is
// left of a value is at most 2^-23 of its block's largest: of bfloat16 numbers nothing, where they are within 2^14 of it, and where
// some are much larger than the rest the digits that these do not need go to the others.
template <typename T>
__global__ void __launch_bounds__(THREADS) mx4_digits_kernel(const RowsParams p) {
  pdl_trigger();
  pdl_wait();
  const int runs = p.steps * (MX4_STEP / RUN);
  const int64_t i = (int64_t)blockIdx.x * THREADS + threadIdx.x;
  const int64_t in = (uint32_t)i / (uint32_t)runs;
  const int run = (int)((uint32_t)i - (uint32_t)in * (uint32_t)runs);
  const bool live = in < p.rows;
  const int64_t row = p.first + (live ? in : 0);
  Eight<T> e;
#pragma unroll
  for (int j = 0; j < RUN; ++j) e.v[j] = 0.f;
  if (live) e = load8<T>(p, row, run * RUN);
#pragma unroll
  for (int t = 0; t < MX4_DIGITS; ++t) {
    uint32_t byte, word;
    mx4_digit(e.v, byte, word);
    const uint32_t s1 = __shfl_down_sync(0xffffffffu, byte, 4), s2 = __shfl_down_sync(0xffffffffu, byte, 8),
                   s3 = __shfl_down_sync(0xffffffffu, byte, 12);
    if (live) {
      const int64_t r = row * MX4_DIGITS + t;
      *reinterpret_cast<uint32_t*>(p.codes + r * (p.steps * 64ll) + run * 4) = word;
      if ((run & 15) == 0)
        *reinterpret_cast<uint32_t*>(p.scales + mx4_scale_at(r, run >> 4, p.steps)) = byte | s1 << 8 | s2 << 16 | s3 << 24;
    }
  }
}

// bfloat16 rows of any stride and alignment into rows that start on 16 bytes, the rest of a row zeros (for the copy engine)
__global__ void __launch_bounds__(THREADS) mx4_align_kernel(const __nv_bfloat16* x, int64_t ldx, __nv_bfloat16* out, int ldo, int cols) {
  pdl_trigger();
  pdl_wait();
  const __nv_bfloat16* src = x + blockIdx.x * ldx;
  __nv_bfloat16* dst = out + (int64_t)blockIdx.x * ldo;
  for (int c = threadIdx.x * RUN; c < ldo; c += THREADS * RUN) {
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < RUN; ++j)
      if (c + j < cols) w[j >> 1] |= (uint32_t)__ldcg(reinterpret_cast<const unsigned short*>(src) + c + j) << (16 * (j & 1));
    *reinterpret_cast<uint4*>(dst + c) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

template <typename T>
__global__ void __launch_bounds__(THREADS) mx4_values_kernel(const RowsParams p) {
  pdl_trigger();
  pdl_wait();
  const int runs = (p.cols + RUN - 1) / RUN;
  const int64_t i = (int64_t)blockIdx.x * THREADS + threadIdx.x;
  const int64_t in = (uint32_t)i / (uint32_t)runs;
  if (in >= p.rows) return;
  const int c = (int)((uint32_t)i - (uint32_t)in * (uint32_t)runs) * RUN;
  const int64_t row = p.first + in;
  const uint32_t word = __ldcg(reinterpret_cast<const uint32_t*>(p.codes + row * (p.steps * 64ll) + c / 2));
  const uint32_t byte = __ldcg(p.scales + mx4_scale_at(row, c >> 7, p.steps) + ((c >> 5) & 3));
  T* dst = (T*)p.out + row * p.ldx + c;
  T v[RUN];
  const float power = mx4_power(byte);
#pragma unroll
  for (int j = 0; j < RUN; ++j) {
    const uint32_t code = word >> (4 * ((j >> 1) + (j & 1) * 4));
    // the code's bits as a 32-bit number times 2^-126, brought up exactly
    const float x = __uint_as_float((code & 8) << 28 | (code & 7) << 22) * 8.507059173023462e+37f;  // 2^126
    v[j] = from_f32<T>(x * power);
  }
  if (p.wide && c + RUN <= p.cols) {
    if constexpr (sizeof(T) == 2) {
      *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(v);
    } else {
      *reinterpret_cast<float4*>(dst) = *reinterpret_cast<const float4*>(v);
      *reinterpret_cast<float4*>(dst + 4) = *reinterpret_cast<const float4*>(v + 4);
    }
  } else {
#pragma unroll
    for (int j = 0; j < RUN; ++j)
      if (c + j < p.cols) dst[j] = v[j];
  }
}

enum Form { QUANTISE, VALUES, DIGITS };

int launch_rows(const CucaMx4Rows* c, Form form) {
  const char* what = form == QUANTISE ? "mx4_quantise" : form == VALUES ? "mx4_values" : "gemm_mx4";
  CUCA_REQUIRE(c->dtype == CUCA_F32 || c->dtype == CUCA_BF16, "%s: unknown dtype %d", what, (int)c->dtype);
  CUCA_REQUIRE(c->rows >= 0 && c->cols > 0 && c->cols < (1ll << 30), "%s: %lld rows of %lld values", what, (long long)c->rows, (long long)c->cols);
  CUCA_REQUIRE(c->ldx >= c->cols || c->rows <= 1, "%s: rows overlap", what);
  CUCA_REQUIRE((((uintptr_t)c->codes | (uintptr_t)c->scales) & 15) == 0, "%s: codes and scales must start on 16 bytes", what);
  const int64_t elem = c->dtype == CUCA_F32 ? 4 : 2, steps = mx4_steps(c->cols);
  const int64_t runs = form == VALUES ? (c->cols + RUN - 1) / RUN : steps * (MX4_STEP / RUN);
  RowsParams p{c->x, c->x, c->codes, c->scales, c->ldx, 0, 0, (int)c->cols, (int)steps, false};
  p.wide = ((uintptr_t)c->x & 15) == 0 && (c->ldx * elem % 16 == 0 || c->rows == 1);
  const bool f32 = c->dtype == CUCA_F32;
  auto kernel = form == QUANTISE ? (f32 ? mx4_quantise_kernel<float> : mx4_quantise_kernel<__nv_bfloat16>)
                : form == VALUES ? (f32 ? mx4_values_kernel<float> : mx4_values_kernel<__nv_bfloat16>)
                                 : (f32 ? mx4_digits_kernel<float> : mx4_digits_kernel<__nv_bfloat16>);
  const int64_t most = (1ll << 31) / runs;  // rows of a launch
  for (int64_t at = 0; at < c->rows; at += most) {
    p.first = at;
    p.rows = c->rows - at < most ? c->rows - at : most;
    const dim3 grid((unsigned)((p.rows * runs + THREADS - 1) / THREADS));
    cuca_launch(kernel, grid, dim3(THREADS), 0, c->stream, true, p);
    CUCA_CHECK_LAUNCH(what);
  }
  return 0;
}

}  // namespace

CUCA_API int cuca_mx4_quantise(const CucaMx4Rows* c) { return launch_rows(c, QUANTISE); }
CUCA_API int cuca_mx4_values(const CucaMx4Rows* c) { return launch_rows(c, VALUES); }
int cuca_mx4_digits(const CucaMx4Rows* c) { return launch_rows(c, DIGITS); }
int cuca_mx4_align(const void* x, int64_t ldx, void* out, int ldo, int rows, int cols, cudaStream_t stream) {
  cuca_launch(mx4_align_kernel, dim3(rows), dim3(THREADS), 0, stream, true, (const __nv_bfloat16*)x, ldx, (__nv_bfloat16*)out, ldo, cols);
  CUCA_CHECK_LAUNCH("gemm_mx4");
  return 0;
}
