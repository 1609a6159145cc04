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
// Both are bound by memory, by the launch where rows are few. A thread takes sixteen values, two threads a block, and eight write the four
// bytes of their step's scales as one word. 2,048 x 14,336 bfloat16 numbers to 4 bits and back take 26.5 us, 5.6 TB/s of what is read and
// written; with eight values a thread, what is done once a thread bound them (43 us).
#include "mx4.cuh"

namespace {

constexpr int THREADS = 256;
constexpr int RUN = 16;         // values of a thread
constexpr int DIGIT_RUN = 8;    // ... that makes digits

struct RowsParams {
  const void* x;
  void* out;
  uint8_t* codes;
  uint8_t* scales;
  int64_t ldx, first;
  uint32_t rows;    // of this launch, from `first` on
  uint32_t runs;    // of a row
  uint32_t magic, shift;  // i / runs = (i * magic >> 32) >> shift, for i below 2^31
  int cols, steps;
  int align;  // rows start on so many bytes: 32, 16 or less
  uint8_t* rest_flags;  // of digits, as Mx4Rest
  __nv_bfloat16* rest;
};

// Row of the launch and run of it that thread i has.
__device__ __forceinline__ uint32_t split(const RowsParams& p, uint32_t i, uint32_t& run) {
  const uint32_t row = __umulhi(i, p.magic) >> p.shift;
  run = i - row * p.runs;
  return row;
}

__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// 32 bytes, past L1.
__device__ __forceinline__ void load32(const void* src, int align, uint32_t (&w)[8]) {
  if (align == 32) {
    asm volatile("ld.relaxed.gpu.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7]) : "l"(src) : "memory");
  } else {
    const uint4 a = __ldcg((const uint4*)src), b = __ldcg((const uint4*)src + 1);
    w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
    w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
  }
}
__device__ __forceinline__ void store32(void* dst, int align, const uint32_t (&w)[8]) {
  if (align == 32) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"l"(dst), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
  } else {
    *(uint4*)dst = make_uint4(w[0], w[1], w[2], w[3]);
    *((uint4*)dst + 1) = make_uint4(w[4], w[5], w[6], w[7]);
  }
}

// N values of a row from c on; zeros past its end.
template <typename T, int N>
__device__ __forceinline__ void load(const RowsParams& p, int64_t row, int c, float (&v)[N]) {
  const T* src = (const T*)p.x + row * p.ldx + c;
  if (p.align >= 16 && c + N <= p.cols) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < N; i += 8) {
        uint32_t w[8];
        load32(src + i, p.align, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i + j] = __uint_as_float(w[j]);
      }
    } else {
      uint32_t w[8];
      if constexpr (N == 16) {
        load32(src, p.align, w);
      } else {
        const uint4 q = __ldcg((const uint4*)src);
        w[0] = q.x; w[1] = q.y; w[2] = q.z; w[3] = q.w;
      }
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = c + i < p.cols ? mx4_read(src + i) : 0.f;
  }
}

// Rows off 16 bytes go through shared memory: the eight threads of a step ask for values next to each other, each eighth of a step at a
// time, and then take their sixteen. (Each asking for its own sixteen, 1,003 x 2,050 32-bit numbers took 25 us to 4 bits and back; so 11.7, the host's pace.)
__device__ __forceinline__ int staged(int value) {  // of a step's 128; sixteen of a thread lie a bank apart from the next thread's
  return (threadIdx.x >> 3) * (MX4_STEP + 8) + value + (value >> 4);
}
constexpr int STAGED = THREADS / 8 * (MX4_STEP + 8);

template <typename T>
__global__ void __launch_bounds__(THREADS) mx4_quantise_kernel(const RowsParams p) {
  pdl_trigger();
  pdl_wait();
  uint32_t run;
  const uint32_t in = split(p, blockIdx.x * THREADS + threadIdx.x, run);
  const bool live = in < p.rows;  // the eight threads of a step alike
  const int64_t row = p.first + in;
  float v[RUN];
  if (p.align < 16) {
    __shared__ float stage[STAGED];
    const int c = (int)(run & ~7u) * RUN + (threadIdx.x & 7);
    const T* src = (const T*)p.x + row * p.ldx + c;
#pragma unroll
    for (int j = 0; j < RUN; ++j) stage[staged(j * 8 + (threadIdx.x & 7))] = live && c + j * 8 < p.cols ? mx4_read(src + j * 8) : 0.f;
    __syncwarp();
#pragma unroll
    for (int j = 0; j < RUN; ++j) v[j] = stage[staged((threadIdx.x & 7) * RUN + j)];
  } else if (live) {
    load<T, RUN>(p, row, run * RUN, v);
  } else {
#pragma unroll
    for (int j = 0; j < RUN; ++j) v[j] = 0.f;
  }
  uint32_t most = 0;
#pragma unroll
  for (int j = 0; j < RUN; ++j) most = max(most, magnitude(v[j]));  // (of a NaN above all others)
  most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
  const bool finite = most < 0x7f800000u;
  const uint32_t field = most >> 23;
  const uint32_t byte = finite ? (field > 2 ? field - 2 : 0) : 255u;
  const float inv = finite ? __uint_as_float((254u - min(byte, 252u)) << 23) : 0.f;  // 2^-e
#pragma unroll
  for (int j = 0; j < RUN; ++j) v[j] *= inv;
  uint2 words = make_uint2(mx4_codes(v), mx4_codes(v + 8));
  if (!finite) words = make_uint2(0, 0);
  // the four blocks' bytes, lowest first, by the step's first thread
  const uint32_t s1 = __shfl_down_sync(0xffffffffu, byte, 2), s2 = __shfl_down_sync(0xffffffffu, byte, 4),
                 s3 = __shfl_down_sync(0xffffffffu, byte, 6);
  if (!live) return;
  *reinterpret_cast<uint2*>(p.codes + row * (p.steps * 64ll) + run * 8) = words;
  if ((run & 7) == 0)
    *reinterpret_cast<uint32_t*>(p.scales + mx4_scale_at(row, run >> 3, p.steps)) = byte | s1 << 8 | s2 << 16 | s3 << 24;
}

// bfloat16 rows as twelve rows in 4 bits each, whose values add up to theirs: digits of three bits (mx4_digit). After twelve what is
// left of a value is at most 2^-35 of its block's largest: nothing, where it is within 2^27 of it. What is left all the same is a
// bfloat16 number too (a multiple of the value's last place, and no larger than it) and is kept beside the digits, for the product
// to add in 32 bits. (Of 32,768 normal values one
// leaves something after eight digits; after twelve one in some six hundred times as many.)
__global__ void __launch_bounds__(THREADS) mx4_digits_kernel(const RowsParams p) {
  pdl_trigger();
  pdl_wait();
  uint32_t run;
  const uint32_t in = split(p, blockIdx.x * THREADS + threadIdx.x, run);
  const bool live = in < p.rows;
  const int64_t row = p.first + in;
  float v[DIGIT_RUN];
#pragma unroll
  for (int j = 0; j < DIGIT_RUN; ++j) v[j] = 0.f;
  if (live) load<__nv_bfloat16, DIGIT_RUN>(p, row, run * DIGIT_RUN, v);
  uint32_t byte = mx4_digit_power(v);
  // the bytes of the step's four blocks, lowest first, for the step's first lane
  uint32_t bytes = byte | __shfl_down_sync(0xffffffffu, byte, 4) << 8 | __shfl_down_sync(0xffffffffu, byte, 8) << 16 |
                   __shfl_down_sync(0xffffffffu, byte, 12) << 24;
  byte = min(byte, 254u);  // (of zeros)
  const bool none = byte == 254;  // a digit could be 2^128: values past 2^127 are left whole
#pragma unroll 3  // (all at once are code that a model's other kernels have pushed out: 0.5 us a product of one row more)
  for (int t = 0; t < MX4_DIGITS; ++t) {
    const uint32_t word = mx4_digit(v, byte, none);
    if (live) {
      const int64_t r = row * MX4_DIGITS + MX4_DIGITS - 1 - t;  // the smallest first
      *reinterpret_cast<uint32_t*>(p.codes + r * (p.steps * 64ll) + run * 4) = word;
      if ((run & 15) == 0) *reinterpret_cast<uint32_t*>(p.scales + mx4_scale_at(r, run >> 4, p.steps)) = bytes;
    }
    byte = max((int)byte - 3, 1);
    bytes = __vmaxu4(__vsubus4(bytes, 0x03030303u), 0x01010101u);
  }
  bool some = false;
#pragma unroll
  for (int j = 0; j < DIGIT_RUN; ++j) some = some || v[j] != 0.f;
  // of this step, which sixteen lanes have
  some = (__ballot_sync(0xffffffffu, some) >> (threadIdx.x & 16) & 0xffffu) != 0;
  if (!live) return;
  const int64_t step = row * p.steps + (run >> 4);
  if ((run & 15) == 0) p.rest_flags[step] = some;
  if (some) {
    uint32_t w[DIGIT_RUN / 2];
#pragma unroll
    for (int j = 0; j < DIGIT_RUN; j += 2) w[j / 2] = __float_as_uint(v[j]) >> 16 | (__float_as_uint(v[j + 1]) & 0xffff0000u);
    *reinterpret_cast<uint4*>(p.rest + step * MX4_STEP + (run & 15) * DIGIT_RUN) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// Rows of any stride and alignment as bfloat16 rows that start on 16 bytes, what is left of a row zeros (for the copy engine). A row of 32
// bits becomes three that add up to it, the smallest first: the bits that bfloat16 has room for, cut off, of the value, of what is left and of what is
// left then. 24 bits are three times eight: nothing is lost from 2^-110 on, below it what lies under 2^-133. (Cut off, not rounded: no
// part is larger than the value.) What is not finite is the first part alone.
template <typename T>
__global__ void __launch_bounds__(THREADS) mx4_spread_kernel(const T* x, int64_t ldx, __nv_bfloat16* out, int ldo, int cols) {
  constexpr int PARTS = sizeof(T) == 4 ? 3 : 1;
  pdl_trigger();
  pdl_wait();
  const T* src = x + blockIdx.x * ldx;
  __nv_bfloat16* dst = out + (int64_t)blockIdx.x * PARTS * ldo;
  for (int c = (blockIdx.y * THREADS + threadIdx.x) * DIGIT_RUN; c < ldo; c += gridDim.y * THREADS * DIGIT_RUN) {
    uint32_t w[PARTS][DIGIT_RUN / 2];
#pragma unroll
    for (int j = 0; j < DIGIT_RUN; ++j) {
      float left = c + j < cols ? mx4_read(src + c + j) : 0.f;
#pragma unroll
      for (int t = 0; t < PARTS; ++t) {
        const uint32_t part = left == left ? __float_as_uint(left) >> 16 : 0x7fffu;
        w[t][j >> 1] = j & 1 ? w[t][j >> 1] | part << 16 : part;
        left = fabsf(left) <= 3.402823466e38f ? left - __uint_as_float(part << 16) : 0.f;
      }
    }
#pragma unroll
    for (int t = 0; t < PARTS; ++t)
      *reinterpret_cast<uint4*>(dst + (int64_t)(PARTS - 1 - t) * ldo + c) = make_uint4(w[t][0], w[t][1], w[t][2], w[t][3]);
  }
}

template <typename T>
__global__ void __launch_bounds__(THREADS) mx4_values_kernel(const RowsParams p) {
  pdl_trigger();
  pdl_wait();
  uint32_t run;
  const uint32_t in = split(p, blockIdx.x * THREADS + threadIdx.x, run);
  const bool live = in < p.rows;
  if (!live && p.align >= 16) return;
  const int64_t row = live ? p.first + in : p.first;
  const int c = (int)run * RUN;
  const uint2 words = __ldcg(reinterpret_cast<const uint2*>(p.codes + row * (p.steps * 64ll) + c / 2));
  const Mx4Factor f = mx4_factor<true>(__ldcg(p.scales + mx4_scale_at(row, c >> 7, p.steps) + ((c >> 5) & 3)));
  uint32_t r[8];  // as bfloat16 numbers, which the values are exactly
  uint32_t t[4];
  mx4_to_bf16<true>(words.x, f, t);
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = t[i];
  mx4_to_bf16<true>(words.y, f, t);
#pragma unroll
  for (int i = 0; i < 4; ++i) r[4 + i] = t[i];
  T* dst = (T*)p.out + row * p.ldx + c;
  if (p.align >= 16 && c + RUN <= p.cols) {
    if constexpr (sizeof(T) == 2) {
      store32(dst, p.align, r);
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          w[2 * i] = r[4 * h + i] << 16;
          w[2 * i + 1] = r[4 * h + i] & 0xffff0000u;
        }
        store32(dst + 8 * h, p.align, w);
      }
    }
  } else if (p.align < 16) {  // as rows come in
    __shared__ float stage[STAGED];
#pragma unroll
    for (int j = 0; j < RUN; ++j)
      stage[staged((threadIdx.x & 7) * RUN + j)] = __uint_as_float(j & 1 ? r[j / 2] & 0xffff0000u : r[j / 2] << 16);
    __syncwarp();
    const int c0 = (int)(run & ~7u) * RUN + (threadIdx.x & 7);
    dst = (T*)p.out + row * p.ldx + c0;
#pragma unroll
    for (int j = 0; j < RUN; ++j)
      if (live && c0 + j * 8 < p.cols) dst[j * 8] = from_f32<T>(stage[staged(j * 8 + (threadIdx.x & 7))]);
  } else {
#pragma unroll
    for (int j = 0; j < RUN; ++j)
      if (c + j < p.cols) dst[j] = from_f32<T>(__uint_as_float(j & 1 ? r[j / 2] & 0xffff0000u : r[j / 2] << 16));
  }
}

enum Form { QUANTISE, VALUES, DIGITS };

int launch_rows(const CucaMx4Rows* c, Form form, const Mx4Rest& rest = {}) {
  const char* what = form == QUANTISE ? "mx4_quantise" : form == VALUES ? "mx4_values" : "gemm_mx4";
  CUCA_REQUIRE(c->dtype == CUCA_F32 || c->dtype == CUCA_BF16, "%s: unknown dtype %d", what, (int)c->dtype);
  CUCA_REQUIRE(c->rows >= 0 && c->cols > 0 && c->cols < (1ll << 30), "%s: %lld rows of %lld values", what, (long long)c->rows, (long long)c->cols);
  CUCA_REQUIRE(c->ldx >= c->cols || c->rows <= 1, "%s: rows overlap", what);
  CUCA_REQUIRE((((uintptr_t)c->codes | (uintptr_t)c->scales) & 15) == 0, "%s: codes and scales must start on 16 bytes", what);
  const int64_t elem = c->dtype == CUCA_F32 ? 4 : 2, steps = mx4_steps(c->cols);
  const int64_t runs = steps * (MX4_STEP / (form == DIGITS ? DIGIT_RUN : RUN));
  RowsParams p{c->x, c->x, c->codes, c->scales, c->ldx, 0, 0, (uint32_t)runs, 0, 0, (int)c->cols, (int)steps, 1,
               const_cast<uint8_t*>(rest.flags), const_cast<__nv_bfloat16*>(rest.values)};
  for (int align = 32; align >= 16 && p.align == 1; align /= 2)
    if ((uintptr_t)c->x % align == 0 && (c->ldx * elem % align == 0 || c->rows == 1)) p.align = align;
  // magic = ceil(2^(32 + shift) / runs) with 2^shift < runs <= 2^(shift + 1) is below 2^32 and off by less than one: exact below 2^31
  while ((2ll << p.shift) < runs) ++p.shift;
  p.magic = (uint32_t)(((1ull << (32 + p.shift)) + runs - 1) / runs);
  const bool f32 = c->dtype == CUCA_F32;
  auto kernel = form == QUANTISE ? (f32 ? mx4_quantise_kernel<float> : mx4_quantise_kernel<__nv_bfloat16>)
                : form == VALUES ? (f32 ? mx4_values_kernel<float> : mx4_values_kernel<__nv_bfloat16>)
                                 : mx4_digits_kernel;
  const int64_t most = ((1ll << 31) - THREADS) / runs;  // rows of a launch
  for (int64_t at = 0; at < c->rows; at += most) {
    p.first = at;
    p.rows = (uint32_t)(c->rows - at < most ? c->rows - at : most);
    const dim3 grid((unsigned)((p.rows * (uint64_t)runs + THREADS - 1) / THREADS));
    cuca_launch(kernel, grid, dim3(THREADS), 0, c->stream, true, p);
    CUCA_CHECK_LAUNCH(what);
  }
  return 0;
}

}  // namespace

CUCA_API int cuca_mx4_quantise(const CucaMx4Rows* c) { return launch_rows(c, QUANTISE); }
CUCA_API int cuca_mx4_values(const CucaMx4Rows* c) { return launch_rows(c, VALUES); }
int cuca_mx4_digits(const CucaMx4Rows* c, const Mx4Rest& rest) { return launch_rows(c, DIGITS, rest); }
int cuca_mx4_spread(const void* x, int64_t ldx, bool f32, void* out, int ldo, int rows, int cols, cudaStream_t stream) {
  int chunks = (ldo + THREADS * DIGIT_RUN - 1) / (THREADS * DIGIT_RUN);
  const dim3 grid(rows, chunks < 64 ? chunks : 64);
  if (f32) cuca_launch(mx4_spread_kernel<float>, grid, dim3(THREADS), 0, stream, true, (const float*)x, ldx, (__nv_bfloat16*)out, ldo, cols);
  else cuca_launch(mx4_spread_kernel<__nv_bfloat16>, grid, dim3(THREADS), 0, stream, true, (const __nv_bfloat16*)x, ldx, (__nv_bfloat16*)out, ldo, cols);
  CUCA_CHECK_LAUNCH("gemm_mx4");
  return 0;
}
