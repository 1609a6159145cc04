// Matrices in microscaled 4-bit floating point: layout, and what the kernels that read and write them share.
//
// A row is cut into blocks of 32 values. A block is a byte e, which stands for 2^(e - 127) (255: NaN), and 32 codes of 4 bits: a
// sign and one of 0, 1/2, 1, 3/2, 2, 3, 4, 6, so that the low three bits are two of exponent and one of mantissa.
//
//   codes   [rows, steps * 64] bytes; a step is 128 values, and what a row's last step has beyond the row is zeros. Eight codes are a
//           32-bit word, in the order 0, 2, 4, 6, 1, 3, 5, 7 from its lowest bits up: the codes sixteen bits apart are next to
//           each other, so masks and multiplications that work on both halves of a word at once leave pairs in their order. To a
//           product of rows in 4 bits the order is nothing, both operands having it;
//   scales  [tiles of 128 rows, steps, 32, 4, 4] bytes: row r, block b of it at [r / 128, b / 4, r % 32, r % 128 / 32, b % 4].
//           512 bytes are the scales of 128 rows and 128 values as the tensor cores take them (four blocks of a row to a 32-bit
//           column of tensor memory), so they go there without being moved about.
#pragma once
#include "common.cuh"
#include <atomic>

#define MX4_BLOCK 32
#define MX4_STEP 128
#define MX4_DIGITS 12  // rows in 4 bits that make up a bfloat16 row (mx4.cu)

// A launch, as Python packs it: one 64-bit word each, in this order (kernels/ops.py:mx4_quantise, mx4_values, gemm_mx4).
struct CucaMx4Rows {
  void* x;  // rows to be quantised, or to be made of codes and scales
  int64_t ldx, dtype;
  uint8_t* codes;
  uint8_t* scales;
  int64_t rows, cols;
  cudaStream_t stream;
};
struct CucaMx4Gemm {
  const void* a;            // rows of `a_kind`: CUCA_F32, CUCA_BF16 or MX4_CODES
  const uint8_t* a_scales;  // of MX4_CODES
  int64_t lda, a_kind;
  const uint8_t* w;
  const uint8_t* w_scales;
  const void* bias;  // 32-bit where `bias_f32`, else bfloat16; or null
  void* out;
  int64_t ldo, out_f32, bias_f32, m, n, k, epilogue;
  void* scratch;  // what cuca_gemm_mx4_scratch asked for
  int* err;
  cudaStream_t stream;
};
// What the digits of bfloat16 rows leave of them (mx4.cu).
struct Mx4Rest {
  const uint8_t* flags;         // [rows, steps]: a step has anything left
  const __nv_bfloat16* values;  // [rows, steps, 128], written where its flag is set
};
static_assert(sizeof(CucaMx4Rows) == 8 * 8 && sizeof(CucaMx4Gemm) == 18 * 8, "one 64-bit word each");

#define MX4_CODES 2
#define EPI_STORE 0
#define EPI_RESIDUAL 1
#define EPI_SWIGLU 2

namespace {

__host__ __device__ inline int64_t mx4_steps(int64_t cols) { return (cols + MX4_STEP - 1) / MX4_STEP; }
// where the four scales of row r in step s lie (one 32-bit word)
__host__ __device__ inline int64_t mx4_scale_at(int64_t r, int64_t s, int64_t steps) {
  return ((r >> 7) * steps + s) * 512 + (r & 31) * 16 + ((r >> 5) & 3) * 4;
}
// Lets a kernel have `smem` bytes of shared memory on the current device; asked of the runtime once for each device.
template <auto KERNEL>
int mx4_configure(int smem) {
  static std::atomic<uint64_t> done{0};
  int device = 0;
  if (cudaGetDevice(&device) == cudaSuccess && device < 64 && (done.load(std::memory_order_relaxed) >> device & 1)) return 0;
  const cudaError_t e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  CUCA_REQUIRE(e == cudaSuccess, "4-bit product: %s", cudaGetErrorString(e));
  if (device < 64) done.fetch_or(1ull << device, std::memory_order_relaxed);
  return 0;
}

// What an earlier kernel may have written is read past L1 in all of these kernels: a launch that started before the one ahead had ended
// does not find L1 invalidated.
__device__ __forceinline__ float mx4_read(const float* at) { return __ldcg(at); }
__device__ __forceinline__ float mx4_read(const __nv_bfloat16* at) {
  return __uint_as_float((uint32_t)__ldcg(reinterpret_cast<const unsigned short*>(at)) << 16);
}

// 2^(e - 127); NaN for 255
__device__ __forceinline__ float mx4_power(uint32_t e) {
  return __uint_as_float(e == 255 ? 0x7fffffffu : e ? e << 23 : 1u << 22);
}

// Eight values' codes as a word: to the nearest, ties to even, at most 6.
__device__ __forceinline__ uint32_t mx4_codes(const float* v) {
  uint32_t w;
  asm("{\n.reg .b8 a, b, c, d;\n"
      "cvt.rn.satfinite.e2m1x2.f32 a, %3, %1;\ncvt.rn.satfinite.e2m1x2.f32 b, %7, %5;\n"
      "cvt.rn.satfinite.e2m1x2.f32 c, %4, %2;\ncvt.rn.satfinite.e2m1x2.f32 d, %8, %6;\n"
      "mov.b32 %0, {a, b, c, d};\n}\n"
      : "=r"(w) : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return w;
}

// The first power of a block's digits, of which this lane and the three beside it have eight values each: with a = max |v|, the byte of
// 2^e, e = max(ceil(log2 a) - 1, -126). A block that is not finite becomes NaN whole: byte 255, and zeros in place of its values.
__device__ __forceinline__ uint32_t mx4_digit_power(float (&v)[8]) {
  uint32_t most = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) most = max(most, __float_as_uint(v[j]) & 0x7fffffffu);
  most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
  most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
  if (most < 0x7f800000u) return max((int)(most >> 23) - ((most & 0x7fffffu) ? 0 : 1), 1);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = 0.f;
  return 255;
}
// A digit of eight values that are 2^(e+1) at most: d = v / 2^e rounded to a multiple of 1/2, v <- v - d 2^e, every step exact. What is
// left is at most 2^(e-2), so the next digit's power is e - 3, whatever the values: digits need no more of each other than what is left.
// `none`: zeros, and everything is left.
__device__ __forceinline__ uint32_t mx4_digit(float (&v)[8], uint32_t byte, bool none) {
  const float down = none ? 0.f : mx4_power(254 - byte), up = mx4_power(byte);  // 2^-e, 2^e
  float d[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    d[j] = __fadd_rn(__fmul_rn(v[j], down), 6291456.f) - 6291456.f;  // 1.5 * 2^22, whose last place is 1/2
    v[j] = fmaf(-d[j], up, v[j]);
  }
  return mx4_codes(d);
}

// Eight codes as bfloat16 numbers times the power of two that a byte stands for, exactly, in their order.
// A code's sign goes to the sign, its other bits to the lowest exponent bits and the highest mantissa bit, which reads as the
// magnitude times 2^-126 (1/2 as a number below the normal ones); the factor brings it up and applies the scale at once. Both
// moves of a code are one multiplication: by 2^6 + 2^12 its copies do not meet, since 15 (2^6 + 2^12) < 2^16. The integer pipe is
// what the conversion is short of: 9 of its operations for eight codes, with shifts in place of multiplications 15.
struct Mx4Factor { uint32_t first, second; };
__device__ __forceinline__ uint32_t mx4_mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// 2^(e - 1) for e below 128, as `first`; LARGE: any byte, 2^127 and the rest as `second`
template <bool LARGE>
__device__ __forceinline__ Mx4Factor mx4_factor(uint32_t e) {
  if (!LARGE) return {e * 0x00800080u + 126u * 0x00800080u, 0u};
  const uint32_t f = e == 255 ? 0x7fffu : (min(e, 128u) + 126u) << 7;
  const uint32_t s = e > 128 && e < 255 ? (e - 1u) << 7 : 0x3f80u;  // 2^(e - 128)
  return {f | f << 16, s | s << 16};
}
template <bool LARGE>
__device__ __forceinline__ void mx4_to_bf16(uint32_t w, const Mx4Factor& f, uint32_t (&r)[4]) {
  const uint32_t h = w >> 8;
  r[0] = (w & 0x000f000fu) * 4160u;
  r[1] = (w & 0x00f000f0u) * 260u;
  r[2] = (h & 0x000f000fu) * 4160u;
  r[3] = (h & 0x00f000f0u) * 260u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    r[i] = mx4_mul_bf16x2(r[i] & 0x81c081c0u, f.first);
    if (LARGE) r[i] = mx4_mul_bf16x2(r[i], f.second);
  }
}

}  // namespace
