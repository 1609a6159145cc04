// The product with a weight in 4 bits: checks of a call, and which form takes it.
#include "mx4.cuh"

int cuca_mx4_digits(const CucaMx4Rows* c, const Mx4Rest& rest);
int cuca_mx4_spread(const void* x, int64_t ldx, bool f32, void* out, int ldo, int rows, int cols, cudaStream_t stream);
int cuca_gemm_mx4_codes(const CucaMx4Gemm* c, const Mx4Rest* rest);
int cuca_gemm_mx4_wide(const CucaMx4Gemm* c, bool parts);

namespace {

// Whether bfloat16 rows go as digits, twelve rows in 4 bits each, which saves converting the weight and costs a launch and columns: from
// 2^24 weights on up to ten rows, up to a tile, 16 rows, where there are 5,120 weight rows too (fewer leave a block so much of K to itself
// that columns count for more). Measured, K x weight rows, us, digits and converted weight: 4096 x 4096 1 row 8.5 and 8.9, 8 rows 8.9 and
// 9.3, 12 rows 10.9 and 9.3; 14336 x 4096 1 row 12.4 and 16.1, 10 rows 15.5 and 16.4, 12 rows 18.6 and 16.5; 4096 x 6144 8 rows 9.8 and
// 10.9, 16 rows 11.0 and 11.3; 13824 x 5120 16 rows 18.9 and 25.8; 4096 x 28672 gated 8 rows 16.9 and 29.1, 16 rows 18.4 and 29.3; smaller
// ones 2048 x 2048 8 rows 7.7 and 6.2, 1024 x 5632 gated 8.2 and 6.7, 2048 x 6000 gated 11.8 and 8.2.
bool as_digits(const CucaMx4Gemm* c) {
  const int64_t rows = c->n * (c->epilogue == EPI_SWIGLU ? 2 : 1);
  // (of longer rows what digits leave, up to 8 us a row and 128 values where all of them leave something, would come near a wait's two seconds)
  return rows * c->k >= 1 << 24 && c->k <= 1 << 18 && c->m <= (rows >= 5120 ? 16 : 10);
}

enum Form { CODES, DIGITS, PARTS, ALIGNED, WIDE };

Form form_of(const CucaMx4Gemm* c) {
  if (c->a_kind == MX4_CODES) return CODES;
  // 32-bit rows are three bfloat16 rows each: digits, which share a power of two, would lose bits beside larger values. What that costs, us,
  // with eight digits in brackets: 4096 x 4096 8 rows 10.8 (8.3), 256 rows 32 (34); 4096 x 14336 gated 8 rows 38 (16), 256 rows 203 (105).
  if (c->a_kind == CUCA_F32) return PARTS;
  if (as_digits(c)) return DIGITS;
  return ((uintptr_t)c->a & 15) == 0 && c->lda % 8 == 0 ? WIDE : ALIGNED;  // rows that the copy engine takes
}
int64_t round256(int64_t n) { return (n + 255) / 256 * 256; }
// scratch of rows as digits: their codes, their scales, and what they leave
struct DigitScratch {
  int64_t scales, flags, rest, end;
  explicit DigitScratch(const CucaMx4Gemm* c) {
    const int64_t steps = mx4_steps(c->k);
    scales = round256(c->m * MX4_DIGITS * steps * 64);
    flags = scales + (c->m * MX4_DIGITS + 127) / 128 * steps * 512;
    rest = flags + round256(c->m * steps);
    end = rest + c->m * steps * MX4_STEP * 2;
  }
};

int64_t scratch_of(const CucaMx4Gemm* c) {
  if (c->m <= 0 || c->n <= 0 || c->k <= 0) return 0;
  switch (form_of(c)) {
    case DIGITS: return DigitScratch(c).end;
    case PARTS: return 3 * c->m * ((c->k + 7) / 8 * 16);
    case ALIGNED: return c->m * ((c->k + 7) / 8 * 16);
    default: return 0;
  }
}

}  // namespace

// Bytes of scratch that a call needs, by its rows' kind, address and stride and its sizes.
CUCA_API long long cuca_gemm_mx4_scratch(const CucaMx4Gemm* c) { return scratch_of(c); }

CUCA_API int cuca_gemm_mx4(const CucaMx4Gemm* c) {
  CUCA_REQUIRE(c->a_kind == CUCA_F32 || c->a_kind == CUCA_BF16 || c->a_kind == MX4_CODES, "gemm_mx4: unknown rows %d", (int)c->a_kind);
  CUCA_REQUIRE(c->epilogue >= EPI_STORE && c->epilogue <= EPI_SWIGLU, "gemm_mx4: unknown epilogue %d", (int)c->epilogue);
  CUCA_REQUIRE(c->m >= 0 && c->n >= 0 && c->k > 0 && c->m < (1ll << 27) && c->n < (1ll << 29) && c->k < (1ll << 30),
               "gemm_mx4: %lld x %lld x %lld", (long long)c->m, (long long)c->n, (long long)c->k);
  CUCA_REQUIRE(c->epilogue != EPI_RESIDUAL || c->out_f32, "gemm_mx4: only a 32-bit stream is added to");
  CUCA_REQUIRE(c->epilogue != EPI_SWIGLU || !c->bias, "gemm_mx4: a gated unit takes no bias");
  CUCA_REQUIRE((((uintptr_t)c->w | (uintptr_t)c->w_scales) & 15) == 0 &&
               (c->a_kind != MX4_CODES || (((uintptr_t)c->a | (uintptr_t)c->a_scales) & 15) == 0),
               "gemm_mx4: codes and scales must start on 16 bytes");
  CUCA_REQUIRE(c->m <= 1 || (c->ldo >= c->n && (c->a_kind == MX4_CODES || c->lda >= c->k)), "gemm_mx4: rows overlap");
  if (c->m == 0 || c->n == 0) return 0;
  const Form form = form_of(c);
  CUCA_REQUIRE(form == CODES || form == WIDE || (c->scratch && ((uintptr_t)c->scratch & 255) == 0),
               "gemm_mx4: these rows need scratch on 256 bytes");
  try {
    CucaMx4Gemm d = *c;
    if (form == DIGITS) {
      d.a = c->scratch;
      const DigitScratch at(c);
      uint8_t* const scratch = (uint8_t*)c->scratch;
      const Mx4Rest rest{scratch + at.flags, (const __nv_bfloat16*)(scratch + at.rest)};
      d.a_scales = scratch + at.scales;
      CucaMx4Rows r{const_cast<void*>(c->a), c->lda, c->a_kind, (uint8_t*)c->scratch, const_cast<uint8_t*>(d.a_scales), c->m, c->k, c->stream};
      if (int e = cuca_mx4_digits(&r, rest)) return e;
      return cuca_gemm_mx4_codes(&d, &rest);
    }
    if (form == CODES) return cuca_gemm_mx4_codes(c, nullptr);
    if (form != WIDE) {
      d.a = c->scratch;
      d.lda = (c->k + 7) / 8 * 8;
      if (int e = cuca_mx4_spread(c->a, c->lda, form == PARTS, c->scratch, (int)d.lda, (int)c->m, (int)c->k, c->stream)) return e;
    }
    return cuca_gemm_mx4_wide(&d, form == PARTS);
  } catch (...) {  // the cache of tensor maps may find no memory
    cuca_set_error("gemm_mx4: out of host memory");
    return 3;
  }
}
