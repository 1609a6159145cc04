// The product with a weight in 4 bits: checks of a call, and which form takes it.
#include "mx4.cuh"
#include <stdlib.h>

int cuca_gemm_mx4_rows(const CucaMx4Gemm* c);
int cuca_gemm_mx4_codes(const CucaMx4Gemm* c);
int cuca_gemm_mx4_wide(const CucaMx4Gemm* c);

CUCA_API int cuca_gemm_mx4(const CucaMx4Gemm* c) {
  CUCA_REQUIRE(c->a_kind == CUCA_F32 || c->a_kind == CUCA_BF16 || c->a_kind == MX4_CODES, "gemm_mx4: unknown rows %d", (int)c->a_kind);
  CUCA_REQUIRE(c->epilogue >= EPI_STORE && c->epilogue <= EPI_SWIGLU, "gemm_mx4: unknown epilogue %d", (int)c->epilogue);
  CUCA_REQUIRE(c->m >= 0 && c->n >= 0 && c->k > 0 && c->m < (1ll << 30) && c->n < (1ll << 29) && c->k < (1ll << 30),
               "gemm_mx4: %lld x %lld x %lld", (long long)c->m, (long long)c->n, (long long)c->k);
  CUCA_REQUIRE(c->epilogue != EPI_RESIDUAL || c->out_f32, "gemm_mx4: only a 32-bit stream is added to");
  CUCA_REQUIRE(c->epilogue != EPI_SWIGLU || !c->bias, "gemm_mx4: a gated unit takes no bias");
  CUCA_REQUIRE((((uintptr_t)c->w | (uintptr_t)c->w_scales) & 15) == 0 &&
               (c->a_kind != MX4_CODES || (((uintptr_t)c->a | (uintptr_t)c->a_scales) & 15) == 0),
               "gemm_mx4: codes and scales must start on 16 bytes");
  if (c->m == 0 || c->n == 0) return 0;
  try {
    if (c->a_kind == MX4_CODES) return cuca_gemm_mx4_codes(c);
    const bool copied = ((uintptr_t)c->a & 15) == 0 && (c->lda % 8 == 0 || c->m == 1);  // rows that the copy engine takes
    if (c->a_kind == CUCA_BF16 && copied && (c->m > 16 || getenv("MXW"))) return cuca_gemm_mx4_wide(c);
    return cuca_gemm_mx4_rows(c);
  } catch (...) {  // the cache of tensor maps may find no memory
    cuca_set_error("gemm_mx4: out of host memory");
    return 3;
  }
}
