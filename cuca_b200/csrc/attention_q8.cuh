// What the attention kernels over 8-bit pages share: their parameters, which rows a block takes, scores and codes.
//
// A cached row is d signed codes and a 32-bit scale (csrc/cache_q8.cu). Codes are whole numbers of at most 127, exact in
// 16-bit floats, and a query times a power of two is too where it came in bfloat16, down to some 2^-20 of its row's largest (in
// 32-bit mode it goes in two 16-bit parts), so the raw score q . codes is as exact as a 32-bit sum of exact products. A row's power
// of two never depends on other rows. The scales never touch the codes:
//
//   s_j = raw_j ks_j (scale log2 e)                 the key's scale multiplies its score (log2 units)
//   vs_j = f_j 2^e_j, 1 <= f_j < 2                  the value's scale goes into the weight: its exponent into the softmax's,
//   z_j = s_j + e_j, u_j = 2^(z_j - max z + LIFT)   its fraction times the weight u_j f_j, which is bounded whatever the scales
//   o   = sum_j (u_j f_j) vcode_j / sum_j u_j 2^-e_j  are, so it fits a 16-bit float
//
// The weights are rounded to 16-bit floats (11 bits; in 32-bit mode to two of them, 22 bits) because the tensor cores take
// them so; every sum, the maximum and the denominator are in 32 bits.
#pragma once
#include "attention_options.cuh"
#include "common.cuh"
#include <cuda_fp16.h>
#include <math.h>

namespace {

// Weights are less than 2^(LIFT + LAG + 1), below 2^15: the running maximum follows a larger one only when it is exceeded by more than
// LAG (rescaling is rare then), and LIFT leaves the largest weight 31 binades above a 16-bit float's least step. Of scores from
// some 2^20 on 32-bit numbers have no steps that small: a score is rounded before the reference is taken off, as the maximum was,
// so that the largest has its exponent to within a step, and a weight that a rounded reference makes too large for a 16-bit float
// becomes the largest one. (Keys that close to the largest share the weight in no certain proportion then: their scores' own steps
// are larger.)
constexpr float Q8_LIFT = 7.f, Q8_LAG = 7.f;

}  // namespace

// A launch, as Python packs it: one 64-bit word each, in this order (kernels/ops.py:attention_q8; so many arguments one by one cost
// the caller 3.6 us, packed 1.1).
struct CucaQ8Attention {
  const void* q;
  int64_t q_stride;  // values between rows
  void* out;
  int64_t out_stride, dtype;
  const int8_t* kpool;
  const int8_t* vpool;
  const float* kscale;
  const float* vscale;
  int64_t n_blocks, bs;
  const int* positions;
  const int* seq_of_row;
  const int* tables;
  int64_t table_stride;
  const int* req_row0;
  const int* req_count;  // null: every request brings one row
  int64_t n_seqs, count_lo, count_hi;  // requests with so many rows are this launch's
  int64_t tile_tokens, n_tiles, tile0;  // rows of a request that a tile takes; how many tiles from which on
  int64_t nh, nkv, d;
  const CucaAttnOptions* opt;
  int64_t heads_per_cta;  // query heads of a key head that a block takes
  int64_t width;          // of a block: column tiles, or query tiles
  int64_t chunk, n_splits;  // keys of a share (the last has the rest) and how many
  float* part;
  int* err;
  cudaStream_t stream;
};
static_assert(sizeof(CucaQ8Attention) == 34 * 8, "one 64-bit word each");

namespace {

struct Q8Params {
  const void* q;
  int q_stride;  // values between rows
  void* out;
  int out_stride;
  const int8_t* kpool;
  const int8_t* vpool;
  const float* kscale;
  const float* vscale;
  int n_blocks, bs;
  int run_shift;  // log2 of bs where it is a power of two, else -1
  const int* tables;
  int table_stride;
  const int* positions;
  const int* seq_of_row;
  const int* req_row0;
  const int* req_count;  // null: every request brings one row
  int n_seqs;
  int count_lo, count_hi;  // requests with so many rows are this launch's
  int tile_tokens;         // rows of a request that a tile takes
  int tile0;               // the launch's first tile
  int width;               // of a block: column tiles, or query tiles
  int nh, nkv, d;
  float scale_log2e;
  float cap;       // > 0: a score s becomes cap tanh(s / cap) ...
  float scale;     // ... of the score with this scale
  float cap_arg;   // 2 log2 e / cap
  int sink;        // the denominator holds one more term exp(0) ...
  const float* sink_val;  // ... or exp(sink_val[head])
  int window, keep;
  const float* slopes;  // slopes[head] * distance is taken off a score
  int heads_per_cta, head_parts;  // a key head's query heads in `head_parts` pieces
  int chunk;       // keys of a block's share (a multiple of 64); 0: all of them
  int n_splits;
  float* part;     // [tiles][kv heads * head parts][splits][columns][d + 2] where a tile's keys are shared out
  int* err;
};

// Which rows tile number `tile` of a launch takes (counted from tile0 on): those of the requests that are the launch's, tile_tokens at a time, a
// request's last ones (which see most keys) first. By every warp for itself.
__device__ __forceinline__ bool q8_rows_of_tile(const Q8Params& p, int tile, int& row0, int& n) {
  tile += p.tile0;
  if (p.req_count == nullptr) {
    row0 = p.req_row0[tile];
    n = 1;
    return true;
  }
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int s0 = 0; s0 < p.n_seqs; s0 += 32) {
    const int s = s0 + lane;
    const int count = s < p.n_seqs ? p.req_count[s] : 0, first = s < p.n_seqs ? p.req_row0[s] : 0;
    const int tiles = count >= p.count_lo && count <= p.count_hi ? (count + p.tile_tokens - 1) / p.tile_tokens : 0;
    int upto = tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    const unsigned past = __ballot_sync(0xffffffffu, before + upto > tile);
    if (past) {
      const int at = __ffs(past) - 1;
      const int its = __shfl_sync(0xffffffffu, tiles, at), its_count = __shfl_sync(0xffffffffu, count, at);
      const int k = its - 1 - (tile - before - (__shfl_sync(0xffffffffu, upto, at) - its));
      row0 = __shfl_sync(0xffffffffu, first, at) + k * p.tile_tokens;
      n = min(p.tile_tokens, its_count - k * p.tile_tokens);
      return true;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  return false;
}

// The keys that some of the rows at positions pos0 .. pos0 + n - 1 see, in groups of U positions counted without the gap
// between the first `keep` and the window: `kept` groups from 0, then those from number `low` on.
struct Q8Keys {
  int kept, low, groups, hi;  // (hi: one past the last position)
  __device__ __forceinline__ int at(int j) const { return j < kept ? j : low + j - kept; }
};
template <int U>
__device__ __forceinline__ Q8Keys q8_keys(const Q8Params& p, int pos0, int n) {
  Q8Keys k;
  k.hi = pos0 + n;
  const int lo = p.window > 0 ? max(0, pos0 - (p.window - 1)) : 0;
  k.low = lo / U;
  k.kept = min((p.keep + U - 1) / U, k.low);
  k.groups = k.kept + (k.hi - 1) / U - k.low + 1;
  return k;
}

// Asynchronous copies into shared memory, and loads from it by address.
__device__ __forceinline__ uint32_t q8_shared(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool ok) {  // zeros where not ok
  const int n = ok ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src, bool ok) {
  const int n = ok ? 4 : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 shared_16(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
  return v;
}
__device__ __forceinline__ uint2 shared_8(uint32_t at) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at));
  return v;
}
__device__ __forceinline__ float shared_f(uint32_t at) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at));
  return v;
}

// Four codes as two pairs of 16-bit floats: x + 128 in the low bits of 1024 (ulp 1), less 1152.
__device__ __forceinline__ uint32_t q8_minus(uint32_t a) {
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(0x64806480u));
  return r;
}
__device__ __forceinline__ uint32_t q8_pair_lo(uint32_t biased) { return q8_minus(__byte_perm(biased, 0x64646464u, 0x4140)); }
__device__ __forceinline__ uint32_t q8_pair_hi(uint32_t biased) { return q8_minus(__byte_perm(biased, 0x64646464u, 0x4342)); }

__device__ __forceinline__ float q8_exp2(float x) {  // 2^x; 0 at -infinity
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t q8_pack(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t q8_pack_weights(float lo, float hi) {  // finite, but for what is no number
  uint32_t r;
  asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float q8_pow2(float e) {  // 2^e, e a whole number of -126 .. 127
  return __uint_as_float((uint32_t)((int)e + 127) << 23);
}
// A value scale as f 2^e (e as a float), and 2^-e for the denominator. e is -60 at least, so that u 2^-e does not leave 32 bits
// where scales are far apart; f is smaller than 1 then, 0 for a row of zeros. (Such a row keeps its part of the denominator beside
// values of up to some 2^80; in 32-bit mode to 20 bits or so, as its exponent in the softmax is that much larger.) A scale that is not finite (2^123 and more, which
// no row has, count as that) makes e, so the weight, NaN where the key is seen; the factors are numbers, so that a masked key's
// weight of zero stays zero.
__device__ __forceinline__ void q8_value_scale(float vs, float& e, float& f, float& inv) {
  const uint32_t bits = (__float_as_uint(vs) >> 23) & 255u, x = max(bits, 67u);
  const bool fine = bits < 250u;
  e = fine ? (float)((int)x - 127) : __uint_as_float(0x7fc00000u);
  inv = fine ? __uint_as_float((254u - x) << 23) : 1.f;
  f = fine ? vs * inv : 1.f;
}
// The power of two that puts magnitudes up to the one with these bits below 2^14, and its inverse (NaN where the row is not
// finite: its scores are NaN then, as they should be).
__device__ __forceinline__ void q8_query_scale(uint32_t top, float& up, float& down) {
  if (top >= 0x7f800000u) {
    up = 0.f;
    down = __uint_as_float(0x7fc00000u);
    return;
  }
  const uint32_t e = max(top >> 23, 14u);
  up = __uint_as_float((267u - e) << 23);
  down = __uint_as_float((e - 13u) << 23);
}
// cap tanh(s / cap) in log2 units. EXACT: for the 32-bit mode; else 1 - 2 / (e^2y + 1), right at both ends, and without a branch
// (a quotient that is rounded right has one, which leaves a warp's threads apart).
template <bool EXACT>
__device__ __forceinline__ float q8_capped(float s, const Q8Params& p) {
  if (EXACT) return p.cap * CUCA_LOG2E * tanhf(s / p.cap);
  return p.cap * CUCA_LOG2E * (1.f - __fdividef(2.f, q8_exp2(s * p.cap_arg) + 1.f));
}
// Two of them through one reciprocal: 1/a = b / (a b). Beyond 2^60 a summand e^2y makes no difference, and the product stays finite.
// (A score that is no number stays none.)
__device__ __forceinline__ float q8_at_most_60(float x) {
  float r;
  asm("min.NaN.f32 %0, %1, 0f42700000;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float2 q8_capped_pair(float2 s, const Q8Params& p) {
  const float2 y = __fmul2_rn(s, make_float2(p.cap_arg, p.cap_arg));
  const float a = q8_exp2(q8_at_most_60(y.x)) + 1.f, b = q8_exp2(q8_at_most_60(y.y)) + 1.f;
  const float r = __fdividef(-2.f * CUCA_LOG2E * p.cap, a * b);
  const float top = p.cap * CUCA_LOG2E;
  return __ffma2_rn(make_float2(r, r), make_float2(b, a), make_float2(top, top));
}
// What a sink adds to a denominator that is relative to the reference m.
__device__ __forceinline__ float q8_sink_term(const Q8Params& p, int head, float m, float lift = Q8_LIFT) {
  return q8_exp2((p.sink_val ? p.sink_val[head] * CUCA_LOG2E : 0.f) - m + lift);
}

// What both entry points check, and the kernels' parameters.
inline int q8_params(const CucaQ8Attention& c, const char* name, int most_d, Q8Params& p) {
  CUCA_REQUIRE(c.dtype == CUCA_F32 || c.dtype == CUCA_BF16, "%s: unknown dtype %lld", name, (long long)c.dtype);
  const CucaAttnOptions* opt = c.opt;
  CUCA_REQUIRE(opt != nullptr && opt->window >= 0 && opt->keep >= 0, "%s: bad options", name);
  CUCA_REQUIRE(opt->gate == nullptr && opt->key_scale == nullptr, "%s: no output gate and no shared rows over 8-bit pages", name);
  CUCA_REQUIRE(c.nkv > 0 && c.nkv <= 65535 && c.nh > 0 && c.nh <= (1 << 20) && c.nh % c.nkv == 0 && c.d >= 16 && c.d <= most_d && c.d % 16 == 0,
               "%s: unsupported shape (heads %lld/%lld, head size %lld)", name, (long long)c.nh, (long long)c.nkv, (long long)c.d);
  CUCA_REQUIRE(c.bs > 0 && c.bs < (1 << 30) && c.n_blocks > 0 && c.n_blocks < (1ll << 31) && c.table_stride > 0 && c.table_stride < (1ll << 31),
               "%s: empty or endless pages or tables", name);
  CUCA_REQUIRE((((uintptr_t)c.kpool | (uintptr_t)c.vpool) & 15) == 0, "%s: pools must be 16-byte aligned", name);
  CUCA_REQUIRE(c.q_stride < (1ll << 31) && c.out_stride < (1ll << 31), "%s: rows too far apart", name);
  CUCA_REQUIRE(c.n_tiles > 0 && c.n_tiles <= 65535 && c.tile0 >= 0 && c.tile0 < (1ll << 30), "%s: %lld tiles from %lld on", name,
               (long long)c.n_tiles, (long long)c.tile0);
  CUCA_REQUIRE(c.chunk >= 0 && c.chunk % 64 == 0 && c.n_splits >= 1 && c.n_splits <= 64 &&
               (c.n_splits == 1 || c.chunk > 0) && ((uintptr_t)c.part & 15) == 0, "%s: bad shares of the keys", name);
  const int group = (int)(c.nh / c.nkv);
  CUCA_REQUIRE(c.heads_per_cta > 0 && c.heads_per_cta <= group && c.tile_tokens > 0 && c.tile_tokens <= 65536, "%s: bad tiles", name);
  p.q = c.q; p.q_stride = (int)c.q_stride; p.out = c.out; p.out_stride = (int)c.out_stride;
  p.kpool = c.kpool; p.vpool = c.vpool; p.kscale = c.kscale; p.vscale = c.vscale;
  p.n_blocks = (int)c.n_blocks; p.bs = (int)c.bs; p.run_shift = (c.bs & (c.bs - 1)) == 0 ? __builtin_ctzll(c.bs) : -1;
  p.tables = c.tables; p.table_stride = (int)c.table_stride; p.positions = c.positions; p.seq_of_row = c.seq_of_row;
  p.req_row0 = c.req_row0; p.req_count = c.req_count; p.n_seqs = (int)c.n_seqs;
  p.count_lo = (int)c.count_lo; p.count_hi = (int)c.count_hi; p.tile_tokens = (int)c.tile_tokens;
  p.tile0 = (int)c.tile0; p.width = (int)c.width;
  p.nh = (int)c.nh; p.nkv = (int)c.nkv; p.d = (int)c.d;
  p.scale = opt->scale; p.scale_log2e = opt->scale * CUCA_LOG2E;
  p.cap = opt->softcap; p.cap_arg = opt->softcap > 0.f ? 2.f * CUCA_LOG2E / opt->softcap : 0.f;
  p.sink = opt->sink ? 1 : 0; p.sink_val = opt->sink ? opt->sink_val : nullptr;
  p.window = opt->window; p.slopes = opt->slopes;
  p.keep = opt->window > 0 ? (opt->keep < 1 << 30 ? opt->keep : 1 << 30) : 0;  // (so that it can be rounded up)
  p.heads_per_cta = (int)c.heads_per_cta; p.head_parts = (group + p.heads_per_cta - 1) / p.heads_per_cta;
  p.n_splits = (int)c.n_splits; p.chunk = c.n_splits > 1 ? (int)c.chunk : 0; p.part = c.part; p.err = c.err;
  return 0;
}

}  // namespace
