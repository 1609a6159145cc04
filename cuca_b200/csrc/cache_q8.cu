// The key/value cache in 8 bits: quantising rows as they are written, and reading them back.
//
// A row (the d keys or values of one position and key head) is d signed 8-bit codes and a 32-bit scale. With a = max |x|,
//
//   scale = a / 127,   code = round(x * (127 / a)) to the nearest, ties to even,   and the row stands for code * scale.
//
// A row with a < 2^-100 is kept as zeros (scale 0). A row that is not finite gets the scale NaN and codes 0, so it reads back
// as NaN whole and never as something plausible; codes are finite whatever happens, so a masked row can be multiplied by zero.
// The rotation, the quotients and the products are rounded one by one in 32 bits (no fused multiply-adds), so the codes do not
// depend on the form that made them. Rounding to 8 bits here is the cache's own choice: against bfloat16 pages it halves the
// bytes a decode step reads; the error of a value is at most half a 127th of its row's largest.
//
// Both kernels do a few operations per byte and are bound by memory, or by latency when there are few rows. Measured, 32 heads of
// 128 over 8: writing 2,048 rows and reading them back 16.2 us (10.6 and 5.0 by themselves; torch's copy of the queries' part alone
// takes 13.1), reading 34,000 positions back 47 us (5.8 TB/s, 0.89 of a copy's rate).
#include "common.cuh"

int cuca_device_sms();

// A launch of either, as Python packs it: one 64-bit word each, in this order (kernels/ops.py:rope_store_q8, read_q8).
struct CucaQ8Store {
  const void* qkv;
  int64_t row_stride;
  void* q_out;
  int64_t q_stride, dtype;
  const int* positions;
  const int* seq_of_row;
  const int* tables;
  int64_t table_stride;
  const float* cos_t;
  const float* sin_t;
  int64_t table_rows, rot, adjacent;
  void* kpool;
  void* vpool;
  float* kscale;
  float* vscale;
  int64_t n_blocks, bs, n_rows, nh, nkv, d;
  int64_t slices, slice_stride;  // > 0: qkv is so many K slices of the rows, 32-bit, to be added (and `bias` to their sum)
  const void* bias;              // of q_out's type, or null
  int* err;
  cudaStream_t stream;
};
struct CucaQ8Read {
  const void* kpool;
  const void* vpool;
  const float* kscale;
  const float* vscale;
  int64_t n_blocks, bs;
  const int* positions;
  const int* seq_of_row;
  const int* tables;
  int64_t table_stride;
  void* k_out;
  int64_t k_stride;
  void* v_out;
  int64_t v_stride, dtype, n_rows, nkv, d;
  int* err;
  cudaStream_t stream;
};
static_assert(sizeof(CucaQ8Store) == 29 * 8 && sizeof(CucaQ8Read) == 20 * 8, "one 64-bit word each");

namespace {

constexpr float CUCA_Q8_TINY = 7.888609052210118e-31f;  // 2^-100
constexpr int STORE_THREADS = 256;

struct StoreParams {
  const void* qkv;
  int row_stride;  // values between rows; q heads, k heads, v heads from a row's start
  void* q_out;
  int q_stride;
  const int* positions;
  const int* seq_of_row;
  const int* tables;
  int table_stride;
  const float* cos_t;
  const float* sin_t;
  int table_rows, rot, adjacent;
  int8_t* kpool;
  int8_t* vpool;
  float* kscale;
  float* vscale;
  int n_blocks, bs, n_rows, nh, nkv, d;
  int seg_shift;  // log2 of a head's lanes: d / 8, rounded up to a power of two
  int slices;
  size_t slice_stride;
  const void* bias;
  int* err;
};

__device__ __forceinline__ void load4(const float* p, float (&v)[4]) {
  const float4 x = *reinterpret_cast<const float4*>(p);
  v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
}
__device__ __forceinline__ void store4(__nv_bfloat16* p, const float (&v)[4]) {
  __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
  *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<uint32_t*>(&a), *reinterpret_cast<uint32_t*>(&b));
}

// Four codes. 1.5 2^23 more, a number is rounded to a whole one, ties to even, and its low byte is the code; no product exceeds
// 127 by so much that it would be 128. Without `inv` (a row of zeros, or one that is not finite, whose products may be NaN): 0.
__device__ __forceinline__ uint32_t codes4(const float (&v)[4], float inv) {
  uint32_t r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = __float_as_uint(__fadd_rn(__fmul_rn(v[i], inv), 12582912.f));
  const uint32_t codes = __byte_perm(__byte_perm(r[0], r[1], 0x0040), __byte_perm(r[2], r[3], 0x0040), 0x5410);
  return inv > 0.f ? codes : 0;
}

// A row's scale from its largest magnitude, and what its values are multiplied by (0: the codes are).
__device__ __forceinline__ void row_scale(uint32_t top, float& scale, float& inv) {
  const float most = __uint_as_float(top);
  scale = inv = 0.f;
  if (top >= 0x7f800000u) {
    scale = __uint_as_float(0x7fc00000u);
  } else if (most >= CUCA_Q8_TINY) {
    scale = __fdiv_rn(most, 127.f);
    inv = __fdiv_rn(127.f, most);
  }
}

// A group of lanes takes one head of a row; a lane has values 4 l .. 4 l + 3 of each half of the head, which are the rotation's
// pairs where the whole head is rotated in halves (VEC, of K slices: 16-byte accesses).
// Else (part of the head rotated, neighbours as pairs, rows that are not aligned) the same values are fetched one by one with
// their partners. A head stays within a warp, and everything is read before anything is written: q_out may be the rows
// themselves. SLICES: the rows are a contraction's K slices, added in their order in 32 bits (and the bias to the sum), and not
// rounded before they are rotated and quantised.
template <typename T, bool SLICES>
__device__ __forceinline__ float row_value(const StoreParams& p, size_t at, int column) {
  if constexpr (!SLICES) {
    return to_f32(((const T*)p.qkv)[at]);
  } else {
    float x = 0.f;
    for (int s = 0; s < p.slices; ++s) x += ((const float*)p.qkv)[s * p.slice_stride + at];
    return p.bias ? x + to_f32(((const T*)p.bias)[column]) : x;
  }
}
template <typename T>
__device__ __forceinline__ void sliced_values(const StoreParams& p, size_t at, int column, float (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = 0.f;
#pragma unroll 4
  for (int s = 0; s < p.slices; ++s) {
    float x[4];
    load4((const float*)p.qkv + s * p.slice_stride + at, x);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] += x[i];
  }
  if (p.bias)
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] += to_f32(((const T*)p.bias)[column + i]);
}
template <typename T, bool VEC, bool SLICES>
__global__ void __launch_bounds__(STORE_THREADS) rope_store_q8_kernel(const StoreParams p) {
  pdl_trigger();
  pdl_wait();
  const int heads = p.nh + 2 * p.nkv;
  const int head = (int)((blockIdx.y * STORE_THREADS + threadIdx.x) >> p.seg_shift);  // gridDim: rows, heads
  const int l = threadIdx.x & ((1 << p.seg_shift) - 1);
  const int half = p.d / 2, row = blockIdx.x;
  const bool lane_ok = head < heads && 4 * l < half;
  const bool is_q = head < p.nh, is_v = head >= p.nh + p.nkv;
  const bool rotate = !is_v && p.rot > 0;
  const int seq = p.seq_of_row[row], pos = p.positions[row];
  const bool live = lane_ok && seq >= 0;
  const size_t from = (size_t)row * p.row_stride + (size_t)head * p.d;
  float a[4] = {0.f, 0.f, 0.f, 0.f}, b[4] = {0.f, 0.f, 0.f, 0.f};
  if (VEC && lane_ok) {  // (whoever's the row is: its numbers need not be known first)
    sliced_values<T>(p, from + 4 * l, head * p.d + 4 * l, a);
    sliced_values<T>(p, from + half + 4 * l, head * p.d + half + 4 * l, b);
  }
  const bool in_table = pos >= 0 && pos < p.table_rows;
  if (rotate && live && !in_table && l == 0 && p.err) atomicExch(p.err, CUCA_ERR_TOKEN_RANGE);
  const float* cr = p.cos_t + (size_t)(in_table ? pos : 0) * (p.rot / 2);
  const float* sr = p.sin_t + (size_t)(in_table ? pos : 0) * (p.rot / 2);
  if (VEC) {
    if (rotate && in_table && lane_ok) {
      float c[4], s[4];
      load4(cr + 4 * l, c);
      load4(sr + 4 * l, s);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = a[i], y = b[i];
        a[i] = __fsub_rn(__fmul_rn(x, c[i]), __fmul_rn(y, s[i]));
        b[i] = __fadd_rn(__fmul_rn(x, s[i]), __fmul_rn(y, c[i]));
      }
    }
  } else if (live) {
    auto src = [&](int e) { return row_value<T, SLICES>(p, from + e, head * p.d + e); };
    auto value = [&](int e) {
      const float x = src(e);
      if (!rotate || !in_table || e >= p.rot) return x;
      const int hr = p.rot / 2;
      const int i = p.adjacent ? e / 2 : (e < hr ? e : e - hr);
      const bool first = p.adjacent ? (e & 1) == 0 : e < hr;
      const float cs = cr[i], sn = sr[i];
      const float y = src(p.adjacent ? e ^ 1 : (first ? e + hr : i));
      return first ? __fsub_rn(__fmul_rn(x, cs), __fmul_rn(y, sn)) : __fadd_rn(__fmul_rn(y, sn), __fmul_rn(x, cs));
    };
#pragma unroll
    for (int i = 0; i < 4; ++i) { a[i] = value(4 * l + i); b[i] = value(half + 4 * l + i); }
  }
  // the largest magnitude of the head, as bits: anything not finite compares above every number
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) top = max(top, max(__float_as_uint(a[i]) & 0x7fffffffu, __float_as_uint(b[i]) & 0x7fffffffu));
  for (int o = (1 << p.seg_shift) >> 1; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));  // (and all has been read)
  if (!live) return;
  if (is_q) {
    T* dst = (T*)p.q_out + (size_t)row * p.q_stride + (size_t)head * p.d;
    if constexpr (VEC) {
      store4(dst + 4 * l, a);
      store4(dst + half + 4 * l, b);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) { dst[4 * l + i] = from_f32<T>(a[i]); dst[half + 4 * l + i] = from_f32<T>(b[i]); }
    }
    return;
  }
  const int entry = pos / p.bs;
  const int blk = pos >= 0 && entry < p.table_stride ? p.tables[(size_t)seq * p.table_stride + entry] : -1;
  if (blk < 0 || blk >= p.n_blocks) {
    if (l == 0 && p.err) atomicExch(p.err, CUCA_ERR_BLOCK_RANGE);
    return;
  }
  float scale, inv;
  row_scale(top, scale, inv);
  const size_t at = ((size_t)blk * p.nkv + (is_v ? head - p.nh - p.nkv : head - p.nh)) * p.bs + (pos - entry * p.bs);
  int8_t* dst = (is_v ? p.vpool : p.kpool) + at * p.d;
  *reinterpret_cast<uint32_t*>(dst + 4 * l) = codes4(a, inv);
  *reinterpret_cast<uint32_t*>(dst + half + 4 * l) = codes4(b, inv);
  if (l == 0) (is_v ? p.vscale : p.kscale)[at] = scale;
}

// The same for rows on 16 bytes that are rotated whole, in halves, or not at all: a lane has eight values of either half of a head.
// gridDim: rows, heads.
// (Blocks of 96 threads: 2,048 rows written and read back 16.4 us; 64 17.8, 128 17.1, 256 20.3; two heads a thread 2 more.)
constexpr int LINE = 8, LINE_THREADS = 96;
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i += 4) {
    const float4 x = *reinterpret_cast<const float4*>(p + i);
    v[i] = x.x; v[i + 1] = x.y; v[i + 2] = x.z; v[i + 3] = x.w;
  }
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&v)[8]) {
  const uint4 x = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&v)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 x = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&x);
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void store_codes8(int8_t* p, const float (&v)[8], float inv) {
  const float lo[4] = {v[0], v[1], v[2], v[3]}, hi[4] = {v[4], v[5], v[6], v[7]};
  *reinterpret_cast<uint2*>(p) = make_uint2(codes4(lo, inv), codes4(hi, inv));
}
template <typename T>
__global__ void __launch_bounds__(LINE_THREADS, 16) rope_store_q8_lines_kernel(const StoreParams p) {
  pdl_trigger();
  pdl_wait();
  const int heads = p.nh + 2 * p.nkv, half = p.d / 2, row = blockIdx.x;
  const int head = (int)((blockIdx.y * LINE_THREADS + threadIdx.x) >> p.seg_shift);
  const int l = threadIdx.x & ((1 << p.seg_shift) - 1);
  const bool lane_ok = head < heads && LINE * l < half;
  const bool is_q = head < p.nh, is_v = head >= p.nh + p.nkv;
  const int seq = p.seq_of_row[row], pos = p.positions[row];
  float a[LINE], b[LINE];
#pragma unroll
  for (int i = 0; i < LINE; ++i) a[i] = b[i] = 0.f;
  if (lane_ok) {  // (whoever's the row is: its numbers need not be known first)
    const T* src = (const T*)p.qkv + (size_t)row * p.row_stride + (size_t)head * p.d + LINE * l;
    load8(src, a);
    load8(src + half, b);
  }
  if (seq < 0) return;
  int blk = -1, entry = 0;
  if (lane_ok && !is_q) {
    entry = pos / p.bs;
    if (pos >= 0 && entry < p.table_stride) blk = p.tables[(size_t)seq * p.table_stride + entry];
  }
  const bool in_table = pos >= 0 && pos < p.table_rows;
  if (p.rot > 0 && !in_table && threadIdx.x == 0 && blockIdx.y == 0 && p.err) atomicExch(p.err, CUCA_ERR_TOKEN_RANGE);
  if (p.rot > 0 && in_table && lane_ok && !is_v) {
    const float *cr = p.cos_t + (size_t)pos * half + LINE * l, *sr = p.sin_t + (size_t)pos * half + LINE * l;
#pragma unroll
    for (int j = 0; j < LINE; j += 4) {
      float c[4], s[4];
      load4(cr + j, c);
      load4(sr + j, s);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = a[j + i], y = b[j + i];
        a[j + i] = __fsub_rn(__fmul_rn(x, c[i]), __fmul_rn(y, s[i]));
        b[j + i] = __fadd_rn(__fmul_rn(x, s[i]), __fmul_rn(y, c[i]));
      }
    }
  }
  if (lane_ok && is_q) {
    T* dst = (T*)p.q_out + (size_t)row * p.q_stride + (size_t)head * p.d + LINE * l;
    store8(dst, a);
    store8(dst + half, b);
  }
  if (!__any_sync(0xffffffffu, lane_ok && !is_q)) return;  // (a warp of queries)
  // the largest magnitude of the head, as bits: anything not finite compares above every number
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < LINE; ++i)
    top = max(top, max(__float_as_uint(a[i]) & 0x7fffffffu, __float_as_uint(b[i]) & 0x7fffffffu));
  for (int o = (1 << p.seg_shift) >> 1; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (!lane_ok || is_q) return;
  if (blk < 0 || blk >= p.n_blocks) {
    if (l == 0 && p.err) atomicExch(p.err, CUCA_ERR_BLOCK_RANGE);
    return;
  }
  float scale, inv;
  row_scale(top, scale, inv);
  const size_t at = ((size_t)blk * p.nkv + (is_v ? head - p.nh - p.nkv : head - p.nh)) * p.bs + (pos - entry * p.bs);
  int8_t* dst = (is_v ? p.vpool : p.kpool) + at * p.d + LINE * l;
  store_codes8(dst, a, inv);
  store_codes8(dst + half, b, inv);
  if (l == 0) (is_v ? p.vscale : p.kscale)[at] = scale;
}

// ------------------------------------------------------------------ reading back
constexpr int READ_WARPS = 2, READ_PIECES = 4;

template <typename T> struct Piece;  // what a thread writes at once: 16 bytes
template <> struct Piece<float> { static constexpr int N = 4; using Codes = uint32_t; };
template <> struct Piece<__nv_bfloat16> { static constexpr int N = 8; using Codes = uint2; };

struct ReadParams {
  const int8_t* pool[2];
  const float* scale[2];
  void* out[2];
  int out_stride[2];
  const int* positions;
  const int* seq_of_row;
  const int* tables;
  int table_stride, n_blocks, bs, n_rows, nkv, d;
  int* err;
};

__device__ __forceinline__ uint32_t word_of(uint32_t w, int) { return w; }
__device__ __forceinline__ uint32_t word_of(const uint2& w, int i) { return i == 0 ? w.x : w.y; }
// What uses the value stays behind this point, and so behind the other loads (34,000 positions: 47 us, left to the compiler 80).
__device__ __forceinline__ void stay(uint32_t& w) { asm volatile("" : "+r"(w)); }
__device__ __forceinline__ void stay(uint2& w) { asm volatile("" : "+r"(w.x), "+r"(w.y)); }

// A warp brings READ_PIECES x 32 pieces of a row, of one tensor, for ROWS rows whose loads go out together: a lane's places in
// the page and in the row are the same for all of them. gridDim: rows, pieces, tensors.
template <typename T, int ROWS>
__global__ void __launch_bounds__(READ_WARPS * 32) read_q8_kernel(const __grid_constant__ ReadParams p) {
  pdl_trigger();
  pdl_wait();
  using P = Piece<T>;
  constexpr int N = P::N;
  const bool values = blockIdx.z != 0;
  T* out = (T*)(values ? p.out[1] : p.out[0]);
  if (!out) return;
  const int8_t* pool = values ? p.pool[1] : p.pool[0];
  const float* scales = values ? p.scale[1] : p.scale[0];
  const int stride = values ? p.out_stride[1] : p.out_stride[0];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per_head = p.d / N, per_row = per_head * p.nkv;
  int head[READ_PIECES], e[READ_PIECES];  // of the lane's pieces: key head (-1: none), first value
#pragma unroll
  for (int i = 0; i < READ_PIECES; ++i) {
    const int piece = (blockIdx.y * READ_PIECES + i) * 32 + lane;
    head[i] = piece < per_row ? piece / per_head : -1;
    e[i] = (piece - max(head[i], 0) * per_head) * N;
  }
  const int row0 = (blockIdx.x * READ_WARPS + warp) * ROWS;
  int seq[ROWS], pos[ROWS], blk[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    seq[r] = row0 + r < p.n_rows ? p.seq_of_row[row0 + r] : -1;
    pos[r] = row0 + r < p.n_rows ? p.positions[row0 + r] : 0;
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int entry = pos[r] / p.bs;
    blk[r] = seq[r] >= 0 && pos[r] >= 0 && entry < p.table_stride ? p.tables[(size_t)seq[r] * p.table_stride + entry] : -1;
  }
  typename P::Codes w[ROWS][READ_PIECES];
  float s[ROWS][READ_PIECES];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const bool there = blk[r] >= 0 && blk[r] < p.n_blocks;
    if (!there && seq[r] >= 0 && lane == 0 && p.err) atomicExch(p.err, CUCA_ERR_BLOCK_RANGE);
    const size_t at = (size_t)(there ? blk[r] : 0) * p.nkv * p.bs + (there ? pos[r] % p.bs : 0);
#pragma unroll
    for (int i = 0; i < READ_PIECES; ++i) {
      w[r][i] = typename P::Codes{};
      s[r][i] = 0.f;  // (a row of no request, or without a page: zeros)
      if (there && head[i] >= 0) {
        const size_t row = at + (size_t)head[i] * p.bs;
        s[r][i] = __ldg(scales + row);
        w[r][i] = __ldg(reinterpret_cast<const typename P::Codes*>(pool + row * p.d + e[i]));
      }
    }
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r)
#pragma unroll
    for (int i = 0; i < READ_PIECES; ++i) stay(w[r][i]);
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    if (row0 + r >= p.n_rows) break;
#pragma unroll
    for (int i = 0; i < READ_PIECES; ++i) {
      if (head[i] < 0) continue;
      float v[N];
#pragma unroll
      for (int n = 0; n < N; ++n) {  // x + 128 in the low bits of 2^23, less those (a conversion instruction is four times slower)
        const uint32_t biased = word_of(w[r][i], n / 4) ^ 0x80808080u;
        v[n] = (__uint_as_float(__byte_perm(biased, 0x4b000000u, 0x7650 | (n & 3))) - 8388736.f) * s[r][i];
      }
      T* dst = out + (size_t)(row0 + r) * stride + (size_t)head[i] * p.d + e[i];
      if constexpr (N == 4) {
        *reinterpret_cast<float4*>(dst) = make_float4(v[0], v[1], v[2], v[3]);
      } else {
        uint32_t o[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          __nv_bfloat162 t = __floats2bfloat162_rn(v[2 * n], v[2 * n + 1]);
          o[n] = *reinterpret_cast<uint32_t*>(&t);
        }
        *reinterpret_cast<uint4*>(dst) = make_uint4(o[0], o[1], o[2], o[3]);
      }
    }
  }
}

}  // namespace

// Rotates q (into q_out, which may be the rows themselves) and k, quantises k and v and writes them to their pages.
// `adjacent`: neighbouring values are the rotation's pairs instead of the halves of the first `rot`.
CUCA_API int cuca_rope_store_q8(const CucaQ8Store* c) {
  const void* qkv = c->qkv;
  void *q_out = c->q_out, *kpool = c->kpool, *vpool = c->vpool;
  const float *cos_t = c->cos_t, *sin_t = c->sin_t;
  const int dtype = (int)c->dtype, n_rows = (int)c->n_rows, nh = (int)c->nh, nkv = (int)c->nkv, d = (int)c->d, bs = (int)c->bs;
  const int n_blocks = (int)c->n_blocks, table_stride = (int)c->table_stride, rot = (int)c->rot, table_rows = (int)c->table_rows;
  const int row_stride = (int)c->row_stride, q_stride = (int)c->q_stride, adjacent = c->adjacent != 0;
  const cudaStream_t stream = c->stream;
  CUCA_REQUIRE(c->row_stride < (1ll << 31) && c->q_stride < (1ll << 31) && c->n_blocks < (1ll << 31) && c->n_rows < (1ll << 31) &&
               c->table_stride < (1ll << 31) && c->table_rows < (1ll << 31), "rope_store_q8: a size beyond 32 bits");
  CUCA_REQUIRE(dtype == CUCA_F32 || dtype == CUCA_BF16, "rope_store_q8: unknown dtype %d", dtype);
  CUCA_REQUIRE(nh > 0 && nkv > 0 && bs > 0 && n_blocks > 0 && table_stride > 0, "rope_store_q8: empty heads, pages or tables");
  CUCA_REQUIRE(d >= 16 && d <= 256 && d % 16 == 0, "rope_store_q8: head size %d is not a multiple of 16 up to 256", d);
  CUCA_REQUIRE(rot >= 0 && rot <= d && rot % 2 == 0 && (rot == 0 || (cos_t && sin_t)), "rope_store_q8: %d rotated values of %d", rot, d);
  CUCA_REQUIRE(((uintptr_t)kpool & 3) == 0 && ((uintptr_t)vpool & 3) == 0, "rope_store_q8: pools must be 4-byte aligned");
  if (n_rows == 0) return 0;
  StoreParams p{qkv, row_stride, q_out, q_stride, c->positions, c->seq_of_row, c->tables, table_stride, cos_t, sin_t, table_rows, rot,
                adjacent, (int8_t*)kpool, (int8_t*)vpool, c->kscale, c->vscale, n_blocks, bs, n_rows, nh, nkv, d, 0, (int)c->slices,
                (size_t)c->slice_stride, c->bias, c->err};
  const bool slices = c->slices > 0, whole = (rot == d || rot == 0) && !adjacent;
  const uintptr_t tables = (uintptr_t)cos_t | (uintptr_t)sin_t;
  CUCA_REQUIRE(!slices || (dtype == CUCA_BF16 && c->slices <= 64 && c->slice_stride >= 0), "rope_store_q8: K slices give bfloat16 queries");
  const int heads = nh + 2 * nkv, line = dtype == CUCA_F32 ? 4 : 8;  // values of 16 bytes
  if (!slices && whole && row_stride % line == 0 && q_stride % line == 0 &&
      (((uintptr_t)qkv | (uintptr_t)q_out | tables) & 15) == 0 && (((uintptr_t)kpool | (uintptr_t)vpool) & 7) == 0) {
    while ((2 * LINE << p.seg_shift) < d) ++p.seg_shift;
    const unsigned blocks = (unsigned)((((long long)heads << p.seg_shift) + LINE_THREADS - 1) / LINE_THREADS);
    auto kernel = dtype == CUCA_F32 ? rope_store_q8_lines_kernel<float> : rope_store_q8_lines_kernel<__nv_bfloat16>;
    CUCA_REQUIRE(blocks <= 65535, "rope_store_q8: too many heads");
    cuca_launch(kernel, dim3(n_rows, blocks), dim3(LINE_THREADS), 0, stream, true, p);
    CUCA_CHECK_LAUNCH("rope_store_q8");
    return 0;
  }
  while ((8 << p.seg_shift) < d) ++p.seg_shift;
  const bool vec = slices && whole && row_stride % 4 == 0 && q_stride % 4 == 0 && (((uintptr_t)qkv | tables) & 15) == 0 &&
                   c->slice_stride % 4 == 0 && ((uintptr_t)q_out & 7) == 0;
  const unsigned blocks = (unsigned)((((long long)heads << p.seg_shift) + STORE_THREADS - 1) / STORE_THREADS);
  CUCA_REQUIRE(blocks <= 65535, "rope_store_q8: too many heads");
  auto kernel = vec ? rope_store_q8_kernel<__nv_bfloat16, true, true> : slices ? rope_store_q8_kernel<__nv_bfloat16, false, true>
      : dtype == CUCA_F32 ? rope_store_q8_kernel<float, false, false> : rope_store_q8_kernel<__nv_bfloat16, false, false>;
  cuca_launch(kernel, dim3(n_rows, blocks), dim3(STORE_THREADS), 0, stream, true, p);
  CUCA_CHECK_LAUNCH("rope_store_q8");
  return 0;
}

// Rows of k_out / v_out (either may be null): the values that the codes of (seq_of_row, positions) stand for; zeros for a row
// of no request (seq < 0).
CUCA_API int cuca_read_q8(const CucaQ8Read* c) {
  const int dtype = (int)c->dtype, n_rows = (int)c->n_rows, nkv = (int)c->nkv, d = (int)c->d, bs = (int)c->bs;
  const int n_blocks = (int)c->n_blocks, table_stride = (int)c->table_stride, k_stride = (int)c->k_stride, v_stride = (int)c->v_stride;
  const void *kpool = c->kpool, *vpool = c->vpool;
  void *k_out = c->k_out, *v_out = c->v_out;
  const cudaStream_t stream = c->stream;
  CUCA_REQUIRE(c->k_stride < (1ll << 31) && c->v_stride < (1ll << 31) && c->n_blocks < (1ll << 31) && c->n_rows < (1ll << 31) &&
               c->table_stride < (1ll << 31), "read_q8: a size beyond 32 bits");
  CUCA_REQUIRE(dtype == CUCA_F32 || dtype == CUCA_BF16, "read_q8: unknown dtype %d", dtype);
  CUCA_REQUIRE(nkv > 0 && bs > 0 && n_blocks > 0 && table_stride > 0, "read_q8: empty heads, pages or tables");
  CUCA_REQUIRE(d >= 16 && d <= 256 && d % 16 == 0, "read_q8: head size %d is not a multiple of 16 up to 256", d);
  const int n = dtype == CUCA_F32 ? 4 : 8;
  CUCA_REQUIRE((((uintptr_t)k_out | (uintptr_t)v_out) & 15) == 0 && (!k_out || k_stride % n == 0) && (!v_out || v_stride % n == 0) &&
               (((uintptr_t)kpool | (uintptr_t)vpool) & 7) == 0, "read_q8: rows must start on 16 bytes, pools on 8");
  if (n_rows == 0 || (!k_out && !v_out)) return 0;
  ReadParams p{{(const int8_t*)kpool, (const int8_t*)vpool}, {c->kscale, c->vscale}, {k_out, v_out}, {k_stride, v_stride},
               c->positions, c->seq_of_row, c->tables, table_stride, n_blocks, bs, n_rows, nkv, d, c->err};
  const int pieces = nkv * d / n;  // of a row
  // Four rows a warp where that leaves 16 warps an SM (34,000 rows of 8 heads of 128: 47 us, with one row 54), else one (2,048 rows:
  // 5.1 us, with four 6.3).
  const unsigned across = (unsigned)((pieces + 32 * READ_PIECES - 1) / (32 * READ_PIECES));
  const int rows = (long long)n_rows / 4 * across * 2 >= 16ll * cuca_device_sms() ? 4 : 1;
  const dim3 grid((n_rows + READ_WARPS * rows - 1) / (READ_WARPS * rows), across, 2);
  CUCA_REQUIRE(grid.y <= 65535, "read_q8: too many heads");
  auto kernel = dtype == CUCA_F32 ? (rows == 4 ? read_q8_kernel<float, 4> : read_q8_kernel<float, 1>)
                                  : (rows == 4 ? read_q8_kernel<__nv_bfloat16, 4> : read_q8_kernel<__nv_bfloat16, 1>);
  cuca_launch(kernel, grid, dim3(READ_WARPS * 32), 0, stream, true, p);
  CUCA_CHECK_LAUNCH("read_q8");
  return 0;
}
