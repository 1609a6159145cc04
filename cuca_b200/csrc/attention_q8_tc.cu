// Causal grouped-query attention over 8-bit pages for portions of tokens, on the 5th-generation tensor cores (bfloat16 rows,
// head sizes up to 128). (Scales, weights and their exactness: attention_q8.cuh.)
//
// A block takes up to 2 x 128 query rows of one request and key head, a row being a (token, head) pair, so that every head of
// the group shares the block's keys and values, and walks the keys in tiles of 64:
//
//   S[128 rows, 64 keys]  = Q K^T      Q and K as 16-bit floats in shared memory (K-major, 128-byte swizzle)
//   O[128 rows, d]       += W V        W from tensor memory, where S was; V as 16-bit floats in shared memory (MN-major)
//
// Four warps fetch the codes (into registers, a tile ahead), turn them into 16-bit floats and store them as operand tiles, with
// each key's factors beside them; four warps per query tile own a row per thread (a lane of tensor memory) and turn scores into
// weights; a warp per query tile issues its products. Where the two query tiles share a converted tile, the conversion is a
// seventh of the block's instructions. Bound by the exponent unit, instruction issue and the tensor pipe, which need about the
// same time for a tile.
//
// Every wait is bounded; when one runs out the kernel records CUCA_ERR_WAIT_TIMEOUT, all roles stop, tensor memory is freed and
// the kernel returns.
#include "attention_q8.cuh"
#include "tcgen05.cuh"

namespace {

constexpr int ROWS = 128;  // query rows of a tile = lanes of tensor memory
constexpr int KEYS = 64;   // keys of a tile
constexpr int NQ = 2;      // query tiles of a block
constexpr int SOFT_WARPS = 4 * NQ, CONV_WARPS = 4;
constexpr int CONV = CONV_WARPS * 32;
constexpr int NTHREADS = (SOFT_WARPS + CONV_WARPS + NQ) * 32;  // softmax, conversion, issue
constexpr int STAGES = 4;
constexpr int TMEM_COLS = 512;  // two score buffers per query tile (4 x 64 columns), results of both (2 x DP)

template <int DP>
struct Shape {
  static constexpr int HALVES = DP / 64;
  static constexpr int Q_HALF = ROWS * 128, Q_BYTES = HALVES * Q_HALF;
  static constexpr int KV_HALF = KEYS * 128, KV_TILE = HALVES * KV_HALF;
  static constexpr int FACTORS = 4 * KEYS * 4;  // of a stage: the keys' factors, the value scales' exponents, 2^-exponents, fractions
  static constexpr int STAGE = 2 * KV_TILE;
  static constexpr int TILES = NQ * Q_BYTES + STAGES * (STAGE + FACTORS);
  static constexpr int SMEM = TILES + 256 + 1024;  // + barriers, + alignment
};

// f16 x f16 -> f32, M = 128, N = n; b_mn: the second operand is MN-major
constexpr uint32_t desc_f16(bool b_mn, int n) {
  return (1u << 4) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}

// 64 columns of a thread's lane. The wait is part of the statement: what uses the registers cannot come before it.
__device__ __forceinline__ void tmem_ld64(uint32_t taddr, uint32_t (&r)[2][32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
      "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, "
      "%22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32, %33, %34, %35, %36, %37, %38, %39, %40, %41, "
      "%42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, "
      "%62, %63"
      "}, [%64];\n\ttcgen05.wait::ld.sync.aligned;"
      :
        "=r"(r[0][0]), "=r"(r[0][1]), "=r"(r[0][2]), "=r"(r[0][3]), "=r"(r[0][4]), "=r"(r[0][5]), "=r"(r[0][6]), "=r"(r[0][7]),
        "=r"(r[0][8]), "=r"(r[0][9]), "=r"(r[0][10]), "=r"(r[0][11]), "=r"(r[0][12]), "=r"(r[0][13]), "=r"(r[0][14]), "=r"(r[0][15]),
        "=r"(r[0][16]), "=r"(r[0][17]), "=r"(r[0][18]), "=r"(r[0][19]), "=r"(r[0][20]), "=r"(r[0][21]), "=r"(r[0][22]), "=r"(r[0][23]),
        "=r"(r[0][24]), "=r"(r[0][25]), "=r"(r[0][26]), "=r"(r[0][27]), "=r"(r[0][28]), "=r"(r[0][29]), "=r"(r[0][30]), "=r"(r[0][31]),
        "=r"(r[1][0]), "=r"(r[1][1]), "=r"(r[1][2]), "=r"(r[1][3]), "=r"(r[1][4]), "=r"(r[1][5]), "=r"(r[1][6]), "=r"(r[1][7]),
        "=r"(r[1][8]), "=r"(r[1][9]), "=r"(r[1][10]), "=r"(r[1][11]), "=r"(r[1][12]), "=r"(r[1][13]), "=r"(r[1][14]), "=r"(r[1][15]),
        "=r"(r[1][16]), "=r"(r[1][17]), "=r"(r[1][18]), "=r"(r[1][19]), "=r"(r[1][20]), "=r"(r[1][21]), "=r"(r[1][22]), "=r"(r[1][23]),
        "=r"(r[1][24]), "=r"(r[1][25]), "=r"(r[1][26]), "=r"(r[1][27]), "=r"(r[1][28]), "=r"(r[1][29]), "=r"(r[1][30]), "=r"(r[1][31])
      : "r"(taddr) : "memory");
}

template <int DP, bool OPT>
__global__ void __launch_bounds__(NTHREADS, 1) attention_q8_tc_kernel(const Q8Params p, const int bs_shift) {
  using SH = Shape<DP>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* q_s = smem;
  uint8_t* kv_s = q_s + NQ * SH::Q_BYTES;
  float* factor_s = (float*)(kv_s + STAGES * SH::STAGE);
  uint64_t* bars = (uint64_t*)((uint8_t*)factor_s + STAGES * SH::FACTORS);
  uint64_t* q_full = bars;                   // [NQ]
  uint64_t* kv_full = q_full + NQ;           // [STAGES]
  uint64_t* kv_empty = kv_full + STAGES;     // [STAGES]
  uint64_t* s_full = kv_empty + STAGES;      // [NQ][2]
  uint64_t* p_full = s_full + 2 * NQ;        // [NQ]
  uint64_t* pv_done = p_full + NQ;           // [NQ]
  uint32_t* tmem_slot = (uint32_t*)(pv_done + NQ);
  volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
  uint32_t* q_top = tmem_slot + 2;           // the largest magnitude of the block's queries, as bits

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_trigger();
  pdl_wait();
  // ---------------------------------------------------------------- rows and keys
  int row0, n_tok;
  if (!q8_rows_of_tile(p, blockIdx.y, row0, n_tok)) return;
  const int kvh = blockIdx.x / p.n_splits, split = blockIdx.x % p.n_splits;
  const int G = p.nh / p.nkv, head0 = kvh * G;
  const int seq = p.seq_of_row[row0];
  const int pos0 = p.positions[row0];
  __nv_bfloat16* out = (__nv_bfloat16*)p.out;
  if (seq < 0 || pos0 < 0) {  // rows of no request
    if (split == 0)
      for (int i = threadIdx.x; i < n_tok * G * p.d; i += NTHREADS)
        out[(size_t)(row0 + i / (G * p.d)) * p.out_stride + (size_t)head0 * p.d + i % (G * p.d)] = __float2bfloat16_rn(0.f);
    return;
  }
  const Q8Keys keys = q8_keys<KEYS>(p, pos0, n_tok);
  const int share = p.chunk > 0 ? p.chunk / KEYS : keys.groups;
  const int first = split * share;
  const int last = split == p.n_splits - 1 ? keys.groups : min(keys.groups, first + share);
  if (first >= last) return;
  const bool alone = share >= keys.groups || p.n_splits == 1;
  const int n_tiles = last - first;
  const int tile_tok = ROWS / G;             // tokens of a query tile
  const int nq = n_tok > tile_tok ? 2 : 1;

  if (warp == SOFT_WARPS + CONV_WARPS) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  if (threadIdx.x == 0) {
    for (int x = 0; x < NQ; ++x) {
      mbar_init(&q_full[x], 128);
      mbar_init(&s_full[2 * x], 1);
      mbar_init(&s_full[2 * x + 1], 1);
      mbar_init(&p_full[x], 128);
      mbar_init(&pv_done[x], 1);
    }
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&kv_full[s], CONV);
      mbar_init(&kv_empty[s], nq);
    }
    *abort_flag = 0;
    *q_top = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  auto tmem_s = [&](int x, int t) { return tmem_base + (uint32_t)((2 * x + (t & 1)) * KEYS); };
  auto tmem_o = [&](int x) { return tmem_base + (uint32_t)(2 * NQ * KEYS + x * DP); };

  if (warp < SOFT_WARPS) {
    // ------------------------------------------------ a query row per thread
    const int x = warp >> 2, quarter = warp & 3;
    const int r = quarter * 32 + lane;  // row of the query tile
    const uint32_t lane_bits = (uint32_t)(quarter * 32) << 16;
    const int tok = x * tile_tok + r / G, head = head0 + r % G;
    const bool row_ok = x < nq && r < tile_tok * G && tok < n_tok;
    uint4 raw_q[DP / 8];
    uint32_t top = 0;
    {
      const __nv_bfloat16* src = (const __nv_bfloat16*)p.q + (size_t)(row0 + (row_ok ? tok : 0)) * p.q_stride + (size_t)head * p.d;
      const bool aligned = ((uintptr_t)p.q & 15) == 0 && p.q_stride % 8 == 0;
#pragma unroll
      for (int c = 0; c < DP / 8; ++c) {
        raw_q[c] = make_uint4(0u, 0u, 0u, 0u);
        if (row_ok && c * 8 < p.d) {
          if (aligned) {
            raw_q[c] = *reinterpret_cast<const uint4*>(src + c * 8);
          } else {
            const unsigned short* h = reinterpret_cast<const unsigned short*>(src + c * 8);
            raw_q[c] = make_uint4(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16, h[4] | (uint32_t)h[5] << 16, h[6] | (uint32_t)h[7] << 16);
          }
        }
        const uint32_t w[4] = {raw_q[c].x, raw_q[c].y, raw_q[c].z, raw_q[c].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) top = max(top, max((w[i] << 16) & 0x7fffffffu, w[i] & 0x7fff0000u));
      }
    }
    // One power of two for the block's rows: what it costs rows much smaller than the largest is far below what a score can
    // show. A row that is not finite goes in as zeros and comes out as NaN.
    const bool bad = top >= 0x7f800000u;
    uint32_t top_w = bad ? 0u : top;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top_w = max(top_w, __shfl_xor_sync(0xffffffffu, top_w, o));
    if (lane == 0) atomicMax(q_top, top_w);
    asm volatile("bar.sync 1, %0;" ::"n"((SOFT_WARPS + CONV_WARPS) * 32) : "memory");
    float up, down;
    q8_query_scale(*q_top, up, down);
    if (x < nq) {
      uint8_t* dst = q_s + x * SH::Q_BYTES + r * 128;
#pragma unroll
      for (int c = 0; c < DP / 8; ++c) {
        const uint32_t w[4] = {raw_q[c].x, raw_q[c].y, raw_q[c].z, raw_q[c].w};
        uint32_t h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          h[i] = bad ? 0u : q8_pack(__uint_as_float(w[i] << 16) * up, __uint_as_float(w[i] & 0xffff0000u) * up);
        *reinterpret_cast<uint4*>(dst + (c / 8) * SH::Q_HALF + (((c & 7) ^ (r & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
      }
      fence_proxy_async();
      mbar_arrive(&q_full[x]);
    }

    const int row_pos = pos0 + tok;
    const int row_lo = p.window > 0 ? row_pos - (p.window - 1) : 0;
    const int least_pos = pos0 + x * tile_tok;  // of the query tile's rows
    const int most_lo = p.window > 0 ? pos0 + min(n_tok, (x + 1) * tile_tok) - 1 - (p.window - 1) : 0;
    const float slope2 = OPT && p.slopes ? p.slopes[head] * CUCA_LOG2E : 0.f;
    float m = -INFINITY, l = 0.f;
    bool ok = x < nq;
    for (int j = 0; ok && j < n_tiles; ++j) {
      const int st = j % STAGES;
      if (!warp_wait(&s_full[2 * x + (j & 1)], (j >> 1) & 1, p.err, abort_flag)) { ok = false; break; }
      tc_fence_after();
      // (long complete: the scores were made from the tile; for the factors that came with it)
      if (!warp_wait(&kv_full[st], (j / STAGES) & 1, p.err, abort_flag)) { ok = false; break; }
      const float4* factor = reinterpret_cast<const float4*>(factor_s + st * 4 * KEYS);
      const int key0 = keys.at(first + j) * KEYS;
      const bool whole = key0 + KEYS - 1 <= least_pos && (p.window <= 0 || key0 >= most_lo || key0 + KEYS <= p.keep);
      uint32_t raw[2][32];
      tmem_ld64(tmem_s(x, j) + lane_bits, raw);
      // z = s + e
      const float bias0 = OPT ? slope2 * (float)(key0 - row_pos) : 0.f;
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float4 kf = factor[c * 8 + i], ve = factor[KEYS / 4 + c * 8 + i];
          const float f[4] = {kf.x, kf.y, kf.z, kf.w}, e[4] = {ve.x, ve.y, ve.z, ve.w};
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int k = 4 * i + 2 * h;
            const float2 r2 = make_float2(__uint_as_float(raw[c][k]), __uint_as_float(raw[c][k + 1]));
            const float2 f2 = make_float2(f[2 * h], f[2 * h + 1]), e2 = make_float2(e[2 * h], e[2 * h + 1]);
            float2 z;
            if (OPT) {
              float2 s2 = __fmul2_rn(r2, f2);
              if (p.cap > 0.f) s2 = make_float2(q8_capped<false>(s2.x, p), q8_capped<false>(s2.y, p));
              s2 = __fadd2_rn(s2, make_float2(fmaf(slope2, (float)(c * 32 + k), bias0), fmaf(slope2, (float)(c * 32 + k + 1), bias0)));
              z = __fadd2_rn(s2, e2);
            } else {
              z = __ffma2_rn(r2, f2, e2);
            }
            raw[c][k] = __float_as_uint(z.x);
            raw[c][k + 1] = __float_as_uint(z.y);
          }
        }
      if (!whole) {
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const int kp = key0 + c * 32 + i;
            if (!(kp <= row_pos && (kp >= row_lo || kp < p.keep))) raw[c][i] = 0xff800000u;
          }
      }
      float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int i = 0; i < 32; i += 2)
          mx4[(i >> 1) & 3] = fmaxf(fmaxf(mx4[(i >> 1) & 3], __uint_as_float(raw[c][i])), __uint_as_float(raw[c][i + 1]));
      const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
      const bool moves = mx > m + Q8_LAG;
      const float corr = moves ? q8_exp2(m - mx) : 1.f;
      if (moves) m = mx;
      const float ref = m == -INFINITY ? 0.f : m - Q8_LIFT;
      const float2 neg2 = make_float2(-ref, -ref);
      float2 sum2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
      uint32_t pw[KEYS / 2];
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float4 vi = factor[2 * KEYS / 4 + c * 8 + i], vf = factor[3 * KEYS / 4 + c * 8 + i];
          const float v[4] = {vi.x, vi.y, vi.z, vi.w}, f[4] = {vf.x, vf.y, vf.z, vf.w};
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int k = 4 * i + 2 * h;
            const float2 x2 = __fadd2_rn(make_float2(__uint_as_float(raw[c][k]), __uint_as_float(raw[c][k + 1])), neg2);
            const float2 u2 = make_float2(q8_exp2(x2.x), q8_exp2(x2.y));
            sum2[h] = __ffma2_rn(u2, make_float2(v[2 * h], v[2 * h + 1]), sum2[h]);
            const float2 w2 = __fmul2_rn(u2, make_float2(f[2 * h], f[2 * h + 1]));
            pw[c * 16 + 2 * i + h] = q8_pack(w2.x, w2.y);
          }
        }
      static_assert(KEYS == 64, "one 32-column store holds a row's weights of a tile");
      __syncwarp();
      tmem_st32_raw(tmem_s(x, j) + lane_bits, pw);
      l = l * corr + (sum2[0].x + sum2[0].y) + (sum2[1].x + sum2[1].y);
      // O is made smaller where a row's maximum moved; only then must the product before have finished (its barrier is never
      // more than a phase ahead: the next product waits for this tile's weights)
      if (j > 0 && __any_sync(0xffffffffu, moves)) {
        if (!warp_wait(&pv_done[x], (j - 1) & 1, p.err, abort_flag)) { ok = false; break; }
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < DP / 32; ++c) {
          float o[32];
          tmem_ld32(tmem_o(x) + lane_bits + c * 32, o);
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] *= corr;
          tmem_st32(tmem_o(x) + lane_bits + c * 32, o);
        }
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&p_full[x]);
    }
    if (ok && warp_wait(&pv_done[x], (n_tiles - 1) & 1, p.err, abort_flag)) {
      tc_fence_after();
      if (alone) {
        if (OPT && p.sink && m != -INFINITY) l += q8_sink_term(p, head, m);
        const float inv = bad ? __uint_as_float(0x7fc00000u) : l == 0.f ? 0.f : 1.f / l;
        __nv_bfloat16* dst = out + (size_t)(row0 + tok) * p.out_stride + (size_t)head * p.d;
        const bool aligned = ((uintptr_t)p.out & 15) == 0 && p.out_stride % 8 == 0;
#pragma unroll
        for (int c = 0; c < DP / 32; ++c) {
          float o[32];
          tmem_ld32(tmem_o(x) + lane_bits + c * 32, o);  // (the whole warp reads)
          if (row_ok) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              if (c * 32 + q * 8 >= p.d) break;
              uint32_t w[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const __nv_bfloat162 t2 = __floats2bfloat162_rn(o[q * 8 + 2 * i] * inv, o[q * 8 + 2 * i + 1] * inv);
                w[i] = *reinterpret_cast<const uint32_t*>(&t2);
              }
              if (aligned) {
                *reinterpret_cast<uint4*>(dst + c * 32 + q * 8) = make_uint4(w[0], w[1], w[2], w[3]);
              } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) dst[c * 32 + q * 8 + i] = __ushort_as_bfloat16((unsigned short)(w[i / 2] >> (16 * (i & 1))));
              }
            }
          }
        }
      } else {
        // [NQ][DP / 4][ROWS][4], then m and l [NQ][2][ROWS]: rows side by side
        float* part = p.part + (((size_t)blockIdx.y * p.nkv + kvh) * p.n_splits + split) * (size_t)(NQ * ROWS * (DP + 2));
        float4* dst = reinterpret_cast<float4*>(part) + (size_t)x * (DP / 4) * ROWS + r;
#pragma unroll
        for (int c = 0; c < DP / 32; ++c) {
          float o[32];
          tmem_ld32(tmem_o(x) + lane_bits + c * 32, o);
#pragma unroll
          for (int q = 0; q < 8; ++q) dst[(c * 8 + q) * ROWS] = make_float4(o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]);
        }
        float* ml = part + NQ * ROWS * DP + x * 2 * ROWS;
        ml[r] = m;
        ml[ROWS + r] = bad ? __uint_as_float(0x7fc00000u) : l;
      }
    }
  } else if (warp < SOFT_WARPS + CONV_WARPS) {
    // ------------------------------------------------ codes to operand tiles
    const int tid = threadIdx.x - SOFT_WARPS * 32;
    constexpr int CHUNKS = DP / 16;                // 16-byte pieces of a row
    constexpr int PER = KEYS * CHUNKS / CONV;      // of a thread, in keys and in values
    constexpr int STEP = CONV / CHUNKS;            // rows between a thread's pieces
    const int c = tid % CHUNKS, r0 = tid / CHUNKS;
    const bool piece = c * 16 < p.d;
    const int* table = p.tables + (size_t)seq * p.table_stride;
    const int lo = p.window > 0 ? max(0, pos0 - (p.window - 1)) : 0;
    // where key number i of tile j stands in the pools, as a row number (-1: nowhere)
    auto entry_of = [&](int j, int i) {  // its page
      if (j >= n_tiles) return -1;
      const int kp = keys.at(first + j) * KEYS + i;
      if (kp >= keys.hi) return -1;
      const int at = bs_shift >= 0 ? kp >> bs_shift : kp / p.bs;
      int blk = at < p.table_stride ? table[at] : -1;
      if (blk < 0 || blk >= p.n_blocks) {
        if ((kp >= lo || kp < p.keep) && p.err) atomicExch(p.err, CUCA_ERR_BLOCK_RANGE);
        blk = -1;
      }
      return blk;
    };
    auto row_of = [&](int blk, int j, int i) -> size_t {
      const int kp = keys.at(first + j) * KEYS + i;
      const int off = bs_shift >= 0 ? kp & (p.bs - 1) : kp % p.bs;
      return ((size_t)blk * p.nkv + kvh) * p.bs + off;
    };
    int blk[PER], blk_f;
    uint4 kn[PER], vn[PER];  // of the tile ahead
    float ksn = 0.f, vsn = 0.f;
    auto look = [&](int j) {
#pragma unroll
      for (int i = 0; i < PER; ++i) blk[i] = entry_of(j, r0 + i * STEP);
      blk_f = tid < KEYS ? entry_of(j, tid) : -1;
    };
    auto fetch = [&](int j) {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        kn[i] = vn[i] = make_uint4(0u, 0u, 0u, 0u);
        if (blk[i] >= 0 && piece) {
          const size_t at = row_of(blk[i], j, r0 + i * STEP) * p.d + c * 16;
          kn[i] = __ldg(reinterpret_cast<const uint4*>(p.kpool + at));
          vn[i] = __ldg(reinterpret_cast<const uint4*>(p.vpool + at));
        }
      }
      ksn = vsn = 0.f;
      if (blk_f >= 0) {
        const size_t at = row_of(blk_f, j, tid);
        ksn = __ldg(p.kscale + at);
        vsn = __ldg(p.vscale + at);
      }
    };
    look(0);
    fetch(0);
    look(1);
    asm volatile("bar.sync 1, %0;" ::"n"((SOFT_WARPS + CONV_WARPS) * 32) : "memory");
    float up, down;
    q8_query_scale(*q_top, up, down);
    const float key_factor = down * (OPT && p.cap > 0.f ? p.scale : p.scale_log2e);
    for (int j = 0; j < n_tiles; ++j) {
      const int st = j % STAGES;
      uint4 k[PER], v[PER];
      const float ks = ksn, vs = vsn;
#pragma unroll
      for (int i = 0; i < PER; ++i) { k[i] = kn[i]; v[i] = vn[i]; }
      if (j + 1 < n_tiles) {
        fetch(j + 1);
        look(j + 2);
      }
      if (j >= STAGES && !warp_wait(&kv_empty[st], ((j / STAGES) & 1) ^ 1, p.err, abort_flag)) break;
      uint8_t* kt = kv_s + st * SH::STAGE;
      auto put = [&](uint8_t* tile, int row, const uint4& w4) {
        // 16 dimensions: two pieces of a 128-byte row of 64. Eight lanes, a row's eight pieces (or two rows' four), must find
        // eight places: lanes of the second half of a wide row go the other way round.
        const int swap = DP == 128 ? c >> 2 : 0;
        const uint32_t w[4] = {(swap ? w4.z : w4.x) ^ 0x80808080u, (swap ? w4.w : w4.y) ^ 0x80808080u,
                               (swap ? w4.x : w4.z) ^ 0x80808080u, (swap ? w4.y : w4.w) ^ 0x80808080u};
        uint8_t* dst = tile + (c / 4) * SH::KV_HALF + row * 128;
        *reinterpret_cast<uint4*>(dst + (((2 * (c & 3) + swap) ^ (row & 7)) << 4)) =
            make_uint4(q8_pair_lo(w[0]), q8_pair_hi(w[0]), q8_pair_lo(w[1]), q8_pair_hi(w[1]));
        *reinterpret_cast<uint4*>(dst + (((2 * (c & 3) + 1 - swap) ^ (row & 7)) << 4)) =
            make_uint4(q8_pair_lo(w[2]), q8_pair_hi(w[2]), q8_pair_lo(w[3]), q8_pair_hi(w[3]));
      };
#pragma unroll
      for (int i = 0; i < PER; ++i) put(kt, r0 + i * STEP, k[i]);
#pragma unroll
      for (int i = 0; i < PER; ++i) put(kt + SH::KV_TILE, r0 + i * STEP, v[i]);
      if (tid < KEYS) {
        float* f = factor_s + st * 4 * KEYS + tid;
        float e, frac, inv;
        q8_value_scale(vs, e, frac, inv);
        f[0] = ks * key_factor;
        f[KEYS] = e;
        f[2 * KEYS] = inv;
        f[3 * KEYS] = frac;
      }
      fence_proxy_async();
      mbar_arrive(&kv_full[st]);
    }
  } else {
    // ------------------------------------------------ products: a warp per query tile; scores run a tile ahead
    const int x = warp - SOFT_WARPS - CONV_WARPS;
    constexpr uint32_t idesc_qk = desc_f16(false, KEYS), idesc_pv = desc_f16(true, DP);
    bool ok = x < nq && warp_wait(&q_full[x], 0, p.err, abort_flag);
    const uint64_t q_desc = smem_desc(smem_u32(q_s + x * SH::Q_BYTES));
    const uint32_t kv_at = smem_u32(kv_s);
    auto scores = [&](int t) {
      const int st = t % STAGES;
      if (!warp_wait(&kv_full[st], (t / STAGES) & 1, p.err, abort_flag)) return false;
      tc_fence_after();
      const uint64_t kd = smem_desc(kv_at + st * SH::STAGE);
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < DP / 16; ++k)
          umma_bf16(tmem_s(x, t), q_desc + (uint64_t)(((k / 4) * SH::Q_HALF + (k % 4) * 32) >> 4),
                    kd + (uint64_t)(((k / 4) * SH::KV_HALF + (k % 4) * 32) >> 4), idesc_qk, k > 0);
        umma_commit(&s_full[2 * x + (t & 1)]);
      }
      __syncwarp();
      return true;
    };
    ok = ok && scores(0) && (n_tiles < 2 || scores(1));
    for (int j = 0; ok && j < n_tiles; ++j) {
      const int st = j % STAGES;
      if (!warp_wait(&p_full[x], j & 1, p.err, abort_flag)) break;
      tc_fence_after();
      const uint64_t vd = desc_mnmajor(kv_at + st * SH::STAGE + SH::KV_TILE, SH::KV_HALF, 1024);
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < KEYS / 16; ++k)
          umma_bf16_tmem_a(tmem_o(x), tmem_s(x, j) + k * 8, vd + (uint64_t)((k * 2048) >> 4), idesc_pv, j > 0 || k > 0);
        umma_commit(&kv_empty[st]);
        umma_commit(&pv_done[x]);
      }
      __syncwarp();
      if (j + 2 < n_tiles && !scores(j + 2)) break;
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {  // what was issued may still be running
    const unsigned long long t0 = global_ns();
    while (global_ns() - t0 < 2000000ull) { }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == SOFT_WARPS + CONV_WARPS) tmem_dealloc(tmem_base, TMEM_COLS);
}

// Joins the shares of a tile's keys, in their order: a thread per query row and eight dimensions.
template <int DP>
__global__ void __launch_bounds__(ROWS) join_q8_tc_kernel(const Q8Params p) {
  pdl_trigger();
  pdl_wait();
  int row0, n_tok;
  if (!q8_rows_of_tile(p, blockIdx.z, row0, n_tok)) return;
  const int kvh = blockIdx.y, G = p.nh / p.nkv;
  const int pos0 = p.positions[row0];
  if (p.seq_of_row[row0] < 0 || pos0 < 0) return;
  const Q8Keys keys = q8_keys<KEYS>(p, pos0, n_tok);
  const int share = p.chunk / KEYS, used = min(p.n_splits, (keys.groups + share - 1) / share);
  if (used <= 1) return;  // written already
  const int x = blockIdx.x % NQ, c8 = blockIdx.x / NQ, r = threadIdx.x;
  const int tile_tok = ROWS / G, tok = x * tile_tok + r / G, head = kvh * G + r % G;
  if (r >= tile_tok * G || tok >= n_tok || c8 * 8 >= p.d) return;
  const size_t step = (size_t)NQ * ROWS * (DP + 2);
  const float* part = p.part + ((size_t)blockIdx.z * p.nkv + kvh) * p.n_splits * step;
  const float* ml = part + NQ * ROWS * DP + x * 2 * ROWS + r;
  float top = -INFINITY;
  for (int s = 0; s < used; ++s) top = fmaxf(top, ml[s * step]);
  float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, den = 0.f;
  for (int s = 0; s < used; ++s) {
    const float ms = ml[s * step], f = ms == top ? 1.f : q8_exp2(ms - top);
    den += f * ml[s * step + ROWS];
    const float4* a = reinterpret_cast<const float4*>(part + s * step) + ((size_t)x * (DP / 4) + 2 * c8) * ROWS + r;
    const float4 lo = a[0], hi = a[ROWS];
    o[0] += f * lo.x; o[1] += f * lo.y; o[2] += f * lo.z; o[3] += f * lo.w;
    o[4] += f * hi.x; o[5] += f * hi.y; o[6] += f * hi.z; o[7] += f * hi.w;
  }
  if (p.sink && top != -INFINITY) den += q8_sink_term(p, head, top);
  const float inv = den == 0.f ? 0.f : 1.f / den;
  __nv_bfloat16* dst = (__nv_bfloat16*)p.out + (size_t)(row0 + tok) * p.out_stride + (size_t)head * p.d + c8 * 8;
  if (((uintptr_t)p.out & 15) == 0 && p.out_stride % 8 == 0) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 t2 = __floats2bfloat162_rn(o[2 * i] * inv, o[2 * i + 1] * inv);
      w[i] = *reinterpret_cast<const uint32_t*>(&t2);
    }
    *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) dst[i] = __float2bfloat16_rn(o[i] * inv);
  }
}

template <int DP, bool OPT>
int launch_q8_tc(const Q8Params& p, int n_tiles, cudaStream_t stream) {
  constexpr int smem = Shape<DP>::SMEM;
  auto kernel = attention_q8_tc_kernel<DP, OPT>;
  static cudaError_t configured = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  CUCA_REQUIRE(configured == cudaSuccess, "attention_q8_tc: cannot reserve %d bytes of shared memory: %s", smem, cudaGetErrorString(configured));
  const int bs_shift = (p.bs & (p.bs - 1)) == 0 ? __builtin_ctz(p.bs) : -1;
  cuca_launch(kernel, dim3(p.nkv * p.n_splits, n_tiles), dim3(NTHREADS), smem, stream, true, p, bs_shift);
  CUCA_CHECK_LAUNCH("attention_q8_tc");
  if (p.n_splits > 1) {
    cuca_launch(join_q8_tc_kernel<DP>, dim3(NQ * DP / 8, p.nkv, n_tiles), dim3(ROWS), 0, stream, true, p);
    CUCA_CHECK_LAUNCH("attention_q8_tc (join)");
  }
  return 0;
}

}  // namespace

// As cuca_attention_q8 for bfloat16 rows and head sizes up to 128, whole groups of at most 128 heads: tile_tokens is
// query_tiles (1 or 2) times the tokens whose rows fit 128. part: [n_tiles][nkv][n_splits][256 (d rounded up to 64 or 128) + 512]
// floats where n_splits > 1.
CUCA_API int cuca_attention_q8_tc(const void* q, int q_stride, void* out, int out_stride, const void* kpool, const void* vpool,
                                  const float* kscale, const float* vscale, int n_blocks, int bs, const int* positions,
                                  const int* seq_of_row, const int* tables, int table_stride, const int* req_row0,
                                  const int* req_count, int n_seqs, int count_lo, int count_hi, int query_tiles, int n_tiles,
                                  int nh, int nkv, int d, const CucaAttnOptions* opt, int chunk, int n_splits, float* part,
                                  int* err, cudaStream_t stream) {
  if (n_tiles == 0) return 0;
  CUCA_REQUIRE(opt != nullptr && opt->window >= 0 && opt->keep >= 0, "attention_q8_tc: bad options");
  CUCA_REQUIRE(opt->gate == nullptr && opt->key_scale == nullptr, "attention_q8_tc: no output gate and no shared rows over 8-bit pages");
  CUCA_REQUIRE(nkv > 0 && nh > 0 && nh % nkv == 0 && nh / nkv <= ROWS && d >= 16 && d <= 128 && d % 16 == 0,
               "attention_q8_tc: unsupported shape (heads %d/%d, head size %d)", nh, nkv, d);
  CUCA_REQUIRE(bs > 0 && n_blocks > 0 && table_stride > 0, "attention_q8_tc: empty pages or tables");
  CUCA_REQUIRE((((uintptr_t)kpool | (uintptr_t)vpool) & 15) == 0, "attention_q8_tc: pools must be 16-byte aligned");
  CUCA_REQUIRE(query_tiles == 1 || query_tiles == NQ, "attention_q8_tc: %d query tiles", query_tiles);
  CUCA_REQUIRE(chunk >= 0 && chunk % KEYS == 0 && n_splits >= 1 && (n_splits == 1 || (chunk > 0 && part && ((uintptr_t)part & 15) == 0)),
               "attention_q8_tc: bad shares of the keys");
  CUCA_REQUIRE(n_tiles <= 65535 && nkv <= 65535, "attention_q8_tc: too many tiles or heads");
  Q8Params p;
  p.q = q; p.q_stride = q_stride; p.out = out; p.out_stride = out_stride;
  p.kpool = (const int8_t*)kpool; p.vpool = (const int8_t*)vpool; p.kscale = kscale; p.vscale = vscale;
  p.n_blocks = n_blocks; p.bs = bs; p.tables = tables; p.table_stride = table_stride; p.positions = positions;
  p.seq_of_row = seq_of_row; p.req_row0 = req_row0; p.req_count = req_count; p.n_seqs = n_seqs; p.count_lo = count_lo;
  p.count_hi = count_hi; p.tile_tokens = query_tiles * (ROWS / (nh / nkv)); p.nh = nh; p.nkv = nkv; p.d = d;
  p.scale = opt->scale; p.scale_log2e = opt->scale * CUCA_LOG2E; p.cap = opt->softcap; p.cap_arg = opt->softcap > 0.f ? 2.f * CUCA_LOG2E / opt->softcap : 0.f; p.sink = opt->sink ? 1 : 0;
  p.sink_val = opt->sink ? opt->sink_val : nullptr; p.window = opt->window; p.keep = opt->window > 0 ? opt->keep : 0;
  p.slopes = opt->slopes; p.heads_per_cta = nh / nkv; p.head_parts = 1; p.chunk = n_splits > 1 ? chunk : 0;
  p.n_splits = n_splits; p.part = part; p.err = err;
  const bool extra = p.cap > 0.f || p.sink || p.slopes;
  if (d <= 64) return extra ? launch_q8_tc<64, true>(p, n_tiles, stream) : launch_q8_tc<64, false>(p, n_tiles, stream);
  return extra ? launch_q8_tc<128, true>(p, n_tiles, stream) : launch_q8_tc<128, false>(p, n_tiles, stream);
}
