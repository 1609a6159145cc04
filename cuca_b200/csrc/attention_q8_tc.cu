// Causal grouped-query attention over 8-bit pages for portions of tokens, on the 5th-generation tensor cores (bfloat16 or 32-bit
// rows, head sizes up to 128). (Scales, weights and their exactness: attention_q8.cuh.)
//
// A block takes up to 2 x 128 query rows of one request and key head, a row being a (token, head) pair, so that every head of
// the group shares the block's keys and values, and walks the keys in tiles of 64:
//
//   S[128 rows, 64 keys]  = Q K^T      Q and K as 16-bit floats in shared memory (K-major, 128-byte swizzle)
//   O[128 rows, d]       += W V        W from tensor memory, where S was; V as 16-bit floats in shared memory (MN-major)
//
// Two warps copy codes from the pages, three tiles ahead; four turn them into 16-bit floats and store them as operand tiles, with
// each key's factors beside them; four warps per query tile own a row per thread (a lane of tensor memory) and turn scores into
// weights; a warp per query tile issues its products. Where the two query tiles share a converted tile, the conversion is a
// sixth of the block's instructions.
//
// A value scale goes into the operand tile here: V = code vs 2^(7 - E) with E the largest exponent of the tile's scales, rounded
// to 11 bits, so that z = s + E for every key of the tile and one multiplication a tile brings the sum of the weights to the
// denominator's unit. Per-key factors in the softmax would each cost 16 loads of 512 bytes a warp and tile: one, the keys' scales,
// is left of four. Where a tile's scales are more than 2^4 apart, or a row is zeros, the exponents stay with the keys (`wide`: the
// portion below 147 us if all tiles are). The keys' scales multiply the scores, so codes of keys are exact.
//
// Measured, 32 heads of 128 over 8: a prompt of 2,048 60 us (576 TFLOP/s), a portion of 512 on 8,192 106 us (668 TFLOP/s; over
// bfloat16 pages, attention_tc.cu, 56 and 138). A tile of 64 keys takes two query tiles some 2,450 clocks, of which the tensor
// pipe and the exponent unit need 1,024 each. No unit sets the pace: without seven eighths of the softmax's arithmetic the portion
// took 20 % less, without most products 9 %, without all three roles' work still 72 us. What is left is the way round: a score
// tile, its weights, their product, and the hand-overs between (barriers, tensor memory's loads and stores), two deep.
//
// Every wait is bounded; when one runs out the kernel records CUCA_ERR_WAIT_TIMEOUT, all roles stop, tensor memory is freed and
// the kernel returns.
#include "attention_q8.cuh"
#include "tcgen05.cuh"
#include <type_traits>

namespace {

constexpr int ROWS = 128;  // query rows of a tile = lanes of tensor memory
constexpr int KEYS = 64;   // keys of a tile
constexpr int NQ = 2;      // query tiles of a block
constexpr int SOFT_WARPS = 4 * NQ, CONV_WARPS = 4;  // (8 that convert, with 144 registers for the softmax: a prompt of 2,048 76 us, not 70)
constexpr int LOAD_WARPS = 2;
constexpr int NTHREADS = (SOFT_WARPS + CONV_WARPS + NQ + LOAD_WARPS) * 32;  // softmax, conversion, issue, copies
// Registers a thread: 128 at launch, then by role; the sum, 2 x 176 + 88 + 64 over groups of 128 threads, is within the 4 x 128
// of the launch.
constexpr int SOFT_REGS = 176, CONV_REGS = 88, ISSUE_REGS = 64;
// Operand tiles: those of keys are free again when their scores are there, those of values after the weights' product. (Two and
// four, three and four with two tiles of codes on their way, four and three: within 2 %.)
constexpr int K_STAGES = 3, V_STAGES = 3;
constexpr int RAW = 3;  // tiles of codes on their way
constexpr float V_LIFT = 7.f;     // values are 2^7 larger in the operand tile: 127 2^7 2 is the most that fits
// A tile's keys take weights relative to the tile's exponent E where their value scales are within 2^WIDE: the reference may be as
// much above a key's own, so a key's weight is good to 2^(WIDE - LIFT - 24) = 2^-28 of the largest weight times value, and what a
// hundred thousand keys lose is under a rounding of the result. (Within 2^20 four thousand keys of 2^-14 of the largest weight lost
// a seventh of theirs beside a key of none with a value 2^18 larger.) Weights are at most 2^(LIFT + LAG). A LAG of 5 and a LIFT of 10
// cost 1 %, 3 and 12 14 %. In 32-bit mode a value scale's fraction goes into the weight, and E is 0.
constexpr int WIDE = 4;
template <bool F32> constexpr float LIFT = F32 ? Q8_LIFT : 8.f;
// bfloat16 queries whose row's largest magnitude is 2^-6 to 2^9, as good as all, go in times 2^6, whatever rows are beside them: what
// 16-bit floats have no steps for is 2^-25 of that magnitude and less. Another row has a power of two of its own, and its warp
// walks the keys in a way of its own, which multiplies by the inverse (a portion of 512 on 8,192 141 us if all do, 106 if none).
constexpr float Q_UNIT = 64.f;
// Scores of such size have steps of an eighth: they are walked in that way too, which rounds a score before the reference is taken off.
constexpr float FAR = 1048576.f;
constexpr int TMEM_COLS = 512;  // two score buffers per query tile (4 x 64 columns), results of both (2 x DP)

__device__ __forceinline__ uint32_t q8_times(uint32_t a, uint32_t hi, uint32_t lo) {  // a (hi + lo), rounded once but for a lo
  uint32_t r;
  asm("{\n.reg .b32 t;\nmul.rn.f16x2 t, %1, %3;\nfma.rn.f16x2 %0, %1, %2, t;\n}" : "=r"(r) : "r"(a), "r"(hi), "r"(lo));
  return r;
}

template <int DP, bool F32>
struct Shape {
  static constexpr int HALVES = DP / 64;
  static constexpr int Q_HALF = ROWS * 128, Q_BYTES = HALVES * Q_HALF;
  static constexpr int KV_HALF = KEYS * 128, KV_TILE = HALVES * KV_HALF;
  // Of a stage: the keys' factors; the value scales' exponents less E and their inverse (of a wide tile, and in 32-bit mode); (there)
  // their fractions; E, its inverse, and whether the tile is wide.
  static constexpr int TILE_E = (F32 ? 4 : 3) * KEYS, FACTORS = (TILE_E + 4) * 4;
  static constexpr int RAW_STAGE = 2 * KEYS * DP + 2 * KEYS * 4;  // codes of a tile's keys and values, their scales
  static constexpr int TILES = NQ * Q_BYTES + (K_STAGES + V_STAGES) * KV_TILE + V_STAGES * FACTORS + RAW * RAW_STAGE;
  static constexpr int SMEM = TILES + 384 + 1024;  // + barriers, + alignment
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

// The same for 32 columns.
__device__ __forceinline__ void tmem_ld32_done(uint32_t taddr, float (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
      "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, "
      "%22, %23, %24, %25, %26, %27, %28, %29, %30, %31"
      "}, [%32];\n\ttcgen05.wait::ld.sync.aligned;"
      :
        "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
        "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]),
        "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]),
        "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(taddr) : "memory");
}

// EXTRA: what a score goes through beside its factor: 1: a distance bias, 2: a cap (and a bias). Constants, as a branch a pair of
// scores keeps their instructions from overlapping (a portion with either took twice the time without).
// F32: 32-bit rows, one query tile a block. A query goes in as two 16-bit parts, in two operand tiles, and so does a weight; the lower
// parts have the second query tile's places in shared and tensor memory. (Sums of their own, as the tensor cores cut off what a
// larger sum has no bits for; the errors are half of those of one sum.) The value scales stay out of the operand tile: their exponents go to the scores and their fractions
// to the weights, so that codes are exact there too. 32 heads of 128 over 8: a prompt of 2,048 237 us, a portion of 512 on 8,192 379
// (attention_q8.cu: 429 and 736), bound by a start and a join every 512 keys, which the errors ask for, and four factors a key.
template <int DP, int EXTRA, bool F32>
__global__ void __launch_bounds__(NTHREADS, 1) attention_q8_tc_kernel(const Q8Params p) {
  using SH = Shape<DP, F32>;
  using T = typename std::conditional<F32, float, __nv_bfloat16>::type;
  extern __shared__ uint8_t smem_raw[];
  // (by an offset, so that the compiler still knows it for shared memory)
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint8_t* q_s = smem;
  uint8_t* k_s = q_s + NQ * SH::Q_BYTES;
  uint8_t* v_s = k_s + K_STAGES * SH::KV_TILE;
  float* factor_s = (float*)(v_s + V_STAGES * SH::KV_TILE);  // [V_STAGES]
  uint8_t* raw_s = (uint8_t*)factor_s + V_STAGES * SH::FACTORS;
  uint64_t* bars = (uint64_t*)(raw_s + RAW * SH::RAW_STAGE);
  uint64_t* q_full = bars;                     // [NQ]
  uint64_t* k_full = q_full + NQ;              // [K_STAGES]
  uint64_t* k_empty = k_full + K_STAGES;       // [K_STAGES]
  uint64_t* v_full = k_empty + K_STAGES;       // [V_STAGES]
  uint64_t* v_empty = v_full + V_STAGES;       // [V_STAGES]
  uint64_t* factor_full = v_empty + V_STAGES;  // [V_STAGES]
  uint64_t* raw_full = factor_full + V_STAGES;   // [RAW]
  uint64_t* raw_empty = raw_full + RAW;          // [RAW]
  uint64_t* s_full = raw_empty + RAW;      // [NQ][2]
  // (a warp can be a tile ahead of the others, so even and odd tiles have a barrier each: its two arrivals must not count for one)
  uint64_t* p_full = s_full + 2 * NQ;        // [NQ][2]
  uint64_t* pv_done = p_full + 2 * NQ;       // [NQ][2]
  uint64_t* ahead = pv_done + 2 * NQ;        // the first query tile has handed over its first weights
  uint32_t* tmem_slot = (uint32_t*)(ahead + 1);
  volatile int* abort_flag = (volatile int*)(tmem_slot + 1);

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
  T* out = (T*)p.out;
  if (seq < 0 || pos0 < 0) {  // rows of no request
    if (split == 0)
      for (int i = threadIdx.x; i < n_tok * G * p.d; i += NTHREADS)
        out[(size_t)(row0 + i / (G * p.d)) * p.out_stride + (size_t)head0 * p.d + i % (G * p.d)] = from_f32<T>(0.f);
    return;
  }
  const Q8Keys keys = q8_keys<KEYS>(p, pos0, n_tok);
  const int share = p.chunk > 0 ? p.chunk / KEYS : keys.groups;
  const int first = split * share;
  const int last = split == p.n_splits - 1 ? keys.groups : min(keys.groups, first + share);
  if (first >= last) return;
  const bool alone = share >= keys.groups || p.n_splits == 1;
  const int n_tiles = last - first;
  const int lo = p.window > 0 ? max(0, pos0 - (p.window - 1)) : 0;  // no row sees positions from p.keep to here
  const int tile_tok = ROWS / G;             // tokens of a query tile
  const int nq = !F32 && n_tok > tile_tok ? 2 : 1;
  const uint32_t per_head = (65536u + G - 1) / G;  // a row of a query tile over G: right for up to 128 of both
  auto token_of = [&](int row) { return (int)(((uint32_t)row * per_head) >> 16); };

  // Pages of a power of two of positions, four at least: a page's part of a tile is a run of bytes in each of the four pools.
  const bool runs = p.run_shift >= 2 && (((uintptr_t)p.kscale | (uintptr_t)p.vscale) & 15) == 0;
  if (warp == SOFT_WARPS + CONV_WARPS) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  if (threadIdx.x == 0) {
    for (int x = 0; x < NQ; ++x) {
      mbar_init(&q_full[x], F32 ? SOFT_WARPS : 4);
      mbar_init(&s_full[2 * x], 1);
      mbar_init(&s_full[2 * x + 1], 1);
      mbar_init(&p_full[2 * x], 4);
      mbar_init(&p_full[2 * x + 1], 4);
      mbar_init(&pv_done[2 * x], 1);
      mbar_init(&pv_done[2 * x + 1], 1);
    }
    for (int s = 0; s < K_STAGES; ++s) {
      mbar_init(&k_full[s], CONV_WARPS);
      mbar_init(&k_empty[s], nq);
    }
    for (int s = 0; s < V_STAGES; ++s) {
      mbar_init(&v_full[s], CONV_WARPS);
      mbar_init(&v_empty[s], nq);
      mbar_init(&factor_full[s], 1);
    }
    for (int s = 0; s < RAW; ++s) {
      mbar_init(&raw_full[s], LOAD_WARPS * (runs ? 1 : 32));
      mbar_init(&raw_empty[s], CONV_WARPS);
    }
    mbar_init(ahead, 4);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  auto tmem_s = [&](int x, int t) { return tmem_base + (uint32_t)((2 * x + (t & 1)) * KEYS); };
  auto tmem_o = [&](int x) { return tmem_base + (uint32_t)(2 * NQ * KEYS + x * DP); };

  // ------------------------------------------------ copies, RAW tiles ahead
  auto load_codes = [&](int lw) {
    const int* table = p.tables + (size_t)seq * p.table_stride;
    if (runs) {
      // A warp for the keys, one for the values (one for both was busy for 1,770 clocks a tile), a lane a page: codes and scales.
      // Positions that no row sees come along where their page does; what converts them takes their scales for 0. (A page behind a
      // window may have gone back, another that is not there is an error: page 0 comes instead; its keys are masked, or the step
      // is lost.)
      const int8_t* pool = lw == 0 ? p.kpool : p.vpool;
      const float* scales = lw == 0 ? p.kscale : p.vscale;
      const int run = min(p.bs, KEYS), n = KEYS / run;
      auto look = [&](int j) {
        const int kp = min(keys.at(first + min(j, n_tiles - 1)) * KEYS + lane * run, keys.hi - 1);
        return (kp >> p.run_shift) < p.table_stride ? __ldg(table + (kp >> p.run_shift)) : -1;
      };
      int page[2] = {look(0), look(1)};  // (two tiles ahead: the next use does not wait for them)
      for (int j = 0; j < n_tiles; ++j) {
        const int kp = keys.at(first + j) * KEYS + lane * run;
        const bool mine = lane < n && kp < keys.hi, paged = page[0] >= 0 && page[0] < p.n_blocks;
        if (mine && !paged && (kp + run > lo || kp < p.keep) && p.err) atomicExch(p.err, CUCA_ERR_BLOCK_RANGE);
        const uint32_t row = ((uint32_t)(paged ? page[0] : 0) * p.nkv + kvh) * p.bs + (kp & (p.bs - 1));
        page[0] = page[1];
        page[1] = look(j + 2);
        if (j >= RAW && !warp_wait(&raw_empty[j % RAW], ((j / RAW) & 1) ^ 1, p.err, abort_flag)) break;
        uint8_t* to = raw_s + (j % RAW) * SH::RAW_STAGE;
        uint64_t* bar = &raw_full[j % RAW];
        const int pages = __popc(__ballot_sync(0xffffffffu, mine));
        if (lane == 0) mbar_expect_tx(bar, pages * run * (p.d + 4));
        __syncwarp();
        if (mine) {
          bulk_load(to + lw * KEYS * DP + lane * run * p.d, pool + (size_t)row * p.d, bar, run * p.d);
          bulk_load(to + 2 * KEYS * DP + (lw * KEYS + lane * run) * 4, scales + row, bar, run * 4);
        }
      }
      return;
    }
    // Two warps, 32 keys of a tile each, a lane a key for pages and scales.
    constexpr int CHUNKS = DP / 16, AT_ONCE = 32 / CHUNKS;  // 16-byte pieces of a row; rows of an instruction
    constexpr uint32_t NOWHERE = 0xffffffffu;
    const int c = lane % CHUNKS, key = lw * 32 + lane;
    auto look = [&](int j) {  // the page of the lane's key: a tile before it is needed
      const int kp = min(keys.at(first + min(j, n_tiles - 1)) * KEYS + key, keys.hi - 1);
      const int entry = p.run_shift >= 0 ? kp >> p.run_shift : kp / p.bs;
      return entry < p.table_stride ? __ldg(table + entry) : -1;
    };
    int page = look(0);
    for (int j = 0; j < n_tiles; ++j) {
      const int kp = keys.at(first + j) * KEYS + key, off = p.run_shift >= 0 ? kp & (p.bs - 1) : kp % p.bs;
      const bool mine = kp < keys.hi, paged = page >= 0 && page < p.n_blocks;
      if (mine && !paged && (kp >= lo || kp < p.keep) && p.err) atomicExch(p.err, CUCA_ERR_BLOCK_RANGE);  // (pages behind a window may have gone back)
      const uint32_t row = mine && paged ? ((uint32_t)page * p.nkv + kvh) * p.bs + off : NOWHERE;
      page = look(j + 1);
      if (j >= RAW && !warp_wait(&raw_empty[j % RAW], ((j / RAW) & 1) ^ 1, p.err, abort_flag)) break;
      const uint32_t to = q8_shared(raw_s) + (j % RAW) * SH::RAW_STAGE, scales = to + 2 * KEYS * DP;
      const bool ok = row != NOWHERE;
      copy4(scales + key * 4, p.kscale + (ok ? row : 0u), ok);
      copy4(scales + (KEYS + key) * 4, p.vscale + (ok ? row : 0u), ok);
#pragma unroll
      for (int i = 0; i < 32 / AT_ONCE; ++i) {
        const int at = i * AT_ONCE + lane / CHUNKS;
        const uint32_t its = __shfl_sync(0xffffffffu, row, at);
        if (c * 16 < p.d) {
          const size_t src = (size_t)(its == NOWHERE ? 0u : its) * p.d + c * 16;  // (a key that is not there: zeros, masked)
          const uint32_t dst = to + (lw * 32 + at) * p.d + c * 16;
          copy16(dst, p.kpool + src, its != NOWHERE);
          copy16(dst + KEYS * DP, p.vpool + src, its != NOWHERE);
        }
      }
      asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&raw_full[j % RAW])) : "memory");
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  };

  if (warp < SOFT_WARPS) {
    // ------------------------------------------------ a query row per thread
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(SOFT_REGS));
    const int x = warp >> 2, quarter = warp & 3;
    const int r = quarter * 32 + lane;  // row of the query tile
    const uint32_t lane_bits = (uint32_t)(quarter * 32) << 16;
    const int tok = x * tile_tok + token_of(r), head = head0 + r - token_of(r) * G;
    // The warp's 32 rows of queries: DP / 8 lanes a row, so that a request for them is whole lines.
    constexpr int LANES = DP / 8, AT_ONCE = 32 / LANES, SETS = 32 / AT_ONCE;
    const int c = lane % LANES;  // 16 bytes of a row
    // In 32-bit mode both halves of the warps read the same rows, the first for the upper parts, the second for the lower.
    float row_down = 1.f;  // of the thread's row
    {
      constexpr int PIECES = F32 ? 2 : 1;                                         // of 16 bytes
      constexpr int AHEAD = F32 ? 4 : SETS, LOG_AHEAD = AHEAD == 4 ? 2 : AHEAD == 8 ? 3 : 4;  // sets whose loads are out together
      const bool aligned = ((uintptr_t)p.q & 15) == 0 && p.q_stride % (16 / (int)sizeof(T)) == 0;
#pragma unroll
      for (int i0 = 0; i0 < SETS; i0 += AHEAD) {
        uint4 raw_q[AHEAD][PIECES];
        uint32_t there = 0;  // a bit a set
        auto piece = [&](int i) {  // where the lane's piece of set i stands (of rows that are not there: another's)
          const int row = quarter * 32 + (i0 + i) * AT_ONCE + lane / LANES, t0 = token_of(row), its_tok = (F32 ? 0 : x * tile_tok) + t0;
          const bool ok = (F32 || x < nq) && row < tile_tok * G && its_tok < n_tok && c * 8 < p.d;
          if (ok) there |= 1u << i;
          return (const T*)p.q + (size_t)(row0 + (ok ? its_tok : 0)) * p.q_stride + (size_t)(head0 + (ok ? row - t0 * G : 0)) * p.d + (ok ? c * 8 : 0);
        };
        if (aligned) {
#pragma unroll
          for (int i = 0; i < AHEAD; ++i) {
            const uint4* src = reinterpret_cast<const uint4*>(piece(i));
#pragma unroll
            for (int n = 0; n < PIECES; ++n) raw_q[i][n] = src[n];
          }
        } else {
#pragma unroll
          for (int i = 0; i < AHEAD; ++i) {
            const T* src = piece(i);
#pragma unroll
            for (int n = 0; n < PIECES; ++n) {
              if constexpr (F32) {
                const uint32_t* h = reinterpret_cast<const uint32_t*>(src) + 4 * n;
                raw_q[i][n] = make_uint4(h[0], h[1], h[2], h[3]);
              } else {
                const unsigned short* h = reinterpret_cast<const unsigned short*>(src);
                raw_q[i][n] = make_uint4(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16, h[4] | (uint32_t)h[5] << 16, h[6] | (uint32_t)h[7] << 16);
              }
            }
          }
        }
        // The rows' largest magnitudes, as bits: of half the sets at each step, so that lane i of a row ends with one set's.
        uint32_t top[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
          top[i] = 0;
#pragma unroll
          for (int n = 0; n < PIECES; ++n) {
            uint4& w = raw_q[i][n];
            if (!((there >> i) & 1u)) w = make_uint4(0u, 0u, 0u, 0u);
            const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int k = 0; k < 4; ++k)
              top[i] = max(top[i], F32 ? words[k] & 0x7fffffffu : max((words[k] << 16) & 0x7fffffffu, words[k] & 0x7fff0000u));
          }
        }
        auto halve = [&](auto size, int o) {  // n sets a lane become n / 2 (one stays one)
          constexpr int n = decltype(size)::value;
          const bool upper = lane & o;
          if constexpr (n == 1) {
            top[0] = max(top[0], __shfl_xor_sync(0xffffffffu, top[0], o));
          } else {
#pragma unroll
            for (int i = 0; i < n / 2; ++i) {
              const uint32_t other = __shfl_xor_sync(0xffffffffu, upper ? top[i] : top[i + n / 2], o);
              top[i] = max(upper ? top[i + n / 2] : top[i], other);
            }
          }
        };
        halve(std::integral_constant<int, AHEAD>{}, 1);
        halve(std::integral_constant<int, AHEAD / 2>{}, 2);
        halve(std::integral_constant<int, (AHEAD > 4 ? AHEAD / 4 : 1)>{}, 4);
        if (LANES == 16) halve(std::integral_constant<int, (AHEAD > 8 ? AHEAD / 8 : 1)>{}, 8);
        auto holder = [&](int i) { return (int)(__brev((uint32_t)i) >> (32 - LOG_AHEAD)); };  // the lane of a row that has set i's
        float its_up, its_down;  // (not finite: 0 and NaN; such a row goes in as zeros and comes out as NaN)
        q8_query_scale(top[0], its_up, its_down);
        if (!F32) {
          const float most = __uint_as_float(top[0]);
          const bool usual = (most >= 1.f / 64.f && most < 512.f) || top[0] == 0;
          its_up = usual ? Q_UNIT : its_up;
          its_down = usual ? 1.f : its_down * Q_UNIT;
        }
        const float mine = __shfl_sync(0xffffffffu, its_down, (lane % AT_ONCE) * LANES + holder((lane / AT_ONCE) % AHEAD));
        if (lane / AT_ONCE / AHEAD == i0 / AHEAD) row_down = mine;
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
          const int row = quarter * 32 + (i0 + i) * AT_ONCE + lane / LANES;
          const float up = __shfl_sync(0xffffffffu, its_up, lane / LANES * LANES + holder(i));
          uint32_t h[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint4& w = raw_q[i][F32 ? k / 2 : 0];
            const uint32_t words[4] = {w.x, w.y, w.z, w.w};
            float lo = F32 ? __uint_as_float(words[2 * k % 4]) : __uint_as_float(words[k] << 16);
            float hi = F32 ? __uint_as_float(words[(2 * k + 1) % 4]) : __uint_as_float(words[k] & 0xffff0000u);
            lo = up == 0.f ? 0.f : lo * up;
            hi = up == 0.f ? 0.f : hi * up;
            if (F32 && x == 1) {
              lo -= __half2float(__float2half_rn(lo));
              hi -= __half2float(__float2half_rn(hi));
            }
            h[k] = q8_pack(lo, hi);
          }
          *reinterpret_cast<uint4*>(q_s + x * SH::Q_BYTES + (c / 8) * SH::Q_HALF + row * 128 + (((c & 7) ^ (row & 7)) << 4)) =
              make_uint4(h[0], h[1], h[2], h[3]);
        }
      }
    }
    const bool bad = !(row_down == row_down);
    if (bad) row_down = 1.f;
    fence_proxy_async();
    __syncwarp();
    if (lane == 0) mbar_arrive(&q_full[F32 ? 0 : x]);

    const int row_pos = pos0 + tok;
    const int row_lo = p.window > 0 ? row_pos - (p.window - 1) : 0;
    const int least_pos = pos0 + x * tile_tok;  // of the query tile's rows
    const int most_lo = p.window > 0 ? pos0 + min(n_tok, (x + 1) * tile_tok) - 1 - (p.window - 1) : 0;
    const float slope2 = EXTRA && p.slopes ? p.slopes[head] * CUCA_LOG2E : 0.f;
    float m = -INFINITY, l = 0.f;
    bool ok = x < nq;
    // The product of tile j - 1. Not every one is waited for and two can be on their way, so even and odd tiles have a barrier
    // each: tile j - 3's product was done before tile j - 1's scores were, so this one's is a phase behind at most.
    auto product_done = [&](int j) {
      return warp_wait(&pv_done[2 * x + ((j - 1) & 1)], ((j - 1) >> 1) & 1, p.err, abort_flag);
    };
    // The tiles from j0 on; returns the one where scores became too large for it. own: for rows with powers of two of their own and
    // scores of any size.
    auto walk = [&](auto own, int j0) {
      for (int j = j0; ok && j < n_tiles; ++j) {
        const int st = j % V_STAGES;
        if (!warp_wait(&s_full[2 * x + (j & 1)], (j >> 1) & 1, p.err, abort_flag)) { ok = false; break; }
        tc_fence_after();
        // (long complete: they were written with the keys)
        if (!warp_wait(&factor_full[st], (j / V_STAGES) & 1, p.err, abort_flag)) { ok = false; break; }
        const float* factor = factor_s + st * (SH::FACTORS / 4);
        const float4* kf4 = reinterpret_cast<const float4*>(factor);
        const float4 tile_e = kf4[SH::TILE_E / 4];  // E, 2^-E, wide
        const int key0 = keys.at(first + j) * KEYS;
        const bool whole = key0 + KEYS - 1 <= least_pos && (p.window <= 0 || key0 >= most_lo || key0 + KEYS <= p.keep);
        const float bias0 = EXTRA ? slope2 * (float)(key0 - row_pos) : 0.f;
        // Weights relative to the maximum of the tiles before, with this tile's maximum beside them, so that the exponents need not
        // wait for it; only where a row exceeds the reference by more than 2^LAG is the tile's row read and worked out again.
        float corr = 1.f;
        bool moved = false;
        float2 sum2[2];
        uint32_t pw[KEYS / 2], pw_lo[F32 ? KEYS / 2 : 1];
#pragma unroll 1
        for (;;) {
          uint32_t raw[2][32];
          if constexpr (F32) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float a[32], b[32];
              tmem_ld32_done(tmem_s(0, j) + lane_bits + h * 32, a);
              tmem_ld32_done(tmem_s(1, j) + lane_bits + h * 32, b);
#pragma unroll
              for (int i = 0; i < 32; ++i) raw[h][i] = __float_as_uint(a[i] + b[i]);
            }
          } else {
            tmem_ld64(tmem_s(x, j) + lane_bits, raw);
          }
          const float ref = m == -INFINITY ? 0.f : m - LIFT<F32>;  // the exponents are z - ref
          const float2 neg2 = make_float2(tile_e.x - ref, tile_e.x - ref);
          float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
          sum2[0] = sum2[1] = make_float2(0.f, 0.f);
          auto row = [&](auto masked, auto wide) {
#pragma unroll
            for (int i = 0; i < KEYS / 4; ++i) {
              const float4 kf = kf4[i];
              const float f[4] = {kf.x, kf.y, kf.z, kf.w};
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const int k = 4 * i + 2 * h;
                float2 x2 = make_float2(__uint_as_float(raw[k / 32][k % 32]), __uint_as_float(raw[k / 32][k % 32 + 1]));
                float2 f2 = make_float2(f[2 * h], f[2 * h + 1]);
                if (decltype(own)::value) {
                  f2 = __fmul2_rn(f2, make_float2(row_down, row_down));
                  x2 = make_float2(__fmul_rn(x2.x, f2.x), __fmul_rn(x2.y, f2.y));  // (a product of two and a sum become one instruction)
                } else if (EXTRA) {
                  x2 = __fmul2_rn(x2, f2);
                }
                // (the key's exponent meets the reference first: their difference is exact where they are large)
                const float2 at2 = decltype(wide)::value ? __fadd2_rn(neg2, *reinterpret_cast<const float2*>(factor + KEYS + k)) : neg2;
                if (EXTRA) {
                  if (EXTRA == 2) x2 = q8_capped_pair(x2, p);
                  x2 = __fadd2_rn(x2, make_float2(fmaf(slope2, (float)k, bias0), fmaf(slope2, (float)(k + 1), bias0)));
                }
                x2 = EXTRA || decltype(own)::value ? __fadd2_rn(x2, at2) : __ffma2_rn(x2, f2, at2);
                if (decltype(masked)::value) {
                  const int kp = key0 + k;
                  if (!(kp <= row_pos && (kp >= row_lo || kp < p.keep))) x2.x = -INFINITY;
                  if (!(kp + 1 <= row_pos && (kp + 1 >= row_lo || kp + 1 < p.keep))) x2.y = -INFINITY;
                }
                const float2 u2 = make_float2(q8_exp2(x2.x), q8_exp2(x2.y));
                mx4[k / 2 & 3] = fmaxf(fmaxf(mx4[k / 2 & 3], x2.x), x2.y);
                if (decltype(wide)::value)
                  sum2[h] = __ffma2_rn(u2, *reinterpret_cast<const float2*>(factor + 2 * KEYS + k), sum2[h]);
                else
                  sum2[h] = __fadd2_rn(sum2[h], u2);
                if (F32) {
                  const float2 w2 = __fmul2_rn(u2, *reinterpret_cast<const float2*>(factor + 3 * KEYS + k));
                  pw[k / 2] = q8_pack_weights(w2.x, w2.y);
                  const float2 upper = __half22float2(*reinterpret_cast<const __half2*>(&pw[k / 2]));
                  pw_lo[F32 ? k / 2 : 0] = q8_pack_weights(w2.x - upper.x, w2.y - upper.y);
                } else {
                  pw[k / 2] = q8_pack_weights(u2.x, u2.y);
                }
              }
            }
          };
          if (F32) {  // (every tile is wide, and E is 0)
            if (!whole) row(std::true_type{}, std::true_type{});
            else row(std::false_type{}, std::true_type{});
          } else if (tile_e.z != 0.f) row(std::true_type{}, std::true_type{});
          else if (decltype(own)::value || !whole) row(std::true_type{}, std::false_type{});
          else row(std::false_type{}, std::false_type{});
          const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) + ref;
          const bool moves = mx > m + Q8_LAG;
          if (!__any_sync(0xffffffffu, moves)) break;
          if (!decltype(own)::value && !moved && __any_sync(0xffffffffu, moves && fabsf(mx) >= FAR)) return j;
          if (moves) {
            corr = q8_exp2(m - mx);
            m = mx;
          }
          moved = true;
        }
        static_assert(KEYS == 64, "one 32-column store holds a row's weights of a tile");
        __syncwarp();
        tmem_st32_raw(tmem_s(x, j) + lane_bits, pw);
        if constexpr (F32) tmem_st32_raw(tmem_s(1, j) + lane_bits, pw_lo);
        l = fmaf((sum2[0].x + sum2[0].y) + (sum2[1].x + sum2[1].y), tile_e.y, l * corr);
        // O is made smaller where a row's maximum moved; only then must the product before have finished
        if (j > 0 && moved) {
          if (!product_done(j)) { ok = false; break; }
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < (F32 ? 2 : 1) * DP / 32; ++c) {  // (the lower parts' results follow the upper's)
            float o[32];
            tmem_ld32_done(tmem_o(x) + lane_bits + c * 32, o);
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] *= corr;
            tmem_st32(tmem_o(x) + lane_bits + c * 32, o);
          }
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&p_full[2 * x + (j & 1)]);
          if (j == 0 && x == 0) mbar_arrive(ahead);
        }
      }
      return n_tiles;
    };
    const int rest = F32 || __any_sync(0xffffffffu, row_down != 1.f) ? 0 : walk(std::false_type{}, 0);
    if (rest < n_tiles) walk(std::true_type{}, rest);
    auto both = [&](int c, float (&o)[32]) {  // 32 dimensions of the results, in 32-bit mode the sum of both parts'
      tmem_ld32_done(tmem_o(x) + lane_bits + c * 32, o);
      if constexpr (F32) {
        float lower[32];
        tmem_ld32_done(tmem_o(1) + lane_bits + c * 32, lower);
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] += lower[i];
      }
    };
    if (ok && product_done(n_tiles)) {
      tc_fence_after();
      if (alone) {
        if (p.sink && m != -INFINITY) l += q8_sink_term(p, head, m, LIFT<F32>);
        const float inv = bad ? __uint_as_float(0x7fc00000u) : l == 0.f ? 0.f : q8_pow2(-V_LIFT) / l;
        if constexpr (F32) {
          const bool mine = r < tile_tok * G && tok < n_tok;
          float* dst = out + (size_t)(row0 + (mine ? tok : 0)) * p.out_stride + (size_t)head * p.d;
          const bool aligned = ((uintptr_t)p.out & 15) == 0 && p.out_stride % 4 == 0;
#pragma unroll
          for (int c0 = 0; c0 < DP / 32; ++c0) {
            float o[32];
            both(c0, o);
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              const int e = c0 * 32 + q * 4;
              if (!mine || e >= p.d) continue;
              if (aligned) {
                *reinterpret_cast<float4*>(dst + e) = make_float4(o[4 * q] * inv, o[4 * q + 1] * inv, o[4 * q + 2] * inv, o[4 * q + 3] * inv);
              } else {
#pragma unroll
                for (int k = 0; k < 4; ++k) dst[e + k] = o[4 * q + k] * inv;
              }
            }
          }
        } else {
        // Through shared memory, where the queries were (every product that read them is done), so that what is stored is whole
        // lines; a row's pieces are turned round by its number, as in the operand tiles.
        uint8_t* mine = q_s + x * SH::Q_BYTES + quarter * 32 * (DP * 2);
#pragma unroll
        for (int c0 = 0; c0 < DP / 32; ++c0) {
          float o[32];
          tmem_ld32_done(tmem_o(x) + lane_bits + c0 * 32, o);  // (the whole warp reads)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const __nv_bfloat162 t2 = __floats2bfloat162_rn(o[q * 8 + 2 * i] * inv, o[q * 8 + 2 * i + 1] * inv);
              w[i] = *reinterpret_cast<const uint32_t*>(&t2);
            }
            *reinterpret_cast<uint4*>(mine + lane * (DP * 2) + (((c0 * 4 + q) ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
        __syncwarp();
        const bool aligned = ((uintptr_t)p.out & 15) == 0 && p.out_stride % 8 == 0;
        auto store = [&](auto whole_lines) {
#pragma unroll
          for (int i = 0; i < SETS; ++i) {
            const int its = i * AT_ONCE + lane / LANES, row = quarter * 32 + its, t0 = token_of(row), its_tok = x * tile_tok + t0;
            const uint4 w = *reinterpret_cast<const uint4*>(mine + its * (DP * 2) + ((c ^ (its & 7)) << 4));
            __nv_bfloat16* dst = out + (size_t)(row0 + its_tok) * p.out_stride + (size_t)(head0 + row - t0 * G) * p.d + c * 8;
            if (row < tile_tok * G && its_tok < n_tok && c * 8 < p.d) {
              if (decltype(whole_lines)::value) {
                *reinterpret_cast<uint4*>(dst) = w;
              } else {
                const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int k = 0; k < 8; ++k) dst[k] = __ushort_as_bfloat16((unsigned short)(v[k / 2] >> (16 * (k & 1))));
              }
            }
          }
        };
        if (aligned) store(std::true_type{});
        else store(std::false_type{});
        }
      } else {
        // [width][DP / 4][ROWS][4], then m and l [width][2][ROWS]: rows side by side
        float* part = p.part + (((size_t)blockIdx.y * p.nkv + kvh) * p.n_splits + split) * (size_t)(p.width * ROWS * (DP + 2));
        float4* dst = reinterpret_cast<float4*>(part) + (size_t)x * (DP / 4) * ROWS + r;
#pragma unroll
        for (int c = 0; c < DP / 32; ++c) {
          float o[32];
          both(c, o);
#pragma unroll
          for (int q = 0; q < 8; ++q) dst[(c * 8 + q) * ROWS] = make_float4(o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]);
        }
        float* ml = part + p.width * ROWS * DP + x * 2 * ROWS;
        ml[r] = m;
        ml[ROWS + r] = bad ? __uint_as_float(0x7fc00000u) : l * q8_pow2(V_LIFT);
      }
    }
  } else if (warp < SOFT_WARPS + CONV_WARPS) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(CONV_REGS));
    // ------------------------------------------------ codes to operand tiles
    // Every warp works for itself: its lanes stand for the tile's keys lane and lane + 32 (scales, the tile's exponent) and hand
    // factors round; it converts every fourth set of rows. It asks for nothing from memory itself: its fence between the two
    // proxies would wait for what is on its way (a prompt of 2,048 62 us so, 60 with copies in warps of their own).
    const int cw = warp - SOFT_WARPS;
    constexpr int ROWS_AT_ONCE = DP == 128 ? 4 : 8;         // of a warp: 16-byte pieces of keys or values
    constexpr int STEP = CONV_WARPS * ROWS_AT_ONCE, PER = KEYS / STEP;
    // (a warp's rows of a set are all among the tile's first 32 keys or all among its last)
    // Eight lanes that read and store together have four pieces each of two neighbouring rows, of different halves: eight places
    // of 128 bytes where the codes are and eight where they go.
    const int half = DP == 128 ? (lane >> 4) ^ ((lane >> 2) & 1) : 0, quad = lane & 3;
    const int r0 = cw * ROWS_AT_ONCE + ((lane >> 2) & (ROWS_AT_ONCE - 1));
    const int place0 = half * SH::KV_HALF + r0 * 128 + (((2 * quad) ^ (r0 & 7)) << 4);
    const int place1 = half * SH::KV_HALF + r0 * 128 + (((2 * quad + 1) ^ (r0 & 7)) << 4);
    const uint32_t raw = q8_shared(raw_s);
    // (beyond the head's size anything will do: the queries are zeros there, and the results are not stored)
    const int piece = (half * 4 + quad) * 16 < p.d ? (half * 4 + quad) * 16 : 0;
    const float key_factor = (F32 ? 1.f : 1.f / Q_UNIT) * (EXTRA == 2 ? p.scale : p.scale_log2e);
    for (int j = 0; j < n_tiles; ++j) {
      const int ks_at = j % K_STAGES, st = j % V_STAGES, from = j % RAW;
      if (!warp_wait(&raw_full[from], (j / RAW) & 1, p.err, abort_flag)) break;
      const uint32_t codes = raw + from * SH::RAW_STAGE, scales = codes + 2 * KEYS * DP;
      float ks[2], vs[2];
      bool seen[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        // (by some row: neither the exponent of the tile nor its bits depend on another, nor on what came for a page that is gone)
        const int kp = keys.at(first + j) * KEYS + lane + 32 * h;
        seen[h] = kp < keys.hi && (kp >= lo || kp < p.keep);
        ks[h] = seen[h] ? shared_f(scales + (lane + 32 * h) * 4) : 0.f;
        vs[h] = seen[h] ? shared_f(scales + (KEYS + lane + 32 * h) * 4) : 0.f;
      }
      uint4 k[PER], v[PER];  // (all asked for before any is used)
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const uint32_t at = codes + (r0 + i * STEP) * p.d + piece;
        k[i] = shared_16(at);
        v[i] = shared_16(at + KEYS * DP);
      }
      // the tile's exponent: the largest of its finite scales other than 0; the least of those that some row sees
      float e[2], f, inv;
      bool fine[2];
      int hi = -60, least = 1000;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        q8_value_scale(vs[h], e[h], f, inv);
        fine[h] = e[h] == e[h];
        if (fine[h] && vs[h] != 0.f) hi = max(hi, (int)e[h]);
        if (fine[h] && seen[h]) least = min(least, (int)e[h]);  // (a row of zeros by its -60: it must not raise the reference)
      }
      hi = F32 ? 0 : __reduce_max_sync(0xffffffffu, hi);
      least = __reduce_min_sync(0xffffffffu, least);
      const bool wide = F32 || hi - least > WIDE;
      // What a key's value codes are multiplied by, twice, and what its rounding left: so a value in the operand tile is rounded once.
      uint32_t factor2[2], left2[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float x = F32 ? q8_pow2(V_LIFT) : fine[h] ? vs[h] * q8_pow2(V_LIFT - (wide ? e[h] : (float)hi)) : 0.f;
        factor2[h] = q8_pack(x, x);
        const float left = x - __half22float2(*reinterpret_cast<const __half2*>(&factor2[h])).x;
        left2[h] = q8_pack(left, left);
      }
      if (j >= V_STAGES && !warp_wait(&v_empty[st], ((j / V_STAGES) & 1) ^ 1, p.err, abort_flag)) break;
      if (j >= K_STAGES && !warp_wait(&k_empty[ks_at], ((j / K_STAGES) & 1) ^ 1, p.err, abort_flag)) break;
      uint8_t* kt = k_s + ks_at * SH::KV_TILE;
      if (cw == j % CONV_WARPS) {
        float* factor = factor_s + st * (SH::FACTORS / 4);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int key = lane + 32 * h;
          // (a value row that is not finite: its scores are NaN for those who see it)
          factor[key] = fine[h] ? ks[h] * key_factor : __uint_as_float(0x7fc00000u);
          if (F32) factor[3 * KEYS + key] = fine[h] ? vs[h] * q8_pow2(-e[h]) : 0.f;
          if (wide) {
            factor[KEYS + key] = fine[h] ? e[h] - (float)hi : 0.f;
            factor[2 * KEYS + key] = fine[h] ? q8_pow2(fmaxf(-126.f, fminf(127.f, (float)hi - e[h]))) : 1.f;
          }
        }
        if (lane == 0) *reinterpret_cast<float4*>(factor + SH::TILE_E) = make_float4((float)hi, q8_pow2(-(float)hi), wide ? 1.f : 0.f, 0.f);
        __syncwarp();
        if (lane == 0) mbar_arrive(&factor_full[st]);
      }
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const uint32_t w[4] = {k[i].x ^ 0x80808080u, k[i].y ^ 0x80808080u, k[i].z ^ 0x80808080u, k[i].w ^ 0x80808080u};
        *reinterpret_cast<uint4*>(kt + place0 + i * STEP * 128) = make_uint4(q8_pair_lo(w[0]), q8_pair_hi(w[0]), q8_pair_lo(w[1]), q8_pair_hi(w[1]));
        *reinterpret_cast<uint4*>(kt + place1 + i * STEP * 128) = make_uint4(q8_pair_lo(w[2]), q8_pair_hi(w[2]), q8_pair_lo(w[3]), q8_pair_hi(w[3]));
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&k_full[ks_at]);
      uint8_t* vt = v_s + st * SH::KV_TILE;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const uint32_t times = __shfl_sync(0xffffffffu, r0 + i * STEP < 32 ? factor2[0] : factor2[1], (r0 + i * STEP) & 31);
        const uint32_t left = F32 ? 0u : __shfl_sync(0xffffffffu, r0 + i * STEP < 32 ? left2[0] : left2[1], (r0 + i * STEP) & 31);
        const uint32_t w[4] = {v[i].x ^ 0x80808080u, v[i].y ^ 0x80808080u, v[i].z ^ 0x80808080u, v[i].w ^ 0x80808080u};
        uint32_t h[8];
#pragma unroll
        for (int n = 0; n < 4; ++n) { h[2 * n] = q8_times(q8_pair_lo(w[n]), times, left); h[2 * n + 1] = q8_times(q8_pair_hi(w[n]), times, left); }
        *reinterpret_cast<uint4*>(vt + place0 + i * STEP * 128) = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4*>(vt + place1 + i * STEP * 128) = make_uint4(h[4], h[5], h[6], h[7]);
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&v_full[st]);
        mbar_arrive(&raw_empty[from]);
      }
    }
  } else {
    // ------------------------------------------------ products: a warp per query tile; scores run a tile ahead
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(ISSUE_REGS));
    if (warp >= SOFT_WARPS + CONV_WARPS + NQ) {
      load_codes(warp - SOFT_WARPS - CONV_WARPS - NQ);
    } else {
    const int x = warp - SOFT_WARPS - CONV_WARPS;
    constexpr uint32_t idesc_qk = desc_f16(false, KEYS), idesc_pv = desc_f16(true, DP);
    bool ok = x < nq && warp_wait(&q_full[x], 0, p.err, abort_flag);
    // The second query tile starts half a tile behind the first, so that one's exponents run beside the other's maxima and sums.
    if (ok && x == 1) ok = warp_wait(ahead, 0, p.err, abort_flag);
    const uint64_t q_desc = smem_desc(smem_u32(q_s + x * SH::Q_BYTES));
    const uint32_t k_at = smem_u32(k_s), v_at = smem_u32(v_s);
    auto scores = [&](int t) {
      const int st = t % K_STAGES;
      if (!warp_wait(&k_full[st], (t / K_STAGES) & 1, p.err, abort_flag)) return false;
      tc_fence_after();
      const uint64_t kd = smem_desc(k_at + st * SH::KV_TILE);
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < DP / 16; ++k)
#pragma unroll
          for (int part = 0; part < (F32 ? 2 : 1); ++part)
            umma_bf16(tmem_s(x + part, t), q_desc + (uint64_t)((part * SH::Q_BYTES + (k / 4) * SH::Q_HALF + (k % 4) * 32) >> 4),
                      kd + (uint64_t)(((k / 4) * SH::KV_HALF + (k % 4) * 32) >> 4), idesc_qk, k > 0);
        umma_commit(&s_full[2 * x + (t & 1)]);
        umma_commit(&k_empty[st]);
      }
      __syncwarp();
      return true;
    };
    ok = ok && scores(0) && (n_tiles < 2 || scores(1));
    for (int j = 0; ok && j < n_tiles; ++j) {
      const int st = j % V_STAGES;
      if (!warp_wait(&p_full[2 * x + (j & 1)], (j >> 1) & 1, p.err, abort_flag) ||
          !warp_wait(&v_full[st], (j / V_STAGES) & 1, p.err, abort_flag)) break;
      tc_fence_after();
      const uint64_t vd = desc_mnmajor(v_at + st * SH::KV_TILE, SH::KV_HALF, 1024);
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < KEYS / 16; ++k)
#pragma unroll
          for (int part = 0; part < (F32 ? 2 : 1); ++part)
            umma_bf16_tmem_a(tmem_o(x + part), tmem_s(x + part, j) + k * 8, vd + (uint64_t)((k * 2048) >> 4), idesc_pv, j > 0 || k > 0);
        umma_commit(&v_empty[st]);
        umma_commit(&pv_done[2 * x + (j & 1)]);
      }
      __syncwarp();
      if (j + 2 < n_tiles && !scores(j + 2)) break;
    }
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
template <int DP, bool F32>
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
  const int x = blockIdx.x % p.width, c8 = blockIdx.x / p.width, r = threadIdx.x;
  const int tile_tok = ROWS / G, tok = x * tile_tok + r / G, head = kvh * G + r % G;
  if (r >= tile_tok * G || tok >= n_tok || c8 * 8 >= p.d) return;
  const size_t step = (size_t)p.width * ROWS * (DP + 2);
  const float* part = p.part + ((size_t)blockIdx.z * p.nkv + kvh) * p.n_splits * step;
  const float* ml = part + p.width * ROWS * DP + x * 2 * ROWS + r;
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
  if (p.sink && top != -INFINITY) den += q8_sink_term(p, head, top, LIFT<F32>) * q8_pow2(V_LIFT);  // (sums come lifted as results do)
  const float inv = den == 0.f ? 0.f : 1.f / den;
  const size_t to = (size_t)(row0 + tok) * p.out_stride + (size_t)head * p.d + c8 * 8;
  if constexpr (F32) {
    float* dst = (float*)p.out + to;
    if (((uintptr_t)p.out & 15) == 0 && p.out_stride % 4 == 0) {
      *reinterpret_cast<float4*>(dst) = make_float4(o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
      *reinterpret_cast<float4*>(dst + 4) = make_float4(o[4] * inv, o[5] * inv, o[6] * inv, o[7] * inv);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) dst[i] = o[i] * inv;
    }
    return;
  }
  __nv_bfloat16* dst = (__nv_bfloat16*)p.out + to;
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

template <int DP, int EXTRA, bool F32>
int launch_q8_tc(const Q8Params& p, int n_tiles, cudaStream_t stream) {
  constexpr int smem = Shape<DP, F32>::SMEM;
  auto kernel = attention_q8_tc_kernel<DP, EXTRA, F32>;
  static cudaError_t configured = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  CUCA_REQUIRE(configured == cudaSuccess, "attention_q8_tc: cannot reserve %d bytes of shared memory: %s", smem, cudaGetErrorString(configured));
  cuca_launch(kernel, dim3(p.nkv * p.n_splits, n_tiles), dim3(NTHREADS), smem, stream, true, p);
  CUCA_CHECK_LAUNCH("attention_q8_tc");
  if (p.n_splits > 1) {
    cuca_launch(join_q8_tc_kernel<DP, F32>, dim3(p.width * DP / 8, p.nkv, n_tiles), dim3(ROWS), 0, stream, true, p);
    CUCA_CHECK_LAUNCH("attention_q8_tc (join)");
  }
  return 0;
}
template <int DP>
int launch_q8_tc_extra(const Q8Params& p, bool f32, int n_tiles, cudaStream_t stream) {
  if (f32) return launch_q8_tc<DP, 0, true>(p, n_tiles, stream);
  if (p.cap > 0.f) return launch_q8_tc<DP, 2, false>(p, n_tiles, stream);
  return p.slopes ? launch_q8_tc<DP, 1, false>(p, n_tiles, stream) : launch_q8_tc<DP, 0, false>(p, n_tiles, stream);
}

}  // namespace

// bfloat16 rows, or 32-bit rows (one query tile, neither cap nor bias), of head sizes up to 128, groups of at most 128 heads whole; `width` (1 or 2) query tiles to a block: tile_tokens is
// that times the tokens whose rows fit 128. part: [n_tiles][nkv][n_splits][width][128 (d rounded up to 64 or 128) + 256] floats where
// n_splits > 1.
CUCA_API int cuca_attention_q8_tc(const CucaQ8Attention* c) {
  if (c->n_tiles == 0) return 0;
  Q8Params p;
  if (const int code = q8_params(*c, "attention_q8_tc", 128, p)) return code;
  const int group = p.nh / p.nkv;
  const bool f32 = c->dtype == CUCA_F32;
  CUCA_REQUIRE(group <= ROWS && p.heads_per_cta == group, "attention_q8_tc: groups of at most %d heads, whole", ROWS);
  CUCA_REQUIRE(!f32 || (c->width == 1 && p.cap == 0.f && !p.slopes), "attention_q8_tc: 32-bit rows one query tile a block, without cap or bias");
  CUCA_REQUIRE(p.n_splits == 1 || p.part, "attention_q8_tc: no place for the shares' results");
  CUCA_REQUIRE((long long)p.n_blocks * p.nkv * p.bs < 0xffffffffll, "attention_q8_tc: more than 2^32 rows in the pools");
  CUCA_REQUIRE((c->width == 1 || c->width == NQ) && p.tile_tokens == (int)c->width * (ROWS / group), "attention_q8_tc: %d rows to %lld query tiles",
               p.tile_tokens, (long long)c->width);
  return p.d <= 64 ? launch_q8_tc_extra<64>(p, f32, (int)c->n_tiles, c->stream) : launch_q8_tc_extra<128>(p, f32, (int)c->n_tiles, c->stream);
}
