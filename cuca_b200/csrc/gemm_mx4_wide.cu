// bfloat16 rows, or 32-bit rows as three bfloat16 rows each (mx4.cu), times a weight in 4 bits on tcgen05: out = epilogue(X W^T).
//
// A code times its power of two is a bfloat16 number exactly, so what the tensor cores multiply is the weight as it is kept and the rows
// as they are. The weight is the 128-row operand and comes out of tensor memory: converter warps take codes from shared memory, a weight
// row a lane, and leave 64 values of it as 32 columns. Shared memory would have to take the converted tile in and give it out again
// beside the rows' own tiles, more than its 128 bytes a clock. The rows of X are the columns, by TMA with 128-byte swizzle.
//
// A tile has 128 features, or 64 gate and 64 up rows of a gated unit, so that one conversion serves up to 256 rows either way.
//
// What bounds it: up to 128 rows in part the conversion, whose 17 instructions for eight codes take a scheduler 22 clocks, at most 46 codes a
// clock and SM where the memory brings 44 (64 rows, 14336 x 4096: 19.0 us, without the conversion's arithmetic 15.7, of which a block's
// start and the join are 6); many rows, the tensor
// cores and their power: a tile of 256 rows converts 16 codes a clock (2,048 rows, 14336 x 4096: 166 us, 1.45 PFLOP/s; 4096 x 14336 gated
// 393 us, 1.22: a tile's results, 7 us of 30, are not hidden). More converting warps or two tiles a block in turn were no faster.
// The multiplying warp is short of time too (a wait takes it 150 clocks, an instruction 60 where eight warps convert beside it), so
// what it waits for is one barrier a step, on which the converted weights and the rows arrive, and a step is 128 values of a row
// but for the largest tiles, whose rows' tiles would leave two steps in shared memory.
// Few tiles: a cluster of up to eight blocks shares K and adds its sums in order out of each other's shared memory.
// The tensor cores cut off what a sum has no bits for (14,336 values in a row: 1.7e-6 off, of one sign 1.6e-5), so 32-bit results leave
// after 8,192 values at most and what follows is added to them with rounding (6e-7; leaving costs a tenth of that), to results in
// memory, or in shared memory where a cluster or a gated unit joins them later. A result, and the stream or bias in it, is so
// rounded once for each 8,192 values begun. Sums of 32-bit rows' parts leave after 2,048, always to shared memory, and are rounded into a
// result once.
#include "mx4.cuh"
#include "mx4_mma.cuh"
#include <type_traits>

namespace {

constexpr int STAGE_BYTES_K = 128;          // bytes of a row of codes in a stage: 256 values
constexpr int STAGE_STEPS = 2;              // of 128 values
constexpr int HALF = TILE_A / 2;            // rows of a box of codes
constexpr int CODE_BYTES = TILE_A * STAGE_BYTES_K;
constexpr int SCALE_BYTES = 512;            // of 128 rows and a step
constexpr int BOX_K = 64;                   // values of a row in a box of X
constexpr int MAX_CODES = 5, MAX_RING = 4, MAX_CLUSTER = 8;
constexpr int MOST_ROWS = 256;              // of X in a tile
constexpr int MOST_WAITING = 240;           // ... whose sums wait in shared memory of their own
constexpr int SUM_STAGES = 32;              // of codes that one 32-bit sum runs over at most
constexpr int SUM_STAGES_F32 = 8;           // ... of 32-bit rows
constexpr int CONVERT_WARP = 2, CONVERT_WARPS = 8, X_WARP = CONVERT_WARP + CONVERT_WARPS;
constexpr int THREADS = 32 * (X_WARP + 1);  // a warp that loads codes, one that multiplies, eight that convert, one that loads rows
constexpr int BARRIERS = 512;

struct Params {
  const uint8_t* w_scales;
  Mx4Out o, more;   // where results go; what is added to them later
  int k_steps, k_stages;
  int nt;  // columns of a whole tile, a multiple of 16
  int mt;  // ... and rows of the result: G columns make one
  int tiles_n, share;
  bool joined;      // what leaves goes to shared memory and is joined later
  int sum_stages;   // stages of codes after which sums leave
  int sums_at;      // bytes into shared memory where sums that leave and are not results yet go: over the stages, where a block leaves once,
  int sums_bytes;   // else so many behind them
  int codes, ring;  // stages of codes; steps in shared (rows) and tensor memory (weights)
  int tmem_cols;
  int* err;
};

// AGAIN: a block's sums leave several times, and wait in shared memory of their own
template <bool DUAL, int KC, int G, bool AGAIN>
__global__ void __launch_bounds__(THREADS, 2) gemm_mx4_wide_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x,
                                                                const Params p) {
  constexpr int BLOCKS = DUAL ? 2 : 1;  // runs of weight rows, each with its scales
  constexpr int CODE_STAGE = CODE_BYTES + BLOCKS * STAGE_STEPS * SCALE_BYTES;
  constexpr int BOXES = KC / BOX_K, COLS = KC / 2;
  constexpr int FEATURES = TILE_A / BLOCKS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const int box_bytes = p.nt * BOX_K * 2, x_bytes = BOXES * box_bytes;
  uint8_t* const code_smem = smem + p.ring * x_bytes;
  uint64_t* code_full = (uint64_t*)(code_smem + p.codes * CODE_STAGE + p.sums_bytes);
  uint64_t* code_empty = code_full + MAX_CODES;
  uint64_t* full = code_empty + MAX_CODES;
  uint64_t* empty = full + MAX_RING;
  uint64_t* done = empty + MAX_RING;
  uint64_t* acc_free = done + 1;
  uint32_t* tmem_slot = (uint32_t*)(acc_free + 1);
  volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
  volatile int* ok_flag = (volatile int*)(tmem_slot + 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = p.share > 1 ? (int)mx4_cluster_rank() : 0;
  const int tile = (int)blockIdx.x / p.share;
  const int n0 = (tile % p.tiles_n) * FEATURES, m0 = (tile / p.tiles_n) * p.mt;
  const int m_here = min(p.mt, p.o.m - m0);
  const int ks0 = (int)((int64_t)p.k_stages * rank / p.share), ks1 = (int)((int64_t)p.k_stages * (rank + 1) / p.share);
  const int steps = (min(ks1 * STAGE_STEPS, p.k_steps) - ks0 * STAGE_STEPS) * (MX4_STEP / KC);  // of KC values
  const int second = DUAL ? p.o.n + n0 : n0 + HALF;  // weight row of the tile's second half
  const bool apart = DUAL && p.o.n % HALF;           // the up rows' scales lie in two runs of 128 rows: lanes read them from memory
  pdl_trigger();
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.codes; ++s) {
      mbar_init(&code_full[s], 1);
      mbar_init(&code_empty[s], CONVERT_WARPS);
    }
    for (int s = 0; s < p.ring; ++s) {
      mbar_init(&full[s], 1 + CONVERT_WARPS / 2);
      mbar_init(&empty[s], 1);
    }
    mbar_init(done, 1);
    mbar_init(acc_free, CONVERT_WARPS);
    *abort_flag = 0;
    *ok_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == X_WARP && lane == 0) {  // the first weights into L2: that needs no wait for the kernel before, whatever it writes
    for (int ks = ks0; ks < ks1 && ks < ks0 + p.codes; ++ks) {
      mx4_prefetch_2d(&tm_w, ks * 64, n0);
      mx4_prefetch_2d(&tm_w, ks * 64, second);
    }
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, p.tmem_cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t acc = *tmem_slot;
  const uint32_t w_cols = acc + p.nt;  // the weights of step b of the ring: w_cols + b * COLS

  if (warp == 0) {
    // ------------------------------------------------ codes and scales
    if (lane == 0) {
      pdl_wait();
      Mx4Ring ring;
      for (int ks = ks0; ks < ks1; ++ks, ring.next(p.codes)) {
        uint8_t* sp = code_smem + ring.at * CODE_STAGE;
        uint64_t* bar = &code_full[ring.at];
        if (!mbar_wait(&code_empty[ring.at], ring.parity ^ 1, p.err, abort_flag)) break;
        const int s0 = ks * STAGE_STEPS;
        const uint32_t sc = min(STAGE_STEPS, p.k_steps - s0) * SCALE_BYTES;
        mbar_expect_tx(bar, CODE_BYTES + sc * (apart ? 1 : BLOCKS));
        tma_load_2d(sp, &tm_w, bar, ks * 64, n0);
        tma_load_2d(sp + CODE_BYTES / 2, &tm_w, bar, ks * 64, second);
        bulk_load(sp + CODE_BYTES, p.w_scales + mx4_scale_at(n0 & ~127, s0, p.k_steps), bar, sc);
        if (DUAL && !apart)
          bulk_load(sp + CODE_BYTES + STAGE_STEPS * SCALE_BYTES, p.w_scales + mx4_scale_at(second & ~127, s0, p.k_steps), bar, sc);
      }
    }
  } else if (warp == X_WARP) {
    // ------------------------------------------------ rows of X
    if (lane == 0) {
      pdl_wait();
      Mx4Ring ring;
      for (int c = 0, k = ks0 * STAGE_STEPS * MX4_STEP; c < steps; ++c, k += KC, ring.next(p.ring)) {
        if (!mbar_wait(&empty[ring.at], ring.parity ^ 1, p.err, abort_flag)) break;
        mbar_expect_tx(&full[ring.at], x_bytes);
#pragma unroll
        for (int b = 0; b < BOXES; ++b)
          tma_load_2d(smem + ring.at * x_bytes + b * box_bytes, &tm_x, &full[ring.at], k + b * BOX_K, m0 * G);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------ products
    pdl_wait();
    const uint32_t idesc = instr_desc((m_here * G + 15) & ~15);
    const uint64_t x0 = smem_desc(smem_u32(smem));
    const uint32_t x_stride = x_bytes >> 4, box_stride = box_bytes >> 4;
    Mx4Ring ring, acc_ring;
    bool ok = true;
    const int run = p.sum_stages * (STAGE_STEPS * MX4_STEP / KC);
    for (int from = 0; ok && from < steps; from += run, acc_ring.next(1)) {
      const int to = min(from + run, steps);
      if (!warp_wait(acc_free, acc_ring.parity ^ 1, p.err, abort_flag)) break;
      tc_fence_after();
      for (int c = from; c < to; ++c, ring.next(p.ring)) {
        if (!warp_wait(&full[ring.at], ring.parity, p.err, abort_flag)) { ok = false; break; }
        tc_fence_after();
        const uint64_t x = x0 + ring.at * x_stride;
        const uint32_t w = w_cols + ring.at * COLS;
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < KC / UMMA_K; ++k)
            umma_bf16_tmem_a(acc, w + k * 8, x + (k >> 2) * box_stride + (uint64_t)((k & 3) * UMMA_K * 2 >> 4), idesc, k > 0 ? 1u : c > from);
          umma_commit(&empty[ring.at]);
        }
        __syncwarp();
      }
      if (ok && elect_one()) umma_commit(done);
      __syncwarp();
    }
  } else {
    // ------------------------------------------------ conversion, a row a lane: two sets of four warps take steps in turn
    pdl_wait();
    const int quarter = warp & 3, set = (warp - CONVERT_WARP) >> 2, row = quarter * 32 + lane;
    const int block = DUAL && row >= HALF;
    const int w_row = DUAL ? min(block ? second + row - HALF : n0 + row, 2 * p.o.n - 1) : n0 + row;
    const bool far = apart && block;
    const uint8_t* far_scales = p.w_scales + mx4_scale_at(w_row, 0, p.k_steps);
    const int scale_at = CODE_BYTES + block * STAGE_STEPS * SCALE_BYTES + (w_row & 31) * 16 + ((w_row >> 5) & 3) * 4;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    Mx4Ring codes_ring, ring, acc_ring;
    if (KC < MX4_STEP) ring.next(p.ring, set);
    bool ok = true;
    for (int from = ks0; ok && from < ks1; from += p.sum_stages, acc_ring.next(1)) {
      const int to = min(from + p.sum_stages, ks1);
      for (int ks = from; ok && ks < to; ++ks, codes_ring.next(p.codes)) {
        const uint8_t* sp = code_smem + codes_ring.at * CODE_STAGE;
        const uint8_t* codes = sp + row * STAGE_BYTES_K;
        if (!warp_wait(&code_full[codes_ring.at], codes_ring.parity, p.err, abort_flag)) { ok = false; break; }
#pragma unroll
        for (int s = 0; s < STAGE_STEPS; ++s) {
          if (ks * STAGE_STEPS + s >= p.k_steps) break;
          if (KC == MX4_STEP && s != set) {
            ring.next(p.ring);
            continue;
          }
          const uint32_t bytes = far ? __ldcg(reinterpret_cast<const uint32_t*>(far_scales + (ks * STAGE_STEPS + s) * 512ll))
                                     : *reinterpret_cast<const uint32_t*>(sp + scale_at + s * SCALE_BYTES);
          const bool large = __any_sync(0xffffffffu, bytes & 0x80808080u);
#pragma unroll
          for (int i = 0; i < KC / BOX_K; ++i) {
            const int h = KC == MX4_STEP ? i : set;  // 64 of the 128 values
            const uint4 q[2] = {*reinterpret_cast<const uint4*>(codes + (((s * 4 + h * 2) ^ (row & 7)) << 4)),
                                *reinterpret_cast<const uint4*>(codes + (((s * 4 + h * 2 + 1) ^ (row & 7)) << 4))};
            uint32_t r[32];
            auto convert = [&](auto is_large) {
#pragma unroll
              for (int b = 0; b < 2; ++b) {
                const Mx4Factor f = mx4_factor<decltype(is_large)::value>((bytes >> (16 * h + 8 * b)) & 255);
                const uint32_t words[4] = {q[b].x, q[b].y, q[b].z, q[b].w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  uint32_t t[4];
                  mx4_to_bf16<decltype(is_large)::value>(words[k], f, t);
#pragma unroll
                  for (int j = 0; j < 4; ++j) r[b * 16 + k * 4 + j] = t[j];
                }
              }
            };
            if (large) convert(std::true_type{});
            else convert(std::false_type{});
            if (i == 0) {
              if (!warp_wait(&empty[ring.at], ring.parity ^ 1, p.err, abort_flag)) { ok = false; break; }
              tc_fence_after();
            }
            tmem_st32_raw(w_cols + ring.at * COLS + i * (BOX_K / 2) + lanes, r);
          }
          if (!ok) break;
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&full[ring.at]);
          ring.next(p.ring, KC == MX4_STEP ? 1 : 2);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&code_empty[codes_ring.at]);
      }
      // ---------------------------------------------- results: the sets take halves of the columns
      if (!ok || !warp_wait(done, acc_ring.parity, p.err, abort_flag)) break;
      tc_fence_after();
      const int half = ((m_here + 1) / 2 + 15) & ~15, first = set * half, last = set ? m_here : min(half, m_here);
      float* const sums = reinterpret_cast<float*>(smem + p.sums_at) + first * TILE_A;
      if (last > first) {
        const uint32_t at = acc + first * G + lanes;
        if (p.joined || from == ks0) mx4_leave<G, false>(p.o, at, m0 + first, last - first, n0, row, !p.joined, sums, AGAIN && from > ks0);
        else mx4_leave<G, false>(p.more, at, m0 + first, last - first, n0, row, true, sums);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(acc_free);
      if (threadIdx.x == CONVERT_WARP * 32) *ok_flag = 1;
    }
  }
  __syncwarp();
  if (*abort_flag) mx4_let_copies_land();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(acc, p.tmem_cols);
  if (p.joined) mx4_join<DUAL>(p.o, reinterpret_cast<const float*>(smem + p.sums_at), m0, m_here, n0, rank, p.share, *ok_flag != 0);
}

template <bool DUAL, int KC, int G>
int launch(const CucaMx4Gemm* c, int nt, int mt) {
  constexpr int CODE_STAGE = CODE_BYTES + (DUAL ? 2 : 1) * STAGE_STEPS * SCALE_BYTES;
  Params p;
  p.w_scales = c->w_scales;
  p.o = Mx4Out{c->out, c->bias, c->ldo, (int)c->m, (int)c->n, (int)c->out_f32, (int)c->epilogue, (int)c->bias_f32};
  p.k_steps = (int)mx4_steps(c->k);
  p.k_stages = (p.k_steps + STAGE_STEPS - 1) / STAGE_STEPS;
  p.err = c->err;
  p.nt = nt;
  p.mt = mt;
  const int features = DUAL ? HALF : TILE_A;
  p.tiles_n = (int)((c->n + features - 1) / features);
  const int64_t tiles = (int64_t)p.tiles_n * ((c->m + mt - 1) / mt);
  CUCA_REQUIRE(tiles * MAX_CLUSTER < (1ll << 31), "gemm_mx4: %lld rows by %lld features are too many", (long long)c->m, (long long)c->n);
  const bool two = nt <= 64;  // blocks an SM
  const int x_bytes = nt * KC * 2, budget = (two ? 108 : 222) * 1024;
  const int slots = cuca_device_sms() * (two ? 2 : 1);
  p.share = 1;
  while (p.share < MAX_CLUSTER && tiles * p.share * 2 <= slots && p.k_stages >= p.share * 4) p.share *= 2;
  const int stages = (p.k_stages + p.share - 1) / p.share;  // of a block, at most
  const int most = G > 1 ? SUM_STAGES_F32 : SUM_STAGES, sums = c->out_f32 ? (stages + most - 1) / most : 1;
  p.sum_stages = (stages + sums - 1) / sums;
  p.more = p.o;
  p.more.bias = nullptr;
  p.more.epilogue = EPI_RESIDUAL;
  p.joined = DUAL || p.share > 1 || (G > 1 && sums > 1);
  p.sums_bytes = p.joined && sums > 1 ? mt * TILE_A * 4 : 0;
  p.ring = ((two ? 256 : 512) - nt) / (KC / 2);
  if (p.ring > MAX_RING) p.ring = MAX_RING;
  while (p.ring > 2 && budget - p.sums_bytes - p.ring * x_bytes < 2 * CODE_STAGE) --p.ring;
  p.codes = (budget - p.sums_bytes - p.ring * x_bytes) / CODE_STAGE;
  if (p.codes > MAX_CODES) p.codes = MAX_CODES;
  p.tmem_cols = 32;
  while (p.tmem_cols < nt + p.ring * (KC / 2)) p.tmem_cols *= 2;
  const int stage_bytes = p.codes * CODE_STAGE + p.ring * x_bytes, data = stage_bytes + p.sums_bytes;
  p.sums_at = p.sums_bytes ? stage_bytes : 0;
  CUCA_REQUIRE(p.codes >= 2 && p.ring >= 2 && p.tmem_cols <= (two ? 256 : 512) && data - p.sums_at >= mt * TILE_A * 4, "gemm_mx4: no room for a tile");
  CUtensorMap tm_w, tm_x;
  const uint64_t cols = (uint64_t)p.k_steps * 32;  // the codes as 16-bit elements
  CUCA_REQUIRE(cuca_tensor_map_2d(c->w, 2, (uint64_t)c->n * (DUAL ? 2 : 1), cols, cols, HALF, &tm_w) &&
               cuca_tensor_map_2d(c->a, 2, (uint64_t)c->m * G, (uint64_t)c->k, (uint64_t)c->lda, nt, &tm_x), "gemm_mx4: tensor map failed");
  const dim3 grid((unsigned)(tiles * p.share));
  const int smem = data + 1024 + BARRIERS;
  auto start = [&](auto again) {
    constexpr auto kernel = gemm_mx4_wide_kernel<DUAL, KC, G, decltype(again)::value>;
    if (int e = mx4_configure<kernel>(227 * 1024)) return e;
    if (p.share > 1) cuca_launch_cluster(kernel, grid, dim3(THREADS), smem, c->stream, true, p.share, tm_w, tm_x, p);
    else cuca_launch(kernel, grid, dim3(THREADS), smem, c->stream, true, tm_w, tm_x, p);
    return 0;
  };
  if (int e = p.sums_bytes ? start(std::true_type{}) : start(std::false_type{})) return e;
  CUCA_CHECK_LAUNCH("gemm_mx4");
  return 0;
}

template <bool DUAL, int G>
int launch_tiles(const CucaMx4Gemm* c) {
  // 32-bit sums of many values that wait beside the stages leave room for fewer rows
  const int64_t features = (c->n + (DUAL ? HALF : TILE_A) - 1) / (DUAL ? HALF : TILE_A);
  const bool waits = c->out_f32 && c->k > SUM_STAGES * STAGE_STEPS * MX4_STEP &&
                     (DUAL || features * ((c->m + MOST_ROWS - 1) / MOST_ROWS) * 2 <= cuca_device_sms());
  const int64_t most = (waits && G == 1 ? MOST_WAITING : MOST_ROWS) / G;
  const int64_t tiles = (c->m + most - 1) / most, rows = (c->m + tiles - 1) / tiles;  // tiles of equal height
  const int nt = (int)(rows * G + 15) / 16 * 16, mt = G > 1 ? (int)rows : nt;
  return nt > 128 ? launch<DUAL, 64, G>(c, nt, mt) : launch<DUAL, 128, G>(c, nt, mt);
}

}  // namespace

// `parts`: X holds three rows for each of c->m
int cuca_gemm_mx4_wide(const CucaMx4Gemm* c, bool parts) {
  if (c->epilogue == EPI_SWIGLU) return parts ? launch_tiles<true, 3>(c) : launch_tiles<true, 1>(c);
  return parts ? launch_tiles<false, 3>(c) : launch_tiles<false, 1>(c);
}
