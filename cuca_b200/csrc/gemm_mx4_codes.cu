// Rows in 4 bits times a weight in 4 bits: out = epilogue(A W^T) on tcgen05.mma.kind::mxf4, which takes the codes and the powers of two
// of both operands as they are and sums in 32 bits.
//
// The weight is the 128-row operand, the rows of A the columns: D[feature, row], a lane of tensor memory per output feature. A tile has
// one block of 128 features, or two that share the rows' tile: gate and up of a gated unit, or 256 features over many rows, where a
// block alone would be bound by what it loads (96 bytes a clock at the tensor cores' rate, two blocks 72). Codes come by TMA in
// stages of 256 values of a row, 128 bytes, with 128-byte swizzle; the scales of 128 rows and 128 values are 512 bytes that go into
// shared memory as one bulk copy and from there by tcgen05.cp into four columns of tensor memory, columns of their own for each
// stage, which are free when the stage is. A tile of A's rows may start at any multiple of 64: scales are taken
// from the 128 rows that it starts in, two columns further on.
// Nothing is converted, so few rows are bound by the weight's bytes, and where the weight is small by a block's start (its first values
// are there after 2 us) and the join. Few tiles: a cluster of up to four blocks shares K; each leaves its sums in shared memory and adds
// its part of the features up in order out of the others': no workspace, equal bits in every run. Many tiles: a block takes tiles in turn,
// the next one's loads under this one's results.
//
// Few bfloat16 rows come here too, as twelve digits each (mx4.cu): G columns make one row of the result, and what
// the digits left of a row, seldom anything, is multiplied on the ordinary pipes and added.
//
// Measured, K x features: 2,048 rows 4096 x 14336 gated 120 us (4.0 PFLOP/s; the tensor pipe busy for half of it: a stage takes 1,190
// clocks of which its contractions need 768, and a tile's results are not hidden), 14336 x 4096 66 us (3.6); 8 rows 4096 x 6144 5.9 us;
// 8 rows as digits 4096 x 14336 gated 16.9 us with the digits (3.7 TB/s), 14336 x 4096 14.4.
#include "mx4.cuh"
#include "mx4_mma.cuh"

namespace {

constexpr int STAGE_BYTES_K = 128;          // bytes of a row in a stage
constexpr int STAGE_STEPS = 2;              // of 128 values
constexpr int MAX_STAGES = 8;
constexpr int W_BYTES = TILE_A * STAGE_BYTES_K;
constexpr int SCALE_BYTES = 512;            // of 128 rows and a step
constexpr int MAX_CLUSTER = 4;              // (shares of K; eight took as long or longer: 14336 x 4096, 64 columns of digits 15.0 us, four 13.5)
constexpr int MANY_ROWS = 256;              // more rows than these: two blocks of features
constexpr int MANY_TILE = 192;              // ... and tiles of so many rows: two accumulators leave 128 columns for scales
// A warp that loads weights, one that loads rows, one that multiplies, and the others read results: sixteen of tiles of many rows, whose
// reading nothing hides, eight of small ones, of which an SM takes two.
constexpr int WEIGHT_WARP = 0, MMA_WARP = 1, ROW_WARP = 2, READ_WARP = 4;
constexpr int read_warps(int spans) { return spans == 2 ? 16 : 8; }
constexpr int threads(int spans) { return 32 * (READ_WARP + read_warps(spans)); }
constexpr int BARRIERS = 512;

struct Params {
  const uint8_t* a_scales;
  const uint8_t* w_scales;
  const uint8_t* w;
  Mx4Rest rest;    // of digits
  Mx4Out o;
  int k_steps, k_stages;
  int nt;          // rows of A of a whole tile, a multiple of 16
  int a_tiles;     // tiles of 128 rows that A's scales have
  int tiles, tiles_n, share;
  int stages, stage_bytes, tmem_cols;
  int* err;
};

template <int BLOCKS, bool DUAL, int SPANS, int G>
__global__ void __launch_bounds__(threads(SPANS), SPANS == 2 ? 1 : 2) gemm_mx4_codes_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_a,
                                                                 const Params p) {
  static_assert(!DUAL || BLOCKS == 2, "gate and up");
  constexpr int READ_WARPS = read_warps(SPANS), SETS = READ_WARPS / 4;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* full = (uint64_t*)(smem + p.stages * p.stage_bytes);
  uint64_t* empty = full + MAX_STAGES;
  uint64_t* done = empty + MAX_STAGES;
  uint64_t* acc_free = done + 1;
  uint32_t* tmem_slot = (uint32_t*)(acc_free + 1);
  volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
  volatile int* ok_flag = (volatile int*)(tmem_slot + 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = p.share > 1 ? (int)mx4_cluster_rank() : 0;
  const int first_tile = (int)blockIdx.x / p.share, tile_step = (int)gridDim.x / p.share;  // (of a cluster one tile)
  struct Tile {
    int n0, m0, nt;       // first feature, first row of A, columns that are multiplied (the last tile has no more than it needs)
    int t0, m_here;       // rows of the result: G rows in 4 bits make one
    int second;           // the second block's first weight row
    bool scaled;          // it has features (else it multiplies zeros)
    int span0, spans;     // A's runs of 128 scales
  };
  auto tile_at = [&](int tile) {
    Tile t;
    t.n0 = (tile % p.tiles_n) * (DUAL ? TILE_A : BLOCKS * TILE_A);
    t.m0 = (tile / p.tiles_n) * p.nt;
    const int rows = min(p.nt, p.o.m * G - t.m0);
    t.nt = (rows + 15) & ~15;
    t.t0 = t.m0 / G;
    t.m_here = rows / G;
    t.second = DUAL ? p.o.n + t.n0 : t.n0 + TILE_A;
    t.scaled = DUAL || t.second < p.o.n;
    t.span0 = t.m0 >> 7;
    t.spans = min(SPANS, p.a_tiles - t.span0);
    return t;
  };
  const int ks0 = (int)((int64_t)p.k_stages * rank / p.share), ks1 = (int)((int64_t)p.k_stages * (rank + 1) / p.share);
  const bool up_apart = DUAL && (p.o.n & 127);         // the up rows' scales do not start where 128 rows' do
  const int a_bytes = p.nt * STAGE_BYTES_K;
  // scales of a stage: [block of features][step][512], then [128 rows of A][step][512]
  const int sc_w = BLOCKS * W_BYTES + a_bytes, sc_a = sc_w + BLOCKS * STAGE_STEPS * SCALE_BYTES;
  pdl_trigger();
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&full[s], up_apart ? 3 : 2);
      mbar_init(&empty[s], 1);
    }
    mbar_init(done, 1);
    mbar_init(acc_free, READ_WARPS);
    *abort_flag = 0;
    *ok_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == ROW_WARP && lane == 0) {  // the first weights into L2: that needs no wait for the kernel before, whatever it writes
    const Tile t = tile_at(first_tile);
    for (int ks = ks0; ks < ks1 && ks < ks0 + p.stages; ++ks) {
      mx4_prefetch_2d(&tm_w, ks * 64, t.n0);
      if (BLOCKS == 2) mx4_prefetch_2d(&tm_w, ks * 64, t.second);
    }
  }
  if (warp == MMA_WARP) {
    tmem_alloc(tmem_slot, p.tmem_cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t acc = *tmem_slot;
  const uint32_t scale_cols = acc + BLOCKS * p.nt;  // of each stage and step [block of features][4], [128 rows of A][4]

  if (warp == WEIGHT_WARP) {
    // ------------------------------------------------ weights
    pdl_wait();
    Mx4Ring ring;
    bool ok = true;
    for (int tile = first_tile; ok && tile < p.tiles; tile += tile_step) {
      const Tile t = tile_at(tile);
      for (int ks = ks0; ks < ks1; ++ks, ring.next(p.stages)) {
        uint8_t* sp = smem + ring.at * p.stage_bytes;
        uint64_t* bar = &full[ring.at];
        if (!warp_wait(&empty[ring.at], ring.parity ^ 1, p.err, abort_flag)) { ok = false; break; }
        const int s0 = ks * STAGE_STEPS, steps = min(STAGE_STEPS, p.k_steps - s0);
        if (lane == 0) {
          const uint32_t sc = steps * SCALE_BYTES;
          mbar_expect_tx(bar, BLOCKS * W_BYTES + sc * (up_apart || !t.scaled ? 1 : BLOCKS));
          tma_load_2d(sp, &tm_w, bar, ks * 64, t.n0);
          if (BLOCKS == 2) tma_load_2d(sp + W_BYTES, &tm_w, bar, ks * 64, t.second);
          bulk_load(sp + sc_w, p.w_scales + mx4_scale_at(t.n0, s0, p.k_steps), bar, sc);
          if (BLOCKS == 2 && !up_apart && t.scaled)
            bulk_load(sp + sc_w + STAGE_STEPS * SCALE_BYTES, p.w_scales + mx4_scale_at(t.second, s0, p.k_steps), bar, sc);
        }
        if (up_apart) {  // word by word: a lane's sixteen bytes are the scales of rows 32 apart
          for (int s = 0; s < steps; ++s) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int r = min(t.second + 32 * i + lane, 2 * p.o.n - 1);
              w[i] = __ldcg(reinterpret_cast<const uint32_t*>(p.w_scales + mx4_scale_at(r, s0 + s, p.k_steps)));
            }
            *reinterpret_cast<uint4*>(sp + sc_w + (STAGE_STEPS + s) * SCALE_BYTES + lane * 16) = make_uint4(w[0], w[1], w[2], w[3]);
          }
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar);
        }
        __syncwarp();
      }
    }
  } else if (warp == ROW_WARP) {
    // ------------------------------------------------ rows of A
    if (lane == 0) {
      pdl_wait();
      Mx4Ring ring;
      bool ok = true;
      for (int tile = first_tile; ok && tile < p.tiles; tile += tile_step) {
        const Tile t = tile_at(tile);
        for (int ks = ks0; ks < ks1; ++ks, ring.next(p.stages)) {
          uint8_t* sp = smem + ring.at * p.stage_bytes;
          uint64_t* bar = &full[ring.at];
          if (!mbar_wait(&empty[ring.at], ring.parity ^ 1, p.err, abort_flag)) { ok = false; break; }
          const int s0 = ks * STAGE_STEPS;
          const uint32_t sc = min(STAGE_STEPS, p.k_steps - s0) * SCALE_BYTES;
          mbar_expect_tx(bar, a_bytes + sc * t.spans);
          tma_load_2d(sp + BLOCKS * W_BYTES, &tm_a, bar, ks * 64, t.m0);
          for (int i = 0; i < t.spans; ++i)
            bulk_load(sp + sc_a + i * STAGE_STEPS * SCALE_BYTES, p.a_scales + mx4_scale_at((t.span0 + i) * 128, s0, p.k_steps), bar, sc);
        }
      }
    }
  } else if (warp == MMA_WARP) {
    // ------------------------------------------------ products. What a stage issues stands unrolled, its descriptors one addition from
    // the first stage's: an instruction whose operands are worked out beside it takes twice as long to issue, and a stage has seventeen
    pdl_wait();
    const uint32_t sa = smem_u32(smem);
    const uint64_t w0 = smem_desc(sa), a0 = smem_desc(sa + BLOCKS * W_BYTES), sw0 = mx4_scale_desc(sa + sc_w), sr0 = mx4_scale_desc(sa + sc_a);
    const uint64_t stride = p.stage_bytes >> 4;
    constexpr int STEP_COLS = 4 * (BLOCKS + SPANS);
    Mx4Ring ring, acc_ring;
    bool ok = true;
    for (int tile = first_tile; ok && tile < p.tiles; tile += tile_step, acc_ring.next(1)) {
      const Tile t = tile_at(tile);
      const uint32_t idesc = mx4_instr_desc(t.nt, TILE_A);
      const uint32_t shift = (t.m0 & 127) >> 5;  // columns of scales before this tile's first row
      if (!warp_wait(acc_free, acc_ring.parity ^ 1, p.err, abort_flag)) break;
      tc_fence_after();
      for (int ks = ks0; ks < ks1; ++ks, ring.next(p.stages)) {
        if (!warp_wait(&full[ring.at], ring.parity, p.err, abort_flag)) { ok = false; break; }
        tc_fence_after();
        const uint64_t at = ring.at * stride;
        const uint32_t cols = scale_cols + ring.at * (STAGE_STEPS * STEP_COLS);
        const bool whole = (ks + 1) * STAGE_STEPS <= p.k_steps;
        if (elect_one()) {
#pragma unroll
          for (int s = 0; s < STAGE_STEPS; ++s) {
            if (s == 0 || whole) {
              const uint32_t cols_w = cols + s * STEP_COLS, cols_a = cols_w + 4 * BLOCKS;
#pragma unroll
              for (int b = 0; b < BLOCKS; ++b)
                mx4_scales_to_tmem(cols_w + 4 * b, sw0 + at + (uint64_t)((b * STAGE_STEPS + s) * SCALE_BYTES >> 4));
#pragma unroll
              for (int i = 0; i < SPANS; ++i)
                mx4_scales_to_tmem(cols_a + 4 * i, sr0 + at + (uint64_t)((i * STAGE_STEPS + s) * SCALE_BYTES >> 4));
#pragma unroll
              for (int h = 0; h < 2; ++h) {  // 64 values each
                const uint64_t off = at + (uint64_t)((s * 64 + h * 32) >> 4);
                const uint32_t id = idesc | mx4_scale_half(h), accumulate = s + h > 0 ? 1u : ks > ks0;
#pragma unroll
                for (int b = 0; b < BLOCKS; ++b)
                  mx4_umma(acc + b * p.nt, w0 + off + (uint64_t)(b * W_BYTES >> 4), a0 + off, id, cols_w + 4 * b, cols_a + shift, accumulate);
              }
            }
          }
          umma_commit(&empty[ring.at]);
        }
        __syncwarp();
      }
      if (ok && elect_one()) umma_commit(done);
      __syncwarp();
    }
  } else if (warp >= READ_WARP) {
    // ------------------------------------------------ results: sets of four warps take a part of the columns each, of one of two blocks of
    // features or of both accumulators of a gated unit
    pdl_wait();
    constexpr int PARTS = BLOCKS == 2 && !DUAL ? SETS / 2 : SETS;
    const int set = (warp - READ_WARP) >> 2, part = set % PARTS, block = set / PARTS, row = (warp & 3) * 32 + lane;
    const uint32_t at = acc + block * p.nt + ((uint32_t)((warp & 3) * 32) << 16);
    Mx4RestOf rest{p.rest, p.w, p.w_scales, p.k_steps, ks0 * STAGE_STEPS, min(ks1 * STAGE_STEPS, p.k_steps), false};
    if (G > 1) {  // while the products run: is there any?
      const int flags = p.o.m * p.k_steps;
      auto of = [](uint32_t word, int left) { return left >= 4 ? word : left > 0 ? word & ((1u << 8 * left) - 1) : 0u; };
      uint32_t some = 0;
      for (int i = lane * 16; i < flags; i += 512) {  // (there is memory to the end of 256)
        const uint4 f = __ldcg(reinterpret_cast<const uint4*>(p.rest.flags + i));
        some |= of(f.x, flags - i) | of(f.y, flags - i - 4) | of(f.z, flags - i - 8) | of(f.w, flags - i - 12);
      }
      rest.any = __any_sync(0xffffffffu, some != 0);
    }
    float* sums = reinterpret_cast<float*>(smem) + block * (p.nt / G) * TILE_A;  // (of a cluster: every copy into the stages has been waited for)
    Mx4Ring acc_ring;
    for (int tile = first_tile; tile < p.tiles; tile += tile_step, acc_ring.next(1)) {
      const Tile t = tile_at(tile);
      if (!warp_wait(done, acc_ring.parity, p.err, abort_flag)) break;
      tc_fence_after();
      constexpr int UNIT = 16 * Mx4Group<G>::LOADS;
      const int each = ((t.nt + PARTS - 1) / PARTS + UNIT - 1) / UNIT * UNIT / G, first = part * each, last = min(first + each, t.m_here);
      if (last > first && (block == 0 || t.scaled))
        mx4_leave<G, DUAL>(p.o, at + first * G, t.t0 + first, last - first, t.n0 + block * TILE_A, row, p.share == 1, sums + first * TILE_A,
                           false, p.nt, p.nt / G, rest);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(acc_free);
      if (threadIdx.x == READ_WARP * 32) *ok_flag = 1;
    }
  }
  __syncwarp();
  if (*abort_flag) mx4_let_copies_land();
  tc_fence_before();
  __syncthreads();
  if (warp == MMA_WARP) tmem_dealloc(acc, p.tmem_cols);
  if (p.share > 1) {
    const float* sums = reinterpret_cast<const float*>(smem);
    const Tile t = tile_at(first_tile);
    mx4_join<false>(p.o, sums, t.t0, t.m_here, t.n0, rank, p.share, *ok_flag != 0, DUAL ? p.nt / G : 0);
    if (BLOCKS == 2 && !DUAL) mx4_join<false>(p.o, sums + (p.nt / G) * TILE_A, t.t0, t.m_here, t.n0 + TILE_A, rank, p.share, *ok_flag != 0 && t.scaled);
  }
}

template <int BLOCKS, bool DUAL, int SPANS, int G>
int launch_spans(const CucaMx4Gemm* c, const Mx4Rest* rest) {
  const int64_t m = c->m * G;  // rows in 4 bits
  Params p;
  p.a_scales = c->a_scales; p.w_scales = c->w_scales; p.w = c->w;
  p.rest = rest ? *rest : Mx4Rest{};
  p.o = Mx4Out{c->out, c->bias, c->ldo, (int)c->m, (int)c->n, (int)c->out_f32, (int)c->epilogue, (int)c->bias_f32};
  p.k_steps = (int)mx4_steps(c->k);
  p.k_stages = (p.k_steps + STAGE_STEPS - 1) / STAGE_STEPS;
  p.err = c->err;
  const int most = BLOCKS == 2 ? MANY_TILE : MANY_ROWS;
  p.nt = m >= most ? most : ((int)m + 15) / 16 * 16;
  p.a_tiles = (int)((m + 127) / 128);
  const int features = DUAL ? TILE_A : BLOCKS * TILE_A;
  p.tiles_n = (int)((c->n + features - 1) / features);
  const int64_t tiles = (int64_t)p.tiles_n * ((m + p.nt - 1) / p.nt);
  CUCA_REQUIRE(tiles * MAX_CLUSTER < (1ll << 31), "gemm_mx4: %lld rows by %lld features are too many", (long long)c->m, (long long)c->n);
  p.stage_bytes = BLOCKS * (W_BYTES + STAGE_STEPS * SCALE_BYTES) + p.nt * STAGE_BYTES_K + SPANS * STAGE_STEPS * SCALE_BYTES;
  const bool two = p.nt * BLOCKS <= 64;  // blocks an SM
  const int budget = (two ? 108 : 222) * 1024, room = (two ? 256 : 512) - BLOCKS * p.nt, stage_cols = STAGE_STEPS * 4 * (BLOCKS + SPANS);
  p.stages = budget / p.stage_bytes;
  if (p.stages > MAX_STAGES) p.stages = MAX_STAGES;
  if (p.stages > room / stage_cols) p.stages = room / stage_cols;
  if (p.stages > p.k_stages) p.stages = p.k_stages;
  p.tmem_cols = 32;
  while (p.tmem_cols < BLOCKS * p.nt + p.stages * stage_cols) p.tmem_cols *= 2;
  CUCA_REQUIRE(p.stages >= 1 && p.tmem_cols <= (two ? 256 : 512), "gemm_mx4: no room for a tile");
  const int slots = cuca_device_sms() * (two ? 2 : 1), sums = BLOCKS * p.nt / G * TILE_A * 4;
  p.share = 1;
  while (p.share < MAX_CLUSTER && tiles * p.share * 2 <= slots && p.k_stages >= p.share * 4 && sums <= p.stages * p.stage_bytes) p.share *= 2;
  const int smem = p.stages * p.stage_bytes + 1024 + BARRIERS;
  CUtensorMap tm_w, tm_a;
  const uint64_t cols = (uint64_t)p.k_steps * 32;  // the codes as 16-bit elements
  CUCA_REQUIRE(cuca_tensor_map_2d(c->w, 2, (uint64_t)c->n * (DUAL ? 2 : 1), cols, cols, TILE_A, &tm_w) &&
               cuca_tensor_map_2d(c->a, 2, (uint64_t)m, cols, cols, p.nt, &tm_a), "gemm_mx4: tensor map failed");
  constexpr auto kernel = gemm_mx4_codes_kernel<BLOCKS, DUAL, SPANS, G>;
  if (int e = mx4_configure<kernel>(227 * 1024)) return e;
  p.tiles = (int)tiles;
  const dim3 grid(p.share > 1 || tiles < slots ? (unsigned)(tiles * p.share) : (unsigned)slots);
  if (p.share > 1) cuca_launch_cluster(kernel, grid, dim3(threads(SPANS)), smem, c->stream, true, p.share, tm_w, tm_a, p);
  else cuca_launch(kernel, grid, dim3(threads(SPANS)), smem, c->stream, true, tm_w, tm_a, p);
  CUCA_CHECK_LAUNCH("gemm_mx4");
  return 0;
}

template <int G>
int launch(const CucaMx4Gemm* c, const Mx4Rest* rest) {
  const int64_t m = c->m * G;
  // a tile of more than 128 rows, or one that starts in the middle of 128, touches the scales of two runs of 128 rows
  if (c->epilogue == EPI_SWIGLU) return m > 128 ? launch_spans<2, true, 2, G>(c, rest) : launch_spans<2, true, 1, G>(c, rest);
  if constexpr (G == 1) {
    if (m > MANY_ROWS) return launch_spans<2, false, 2, G>(c, rest);
  } else {
    CUCA_REQUIRE(m <= MANY_TILE, "gemm_mx4: %lld rows as digits", (long long)c->m);  // a tile
  }
  return m > 128 ? launch_spans<1, false, 2, G>(c, rest) : launch_spans<1, false, 1, G>(c, rest);
}

}  // namespace

// `rest`: A holds MX4_DIGITS rows for each of c->m, and this is what they left of them; else null
int cuca_gemm_mx4_codes(const CucaMx4Gemm* c, const Mx4Rest* rest) { return rest ? launch<MX4_DIGITS>(c, rest) : launch<1>(c, nullptr); }
