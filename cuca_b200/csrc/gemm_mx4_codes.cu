// Rows in 4 bits times a weight in 4 bits: out = epilogue(A W^T) on tcgen05.mma.kind::mxf4, which takes the codes and the powers of two
// of both operands as they are and sums in 32 bits.
//
// The weight is the 128-row operand, the rows of A the columns: D[feature, row], a lane of tensor memory per output feature (of a gated
// unit two accumulators side by side, gate and up). Codes come by TMA in stages of 256 values of a row, 128 bytes, with 128-byte
// swizzle; the scales of 128 rows and 128 values are 512 bytes that go into shared memory as one bulk copy and from there by
// tcgen05.cp into four columns of tensor memory, in columns of their own for each stage, which are free when the stage is. Nothing is
// converted, so few rows are bound by the weight's bytes; a block an SM has up to eight stages in flight, or two blocks five each.
// Few tiles: a cluster of up to eight blocks shares K; each leaves its sums in shared memory and adds an eighth of the features up in
// order out of the others': no workspace, equal bits in every run.
#include "mx4.cuh"
#include "mx4_mma.cuh"

namespace {

constexpr int STAGE_BYTES_K = 128;          // bytes of a row in a stage
constexpr int STAGE_STEPS = 2;              // of 128 values
constexpr int MAX_STAGES = 8;
constexpr int A_BYTES = TILE_A * STAGE_BYTES_K;
constexpr int SCALE_BYTES = 512;            // of 128 rows and a step
constexpr int MAX_CLUSTER = 8;
constexpr int THREADS = 192;                // a warp that loads, one that multiplies, four that read tensor memory
constexpr int BARRIERS = 512;

struct Params {
  const uint8_t* a_scales;
  const uint8_t* w_scales;
  Mx4Out o;
  int k_steps, k_stages;
  int nt;          // columns of a tile: rows of A, a multiple of 16
  int a_tiles;     // tiles of 128 rows that A's scales have
  int tiles_n, share;
  int stages, stage_bytes, tmem_cols;
  int* err;
};

template <bool DUAL>
__global__ void __launch_bounds__(THREADS) gemm_mx4_codes_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_a,
                                                                 const Params p) {
  constexpr int BLOCKS = DUAL ? 2 : 1;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* full = (uint64_t*)(smem + p.stages * p.stage_bytes);
  uint64_t* empty = full + MAX_STAGES;
  uint64_t* done = empty + MAX_STAGES;
  uint32_t* tmem_slot = (uint32_t*)(done + 1);
  volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
  volatile int* ok_flag = (volatile int*)(tmem_slot + 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = p.share > 1 ? (int)mx4_cluster_rank() : 0;
  const int tile = (int)blockIdx.x / p.share;
  const int n0 = (tile % p.tiles_n) * TILE_A, m0 = (tile / p.tiles_n) * p.nt;
  const int ks0 = (int)((int64_t)p.k_stages * rank / p.share), ks1 = (int)((int64_t)p.k_stages * (rank + 1) / p.share);
  const int up0 = p.o.n + n0;                     // the first up row
  const bool up_apart = DUAL && (p.o.n & 127);    // the up rows' scales do not start where 128 rows' do
  const int scale_tiles = min((p.nt + 127) >> 7, p.a_tiles - (m0 >> 7));
  const int b_bytes = p.nt * STAGE_BYTES_K;
  // scales of a stage: [block of weight rows][step][512], then [tile of 128 rows of A][step][512]
  const int sc_w = BLOCKS * A_BYTES + b_bytes, sc_a = sc_w + BLOCKS * STAGE_STEPS * SCALE_BYTES;
  pdl_trigger();
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&full[s], up_apart ? 2 : 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(done, 1);
    *abort_flag = 0;
    *ok_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, p.tmem_cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t acc = *tmem_slot;
  // columns: the accumulators, then a stage's scales in turn
  const int b_cols = 4 * ((p.nt + 127) >> 7);  // of a step
  const int stage_cols = STAGE_STEPS * (4 * BLOCKS + b_cols);
  const uint32_t scale_cols = acc + BLOCKS * p.nt;

  if (warp == 0) {
    if (lane == 0) {  // the first weights into L2: that needs no wait for the kernel before, whatever it writes
      for (int ks = ks0; ks < ks1 && ks < ks0 + p.stages; ++ks) {
        mx4_prefetch_2d(&tm_w, ks * 64, n0);
        if (DUAL) mx4_prefetch_2d(&tm_w, ks * 64, up0);
      }
    }
    __syncwarp();
    pdl_wait();
    for (int ks = ks0, it = 0; ks < ks1; ++ks, ++it) {
      const int st = it % p.stages;
      uint8_t* sp = smem + st * p.stage_bytes;
      if (it >= p.stages && !warp_wait(&empty[st], ((it / p.stages) & 1) ^ 1, p.err, abort_flag)) break;
      const int s0 = ks * STAGE_STEPS, steps = min(STAGE_STEPS, p.k_steps - s0);
      if (lane == 0) {
        const uint32_t sc = steps * SCALE_BYTES;
        mbar_expect_tx(&full[st], BLOCKS * A_BYTES + b_bytes + sc * ((up_apart ? 1 : BLOCKS) + scale_tiles));
        tma_load_2d(sp, &tm_w, &full[st], ks * 64, n0);
        if (DUAL) tma_load_2d(sp + A_BYTES, &tm_w, &full[st], ks * 64, up0);
        tma_load_2d(sp + BLOCKS * A_BYTES, &tm_a, &full[st], ks * 64, m0);
        bulk_load(sp + sc_w, p.w_scales + mx4_scale_at(n0, s0, p.k_steps), &full[st], sc);
        if (DUAL && !up_apart)
          bulk_load(sp + sc_w + STAGE_STEPS * SCALE_BYTES, p.w_scales + mx4_scale_at(up0, s0, p.k_steps), &full[st], sc);
        for (int t = 0; t < scale_tiles; ++t)
          bulk_load(sp + sc_a + t * STAGE_STEPS * SCALE_BYTES, p.a_scales + mx4_scale_at(m0 + 128 * t, s0, p.k_steps), &full[st], sc);
      }
      if (up_apart) {  // word by word: a lane's sixteen bytes are the scales of rows 32 apart
        for (int s = 0; s < steps; ++s) {
          uint32_t w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = min(up0 + 32 * i + lane, 2 * p.o.n - 1);
            w[i] = __ldcg(reinterpret_cast<const uint32_t*>(p.w_scales + mx4_scale_at(r, s0 + s, p.k_steps)));
          }
          *reinterpret_cast<uint4*>(sp + sc_w + (STAGE_STEPS + s) * SCALE_BYTES + lane * 16) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&full[st]);
      }
      __syncwarp();
    }
  } else if (warp == 1) {
    pdl_wait();
    const uint32_t idesc = mx4_instr_desc(p.nt, TILE_A);
    bool ok = true;
    for (int ks = ks0, it = 0; ks < ks1; ++ks, ++it) {
      const int st = it % p.stages;
      if (!warp_wait(&full[st], (it / p.stages) & 1, p.err, abort_flag)) { ok = false; break; }
      tc_fence_after();
      const uint32_t sa = smem_u32(smem + st * p.stage_bytes);
      const uint64_t adesc = smem_desc(sa), adesc2 = smem_desc(sa + A_BYTES), bdesc = smem_desc(sa + BLOCKS * A_BYTES);
      const uint32_t cols = scale_cols + st * stage_cols, cols_b = cols + STAGE_STEPS * 4 * BLOCKS;
      const int steps = min(STAGE_STEPS, p.k_steps - ks * STAGE_STEPS);
      if (elect_one()) {
        for (int s = 0; s < steps; ++s) {
          for (int b = 0; b < BLOCKS; ++b)
            mx4_scales_to_tmem(cols + (b * STAGE_STEPS + s) * 4, mx4_scale_desc(sa + sc_w + (b * STAGE_STEPS + s) * SCALE_BYTES));
          for (int t = 0; t < scale_tiles; ++t)
            mx4_scales_to_tmem(cols_b + s * b_cols + 4 * t, mx4_scale_desc(sa + sc_a + (t * STAGE_STEPS + s) * SCALE_BYTES));
        }
        for (int j = 0; j < 2 * steps; ++j) {  // 64 values each
          const uint64_t off = (uint64_t)(j * 32 >> 4);
          const uint32_t id = idesc | mx4_scale_half(j & 1), sb = cols_b + (j >> 1) * b_cols;
          const uint32_t accumulate = it > 0 || j > 0;
          mx4_umma(acc, adesc + off, bdesc + off, id, cols + (j >> 1) * 4, sb, accumulate);
          if (DUAL) mx4_umma(acc + p.nt, adesc2 + off, bdesc + off, id, cols + (STAGE_STEPS + (j >> 1)) * 4, sb, accumulate);
        }
        umma_commit(&empty[st]);
      }
      __syncwarp();
    }
    if (ok && elect_one()) umma_commit(done);
    __syncwarp();
  } else {
    pdl_wait();
    if (warp_wait(done, 0, p.err, abort_flag)) {
      tc_fence_after();
      const int row = (warp & 3) * 32 + lane;
      const uint32_t at = acc + ((uint32_t)((warp & 3) * 32) << 16);
      mx4_leave<DUAL>(p.o, at, p.nt, m0, min(p.nt, p.o.m - m0), n0, row, p.share == 1, reinterpret_cast<float*>(smem));
      if (row == 0) *ok_flag = 1;
    }
  }
  __syncwarp();
  if (*abort_flag) mx4_let_copies_land();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(acc, p.tmem_cols);
  if (p.share > 1) mx4_join<DUAL>(p.o, reinterpret_cast<const float*>(smem), p.nt, m0, min(p.nt, p.o.m - m0), n0, rank, p.share, *ok_flag != 0);
}

template <bool DUAL>
int launch(const CucaMx4Gemm* c) {
  Params p;
  p.a_scales = c->a_scales; p.w_scales = c->w_scales;
  p.o = Mx4Out{c->out, c->bias, c->ldo, (int)c->m, (int)c->n, (int)c->out_f32, (int)c->epilogue, 0};
  p.k_steps = (int)mx4_steps(c->k);
  p.k_stages = (p.k_steps + STAGE_STEPS - 1) / STAGE_STEPS;
  p.err = c->err;
  const int most = DUAL ? 128 : 256;
  p.nt = c->m >= most ? most : ((int)c->m + 15) / 16 * 16;
  p.a_tiles = (int)((c->m + 127) / 128);
  p.tiles_n = (int)((c->n + TILE_A - 1) / TILE_A);
  const int64_t tiles = (int64_t)p.tiles_n * ((c->m + p.nt - 1) / p.nt);
  CUCA_REQUIRE(tiles * MAX_CLUSTER < (1ll << 31), "gemm_mx4: %lld rows by %lld features are too many", (long long)c->m, (long long)c->n);
  const int blocks = DUAL ? 2 : 1, scale_tiles = (p.nt + 127) / 128;
  p.stage_bytes = blocks * (A_BYTES + STAGE_STEPS * SCALE_BYTES) + p.nt * STAGE_BYTES_K + scale_tiles * STAGE_STEPS * SCALE_BYTES;
  // two blocks an SM where tiles are small
  const bool two = p.nt * blocks <= 64;
  const int budget = (two ? 108 : 210) * 1024;
  p.stages = budget / p.stage_bytes < MAX_STAGES ? budget / p.stage_bytes : MAX_STAGES;
  if (p.stages > p.k_stages) p.stages = p.k_stages;
  const int need = blocks * p.nt + p.stages * STAGE_STEPS * 4 * (blocks + scale_tiles);
  p.tmem_cols = 32;
  while (p.tmem_cols < need) p.tmem_cols *= 2;
  CUCA_REQUIRE(p.stages >= 1 && p.tmem_cols <= (two ? 256 : 512), "gemm_mx4: no room for a tile");
  const int slots = cuca_device_sms() * (two ? 2 : 1);
  p.share = 1;
  while (p.share < MAX_CLUSTER && tiles * p.share * 2 <= slots && p.k_stages >= p.share * 4) p.share *= 2;
  // (shares are cut from four stages on, so a block has that many, or two of a gated unit: sums fit)
  CUCA_REQUIRE(p.share == 1 || p.stages * p.stage_bytes >= blocks * p.nt * TILE_A * 4, "gemm_mx4: sums do not fit");
  const int smem = p.stages * p.stage_bytes + 1024 + BARRIERS;
  CUtensorMap tm_w, tm_a;
  const uint64_t cols = (uint64_t)p.k_steps * 32;  // the codes as 16-bit elements
  CUCA_REQUIRE(cuca_tensor_map_2d(c->w, 2, (uint64_t)c->n * blocks, cols, cols, TILE_A, &tm_w) &&
               cuca_tensor_map_2d(c->a, 2, (uint64_t)c->m, cols, cols, p.nt, &tm_a), "gemm_mx4: tensor map failed");
  constexpr auto kernel = gemm_mx4_codes_kernel<DUAL>;
  if (int e = mx4_configure<kernel>(227 * 1024)) return e;
  const dim3 grid((unsigned)(tiles * p.share));
  if (p.share > 1) cuca_launch_cluster(kernel, grid, dim3(THREADS), smem, c->stream, true, p.share, tm_w, tm_a, p);
  else cuca_launch(kernel, grid, dim3(THREADS), smem, c->stream, true, tm_w, tm_a, p);
  CUCA_CHECK_LAUNCH("gemm_mx4");
  return 0;
}

}  // namespace

int cuca_gemm_mx4_codes(const CucaMx4Gemm* c) { return c->epilogue == EPI_SWIGLU ? launch<true>(c) : launch<false>(c); }
