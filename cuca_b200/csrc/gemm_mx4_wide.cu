// bfloat16 rows times a weight in 4 bits on tcgen05: out = epilogue(X W^T).
//
// A code times its power of two is a bfloat16 number exactly, so what the tensor cores multiply is the weight as it is kept and the rows
// as they are. The weight is the 128-row operand and comes out of tensor memory: converter warps take codes from shared memory, a weight
// row a lane, and leave 64 values of it as 32 columns. Shared memory would have to take the converted tile in and give it out again
// beside the rows' own tiles, more than its 128 bytes a clock. The rows of X are the columns, by TMA with 128-byte swizzle.
//
// What bounds it: few rows, the weight's bytes (17 bits for 32 values) and the conversion's instructions, 17 for eight codes, 2.9 of four
// issue slots a clock at the memory's full rate; many rows, the tensor cores: a tile of 256 rows converts 16 codes a clock.
// Few tiles: a cluster of up to eight blocks shares K and adds its sums in order out of each other's shared memory.
#include "mx4.cuh"
#include "mx4_mma.cuh"

namespace {

constexpr int CHUNK = 64;                   // values that a buffer in tensor memory and a tile of X hold of a row
constexpr int CHUNK_COLS = CHUNK / 2;
constexpr int STAGE_BYTES_K = 128;          // bytes of a row of codes in a stage: 256 values
constexpr int STAGE_STEPS = 2, STAGE_CHUNKS = 4;
constexpr int CODE_BYTES = TILE_A * STAGE_BYTES_K;
constexpr int SCALE_BYTES = 512;            // of 128 rows and a step
constexpr int MAX_CODES = 4, MAX_X = 8, MAX_A = 4, MAX_CLUSTER = 8;
constexpr int CONVERT_WARP = 2, CONVERT_WARPS = 8, X_WARP = CONVERT_WARP + CONVERT_WARPS;
constexpr int THREADS = 32 * (X_WARP + 1);  // a warp that loads codes, one that multiplies, eight that convert, one that loads rows
constexpr int BARRIERS = 512;

struct Params {
  const uint8_t* w_scales;
  Mx4Out o;
  int k_steps, k_stages;
  int nt;  // columns of a tile: rows of X, a multiple of 16
  int tiles_n, share;
  int codes, xs, bufs;  // stages of codes, tiles of X, buffers in tensor memory
  int tmem_cols;
  int* err;
};

template <bool DUAL>
__global__ void __launch_bounds__(THREADS) gemm_mx4_wide_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x,
                                                                const Params p) {
  constexpr int BLOCKS = DUAL ? 2 : 1;
  constexpr int CODE_STAGE = BLOCKS * (CODE_BYTES + STAGE_STEPS * SCALE_BYTES);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const int x_bytes = p.nt * CHUNK * 2;
  uint8_t* const x_smem = smem + p.codes * CODE_STAGE;
  uint64_t* code_full = (uint64_t*)(x_smem + p.xs * x_bytes);
  uint64_t* code_empty = code_full + MAX_CODES;
  uint64_t* x_full = code_empty + MAX_CODES;
  uint64_t* x_empty = x_full + MAX_X;
  uint64_t* a_full = x_empty + MAX_X;
  uint64_t* a_empty = a_full + MAX_A;
  uint64_t* done = a_empty + MAX_A;
  uint32_t* tmem_slot = (uint32_t*)(done + 1);
  volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
  volatile int* ok_flag = (volatile int*)(tmem_slot + 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = p.share > 1 ? (int)mx4_cluster_rank() : 0;
  const int tile = (int)blockIdx.x / p.share;
  const int n0 = (tile % p.tiles_n) * TILE_A, m0 = (tile / p.tiles_n) * p.nt;
  const int ks0 = (int)((int64_t)p.k_stages * rank / p.share), ks1 = (int)((int64_t)p.k_stages * (rank + 1) / p.share);
  const int c0 = ks0 * STAGE_CHUNKS, c1 = min(ks1 * STAGE_CHUNKS, 2 * p.k_steps);  // chunks of this block
  const int up0 = p.o.n + n0;
  const bool up_apart = DUAL && (p.o.n & 127);  // the up rows' scales do not start where 128 rows' do: lanes read them from memory
  pdl_trigger();
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.codes; ++s) {
      mbar_init(&code_full[s], 1);
      mbar_init(&code_empty[s], CONVERT_WARPS);
    }
    for (int s = 0; s < p.xs; ++s) {
      mbar_init(&x_full[s], 1);
      mbar_init(&x_empty[s], 1);
    }
    for (int s = 0; s < p.bufs; ++s) {
      mbar_init(&a_full[s], DUAL ? CONVERT_WARPS : CONVERT_WARPS / 2);
      mbar_init(&a_empty[s], 1);
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
  const uint32_t a_cols = acc + BLOCKS * p.nt;  // buffer b of block i: a_cols + (b * BLOCKS + i) * CHUNK_COLS

  if (warp == 0) {
    // ------------------------------------------------ codes and scales
    if (lane == 0) {
      // the first weights into L2: that needs no wait for the kernel before, whatever it writes
      for (int ks = ks0; ks < ks1 && ks < ks0 + p.codes; ++ks) {
        mx4_prefetch_2d(&tm_w, ks * 64, n0);
        if (DUAL) mx4_prefetch_2d(&tm_w, ks * 64, up0);
      }
      pdl_wait();
      Mx4Ring ring;
      for (int ks = ks0; ks < ks1; ++ks, ring.next(p.codes)) {
        const int st = ring.at;
        uint8_t* sp = smem + st * CODE_STAGE;
        if (!mbar_wait(&code_empty[st], ring.parity ^ 1, p.err, abort_flag)) break;
        const int s0 = ks * STAGE_STEPS;
        const uint32_t sc = min(STAGE_STEPS, p.k_steps - s0) * SCALE_BYTES;
        mbar_expect_tx(&code_full[st], BLOCKS * CODE_BYTES + sc * (up_apart ? 1 : BLOCKS));
        tma_load_2d(sp, &tm_w, &code_full[st], ks * 64, n0);
        if (DUAL) tma_load_2d(sp + CODE_BYTES, &tm_w, &code_full[st], ks * 64, up0);
        bulk_load(sp + BLOCKS * CODE_BYTES, p.w_scales + mx4_scale_at(n0, s0, p.k_steps), &code_full[st], sc);
        if (DUAL && !up_apart)
          bulk_load(sp + BLOCKS * CODE_BYTES + STAGE_STEPS * SCALE_BYTES, p.w_scales + mx4_scale_at(up0, s0, p.k_steps), &code_full[st], sc);
      }
    }
  } else if (warp == X_WARP) {
    // ------------------------------------------------ rows of X
    if (lane == 0) {
      pdl_wait();
      Mx4Ring ring;
      for (int c = c0; c < c1; ++c, ring.next(p.xs)) {
        if (!mbar_wait(&x_empty[ring.at], ring.parity ^ 1, p.err, abort_flag)) break;
        mbar_expect_tx(&x_full[ring.at], x_bytes);
        tma_load_2d(x_smem + ring.at * x_bytes, &tm_x, &x_full[ring.at], c * CHUNK, m0);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------ products
    pdl_wait();
    const uint32_t idesc = instr_desc(p.nt);
    bool ok = true;
    Mx4Ring x_ring, a_ring;
    for (int c = c0; c < c1; ++c, x_ring.next(p.xs), a_ring.next(p.bufs)) {
      const int xs = x_ring.at, buf = a_ring.at;
      if (!warp_wait(&x_full[xs], x_ring.parity, p.err, abort_flag)) { ok = false; break; }
      if (!warp_wait(&a_full[buf], a_ring.parity, p.err, abort_flag)) { ok = false; break; }
      tc_fence_after();
      const uint64_t bdesc = smem_desc(smem_u32(x_smem + xs * x_bytes));
      const uint32_t a = a_cols + buf * BLOCKS * CHUNK_COLS;
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < CHUNK / UMMA_K; ++k) {
          const uint64_t off = (uint64_t)(k * UMMA_K * 2 >> 4);
          umma_bf16_tmem_a(acc, a + k * 8, bdesc + off, idesc, c > c0 || k > 0);
          if (DUAL) umma_bf16_tmem_a(acc + p.nt, a + CHUNK_COLS + k * 8, bdesc + off, idesc, c > c0 || k > 0);
        }
        umma_commit(&x_empty[xs]);
        umma_commit(&a_empty[buf]);
      }
      __syncwarp();
    }
    if (ok && elect_one()) umma_commit(done);
    __syncwarp();
  } else {
    // ------------------------------------------------ conversion: of a gated unit a set of warps takes the gate rows and one the up rows,
    // else the sets take chunks in turn
    pdl_wait();
    const int quarter = warp & 3, set = (warp - CONVERT_WARP) >> 2, row = quarter * 32 + lane;
    const int block = DUAL ? set : 0;
    const bool apart = up_apart && block == 1;
    const uint8_t* scales_of_row = p.w_scales + mx4_scale_at(min(up0 + row, 2 * p.o.n - 1), 0, p.k_steps);
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    bool ok = true;
    Mx4Ring ring, a_ring;
    if (!DUAL) a_ring.next(p.bufs, set);
    for (int ks = ks0; ok && ks < ks1; ++ks, ring.next(p.codes)) {
      const int st = ring.at;
      const uint8_t* sp = smem + st * CODE_STAGE;
      const uint8_t* codes = sp + block * CODE_BYTES + row * STAGE_BYTES_K;
      const int steps = min(STAGE_STEPS, p.k_steps - ks * STAGE_STEPS);
      if (!warp_wait(&code_full[st], ring.parity, p.err, abort_flag)) { ok = false; break; }
      for (int s = 0; s < steps; ++s) {
        const uint32_t bytes = apart ? __ldcg(reinterpret_cast<const uint32_t*>(scales_of_row + (ks * STAGE_STEPS + s) * 512ll))
                                     : *reinterpret_cast<const uint32_t*>(sp + BLOCKS * CODE_BYTES + (block * STAGE_STEPS + s) * SCALE_BYTES +
                                                                          lane * 16 + quarter * 4);
        for (int h = DUAL ? 0 : set; h < (DUAL ? 2 : set + 1); ++h, a_ring.next(p.bufs, DUAL ? 1 : 2)) {  // halves of a step: chunks
          const int chunk = s * 2 + h, buf = a_ring.at;
          uint32_t r[32];
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const uint4 q = *reinterpret_cast<const uint4*>(codes + (((chunk * 2 + b) ^ (row & 7)) << 4));
            const uint32_t byte = (bytes >> (8 * (h * 2 + b))) & 255;
            const Mx4Factor f = mx4_factor(byte);
            const uint32_t words[4] = {q.x, q.y, q.z, q.w};
            const bool large = byte > 128 && byte < 255;
            uint32_t t[4];
            if (__any_sync(0xffffffffu, large)) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                mx4_to_bf16<true>(words[i], f, t);
#pragma unroll
                for (int j = 0; j < 4; ++j) r[b * 16 + i * 4 + j] = t[j];
              }
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                mx4_to_bf16<false>(words[i], f, t);
#pragma unroll
                for (int j = 0; j < 4; ++j) r[b * 16 + i * 4 + j] = t[j];
              }
            }
          }
          if (!warp_wait(&a_empty[buf], a_ring.parity ^ 1, p.err, abort_flag)) { ok = false; break; }
          tc_fence_after();
          tmem_st32_raw(a_cols + (buf * BLOCKS + block) * CHUNK_COLS + lanes, r);
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&a_full[buf]);
        }
        if (!ok) break;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&code_empty[st]);
    }
    // ------------------------------------------------ results: the sets take halves of the columns
    if (ok && warp_wait(done, 0, p.err, abort_flag)) {
      tc_fence_after();
      const int m_here = min(p.nt, p.o.m - m0), half = (p.nt / 2 + 15) / 16 * 16;
      const int first = set * half, last = set ? m_here : min(half, m_here);
      if (last > first)
        mx4_leave<DUAL>(p.o, acc + first + lanes, p.nt, m0 + first, last - first, n0, row, p.share == 1,
                        reinterpret_cast<float*>(smem) + first * TILE_A);
      if (threadIdx.x == CONVERT_WARP * 32) *ok_flag = 1;
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
  constexpr int BLOCKS = DUAL ? 2 : 1;
  constexpr int CODE_STAGE = BLOCKS * (CODE_BYTES + STAGE_STEPS * SCALE_BYTES);
  Params p;
  p.w_scales = c->w_scales;
  p.o = Mx4Out{c->out, c->bias, c->ldo, (int)c->m, (int)c->n, (int)c->out_f32, (int)c->epilogue, 0};
  p.k_steps = (int)mx4_steps(c->k);
  p.k_stages = (p.k_steps + STAGE_STEPS - 1) / STAGE_STEPS;
  p.err = c->err;
  const int most = DUAL ? 128 : 256;
  p.nt = c->m >= most ? most : ((int)c->m + 15) / 16 * 16;
  p.tiles_n = (int)((c->n + TILE_A - 1) / TILE_A);
  const int64_t tiles = (int64_t)p.tiles_n * ((c->m + p.nt - 1) / p.nt);
  CUCA_REQUIRE(tiles * MAX_CLUSTER < (1ll << 31), "gemm_mx4: %lld rows by %lld features are too many", (long long)c->m, (long long)c->n);
  const bool two = p.nt * BLOCKS <= 64;  // blocks an SM
  const int x_bytes = p.nt * CHUNK * 2, budget = (two ? 108 : 210) * 1024;
  p.codes = two ? (DUAL ? 2 : 4) : 3;
  p.xs = (budget - p.codes * CODE_STAGE) / x_bytes;
  if (p.xs > MAX_X) p.xs = MAX_X;
  p.bufs = ((two ? 256 : 512) - BLOCKS * p.nt) / (BLOCKS * CHUNK_COLS);
  if (p.bufs > MAX_A) p.bufs = MAX_A;
  p.tmem_cols = 32;
  while (p.tmem_cols < BLOCKS * (p.nt + p.bufs * CHUNK_COLS)) p.tmem_cols *= 2;
  const int slots = cuca_device_sms() * (two ? 2 : 1);
  p.share = 1;
  while (p.share < MAX_CLUSTER && tiles * p.share * 2 <= slots && p.k_stages >= p.share * 4) p.share *= 2;
  const int data = p.codes * CODE_STAGE + p.xs * x_bytes;
  CUCA_REQUIRE(p.xs >= 2 && p.bufs >= 2 && p.tmem_cols <= (two ? 256 : 512) && data >= BLOCKS * p.nt * TILE_A * 4, "gemm_mx4: no room for a tile");
  const uint64_t lda = c->m == 1 ? (c->k + 7) / 8 * 8 : c->lda;  // (of one row there is no stride)
  CUtensorMap tm_w, tm_x;
  const uint64_t cols = (uint64_t)p.k_steps * 32;  // the codes as 16-bit elements
  CUCA_REQUIRE(cuca_tensor_map_2d(c->w, 2, (uint64_t)c->n * BLOCKS, cols, cols, TILE_A, &tm_w) &&
               cuca_tensor_map_2d(c->a, 2, (uint64_t)c->m, (uint64_t)c->k, lda, p.nt, &tm_x), "gemm_mx4: tensor map failed");
  constexpr auto kernel = gemm_mx4_wide_kernel<DUAL>;
  if (int e = mx4_configure<kernel>(227 * 1024)) return e;
  const dim3 grid((unsigned)(tiles * p.share));
  const int smem = data + 1024 + BARRIERS;
  if (p.share > 1) cuca_launch_cluster(kernel, grid, dim3(THREADS), smem, c->stream, true, p.share, tm_w, tm_x, p);
  else cuca_launch(kernel, grid, dim3(THREADS), smem, c->stream, true, tm_w, tm_x, p);
  CUCA_CHECK_LAUNCH("gemm_mx4");
  return 0;
}

}  // namespace

int cuca_gemm_mx4_wide(const CucaMx4Gemm* c) { return c->epilogue == EPI_SWIGLU ? launch<true>(c) : launch<false>(c); }
