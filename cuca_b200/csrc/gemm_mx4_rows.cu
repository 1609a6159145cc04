// Few rows of 16 or 32 bits times a weight in 4 bits: out = epilogue(X W^T); W as mx4.cuh lays it out.
//
// Bound by the weight's bytes, 17 bits for 32 values, and by the instructions that make bfloat16 numbers of codes (17 for eight codes:
// see mx4_to_bf16). Codes times their power of two are bfloat16 numbers exactly, so a product with a bfloat16 row is exact and is
// summed in 32 bits. A 32-bit value is the sum of three bfloat16 parts (exact from 2^-110 on), three rows of one product, whose sums
// are added at the end. Nothing here passes through tensor memory: one row takes some 3 us less than in the form for many.
//
// A block has eight warps: four take 32 weight rows each of a tile of 128 (of a gated unit 64 gate and 64 up rows), and two sets of four
// take the steps of 128 values in turn. A lane's 16 bytes are one block of 32 codes of one weight row, so a warp reads 64 bytes of 32
// rows at a time and every lane has one scale per row. Few tiles: a cluster of up to eight blocks shares K, and adds its sums in
// order out of each other's shared memory: no workspace, and equal bits in every run.
#include "mx4_mma.cuh"
#include <type_traits>

namespace {

constexpr int WARPS = 8, THREADS = 32 * WARPS;
constexpr int ROWS = 16;       // of X at most: two runs of eight, as the matrix instruction takes them
constexpr int TILE = 128;      // weight rows of a block
constexpr int GROUPS = 4;      // of eight weight rows a warp, two to a matrix instruction
constexpr int KEPT = 16;       // steps of A in shared memory at a time
constexpr int A_STRIDE = KEPT * MX4_STEP * 2 + 64;  // bytes: rows next to each other lie 16 banks apart
constexpr int SUM_STRIDE = TILE + 4;
constexpr int MAX_CLUSTER = 8;
constexpr int SMEM = ROWS * A_STRIDE;
static_assert(ROWS * SUM_STRIDE * 4 * 2 <= SMEM, "two sets' sums lie where A lay");

struct Params {
  const void* a;
  int64_t lda;
  const uint8_t* w;
  const uint8_t* w_scales;
  const void* bias;
  void* out;
  int64_t ldo;
  int m, n, k, steps;
  int out_f32, epilogue;
  int share;  // blocks of a cluster
  bool wide;  // rows of A start on 16 bytes
};

// 16 weight rows (a0..a3: rows g, g + 8 of the lower, then of the upper eight values) times eight rows of X
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const __nv_bfloat162 t = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&t);
}
// Values c .. c + 7 of row m into the rows of shared memory from `at` on, one for each of its parts.
template <int KIND>
__device__ __forceinline__ void fill8(const Params& p, uint8_t* at, int m, int c) {
  uint32_t w[4] = {0, 0, 0, 0};
  if (KIND == CUCA_BF16) {
    if (m < p.m) {
      const __nv_bfloat16* src = (const __nv_bfloat16*)p.a + m * p.lda + c;
      if (p.wide && c + 8 <= p.k) {
        const uint4 q = __ldcg(reinterpret_cast<const uint4*>(src));
        w[0] = q.x; w[1] = q.y; w[2] = q.z; w[3] = q.w;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (c + j < p.k) w[j >> 1] |= (uint32_t)__ldcg(reinterpret_cast<const unsigned short*>(src) + j) << (16 * (j & 1));
      }
    }
    *reinterpret_cast<uint4*>(at) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 0.f;
    if (m < p.m) {
      const float* src = (const float*)p.a + m * p.lda + c;
      if (p.wide && c + 8 <= p.k) {
        const float4 f = __ldcg(reinterpret_cast<const float4*>(src)), g = __ldcg(reinterpret_cast<const float4*>(src) + 1);
        v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w; v[4] = g.x; v[5] = g.y; v[6] = g.z; v[7] = g.w;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (c + j < p.k) v[j] = __ldcg(src + j);
      }
    }
#pragma unroll
    for (int part = 0; part < 3; ++part) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        w[j] = pack2(v[2 * j], v[2 * j + 1]);
        v[2 * j] -= __uint_as_float(w[j] << 16);
        v[2 * j + 1] -= __uint_as_float(w[j] & 0xffff0000u);
      }
      *reinterpret_cast<uint4*>(at + part * A_STRIDE) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

struct Codes {
  uint4 w[GROUPS];
  uint32_t s[GROUPS];
};

// RUNS of eight rows of shared memory: so many rows of bfloat16, or a third of 32 bits
template <int KIND, int RUNS>
__global__ void __launch_bounds__(THREADS, 2) gemm_mx4_rows_kernel(const Params p) {
  extern __shared__ __align__(16) uint8_t smem[];
  constexpr int PARTS = KIND == CUCA_F32 ? 3 : 1;
  constexpr int TOKENS = 8 * RUNS / PARTS;  // rows of X that a block takes
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int set = warp >> 2;
  const int rank = p.share > 1 ? (int)mx4_cluster_rank() : 0;
  const int tile = (int)blockIdx.x / p.share;
  const bool dual = p.epilogue == EPI_SWIGLU;
  const int m0 = (int)blockIdx.y * TOKENS;
  const int m_here = min(TOKENS, p.m - m0);
  // weight row of place v of the tile: 128 rows, or 64 of the gate and 64 of the up part
  auto weight_row = [&](int v) {
    if (!dual) return min(tile * TILE + v, p.n - 1);
    return v < TILE / 2 ? min(tile * (TILE / 2) + v, p.n - 1) : p.n + min(tile * (TILE / 2) + v - TILE / 2, p.n - 1);
  };
  const int s0 = (int)((int64_t)p.steps * rank / p.share), s1 = (int)((int64_t)p.steps * (rank + 1) / p.share);
  const uint8_t* w_at[GROUPS];  // of the next step to be fetched
  const uint8_t* s_at[GROUPS];
#pragma unroll
  for (int j = 0; j < GROUPS; ++j) {
    const int r = weight_row((warp & 3) * 32 + j * 8 + g);
    w_at[j] = p.w + (r * (int64_t)p.steps + s0 + set) * 64 + q * 16;
    s_at[j] = p.w_scales + mx4_scale_at(r, s0 + set, p.steps) + q;
  }
  pdl_trigger();
  // what the first steps read, into L2: that needs no wait for the kernel before, whatever it writes
  if (s0 + set < s1) {
#pragma unroll
    for (int j = 0; j < GROUPS; ++j) asm volatile("prefetch.global.L2 [%0];" ::"l"(w_at[j]));
  }
  pdl_wait();

  auto fetch = [&](Codes& c) {
#pragma unroll
    for (int j = 0; j < GROUPS; ++j) {
      c.w[j] = __ldcg(reinterpret_cast<const uint4*>(w_at[j]));
      c.s[j] = __ldcg(s_at[j]);
      w_at[j] += 2 * 64;
      s_at[j] += 2 * 512;
    }
  };
  float acc[GROUPS / 2][RUNS][4];
#pragma unroll
  for (int j = 0; j < GROUPS / 2; ++j)
#pragma unroll
    for (int r = 0; r < RUNS; ++r)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[j][r][i] = 0.f;
  // a step's products: the matrix instruction cuts off what its sum has no bits for, so sums of 128 products meet the others with rounding
  auto multiply = [&](const Codes& c, const uint8_t* x) {
    float part[GROUPS / 2][RUNS][4];
#pragma unroll
    for (int j = 0; j < GROUPS / 2; ++j)
#pragma unroll
      for (int r = 0; r < RUNS; ++r)
#pragma unroll
        for (int i = 0; i < 4; ++i) part[j][r][i] = 0.f;
    auto step = [&](auto large) {
      constexpr bool LARGE = decltype(large)::value;
      Mx4Factor f[GROUPS];
#pragma unroll
      for (int j = 0; j < GROUPS; ++j) f[j] = mx4_factor<LARGE>(c.s[j]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint4 b[RUNS];
#pragma unroll
        for (int r = 0; r < RUNS; ++r) b[r] = *reinterpret_cast<const uint4*>(x + r * 8 * A_STRIDE + i * 64);
#pragma unroll
        for (int j = 0; j < GROUPS / 2; ++j) {
          uint32_t lo[4], hi[4];  // weight rows g and g + 8 of sixteen
          mx4_to_bf16<LARGE>((&c.w[2 * j].x)[i], f[2 * j], lo);
          mx4_to_bf16<LARGE>((&c.w[2 * j + 1].x)[i], f[2 * j + 1], hi);
#pragma unroll
          for (int r = 0; r < RUNS; ++r) {
            mma(part[j][r], lo[0], hi[0], lo[1], hi[1], b[r].x, b[r].y);
            mma(part[j][r], lo[2], hi[2], lo[3], hi[3], b[r].z, b[r].w);
          }
        }
      }
    };
    if (__any_sync(0xffffffffu, (c.s[0] | c.s[1] | c.s[2] | c.s[3]) & 128)) step(std::true_type{});
    else step(std::false_type{});
#pragma unroll
    for (int j = 0; j < GROUPS / 2; ++j)
#pragma unroll
      for (int r = 0; r < RUNS; ++r)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[j][r][i] += part[j][r][i];
  };

  Codes even, odd;
  int s = s0 + set;
  if (s < s1) fetch(even);
  for (int k0 = s0; k0 < s1; k0 += KEPT) {
    const int kept = min(KEPT, s1 - k0);
    if (k0 > s0) __syncthreads();
    // A thread has a run of eight values of every row. (Of 32-bit rows' parts the last places may stay as they are: their sums are not
    // read.) A lane's blocks lie in four places 64 bytes apart: four lanes next to each other read 64 bytes.
    static_assert(KEPT * 16 == THREADS, "a run of eight values for each thread");
    if ((int)threadIdx.x < kept * 16) {
      const int step = threadIdx.x >> 4, run = threadIdx.x & 15;
      uint8_t* at = smem + step * (MX4_STEP * 2) + ((run >> 2) | (run & 3) << 2) * 16;
#pragma unroll 4
      for (int t = 0; t < TOKENS; ++t)
        fill8<KIND>(p, at + t * PARTS * A_STRIDE, t < m_here ? m0 + t : p.m, (k0 + step) * MX4_STEP + run * 8);
    }
    __syncthreads();
    const uint8_t* x = smem + g * A_STRIDE + (s - k0) * (MX4_STEP * 2) + q * 16;
    // (KEPT is a multiple of four: of a set's steps in it, all but the last call's are an even number)
    for (; s < k0 + kept; s += 4, x += 4 * MX4_STEP * 2) {
      if (s + 2 < s1) fetch(odd);
      multiply(even, x);
      if (s + 4 < s1) fetch(even);
      if (s + 2 < k0 + kept) multiply(odd, x + 2 * MX4_STEP * 2);
    }
  }

  // the two sets' sums, [set][row][weight row], where A lay
  __syncthreads();
  float* sums = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int j = 0; j < GROUPS / 2; ++j)
#pragma unroll
    for (int r = 0; r < RUNS; ++r) {
      float* at = sums + (set * ROWS + r * 8 + q * 2) * SUM_STRIDE + (warp & 3) * 32 + j * 16 + g;
      at[0] = acc[j][r][0];
      at[SUM_STRIDE] = acc[j][r][1];
      at[8] = acc[j][r][2];
      at[SUM_STRIDE + 8] = acc[j][r][3];
    }
  __syncthreads();
  if (p.share > 1) mx4_cluster_sync();
  const int cols = dual ? TILE / 2 : TILE;  // output columns of a tile; this block finishes `mine` of them
  const int mine = cols / p.share, c0 = rank * mine;
  auto total = [&](int row, int v) {
    float y = 0.f;
    for (int part = PARTS - 1; part >= 0; --part) {  // (small parts first)
      const float* at = sums + (row + part) * SUM_STRIDE + v;
      for (int r = 0; r < p.share; ++r) {
        if (p.share > 1) y += mx4_peer_f32(at, r), y += mx4_peer_f32(at + ROWS * SUM_STRIDE, r);
        else y += at[0], y += at[ROWS * SUM_STRIDE];
      }
    }
    return y;
  };
  for (int i = threadIdx.x; i < m_here * mine; i += THREADS) {
    const int t = i / mine, v = c0 + i - t * mine, n = tile * cols + v;
    if (n >= p.n) continue;
    float y = total(t * PARTS, v);
    const int64_t o = (m0 + t) * p.ldo + n;
    if (dual) {
      const float u = total(t * PARTS, v + TILE / 2);
      y = KIND == CUCA_F32 ? y / (1.f + expf(-y)) * u : __fdividef(y, 1.f + __expf(-y)) * u;
    } else if (p.bias) {
      y += KIND == CUCA_F32 ? ((const float*)p.bias)[n] : __bfloat162float(((const __nv_bfloat16*)p.bias)[n]);
    }
    if (p.epilogue == EPI_RESIDUAL) ((float*)p.out)[o] += y;
    else if (p.out_f32) ((float*)p.out)[o] = y;
    else ((__nv_bfloat16*)p.out)[o] = __float2bfloat16_rn(y);
  }
  if (p.share > 1) mx4_cluster_sync();  // until nobody reads these sums any more
}

template <int KIND, int RUNS>
int launch(const CucaMx4Gemm* c) {
  const int64_t elem = KIND == CUCA_F32 ? 4 : 2;
  Params p{c->a, c->lda, c->w, c->w_scales, c->bias, c->out, c->ldo, (int)c->m, (int)c->n, (int)c->k, (int)mx4_steps(c->k),
           (int)c->out_f32, (int)c->epilogue, 1, ((uintptr_t)c->a & 15) == 0 && (c->m == 1 || c->lda * elem % 16 == 0)};
  const int cols = p.epilogue == EPI_SWIGLU ? TILE / 2 : TILE, tokens = 8 * RUNS / (KIND == CUCA_F32 ? 3 : 1);
  const int tiles = (p.n + cols - 1) / cols, groups = (p.m + tokens - 1) / tokens;
  CUCA_REQUIRE(groups <= 65535 && (int64_t)tiles * MAX_CLUSTER < (1ll << 31), "gemm_mx4: %d rows by %d features are too many", p.m, p.n);
  // shares of K until two blocks an SM have work, of two steps at least (one for each set of warps)
  while (p.share < MAX_CLUSTER && (int64_t)tiles * groups * p.share < 2 * cuca_device_sms() && p.steps >= p.share * 4) p.share *= 2;
  constexpr auto kernel = gemm_mx4_rows_kernel<KIND, RUNS>;
  if (int e = mx4_configure<kernel>(SMEM)) return e;
  const dim3 grid(tiles * p.share, groups);
  if (p.share > 1) cuca_launch_cluster(kernel, grid, dim3(THREADS), SMEM, c->stream, true, p.share, p);
  else cuca_launch(kernel, grid, dim3(THREADS), SMEM, c->stream, true, p);
  CUCA_CHECK_LAUNCH("gemm_mx4");
  return 0;
}

}  // namespace

int cuca_gemm_mx4_rows(const CucaMx4Gemm* c) {
  if (c->a_kind == CUCA_F32) return c->m <= 2 ? launch<CUCA_F32, 1>(c) : launch<CUCA_F32, 2>(c);
  return c->m <= 8 ? launch<CUCA_BF16, 1>(c) : launch<CUCA_BF16, 2>(c);
}
