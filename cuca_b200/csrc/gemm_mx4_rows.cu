// Few rows times a weight in 4 bits: out = epilogue(A W^T), A of 16 or 32 bits or in 4 bits itself, W as mx4.cuh lays it out.
//
// Bound by the weight's bytes, 17 bits for 32 values, and by the instructions that make bfloat16 numbers of codes (17 for eight codes:
// see mx4_to_bf16). Codes times their power of two are bfloat16 numbers exactly, so a product with a bfloat16 row is exact and is
// summed in 32 bits. A 32-bit value is the sum of three bfloat16 parts (exact from 2^-110 on), three rows of one product, whose sums
// are added at the end; so it is with a row in 4 bits, of one part.
//
// A block has eight warps: four take 32 weight rows each of a tile of 128, and two sets of four take the steps of 128 values in turn.
// A lane's 16 bytes are one block of 32 codes of one weight row, so a warp reads 64 bytes of 32 rows at a time and every lane has one
// scale per row. Few tiles: a cluster of up to eight blocks shares K, and adds its sums in order out of each other's shared memory: no workspace, and
// equal bits in every run.
#include "mx4_mma.cuh"
#include <type_traits>

namespace {

constexpr int WARPS = 8, THREADS = 32 * WARPS;
constexpr int ROWS = 16;       // of A, as the matrix instruction takes them
constexpr int TILE = 128;      // weight rows of a block
constexpr int GROUPS = 4;      // of eight weight rows a warp
constexpr int KEPT = 16;       // steps of A in shared memory at a time
constexpr int A_STRIDE = KEPT * MX4_STEP * 2 + 64;  // bytes: rows next to each other lie 16 banks apart
constexpr int SUM_STRIDE = TILE + 4;
constexpr int MAX_CLUSTER = 8;
constexpr int SMEM = ROWS * A_STRIDE;
static_assert(ROWS * SUM_STRIDE * 4 * 2 <= SMEM, "two sets' sums lie where A lay");

struct Params {
  const void* a;
  const uint8_t* a_scales;
  int64_t lda;
  const uint8_t* w;
  const uint8_t* w_scales;
  const void* bias;
  void* out;
  int64_t ldo;
  int m, n, k, steps;
  int out_f32, epilogue;
  int share;  // blocks of a cluster
};

__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const __nv_bfloat162 t = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&t);
}
// Values c .. c + 7 of row m into the rows of shared memory that belong to it, one for each of its parts.
template <int KIND>
__device__ __forceinline__ void fill8(const Params& p, uint8_t* smem, int row, int m, int c, int at) {
  uint32_t w[4] = {0, 0, 0, 0};
  if (KIND == MX4_CODES) {
    uint4 q = make_uint4(0, 0, 0, 0);
    if (m < p.m) {
      const uint32_t word = __ldcg(reinterpret_cast<const uint32_t*>((const uint8_t*)p.a + m * (p.steps * 64ll) + c / 2));
      const uint32_t byte = __ldcg(p.a_scales + mx4_scale_at(m, c >> 7, p.steps) + ((c >> 5) & 3));
      uint32_t r[4];
      mx4_to_bf16<true>(word, mx4_factor(byte), r);
      q = make_uint4(r[0], r[1], r[2], r[3]);
    }
    *reinterpret_cast<uint4*>(smem + row * A_STRIDE + at) = q;
  } else if (KIND == CUCA_BF16) {
    if (m < p.m) {
      const __nv_bfloat16* src = (const __nv_bfloat16*)p.a + m * p.lda + c;
      if (c + 8 <= p.k && ((uintptr_t)src & 15) == 0) {
        const uint4 q = __ldcg(reinterpret_cast<const uint4*>(src));
        w[0] = q.x; w[1] = q.y; w[2] = q.z; w[3] = q.w;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (c + j < p.k) w[j >> 1] |= (uint32_t)__ldcg(reinterpret_cast<const unsigned short*>(src) + j) << (16 * (j & 1));
      }
    }
    *reinterpret_cast<uint4*>(smem + row * A_STRIDE + at) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 0.f;
    if (m < p.m) {
      const float* src = (const float*)p.a + m * p.lda + c;
      if (c + 8 <= p.k && ((uintptr_t)src & 15) == 0) {
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
      *reinterpret_cast<uint4*>(smem + (row + part) * A_STRIDE + at) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

struct Codes {
  uint4 w[GROUPS];
  uint32_t s[GROUPS];
};

template <int KIND>
__global__ void __launch_bounds__(THREADS, 2) gemm_mx4_rows_kernel(const Params p) {
  extern __shared__ __align__(16) uint8_t smem[];
  constexpr int PARTS = KIND == CUCA_F32 ? 3 : 1;
  constexpr int TOKENS = ROWS / PARTS;  // rows of A that a block takes
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
  const int64_t row_bytes = p.steps * 64ll;
  const uint8_t* w_at[GROUPS];
  const uint8_t* s_at[GROUPS];
#pragma unroll
  for (int j = 0; j < GROUPS; ++j) {
    const int r = weight_row((warp & 3) * 32 + j * 8 + g);
    w_at[j] = p.w + r * row_bytes + q * 16;
    s_at[j] = p.w_scales + mx4_scale_at(r, 0, p.steps) + q;
  }
  pdl_trigger();
  // what the first steps read, into L2: that needs no wait for the kernel before, whatever it writes
  if (s0 + set < s1) {
#pragma unroll
    for (int j = 0; j < GROUPS; ++j) asm volatile("prefetch.global.L2 [%0];" ::"l"(w_at[j] + (s0 + set) * 64ll));
  }
  pdl_wait();

  auto fetch = [&](Codes& c, int s) {
#pragma unroll
    for (int j = 0; j < GROUPS; ++j) {
      c.w[j] = __ldcg(reinterpret_cast<const uint4*>(w_at[j] + s * 64ll));
      c.s[j] = __ldcg(s_at[j] + s * 512ll);
    }
  };
  float acc[GROUPS][4];
#pragma unroll
  for (int j = 0; j < GROUPS; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[j][i] = 0.f;

  Codes now, next;
  int s = s0 + set;
  if (s < s1) fetch(now, s);
  for (int k0 = s0; k0 < s1; k0 += KEPT) {
    const int kept = min(KEPT, s1 - k0);
    if (k0 > s0) __syncthreads();
    // (an odd 32-bit row of the sixteen stays as it is: its sums are not read)
    for (int i = threadIdx.x; i < TOKENS * kept * 16; i += THREADS) {
      const int t = i / (kept * 16), c = i - t * (kept * 16);  // token, run of eight values
      const int step = c >> 4, run = c & 15;
      // a lane's blocks lie in four places 64 bytes apart: four lanes next to each other read 64 bytes
      fill8<KIND>(p, smem, t * PARTS, t < m_here ? m0 + t : p.m, (k0 + step) * MX4_STEP + run * 8,
                  step * (MX4_STEP * 2) + ((run >> 2) | (run & 3) << 2) * 16);
    }
    __syncthreads();
    for (; s < k0 + kept; s += 2) {
      if (s + 2 < s1) fetch(next, s + 2);
      Mx4Factor f[GROUPS];
      bool large = false;
#pragma unroll
      for (int j = 0; j < GROUPS; ++j) {
        f[j] = mx4_factor(now.s[j]);
        large |= now.s[j] > 128 && now.s[j] < 255;
      }
      float part[GROUPS][4];
#pragma unroll
      for (int j = 0; j < GROUPS; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) part[j][i] = 0.f;
      const uint8_t* row = smem + g * A_STRIDE + (s - k0) * (MX4_STEP * 2) + q * 16;
      auto step = [&](auto is_large) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint4 x = *reinterpret_cast<const uint4*>(row + i * 64);
          const uint4 y = *reinterpret_cast<const uint4*>(row + 8 * A_STRIDE + i * 64);
          const uint32_t a0[4] = {x.x, y.x, x.y, y.y}, a1[4] = {x.z, y.z, x.w, y.w};
#pragma unroll
          for (int j = 0; j < GROUPS; ++j) {
            const uint32_t words[4] = {now.w[j].x, now.w[j].y, now.w[j].z, now.w[j].w};
            uint32_t b[4];
            mx4_to_bf16<decltype(is_large)::value>(words[i], f[j], b);
            mma(part[j], a0, b[0], b[1]);
            mma(part[j], a1, b[2], b[3]);
          }
        }
      };
      if (__any_sync(0xffffffffu, large)) step(std::true_type{});
      else step(std::false_type{});
      // the matrix instruction cuts off what its sum has no bits for: sums of 128 products meet the others with rounding
#pragma unroll
      for (int j = 0; j < GROUPS; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[j][i] += part[j][i];
      now = next;
    }
  }

  // the two sets' sums, [set][row][weight row], where A lay
  __syncthreads();
  float* sums = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int j = 0; j < GROUPS; ++j) {
    float* at = sums + (set * ROWS + g) * SUM_STRIDE + (warp & 3) * 32 + j * 8 + q * 2;
    *reinterpret_cast<float2*>(at) = make_float2(acc[j][0], acc[j][1]);
    *reinterpret_cast<float2*>(at + 8 * SUM_STRIDE) = make_float2(acc[j][2], acc[j][3]);
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

template <int KIND>
int launch(const CucaMx4Gemm* c) {
  Params p{c->a, c->a_scales, c->lda, c->w, c->w_scales, c->bias, c->out, c->ldo, (int)c->m, (int)c->n, (int)c->k,
           (int)mx4_steps(c->k), (int)c->out_f32, (int)c->epilogue, 1};
  const int cols = p.epilogue == EPI_SWIGLU ? TILE / 2 : TILE, tokens = KIND == CUCA_F32 ? ROWS / 3 : ROWS;
  const int tiles = (p.n + cols - 1) / cols, groups = (p.m + tokens - 1) / tokens;
  CUCA_REQUIRE(groups <= 65535 && (int64_t)tiles * MAX_CLUSTER < (1ll << 31), "gemm_mx4: %d rows by %d features are too many", p.m, p.n);
  // shares of K until two blocks an SM have work, of two steps at least (one for each set of warps)
  while (p.share < MAX_CLUSTER && (int64_t)tiles * groups * p.share < 2 * cuca_device_sms() && p.steps >= p.share * 4) p.share *= 2;
  auto kernel = gemm_mx4_rows_kernel<KIND>;
  if (int e = mx4_configure<gemm_mx4_rows_kernel<KIND>>(SMEM)) return e;
  const dim3 grid(tiles * p.share, groups);
  if (p.share > 1) cuca_launch_cluster(kernel, grid, dim3(THREADS), SMEM, c->stream, true, p.share, p);
  else cuca_launch(kernel, grid, dim3(THREADS), SMEM, c->stream, true, p);
  CUCA_CHECK_LAUNCH("gemm_mx4");
  return 0;
}

}  // namespace

int cuca_gemm_mx4_rows(const CucaMx4Gemm* c) {
  return c->a_kind == MX4_CODES ? launch<MX4_CODES>(c) : c->a_kind == CUCA_F32 ? launch<CUCA_F32>(c) : launch<CUCA_BF16>(c);
}
