// What the tensor-core products with 4-bit weights share: block-scaled contractions, clusters, results.
#pragma once
#include "mx4.cuh"
#include "tcgen05.cuh"

namespace {

__device__ __forceinline__ uint32_t mx4_cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// (.aligned: a warp's lanes come here together, whatever they did before)
__device__ __forceinline__ void mx4_cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float2 mx4_peer_f32x2(uint32_t at) {  // an address that mapa made
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void mx4_prefetch_2d(const CUtensorMap* map, int c0, int c1) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(map), "r"(c0), "r"(c1) : "memory");
}
// After a wait gave up: copies in flight land before the shared memory is handed on.
__device__ __forceinline__ void mx4_let_copies_land() {
  const unsigned long long t0 = global_ns();
  while (global_ns() - t0 < 2000000ull) { }
}

// A place in a ring of n, and the parity of the phase that is being filled (a remainder costs some 100 clocks a turn). Those who
// wait for a place to be full wait for `parity`, those who wait for it to be free for its opposite, which a new barrier grants.
struct Mx4Ring {
  int at;
  uint32_t parity;
  __device__ Mx4Ring() : at(0), parity(0) {}
  __device__ void next(int n, int by = 1) {
    at += by;
    if (at >= n) { at -= n; parity ^= 1; }
  }
};

// ---- kind::mxf4: both operands e2m1, a power of two for 32 values
// M rows by n columns, both K-major.
__host__ __device__ constexpr uint32_t mx4_instr_desc(int n, int m) {
  return (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | ((uint32_t)(m >> 4) << 24);
}
// which two of a column's four bytes the 64 values of an instruction go by, in both operands
__host__ __device__ constexpr uint32_t mx4_scale_half(int half) { return half ? (2u << 4) | (2u << 29) : 0u; }
__device__ __forceinline__ void mx4_umma(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t scale_a, uint32_t scale_b,
                                         uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %6, 0;\n"
      "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}\n"
      ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(scale_a), "r"(scale_b), "r"(accumulate) : "memory");
}
// 512 bytes of scales: 32 rows of 16 bytes, eight rows to 128 bytes, not swizzled
__device__ __forceinline__ uint64_t mx4_scale_desc(uint32_t addr) {
  uint64_t d = 0;
  d |= (uint64_t)((addr & 0x3FFFFu) >> 4);
  d |= (uint64_t)(128 >> 4) << 32;  // between groups of eight rows
  d |= (uint64_t)1 << 46;
  return d;
}
// ... into four columns of tensor memory, the same in each quarter of the lanes
__device__ __forceinline__ void mx4_scales_to_tmem(uint32_t col, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(col), "l"(desc) : "memory");
}

// ---- results
struct Mx4Out {
  void* out;
  const void* bias;  // 32-bit where `bias_f32`, else bfloat16
  int64_t ldo;
  int m, n, out_f32, epilogue, bias_f32;
};
// silu(g) u. For 32-bit results g / (1 + e^-|g|) u, times e^-|g| where g is negative, so that no exponential is past the range: good to 2^-21
// down to where e^-|g| lies under 2^-126 and has fewer bits of its own. For bfloat16 results the approximate reciprocal and exponential:
// good to 2^-20 and |g| 2^-23 more, which the rounded product in the exponent costs (2^-16 at -100); below -87.3, where silu lies under
// 2^-119, they give zero. (The other form for these too: 2,048 gated rows in 4 bits of 4096 x 14336 took 125 us, 115.)
__device__ __forceinline__ float mx4_gate(bool exact, float g, float u) {
  if (exact) {
    const float z = expf(-fabsf(g));
    return (g < 0.f ? g * z : g) / (1.f + z) * u;
  }
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + fast_exp2(-1.4426950408889634f * g)));
  return g * r * u;
}
// Where a feature's results go, one row of A after the other. What does not change from row to row is settled once: with the checks at
// each result a tile's results took longer than its products (14 us of 26 for 192 x 256).
struct Mx4Column {
  char* at;
  int64_t step;  // bytes from row to row
  float bias;
  bool f32, add;
  __device__ Mx4Column(const Mx4Out& o, int m, int n) {
    const int size = o.out_f32 ? 4 : 2;
    at = (char*)o.out + (m * o.ldo + n) * size;
    step = o.ldo * size;
    bias = !o.bias ? 0.f : o.bias_f32 ? mx4_read((const float*)o.bias + n) : mx4_read((const __nv_bfloat16*)o.bias + n);
    f32 = o.out_f32;
    add = o.epilogue == EPI_RESIDUAL;
  }
  // (an atomic takes and leaves numbers below 2^-126 as zeros)
  __device__ void put(float y) const {
    y += bias;
    if (!f32) *(__nv_bfloat16*)at = __float2bfloat16_rn(y);
    else if (add) atomicAdd((float*)at, y);  // one thread owns the place: its result is not waited for, as that of a load would be
    else *(float*)at = y;
  }
  __device__ void put2(float y, float z) const {  // z: of the next feature, its bias added; for places on two results' size
    y += bias;
    if (!f32) {
      *(__nv_bfloat162*)at = __floats2bfloat162_rn(y, z);
    } else {
      if (add) {
        atomicAdd((float*)at, y);
        atomicAdd((float*)at + 1, z);
        return;
      }
      *(float2*)at = make_float2(y, z);
    }
  }
};

__device__ __forceinline__ void mx4_ask16(uint32_t at, uint32_t (&r)[16]) {  // to be waited for
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(at) : "memory");
}
// Results out of sixteens of columns: G columns are one row of A (its digits or parts, the smallest first), added up as they come.
template <int G>
struct Mx4Group {
  static constexpr int LOADS = G == 1 ? 1 : 3, ROWS = LOADS * 16 / G;  // what whole rows take
};
template <int G, int LOAD>
__device__ __forceinline__ void mx4_sum16(const uint32_t (&r)[16], float (&y)[Mx4Group<G>::ROWS]) {
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const int c = LOAD * 16 + j;
    y[c / G] = c % G ? y[c / G] + __uint_as_float(r[j]) : __uint_as_float(r[j]);
  }
}
// `rows`: how many there are to have
template <int G, int LOAD = 0>
__device__ __forceinline__ void mx4_rows_of(uint32_t at, int rows, float (&y)[Mx4Group<G>::ROWS]) {
  if constexpr (LOAD < Mx4Group<G>::LOADS) {
    if (LOAD == 0 || LOAD * 16 < rows * G) {
      uint32_t r[16];
      mx4_ask16(at + LOAD * 16, r);
      tmem_ld_wait();
      mx4_sum16<G, LOAD>(r, y);
      mx4_rows_of<G, LOAD + 1>(at, rows, y);
    }
  }
}
// What the digits of a row left in steps s0..s1, times a weight row: sixteen codes' words a step, products exact, added up in 32 bits. Seldom
// there is any: not fast (8 rows of 4096 x 14336 gated of which every block leaves something 2.1 ms; all of a block's codes asked for at once 0.7,
// but then the rows that leave nothing pay for the registers: 2 % of a model's step).
struct Mx4RestOf {
  Mx4Rest rest;
  const uint8_t* w;
  const uint8_t* w_scales;
  int steps, s0, s1;
  bool any;
};
__device__ __noinline__ float mx4_rest_product(const Mx4RestOf r, int row, int n) {
  float y = 0.f;
  for (int s = r.s0; s < r.s1; ++s) {
    const int64_t step = (int64_t)row * r.steps + s;
    if (!__ldcg(r.rest.flags + step)) continue;
    const uint4* x = reinterpret_cast<const uint4*>(r.rest.values + step * MX4_STEP);
    const uint32_t* w = reinterpret_cast<const uint32_t*>(r.w + ((int64_t)n * r.steps + s) * 64);
    const uint32_t bytes = __ldcg(reinterpret_cast<const uint32_t*>(r.w_scales + mx4_scale_at(n, s, r.steps)));
    for (int i = 0; i < 16; ++i) {
      const uint4 q = __ldcg(x + i);
      if (!(q.x | q.y | q.z | q.w)) continue;
      const uint32_t v[4] = {q.x, q.y, q.z, q.w};
      uint32_t c[4];
      mx4_to_bf16<true>(__ldcg(w + i), mx4_factor<true>(bytes >> (i >> 2) * 8 & 255), c);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        y = fmaf(__uint_as_float(v[j] << 16), __uint_as_float(c[j] << 16), y);
        y = fmaf(__uint_as_float(v[j] & 0xffff0000u), __uint_as_float(c[j] & 0xffff0000u), y);
      }
    }
  }
  return y;
}
// A finished tile: lane `row` (0..127) of tensor memory holds weight row `row` of the tile, G columns `at`.. each of the m_here rows of A
// from m0 on. Alone they are results, features from n0 on; else they go to shared memory, [row of A][128], for mx4_join (`again`: are added
// to what this thread left there). GATED: the up part's accumulator lies `apart` columns further on, in shared memory `up` rows. `rest`: of digits, what they left of these rows.
template <int G, bool GATED>
__device__ __forceinline__ void mx4_leave(const Mx4Out& o, uint32_t at, int m0, int m_here, int n0, int row, bool alone, float* sums,
                                          bool again = false, int apart = 0, int up = 0, const Mx4RestOf& rest = {}) {
  constexpr int N = Mx4Group<G>::ROWS;
  const bool live = n0 + row < o.n;
  Mx4Column out(o, m0, live ? n0 + row : 0);
  for (int c = 0; c < m_here; c += N) {
    float v[N], u[N];
    if constexpr (Mx4Group<G>::LOADS == 1) {
      uint32_t r[16], q[16];
      mx4_ask16(at + c * G, r);
      if (GATED) mx4_ask16(at + apart + c * G, q);
      tmem_ld_wait();
      mx4_sum16<G, 0>(r, v);
      if (GATED) mx4_sum16<G, 0>(q, u);
    } else {
      mx4_rows_of<G>(at + c * G, m_here - c, v);
      if (GATED) mx4_rows_of<G>(at + apart + c * G, m_here - c, u);
    }
    if constexpr (G == MX4_DIGITS) {
      if (rest.any && live) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
          if (c + j < m_here) {
            v[j] += mx4_rest_product(rest, m0 + c + j, n0 + row);
            if (GATED) u[j] += mx4_rest_product(rest, m0 + c + j, o.n + n0 + row);
          }
        }
      }
    }
    if (!alone) {
      float* const sum = sums + c * TILE_A + row;
      if (again) {
#pragma unroll
        for (int j = 0; j < N; ++j)
          if (G == 1 || c + j < m_here) v[j] += sum[j * TILE_A];
      }
#pragma unroll
      for (int j = 0; j < N; ++j) {
        if (G == 1 || c + j < m_here) {  // (where each column is a row there is room for whole sixteens of them)
          sum[j * TILE_A] = v[j];
          if (GATED) sum[(up + j) * TILE_A] = u[j];
        }
      }
    } else if (live) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        if (c + j < m_here) out.put(GATED ? mx4_gate(out.f32, v[j], u[j]) : v[j]);
        out.at += out.step;
      }
    }
    __syncwarp();  // what is asked of tensor memory next is asked by all lanes together
  }
}
// The sums that the blocks of a cluster left, added up in order, each block for its part of the features; a block alone finishes its own.
// All threads of all blocks of the cluster come here. HALVES: weight rows 64.. of the tile are the up part of rows 0..63; with `up` the
// up part stands so many rows of A further on.
template <bool HALVES>
__device__ __forceinline__ void mx4_join(const Mx4Out& o, const float* sums, int m0, int m_here, int n0, int rank, int share, bool ok, int up = 0) {
  constexpr int THREADS = 256, MOST = 8;
  if (share > 1) mx4_cluster_sync();
  // a thread has two features, and rows of A in turn with the other threads that have them
  const int mine = (HALVES ? TILE_A / 2 : TILE_A) / share, shift = 30 - __clz(mine);
  const int row = rank * mine + 2 * (threadIdx.x & (mine / 2 - 1)), turn = THREADS >> shift;
  const int second = HALVES ? TILE_A / 2 : up * TILE_A;
  int c = threadIdx.x >> shift;
  if (ok && threadIdx.x < THREADS && n0 + row < o.n && c < m_here) {
    Mx4Column out(o, m0 + c, n0 + row), next(o, m0 + c, min(n0 + row + 1, o.n - 1));
    const bool both = n0 + row + 1 < o.n, wide = both && !(((uintptr_t)out.at | out.step) & (out.f32 ? 7 : 3));
    const uint32_t at = smem_u32(sums + c * TILE_A + row), apart = second * 4;
    uint32_t peer[MOST];
#pragma unroll
    for (int r = 0; r < MOST; ++r) {
      peer[r] = at;
      if (share > 1) asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer[r]) : "r"(at), "r"(r < share ? r : 0));
    }
    const float* here = sums + c * TILE_A + row;
    for (; c < m_here; c += turn) {
      float2 v = make_float2(0.f, 0.f), u = v;
      if (share == 1) {
        v = *reinterpret_cast<const float2*>(here);
        if (second) u = *reinterpret_cast<const float2*>(here + second);
        here += turn * TILE_A;
      } else {
#pragma unroll
        for (int r = 0; r < MOST; ++r) {
          if (r < share) {
            const float2 a = mx4_peer_f32x2(peer[r]);
            v.x += a.x;
            v.y += a.y;
            if (second) {
              const float2 b = mx4_peer_f32x2(peer[r] + apart);
              u.x += b.x;
              u.y += b.y;
            }
            peer[r] += turn * TILE_A * 4;
          }
        }
      }
      if (second) v = make_float2(mx4_gate(out.f32, v.x, u.x), mx4_gate(out.f32, v.y, u.y));
      if (wide) {
        out.put2(v.x, v.y + next.bias);
      } else {
        out.put(v.x);
        if (both) next.put(v.y);
      }
      out.at += turn * out.step;
      next.at += turn * out.step;
    }
  }
  if (share > 1) mx4_cluster_sync();  // until nobody reads these sums any more
}

}  // namespace
