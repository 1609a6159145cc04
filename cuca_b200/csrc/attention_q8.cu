// Causal grouped-query attention over 8-bit pages for few query rows: single tokens and short portions; and portions that
// attention_q8_tc.cu does not take (heads beyond 128, 32-bit rows with a score cap or a distance bias).
// (Scales, weights and their exactness: attention_q8.cuh.)
//
// Both products run turned round on mma.sync.m16n8k16 (16-bit floats, 32-bit sums): the 16 rows are keys (then dimensions of
// the values), the 8 columns are query rows, i.e. (token, head) pairs of one key head; S^T = K Q^T, O^T = V^T W^T. So a key
// head's few query rows fill half an instruction instead of a quarter, and in 32-bit mode a row's two 16-bit parts are simply
// two neighbouring columns: the same instructions serve both types.
//
// A block (4 warps) takes one tile of rows, one key head and a share of the keys; its warps take the groups of 16 keys in
// turn, each through a ring of its own (16-byte asynchronous copies straight from the pages, no barrier in the loop), and are
// joined at the end; shares of a tile's keys are joined through distributed shared memory, their blocks being a cluster, where
// there are 2, 4 or 8 of them and all blocks are resident at once, else by a second small launch. A thread's values sit in shared memory so
// that it reads its fragments 16 bytes at a time without bank conflicts (`place`), and the order of dimensions and keys
// within an instruction is chosen to match: a contraction may be summed in any order.
//
// Decoding would be bound by the pages' bytes (16 keys of 128 are 4.2 KB, 183 clocks of an SM's share of memory) but for the
// instructions that turn codes into 16-bit floats: some 320 a warp and group, 176 of them conversion. Measured, 32 heads of 128 over 8,
// pages of 16: 64 requests of up to 8,192 positions 111 us (5.1 TB/s, 0.78 of a copy's rate; with nothing fetched 98), 8 of 1,152
// 12.7 us (latency: three groups a warp), one of 77 4.7 us; over bfloat16 pages 190, 12.9 and 6.9 us.
#include "attention_q8.cuh"
#include <type_traits>

namespace {

constexpr int GROUP = 16;     // keys of a step
constexpr int STAGES = 3;     // of a warp's ring (four, with three blocks an SM: 64 ragged requests 118 us, not 114; five 134)
constexpr int WARPS = 4;

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t turned_8x8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

// 16 bytes (none, and zeros: bytes 0) with constant offsets on both sides
template <int DST, int SRC>
__device__ __forceinline__ void copy16_at(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0+%2], [%1+%3], 16, %4;" ::"r"(dst), "l"(src), "n"(DST), "n"(SRC), "r"(bytes) : "memory");
}
template <int N, int I = 0, typename F>
__device__ __forceinline__ void for_each(F f) {  // f(0), .. f(N - 1), each a constant
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    for_each<N, I + 1>(f);
  }
}
// A barrier over every thread of the cluster, and loads from the shared memory of one of its blocks.
constexpr int MOST_CLUSTER = 8;
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_at(uint32_t at, int rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(at), "r"(rank));
  return r;
}
__device__ __forceinline__ float2 cluster_2(uint32_t at, int rank) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(cluster_at(at, rank)) : "memory");
  return v;
}
__device__ __forceinline__ float4 cluster_4(uint32_t at, int rank) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(cluster_at(at, rank)) : "memory");
  return v;
}

// DP: the head size rounded up to 64, 128 or 256 (what is beyond d stays zero).
template <int DP>
struct Ring {
  static constexpr int CHUNKS = DP / 16;                 // 16-byte pieces of a row
  static constexpr int TENSOR = GROUP * DP;              // bytes of a group's keys
  static constexpr int STAGE = 2 * TENSOR + 2 * GROUP * 4;  // keys, values, their scales
  static constexpr int WARP = STAGES * STAGE;
  // Where piece c of key k stands. A thread (g, t) of a warp reads keys g and g + 8 at pieces t, t + 4, .. and, for the values,
  // keys 2t, 2t + 1, 2t + 8, 2t + 9 at piece g (half a piece with DP = 64): the eight lanes that are served together must find
  // their pieces in eight different places of 128 bytes, for both.
  static __device__ __forceinline__ uint32_t place(int k, int c) {
    const int k0 = k & 1, k1 = (k >> 1) & 1, k2 = (k >> 2) & 1;
    if (DP == 64) return (uint32_t)(((k & ~1) | (k0 ^ k1)) * 64 + ((c ^ (k2 << 1)) * 16));
    return (uint32_t)(k * DP + ((c ^ (((k0 ^ k2) << 2) | (k1 << 1))) * 16));
  }
};

// NT: tiles of 8 columns. PARTS: 1: bfloat16 rows, a column each; 2: 32-bit rows, two columns each. OPT: score cap and
// distance bias.
template <int DP, int NT, int PARTS, bool OPT>
__global__ void __launch_bounds__(WARPS * 32)
attention_q8_kernel(const Q8Params p) {
  extern __shared__ __align__(16) uint8_t smem[];
  using R = Ring<DP>;
  using T = typename std::conditional<PARTS == 2, float, __nv_bfloat16>::type;
  constexpr int CHUNKS = R::CHUNKS;
  constexpr int QC = CHUNKS / 4;         // pieces of a key row that a thread reads
  constexpr int TILES = DP / 16;         // of 16 dimensions
  constexpr int COLS = NT * 8 / PARTS;   // query rows
  constexpr int LC = 2 / PARTS;          // of a thread and column tile
  constexpr bool Q_SHARED = NT * DP > 256;  // the queries' fragments do not fit the registers: they are read from shared memory
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  pdl_trigger();
  pdl_wait();

  // ---------------------------------------------------------------- rows, heads, keys
  int row0, n_tok;
  if (!q8_rows_of_tile(p, blockIdx.z, row0, n_tok)) return;
  const int kvh = blockIdx.y / p.head_parts, hp = blockIdx.y % p.head_parts;
  const int group_heads = p.nh / p.nkv;
  const int head0 = kvh * group_heads + hp * p.heads_per_cta;
  const int heads = min(p.heads_per_cta, group_heads - hp * p.heads_per_cta);
  const int seq = p.seq_of_row[row0];
  const int pos0 = p.positions[row0];
  const int n_cols = n_tok * heads;
  const bool nothing = seq < 0 || pos0 < 0;  // rows of no request
  if (nothing) {
    if (blockIdx.x == 0)
      for (int i = threadIdx.x; i < n_cols * p.d; i += WARPS * 32) {
        const int c = i / p.d;
        ((T*)p.out)[(size_t)(row0 + c / heads) * p.out_stride + (size_t)(head0 + c % heads) * p.d + i % p.d] = from_f32<T>(0.f);
      }
    return;
  }
  const Q8Keys keys = q8_keys<GROUP>(p, pos0, n_tok);
  const int share = p.chunk > 0 ? p.chunk / GROUP : keys.groups;
  const int first = blockIdx.x * share;
  const int last = (int)blockIdx.x == p.n_splits - 1 ? keys.groups : min(keys.groups, first + share);
  const bool alone = share >= keys.groups || p.n_splits == 1;
  const bool as_cluster = !alone && p.part == nullptr;  // the shares' blocks are a cluster
  if (first >= last) {  // a share that this tile does not have
    if (as_cluster) {
      cluster_sync();
      cluster_sync();
    }
    return;
  }
  const int* table = p.tables + (size_t)seq * p.table_stride;

  // ---------------------------------------------------------------- queries: the second operand's fragments
  // column c of tile j is query row (8 j + c) / PARTS: token (..) / heads, head (..) % heads
  uint8_t* my_ring = smem + warp * R::WARP;
  uint32_t* q_shared = reinterpret_cast<uint32_t*>(smem + WARPS * R::WARP);  // [TILES][NT][32 lanes][2]
  uint32_t qf[Q_SHARED ? 1 : TILES][Q_SHARED ? 1 : NT][2];
  float q_down[NT][LC];
  const bool q_aligned = ((uintptr_t)p.q & 15) == 0 && p.q_stride % (16 / (int)sizeof(T)) == 0;
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int col = (8 * j + g) / PARTS;
    const bool ok = col < n_cols;
    const T* src = (const T*)p.q + (size_t)(row0 + (ok ? col / heads : 0)) * p.q_stride + (size_t)(head0 + (ok ? col % heads : 0)) * p.d;
    float v[QC][16];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < QC; ++i) {
      const int e0 = (t + 4 * i) * 16;
      const bool mine = ok && e0 < p.d;
      if (q_aligned) {
        constexpr int N = 16 / sizeof(T);  // values of 16 bytes
#pragma unroll
        for (int n = 0; n < 16 / N; ++n) {
          const uint4 w = mine ? *reinterpret_cast<const uint4*>(src + e0 + n * N) : make_uint4(0u, 0u, 0u, 0u);
          const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (PARTS == 2) {
              v[i][n * N + e] = __uint_as_float(x[e]);
            } else {
              v[i][n * N + (2 * e) % N] = __uint_as_float(x[e] << 16);
              v[i][n * N + (2 * e + 1) % N] = __uint_as_float(x[e] & 0xffff0000u);
            }
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) v[i][e] = mine ? to_f32(src[e0 + e]) : 0.f;
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) top = max(top, __float_as_uint(v[i][e]) & 0x7fffffffu);
    }
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    float up, down;
    q8_query_scale(top, up, down);
#pragma unroll
    for (int c = 0; c < LC; ++c) q_down[j][c] = __shfl_sync(0xffffffffu, down, (2 * t + c) * 4);
#pragma unroll
    for (int i = 0; i < QC; ++i)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = top >= 0x7f800000u ? 0.f : v[i][4 * w + e] * up;
          if (PARTS == 2 && (g & 1)) x[e] -= __half2float(__float2half_rn(x[e]));  // the second part
        }
        const uint32_t lo = q8_pack(x[0], x[1]), hi = q8_pack(x[2], x[3]);
        if (Q_SHARED) {
          if (warp == 0) *reinterpret_cast<uint2*>(q_shared + (((4 * i + w) * NT + j) * 32 + lane) * 2) = make_uint2(lo, hi);
        } else {
          qf[Q_SHARED ? 0 : 4 * i + w][Q_SHARED ? 0 : j][0] = lo;
          qf[Q_SHARED ? 0 : 4 * i + w][Q_SHARED ? 0 : j][1] = hi;
        }
      }
  }
  // positions that bound what a column sees
  int col_pos[NT][LC], col_lo[NT][LC], col_head[NT][LC];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int c = 0; c < LC; ++c) {
      const int col = 8 * j / PARTS + LC * t + c;
      const bool ok = col < n_cols;
      col_pos[j][c] = ok ? pos0 + col / heads : -1;
      col_lo[j][c] = p.window > 0 ? col_pos[j][c] - (p.window - 1) : 0;
      col_head[j][c] = head0 + (ok ? col % heads : 0);
    }
  const int least_pos = pos0, most_lo = p.window > 0 ? pos0 + n_tok - 1 - (p.window - 1) : 0;

  // ---------------------------------------------------------------- the ring
  const uint32_t ring = q8_shared(my_ring);
  if (p.d < DP) {
    for (int i = lane; i < R::WARP / 16; i += 32) reinterpret_cast<uint4*>(my_ring)[i] = make_uint4(0u, 0u, 0u, 0u);
    __syncwarp();
  }
  // Groups that lie within a page (its size a power of two, 16 at least) and whose rows have no gap: one look at the table and two
  // runs of bytes a group. `find` gives the page, `fetch` checks it and asks for the rows; the look goes out a step before.
  const bool in_page = p.run_shift >= 4 && p.d == DP;
  constexpr int KEYS_AT_ONCE = 32 / CHUNKS;
  const uint32_t place_even = R::place(lane / CHUNKS, lane % CHUNKS);
  const uint32_t place_odd = R::place(4 + lane / CHUNKS, lane % CHUNKS) - 4 * DP;
  const int lo = p.window > 0 ? pos0 - (p.window - 1) : 0;
  // Else lane k of 16: the page of key k of the group.
  auto find = [&](int j) -> int {
    if (j >= last) return -1;
    if (in_page) {
      const int entry = (keys.at(j) * GROUP) >> p.run_shift;
      return entry < p.table_stride ? table[entry] : -1;
    }
    const int kp = keys.at(j) * GROUP + (lane & 15), entry = kp / p.bs;
    return kp < keys.hi && entry < p.table_stride ? table[entry] : -1;
  };
  auto fetch = [&](int j, int stage, int blk) {
    const uint32_t at = ring + stage * R::STAGE;
    const int key0 = keys.at(j) * GROUP;
    const bool paged = blk >= 0 && blk < p.n_blocks;
    const int c = lane % CHUNKS;
    if (in_page) {
      // (pages behind a window may have gone back; their keys are masked. Any other that is not there is an error.)
      if (!paged && (key0 + GROUP > lo || key0 < p.keep) && lane == 0 && p.err) atomicExch(p.err, CUCA_ERR_BLOCK_RANGE);
      const size_t row = ((size_t)(paged ? blk : 0) * p.nkv + kvh) * p.bs + (key0 & (p.bs - 1));
      const int8_t* kr = p.kpool + row * DP + lane * 16;
      const int8_t* vr = p.vpool + row * DP + lane * 16;
      const uint32_t bytes = paged ? 16u : 0u;
      for_each<GROUP / KEYS_AT_ONCE>([&](auto n) {
        constexpr int i = decltype(n)::value;
        // Where the lane's piece of row i * KEYS_AT_ONCE + lane / CHUNKS goes, less i * 512: the place turns with the row's lowest
        // three bits, of which the lane gives all but the highest (all, with half rows; the lowest, with rows of 256).
        const uint32_t to = at + (DP == 256 ? R::place(i * KEYS_AT_ONCE + lane / CHUNKS, c) - i * 512 :
                                  (i * KEYS_AT_ONCE) & 4 ? place_odd : place_even);
        copy16_at<i * 512, i * 512>(to, kr, bytes);
        copy16_at<R::TENSOR + i * 512, i * 512>(to, vr, bytes);
      });
      copy4(at + 2 * R::TENSOR + lane * 4, (lane < 16 ? p.kscale : p.vscale) + row + (lane & 15), paged);
      return;
    }
    const int kp = key0 + (lane & 15);
    if (!paged && kp < keys.hi && (kp >= lo || kp < p.keep) && p.err) atomicExch(p.err, CUCA_ERR_BLOCK_RANGE);
    const long long mine = paged ? ((long long)blk * p.nkv + kvh) * p.bs + kp % p.bs : -1;
#pragma unroll
    for (int i = 0; i < GROUP / KEYS_AT_ONCE; ++i) {
      const int k = i * KEYS_AT_ONCE + lane / CHUNKS;
      const long long row = __shfl_sync(0xffffffffu, mine, k);
      const bool ok = row >= 0;
      const size_t off = (size_t)(ok ? row : 0) * p.d + c * 16;
      if (c * 16 < p.d) {
        copy16(at + R::place(k, c), p.kpool + off, ok);
        copy16(at + R::TENSOR + R::place(k, c), p.vpool + off, ok);
      }
    }
    const float* scales = lane < 16 ? p.kscale : p.vscale;
    copy4(at + 2 * R::TENSOR + lane * 4, scales + (mine >= 0 ? mine : 0), mine >= 0);
  };

  float acc[TILES][NT][4];
#pragma unroll
  for (int i = 0; i < TILES; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[i][j][c] = 0.f;
  float m[NT][LC], l[NT][LC];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int c = 0; c < LC; ++c) { m[j][c] = -INFINITY; l[j][c] = 0.f; }

  int next;
  {
    int at[STAGES - 1];
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) at[s] = find(first + warp + WARPS * s);
    next = find(first + warp + WARPS * (STAGES - 1));
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) {
      if (first + warp + WARPS * s < last) fetch(first + warp + WARPS * s, s, at[s]);
      copies_commit();
    }
  }
  if (Q_SHARED) __syncthreads();

  int stage = 0;
  for (int j0 = first + warp; j0 < last; j0 += WARPS) {
    copies_wait<STAGES - 2>();
    __syncwarp();
    {  // the stage that was read in the last turn
      const int ahead = stage == 0 ? STAGES - 1 : stage - 1;
      if (j0 + WARPS * (STAGES - 1) < last) fetch(j0 + WARPS * (STAGES - 1), ahead, next);
      copies_commit();
      next = find(j0 + WARPS * STAGES);
    }
    const uint32_t at = ring + stage * R::STAGE;
    stage = stage + 1 == STAGES ? 0 : stage + 1;

    // ------------------------------------------------ raw scores: rows g and g + 8 are the group's keys, columns query rows
    float s[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) s[j][c] = 0.f;
#pragma unroll
    for (int i = 0; i < QC; ++i) {
      const uint4 a4 = shared_16(at + R::place(g, t + 4 * i)), b4 = shared_16(at + R::place(g + 8, t + 4 * i));
      const uint32_t a[4] = {a4.x, a4.y, a4.z, a4.w}, b[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t x = a[w] ^ 0x80808080u, y = b[w] ^ 0x80808080u;
        const uint32_t a0 = q8_pair_lo(x), a1 = q8_pair_lo(y), a2 = q8_pair_hi(x), a3 = q8_pair_hi(y);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          uint32_t b0, b1;
          if (Q_SHARED) {
            const uint2 f = *reinterpret_cast<const uint2*>(q_shared + (((4 * i + w) * NT + j) * 32 + lane) * 2);
            b0 = f.x; b1 = f.y;
          } else {
            b0 = qf[Q_SHARED ? 0 : 4 * i + w][Q_SHARED ? 0 : j][0];
            b1 = qf[Q_SHARED ? 0 : 4 * i + w][Q_SHARED ? 0 : j][1];
          }
          mma_f16(s[j], a0, a1, a2, a3, b0, b1);
        }
      }
    }

    // ------------------------------------------------ scores in log2 units with the values' scales, masks
    const int key0 = keys.at(j0) * GROUP;
    float ks[2], ve[2], vf[2], vi[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      ks[r] = shared_f(at + 2 * R::TENSOR + (g + 8 * r) * 4) * (OPT && p.cap > 0.f ? p.scale : p.scale_log2e);
      q8_value_scale(shared_f(at + 2 * R::TENSOR + GROUP * 4 + (g + 8 * r) * 4), ve[r], vf[r], vi[r]);
    }
    const bool whole = key0 + GROUP - 1 <= least_pos && (p.window <= 0 || key0 >= most_lo || key0 + GROUP <= p.keep);
    float z[NT][LC][2], zs[NT][LC][2];  // (in 32-bit mode the scores without the values' exponents too)
    bool higher = false;
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int c = 0; c < LC; ++c)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float raw = PARTS == 2 ? s[j][2 * r] + s[j][2 * r + 1] : s[j][2 * r + c];
          const float f = ks[r] * q_down[j][c];
          float x;
          if (OPT) {
            x = raw * f;
            if (p.cap > 0.f) x = q8_capped<PARTS == 2>(x, p);
            if (p.slopes) x -= p.slopes[col_head[j][c]] * CUCA_LOG2E * (float)(col_pos[j][c] - (key0 + g + 8 * r));
            if (PARTS == 2) zs[j][c][r] = x;
            x += ve[r];
          } else if (PARTS == 2) {
            zs[j][c][r] = raw * f;
            x = zs[j][c][r] + ve[r];
          } else {
            x = fmaf(raw, f, ve[r]);
          }
          if (!whole) {
            const int kp = key0 + g + 8 * r;
            if (!(kp <= col_pos[j][c] && (kp >= col_lo[j][c] || kp < p.keep))) x = -INFINITY;
          }
          z[j][c][r] = x;
          higher |= x > m[j][c] + Q8_LAG;
        }
    if (__any_sync(0xffffffffu, higher)) {
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        float corr[LC];
#pragma unroll
        for (int c = 0; c < LC; ++c) {
          float top = fmaxf(z[j][c][0], z[j][c][1]);
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
          const bool moves = top > m[j][c] + Q8_LAG;  // (each column by its own scores alone)
          corr[c] = moves ? q8_exp2(m[j][c] - top) : 1.f;
          if (moves) m[j][c] = top;
          l[j][c] *= corr[c];
        }
#pragma unroll
        for (int i = 0; i < TILES; ++i) {
          acc[i][j][0] *= corr[0]; acc[i][j][1] *= corr[LC - 1];
          acc[i][j][2] *= corr[0]; acc[i][j][3] *= corr[LC - 1];
        }
      }
    }

    // ------------------------------------------------ weights, as the second operand of the values' product
    uint32_t wb[NT][2];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float w[LC];
#pragma unroll
        for (int c = 0; c < LC; ++c) {
          const float ref = m[j][c] == -INFINITY ? 0.f : m[j][c] - Q8_LIFT;
          // In 32-bit mode an exponent meets the reference first: their difference is exact where values are large, and z is not.
          w[c] = PARTS == 2 && z[j][c][r] != -INFINITY ? q8_exp2(zs[j][c][r] + (ve[r] - ref)) : q8_exp2(z[j][c][r] - ref);
          l[j][c] = fmaf(w[c], vi[r], l[j][c]);
          w[c] *= vf[r];
        }
        uint32_t packed;
        if (PARTS == 2) {
          const uint32_t upper = q8_pack_weights(w[0], 0.f);
          packed = (upper & 0xffffu) | q8_pack_weights(0.f, w[0] - __half22float2(*reinterpret_cast<const __half2*>(&upper)).x);
        } else {
          packed = q8_pack_weights(w[0], w[LC - 1]);
        }
        wb[j][r] = turned_8x8(packed);
      }
    // ------------------------------------------------ values: rows are dimensions, from keys 2t, 2t + 1, 2t + 8, 2t + 9
    const uint32_t vat = at + R::TENSOR;
    auto products = [&](int tile0, uint32_t ka, uint32_t kb, uint32_t kc, uint32_t kd) {  // four dimensions: two tiles
      ka ^= 0x80808080u; kb ^= 0x80808080u; kc ^= 0x80808080u; kd ^= 0x80808080u;
      const uint32_t ab0 = __byte_perm(ka, kb, 0x5140), ab1 = __byte_perm(ka, kb, 0x7362);
      const uint32_t cd0 = __byte_perm(kc, kd, 0x5140), cd1 = __byte_perm(kc, kd, 0x7362);
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        mma_f16(acc[tile0][j], q8_pair_lo(ab0), q8_pair_hi(ab0), q8_pair_lo(cd0), q8_pair_hi(cd0), wb[j][0], wb[j][1]);
        mma_f16(acc[tile0 + 1][j], q8_pair_lo(ab1), q8_pair_hi(ab1), q8_pair_lo(cd1), q8_pair_hi(cd1), wb[j][0], wb[j][1]);
      }
    };
    if (DP == 64) {
      uint2 x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = shared_8(vat + R::place(2 * t + (i & 1) + 8 * (i >> 1), g >> 1) + (g & 1) * 8);
      products(0, x[0].x, x[1].x, x[2].x, x[3].x);
      products(2, x[0].y, x[1].y, x[2].y, x[3].y);
    } else {
#pragma unroll
      for (int h = 0; h < DP / 128; ++h) {
        uint4 x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = shared_16(vat + R::place(2 * t + (i & 1) + 8 * (i >> 1), g + 8 * h));
        products(8 * h, x[0].x, x[1].x, x[2].x, x[3].x);
        products(8 * h + 2, x[0].y, x[1].y, x[2].y, x[3].y);
        products(8 * h + 4, x[0].z, x[1].z, x[2].z, x[3].z);
        products(8 * h + 6, x[0].w, x[1].w, x[2].w, x[3].w);
      }
    }
  }

  // ---------------------------------------------------------------- the warps' results joined, in their order
  copies_wait<0>();
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int c = 0; c < LC; ++c) {
      l[j][c] += __shfl_xor_sync(0xffffffffu, l[j][c], 4);
      l[j][c] += __shfl_xor_sync(0xffffffffu, l[j][c], 8);
      l[j][c] += __shfl_xor_sync(0xffffffffu, l[j][c], 16);
    }
  __syncthreads();  // the rings are free
  constexpr int OS = DP + 4;  // floats between columns
  float* o_s = reinterpret_cast<float*>(smem);             // [WARPS][COLS][OS]
  float* ml_s = o_s + WARPS * COLS * OS;                   // [WARPS][COLS][2]
  float* ml_all = ml_s + WARPS * COLS * 2;                 // [COLS][2]: of the block
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int c = 0; c < LC; ++c) {
      const int col = 8 * j / PARTS + LC * t + c;
      float* dst = o_s + (warp * COLS + col) * OS;
#pragma unroll
      for (int i = 0; i < TILES; ++i) {
        // dimensions of the thread: DP / 8 from piece (half a piece) g, eight tiles a piece
        const int e = DP == 64 ? 8 * g + 2 * i : 128 * (i / 8) + 16 * g + 2 * (i % 8);
        const float lo = PARTS == 2 ? acc[i][j][0] + acc[i][j][1] : acc[i][j][c];
        const float hi = PARTS == 2 ? acc[i][j][2] + acc[i][j][3] : acc[i][j][2 + c];
        *reinterpret_cast<float2*>(dst + e) = make_float2(lo, hi);
      }
      if (g == 0) {
        ml_s[(warp * COLS + col) * 2] = m[j][c];
        ml_s[(warp * COLS + col) * 2 + 1] = l[j][c];
      }
    }
  __syncthreads();
  const int per_col = p.d / 4;
  for (int i = threadIdx.x; i < n_cols * per_col; i += WARPS * 32) {
    const int col = i / per_col, e = (i % per_col) * 4;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) top = fmaxf(top, ml_s[(w * COLS + col) * 2]);
    float o[4] = {0.f, 0.f, 0.f, 0.f}, den = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float mw = ml_s[(w * COLS + col) * 2];
      const float f = mw == top ? 1.f : q8_exp2(mw - top);  // (a warp without keys has zeros)
      const float4 v = *reinterpret_cast<const float4*>(o_s + (w * COLS + col) * OS + e);
      o[0] += f * v.x; o[1] += f * v.y; o[2] += f * v.z; o[3] += f * v.w;
      den += f * ml_s[(w * COLS + col) * 2 + 1];
    }
    const int head = head0 + col % heads;
    if (alone) {
      if (p.sink && top != -INFINITY) den += q8_sink_term(p, head, top);
      const float inv = den == 0.f ? 0.f : 1.f / den;  // (a column that saw nothing has zeros)
      T* dst = (T*)p.out + (size_t)(row0 + col / heads) * p.out_stride + (size_t)head * p.d + e;
#pragma unroll
      for (int k = 0; k < 4; ++k) dst[k] = from_f32<T>(o[k] * inv);
    } else if (as_cluster) {  // (the first warp's place: nobody else reads it)
      *reinterpret_cast<float4*>(o_s + col * OS + e) = make_float4(o[0], o[1], o[2], o[3]);
      if (e == 0) *reinterpret_cast<float2*>(ml_all + 2 * col) = make_float2(top, den);
    } else {
      float* part = p.part + (((size_t)blockIdx.z * gridDim.y + blockIdx.y) * p.n_splits + blockIdx.x) * (COLS * (p.d + 2));
      *reinterpret_cast<float4*>(part + col * p.d + e) = make_float4(o[0], o[1], o[2], o[3]);
      if (e == 0) *reinterpret_cast<float2*>(part + COLS * p.d + 2 * col) = make_float2(top, den);
    }
  }
  if (!as_cluster) return;

  // ---------------------------------------------------------------- the shares joined, in their order, out of one another's
  // shared memory; each block of the cluster writes a part of the rows
  cluster_sync();
  const int used = min(p.n_splits, (keys.groups + share - 1) / share);
  const uint32_t o_at = q8_shared(o_s), ml_at = q8_shared(ml_all);
  for (int i = blockIdx.x * WARPS * 32 + threadIdx.x; i < n_cols * per_col; i += used * WARPS * 32) {
    const int col = i / per_col, e = (i % per_col) * 4;
    float2 ml[MOST_CLUSTER];
    float4 v[MOST_CLUSTER];
    float top = -INFINITY;
#pragma unroll
    for (int s = 0; s < MOST_CLUSTER; ++s) {
      ml[s] = make_float2(-INFINITY, 0.f);
      v[s] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (s < used) {
        ml[s] = cluster_2(ml_at + col * 8, s);
        v[s] = cluster_4(o_at + (col * OS + e) * 4, s);
      }
      top = fmaxf(top, ml[s].x);
    }
    float o[4] = {0.f, 0.f, 0.f, 0.f}, den = 0.f;
#pragma unroll
    for (int s = 0; s < MOST_CLUSTER; ++s) {
      const float f = ml[s].x == top ? 1.f : q8_exp2(ml[s].x - top);
      o[0] += f * v[s].x; o[1] += f * v[s].y; o[2] += f * v[s].z; o[3] += f * v[s].w;
      den += f * ml[s].y;
    }
    const int head = head0 + col % heads;
    if (p.sink && top != -INFINITY) den += q8_sink_term(p, head, top);
    const float inv = den == 0.f ? 0.f : 1.f / den;
    T* dst = (T*)p.out + (size_t)(row0 + col / heads) * p.out_stride + (size_t)head * p.d + e;
#pragma unroll
    for (int k = 0; k < 4; ++k) dst[k] = from_f32<T>(o[k] * inv);
  }
  cluster_sync();  // nobody leaves while another reads its memory
}

// Joins the shares of a tile's keys, in their order: a warp per query row. Its lanes take two shares' maxima and sums each (there
// are 64 at most), then four dimensions (of each 128).
template <typename T>
__global__ void __launch_bounds__(WARPS * 32) join_q8_kernel(const Q8Params p, int cols) {
  pdl_trigger();
  pdl_wait();
  const int col = blockIdx.x * WARPS + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  int row0, n_tok;
  if (!q8_rows_of_tile(p, blockIdx.z, row0, n_tok)) return;
  const int kvh = blockIdx.y / p.head_parts, hp = blockIdx.y % p.head_parts;
  const int group_heads = p.nh / p.nkv;
  const int head0 = kvh * group_heads + hp * p.heads_per_cta;
  const int heads = min(p.heads_per_cta, group_heads - hp * p.heads_per_cta);
  const int pos0 = p.positions[row0];
  if (p.seq_of_row[row0] < 0 || pos0 < 0 || col >= n_tok * heads) return;
  const Q8Keys keys = q8_keys<GROUP>(p, pos0, n_tok);
  const int share = p.chunk / GROUP, used = min(p.n_splits, (keys.groups + share - 1) / share);
  if (used <= 1) return;  // written already
  const size_t step = (size_t)cols * (p.d + 2);
  const float* part = p.part + ((size_t)blockIdx.z * gridDim.y + blockIdx.y) * p.n_splits * step;
  float2 ml[2];
#pragma unroll
  for (int h = 0; h < 2; ++h)
    ml[h] = lane + 32 * h < used ? *reinterpret_cast<const float2*>(part + (lane + 32 * h) * step + cols * p.d + 2 * col)
                                 : make_float2(-INFINITY, 0.f);
  const float top = warp_max(fmaxf(ml[0].x, ml[1].x));
  float f[2], den = 0.f;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    f[h] = lane + 32 * h < used ? (ml[h].x == top ? 1.f : q8_exp2(ml[h].x - top)) : 0.f;
    den += lane + 32 * h < used ? f[h] * ml[h].y : 0.f;
  }
  den = warp_sum(den);
  const int head = head0 + col % heads;
  if (p.sink && top != -INFINITY) den += q8_sink_term(p, head, top);
  const float inv = den == 0.f ? 0.f : 1.f / den;
  for (int e0 = 0; e0 < p.d; e0 += 128) {
    const int e = e0 + 4 * lane;
    const float* src = part + col * p.d + (e < p.d ? e : 0);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int s = 0; s < used; ++s) {
      const float fs = __shfl_sync(0xffffffffu, s < 32 ? f[0] : f[1], s & 31);
      const float4 v = *reinterpret_cast<const float4*>(src + s * step);
      o.x += fs * v.x; o.y += fs * v.y; o.z += fs * v.z; o.w += fs * v.w;
    }
    if (e >= p.d) continue;
    T* dst = (T*)p.out + (size_t)(row0 + col / heads) * p.out_stride + (size_t)head * p.d + e;
    dst[0] = from_f32<T>(o.x * inv); dst[1] = from_f32<T>(o.y * inv);
    dst[2] = from_f32<T>(o.z * inv); dst[3] = from_f32<T>(o.w * inv);
  }
}

// ------------------------------------------------------------------ host side
template <int DP, int NT, int PARTS>
constexpr int smem_bytes() {
  const int ring = WARPS * Ring<DP>::WARP + (NT * DP > 256 ? (DP / 16) * NT * 32 * 8 : 0);
  const int cols = NT * 8 / PARTS;
  const int join = (WARPS * cols * (DP + 4 + 2) + cols * 2) * 4;
  return ring > join ? ring : join;
}

template <int DP, int NT, int PARTS, bool OPT>
int launch_q8(const Q8Params& p, int n_tiles, cudaStream_t stream) {
  constexpr int smem = smem_bytes<DP, NT, PARTS>();
  auto kernel = attention_q8_kernel<DP, NT, PARTS, OPT>;
  static cudaError_t configured = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  CUCA_REQUIRE(configured == cudaSuccess, "attention_q8: cannot reserve %d bytes of shared memory: %s", smem, cudaGetErrorString(configured));
  const dim3 grid(p.n_splits, p.nkv * p.head_parts, n_tiles);
  if (p.n_splits > 1 && p.part == nullptr) {
    CUCA_REQUIRE(p.n_splits <= MOST_CLUSTER, "attention_q8: %d shares do not join as a cluster", p.n_splits);
    cuca_launch_cluster(kernel, grid, dim3(WARPS * 32), smem, stream, true, p.n_splits, p);
    CUCA_CHECK_LAUNCH("attention_q8");
    return 0;
  }
  cuca_launch(kernel, grid, dim3(WARPS * 32), smem, stream, true, p);
  CUCA_CHECK_LAUNCH("attention_q8");
  if (p.n_splits > 1) {
    auto join = join_q8_kernel<typename std::conditional<PARTS == 2, float, __nv_bfloat16>::type>;
    cuca_launch(join, dim3((p.tile_tokens * p.heads_per_cta + WARPS - 1) / WARPS, p.nkv * p.head_parts, n_tiles), dim3(WARPS * 32), 0, stream, true, p, NT * 8 / PARTS);
    CUCA_CHECK_LAUNCH("attention_q8 (join)");
  }
  return 0;
}
template <int DP, int NT, int PARTS>
int launch_q8_opt(const Q8Params& p, int n_tiles, cudaStream_t stream) {
  return p.cap > 0.f || p.slopes ? launch_q8<DP, NT, PARTS, true>(p, n_tiles, stream)
                                           : launch_q8<DP, NT, PARTS, false>(p, n_tiles, stream);
}
template <int DP, int PARTS>
int launch_q8_nt(const Q8Params& p, int nt, int n_tiles, cudaStream_t stream) {
  if (nt == 1) return launch_q8_opt<DP, 1, PARTS>(p, n_tiles, stream);
  if constexpr (DP <= 128) {
    if (nt == 4) return launch_q8_opt<DP, 4, PARTS>(p, n_tiles, stream);
  }
  return launch_q8_opt<DP, 2, PARTS>(p, n_tiles, stream);
}

}  // namespace


// bfloat16 or 32-bit rows; tile_tokens rows of a request and heads_per_cta query heads to a block of `width` (1, 2, 4; not 4 beyond
// 128 dimensions) column tiles. part: [n_tiles][nkv * pieces of a group][n_splits][8 width / parts][d + 2] floats where
// n_splits > 1 (parts: 2 for 32-bit rows, else 1), or null: the shares (8 at most) join as a cluster.
CUCA_API int cuca_attention_q8(const CucaQ8Attention* c) {
  if (c->n_tiles == 0) return 0;
  Q8Params p;
  if (const int code = q8_params(*c, "attention_q8", 256, p)) return code;
  const int nt = (int)c->width, parts = c->dtype == CUCA_F32 ? 2 : 1, n_tiles = (int)c->n_tiles, d = p.d;
  CUCA_REQUIRE(nt == 1 || nt == 2 || (nt == 4 && d <= 128), "attention_q8: %d column tiles", nt);
  CUCA_REQUIRE((long long)p.tile_tokens * p.heads_per_cta * parts <= 8 * nt, "attention_q8: %d rows of %d heads do not fit %d columns",
               p.tile_tokens, p.heads_per_cta, 8 * nt / parts);
  CUCA_REQUIRE((long long)p.nkv * p.head_parts <= 65535, "attention_q8: too many heads");
  if (parts == 2) {
    if (d <= 64) return launch_q8_nt<64, 2>(p, nt, n_tiles, c->stream);
    if (d <= 128) return launch_q8_nt<128, 2>(p, nt, n_tiles, c->stream);
    return launch_q8_nt<256, 2>(p, nt, n_tiles, c->stream);
  }
  if (d <= 64) return launch_q8_nt<64, 1>(p, nt, n_tiles, c->stream);
  if (d <= 128) return launch_q8_nt<128, 1>(p, nt, n_tiles, c->stream);
  return launch_q8_nt<256, 1>(p, nt, n_tiles, c->stream);
}
