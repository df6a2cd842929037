// nvfp4_matvec.cu -- a few rows of activations times an NVFP4 weight matrix, activations in their own type:
//   y[m][n] = alpha * sum_k x[m][k] * e2m1(values[n][k]) * e4m3(scales[n][k / 16])
// for one token to a draft tree's 32 rows.  The weights are read once, N * K * 9 / 16 bytes: at these row counts that
// stream is the floor (the prefill chunk's GEMM in nvfp4.cu pays a 128-row tile and an activation quantizer instead).
//
//   tensor cores  mma.sync m16n8k16 in FP16 with fp32 sums: 16 weight rows are the MMA's M, 8 activation columns its N.  A thread
//                 builds its A fragments in registers from the codes as the matrix holds them: 32 neighbouring codes of a
//                 row (16 bytes, two scales), four to an MMA; the order of k is free as long as the activations follow it.  A
//                 weight is exact in FP16 (E2M1 x E4M3 has 6 significant bits).
//   activations   FP16 as they are; BF16 and fp32 times a power of two per row and warp that brings the largest into FP16's top
//                 binade, fp32 as the sum of two FP16 columns (22 bits and more): what that drops lies 2^-39 and 2^-23 below the
//                 row's largest value and the element, under what the fp32 sum keeps.  They are converted once into shared
//                 memory (where they do not fit, panel by panel) and serve every weight row of the CTA.
//   K             is cut over the 8 warps of a CTA and the 1, 2, 4 or 8 CTAs of a cluster, whose sums meet in shared memory and
//                 distributed shared memory: no workspace, one launch, an order of additions that depends on the shape alone.
//   loads         every warp streams 32 rows x 256 k (4.5 KB) at a time by cp.async through a private ring, across the rows of
//                 the CTA; nothing waits for another warp until 128 rows are summed.
#include <algorithm>

#include <cooperative_groups.h>

#include "decode4.cuh"

namespace lb {
namespace {
using namespace d4;

constexpr int kWarps = 8, kThreads = kWarps * 32;
constexpr int kUnit = 32;        // k of a unit: 16 bytes of a row
constexpr int kChunkUnits = 8;   // units of a stage
constexpr int kStageBytes = 32 * 128 + 32 * 16;  // 32 rows: codes, scales

// By 8-column tiles of activations: weight tiles (16 rows) summed at a time, ring stages, units of a panel.
__host__ __device__ constexpr int mv_tiles(int nt) { return nt <= 4 ? 8 : 4; }
__host__ __device__ constexpr int mv_stages(int nt) { return nt <= 4 ? 3 : 2; }
__host__ __device__ constexpr int mv_panel(int nt) { return nt == 1 ? 21 : nt == 2 ? 11 : nt == 4 ? 5 : 3; }  // (odd: a column is a multiple of 128 bytes)
__host__ __device__ constexpr int mv_x_stride(int nt) { return (mv_panel(nt) + 1) * 64; }  // bytes of a column: its units and one of zeros
__host__ __device__ constexpr int mv_x_bytes(int nt) { return 8 * nt * mv_x_stride(nt); }
constexpr int kJoin = 4;  // (tile, column tile) blocks whose sums meet at a time
constexpr int kJoinBytes = kWarps * kJoin * 512;
__host__ __device__ constexpr int mv_smem(int nt) { return kWarps * (mv_stages(nt) * kStageBytes + mv_x_bytes(nt)) + kJoinBytes; }

struct MatvecArgs {
  const void* x;
  long long ldx;
  int M;
  const uint8_t *values, *scales;
  float alpha;
  int N, K;
  void* y;
  long long ldy;
  int y_type, accumulate;
  bool x_vec;  // every row of x starts on a 16-byte boundary
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, int bytes) {  // the rest of the 16 is zero
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp8(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t h2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t h2_mul(uint32_t a, uint32_t b) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ float load_y(const void* y, int type, long long i) {
  return type == LING_B200_F32 ? static_cast<const float*>(y)[i] : type == LING_B200_BF16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(y)[i]) : __half2float(static_cast<const __half*>(y)[i]);
}
__device__ __forceinline__ void store_y(void* y, int type, long long i, float v) {
  if (type == LING_B200_F32) static_cast<float*>(y)[i] = v;
  else if (type == LING_B200_BF16) static_cast<__nv_bfloat16*>(y)[i] = __float2bfloat16_rn(v);
  else static_cast<__half*>(y)[i] = __float2half_rn(v);
}

// Eight elements of a row from k on (zeros from K on) as floats.
template <typename TX>
__device__ __forceinline__ void load_x8(const TX* row, int k, int K, bool vec, float (&v)[8]) {
  if (vec && k + 8 <= K) {
    constexpr int kPer = 16 / sizeof(TX);
#pragma unroll
    for (int i = 0; i < 8 / kPer; ++i) {
      const uint4 w = reinterpret_cast<const uint4*>(row + k)[i];
#pragma unroll
      for (int j = 0; j < kPer; ++j) v[i * kPer + j] = to_f32<TX>(reinterpret_cast<const TX*>(&w)[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = k + j < K ? to_f32<TX>(row[k + j]) : 0.f;
  }
}

// kRow16: rows of codes start on 16-byte boundaries (else on 8).
template <typename TX, int NT, bool kRow16>
__global__ void __launch_bounds__(kThreads, 1) nvfp4_matvec_kernel(MatvecArgs a) {
  pdl_sync();  // first statement: see common.cuh
  namespace cg = cooperative_groups;
  constexpr int TB = mv_tiles(NT), S = mv_stages(NT), PU = mv_panel(NT), XS = mv_x_stride(NT);
  constexpr bool kF32 = sizeof(TX) == 4, kScaled = !std::is_same<TX, __half>::value;
  constexpr int kCols = kF32 ? 2 : 1;  // columns of a row
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float4 cluster_sums[2][kJoin * 32];
  __shared__ float x_inv[kWarps][8 * NT];
  cg::cluster_group cluster = cg::this_cluster();
  const int c = int(cluster.num_blocks()), rank = int(cluster.block_rank()), cid = int(blockIdx.x) / c, clusters = int(gridDim.x) / c;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  uint8_t* ring = smem + warp * (S * kStageBytes);
  uint8_t* xs = smem + kWarps * S * kStageBytes + warp * mv_x_bytes(NT);
  float4* join = reinterpret_cast<float4*>(smem + kWarps * (S * kStageBytes + mv_x_bytes(NT)));
  const uint32_t ring_u32 = static_cast<uint32_t>(__cvta_generic_to_shared(ring));

  // ---- this cluster's weight tiles, this warp's units
  const int tiles = (a.N + 15) / 16, units = (a.K + kUnit - 1) / kUnit;
  const int tile0 = int((long long)tiles * cid / clusters), tile1 = int((long long)tiles * (cid + 1) / clusters);
  const int u0 = int((long long)units * (rank * kWarps + warp) / (c * kWarps)), u1 = int((long long)units * (rank * kWarps + warp + 1) / (c * kWarps));
  const int panels = (u1 - u0 + PU - 1) / PU;
  const size_t row_bytes = size_t(a.K) / 2, scale_bytes = size_t(a.K) / 16;

  // ---- the loading side: batch of TB tiles by batch, panel by panel, chunk by chunk, pair of tiles by pair
  int in_tile = tile0, in_panel = 0, in_unit = u0, in_pair = 0, put = 0;
  uint32_t words[5];             // the scales of the stage issued last: one row a lane, 16 bytes and what is before them in their word
  int words_shift = 0, words_units = 0;
  uint8_t* words_to = nullptr;
  auto issue = [&]() {
    if (in_tile < tile1 && panels > 0) {
      const int end = min(u1, u0 + (in_panel + 1) * PU), n = min(kChunkUnits, end - in_unit);
      const int row0 = (in_tile + in_pair * 2) * 16, rows = min(a.N, tile1 * 16) - row0;  // rows that are there
      const uint32_t st = ring_u32 + put * kStageBytes;
      // codes: four rows of 8 units an instruction; chunk u of row r lies at u ^ 4 (r & 1)
      const int r = lane >> 3, u = lane & 7;
      const uint8_t* src = a.values + size_t(row0 + r) * row_bytes + size_t(in_unit + u) * 16;
      const uint32_t dst = st + r * 128 + ((u ^ (r & 1) * 4) * 16);
      const int left = u < n ? int(min((long long)row_bytes - (long long)(in_unit + u) * 16, 16ll)) : 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool there = i * 4 + r < rows && left > 0;
        const uint8_t* from = there ? src + size_t(i * 4) * row_bytes : a.values;
        if constexpr (kRow16) {
          cp16(dst + i * 512, from, there ? 16 : 0);
        } else {
          cp8(dst + i * 512, from, there ? 8 : 0);
          cp8(dst + i * 512 + 8, there && left == 16 ? from + 8 : a.values, there && left == 16 ? 8 : 0);
        }
      }
      // scales: a row a lane, whole words that hold at least one of its bytes
      const int bytes = int(min((long long)scale_bytes - (long long)in_unit * 2, (long long)n * 2));
      words_units = lane < rows ? bytes : 0;
      const uintptr_t at = reinterpret_cast<uintptr_t>(a.scales) + size_t(row0 + (lane < rows ? lane : 0)) * scale_bytes + size_t(in_unit) * 2;
      words_shift = int(at & 3) * 8;
      const uint32_t* w = reinterpret_cast<const uint32_t*>(at & ~uintptr_t(3));
#pragma unroll
      for (int i = 0; i < 5; ++i) words[i] = i * 4 < int(at & 3) + words_units ? w[i] : 0u;
      words_to = ring + put * kStageBytes + 32 * 128 + lane * 16;
      put = put + 1 == S ? 0 : put + 1;
      // the next stage
      const int batch_tiles = min(TB, tile1 - in_tile);
      if (++in_pair * 2 >= batch_tiles) {
        in_pair = 0, in_unit += n;
        if (in_unit == end && ++in_panel == panels) in_panel = 0, in_unit = u0, in_tile += TB;
      }
    } else {
      words_to = nullptr;
    }
    cp_commit();
  };
  auto store_scales = [&]() {  // of the stage issued last
    if (words_to) {
      uint4 v;
      uint32_t* e = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t x = __funnelshift_r(words[i], words[i + 1], words_shift);
        const int left = words_units - i * 4;  // bytes of this word that are there
        e[i] = left >= 4 ? x : left <= 0 ? 0u : x & ((1u << (8 * left)) - 1u);
      }
      *reinterpret_cast<uint4*>(words_to) = v;
    }
  };
#pragma unroll
  for (int i = 0; i < S - 1; ++i) store_scales(), issue();

  // ---- the activations of a panel as FP16 columns: unit u, 16-byte piece q of column n lies at piece (4 u + q) ^ (u / 2 & 1 | 2 (n & 1))
  const int cols = a.M * kCols;
  auto x_at = [&](int n, int u, int q) { return xs + n * XS + (((u * 4 + q) ^ ((u >> 1 & 1) | (n & 1) << 1)) * 16); };
  for (int i = lane; i < 8 * NT * (XS / 16); i += 32) reinterpret_cast<uint4*>(xs)[i] = make_uint4(0, 0, 0, 0);  // columns and units that are not there
  if (lane < 8) {
#pragma unroll
    for (int n = 0; n < NT; ++n) x_inv[warp][n * 8 + lane] = 1.f;
  }
  __syncwarp();
  auto stage_x = [&](int pu0, int n, bool opening) {  // units pu0 .. pu0 + n; opening: no sums count in earlier ones' powers
    constexpr int kFly = (PU * 4 + 31) / 32;
    const int pieces = n * 4, k0 = pu0 * kUnit;
    constexpr int kRows = kF32 ? 2 : 4;  // rows whose loads are in flight
    for (int m0 = 0; m0 < a.M; m0 += kRows) {
      float v[kRows][kFly][8];
#pragma unroll
      for (int r = 0; r < kRows; ++r)
#pragma unroll
        for (int i = 0; i < kFly; ++i)
          if (m0 + r < a.M && lane + i * 32 < pieces) load_x8(static_cast<const TX*>(a.x) + (m0 + r) * a.ldx, k0 + (lane + i * 32) * 8, a.K, a.x_vec, v[r][i]);
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        if (m0 + r >= a.M) break;
        float mul = 1.f, inv = 1.f;
        if constexpr (kScaled) {
          uint32_t top = 0;  // bits of the largest finite magnitude
#pragma unroll
          for (int i = 0; i < kFly; ++i)
            if (lane + i * 32 < pieces) {
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const uint32_t b = __float_as_uint(v[r][i][j]) & 0x7fffffffu;
                top = b < 0x7f800000u ? max(top, b) : top;
              }
            }
          top = __reduce_max_sync(0xffffffffu, top);
          inv = __uint_as_float(uint32_t(max(int(top >> 23) - 14, 1)) << 23);  // 2^(exponent - 14)
          if (!opening) inv = fmaxf(inv, x_inv[warp][(m0 + r) * kCols]);       // sums only ever count in larger powers
          mul = 1.f / inv;
        }
#pragma unroll
        for (int i = 0; i < kFly; ++i) {
          const int p = lane + i * 32;
          if (p >= pieces) continue;
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float e0 = v[r][i][2 * j] * mul, e1 = v[r][i][2 * j + 1] * mul;
            hi[j] = h2(e0, e1);
            if constexpr (kF32) {
              const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi[j]));
              lo[j] = h2(fabsf(e0) < INFINITY ? e0 - f.x : 0.f, fabsf(e1) < INFINITY ? e1 - f.y : 0.f);
            }
          }
          *reinterpret_cast<uint4*>(x_at((m0 + r) * kCols, p >> 2, p & 3)) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          if constexpr (kF32) *reinterpret_cast<uint4*>(x_at((m0 + r) * kCols + 1, p >> 2, p & 3)) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
        __syncwarp();
        if (lane < kCols) x_inv[warp][(m0 + r) * kCols + lane] = inv;
      }
    }
    __syncwarp();
  };

  int stage = 0, buffer = 0;
  for (int tile = tile0; tile < tile1; tile += TB) {
    const int batch_tiles = min(TB, tile1 - tile);
    float acc[TB][NT][4] = {};
    for (int panel = 0; panel < panels; ++panel) {
      const int p0 = u0 + panel * PU, pn = min(PU, u1 - p0);
      if (panels > 1 || tile == tile0) {
        float was[NT][2];  // the sums so far count in the last panel's powers of two
#pragma unroll
        for (int n = 0; n < NT; ++n) was[n][0] = x_inv[warp][n * 8 + 2 * t], was[n][1] = x_inv[warp][n * 8 + 2 * t + 1];
        __syncwarp();
        stage_x(p0, pn, panel == 0);
        if constexpr (kScaled) {
          if (panel > 0) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const float f0 = was[n][0] / x_inv[warp][n * 8 + 2 * t], f1 = was[n][1] / x_inv[warp][n * 8 + 2 * t + 1];
#pragma unroll
              for (int i = 0; i < TB; ++i) acc[i][n][0] *= f0, acc[i][n][2] *= f0, acc[i][n][1] *= f1, acc[i][n][3] *= f1;
            }
          }
        }
      }
      for (int done = 0; done < pn; done += kChunkUnits) {
        const int pieces = (min(kChunkUnits, pn - done) + 3) / 4;
#pragma unroll
        for (int pair = 0; pair < TB / 2; ++pair) {
          if (pair * 2 >= batch_tiles) break;
          store_scales();
          cp_wait<S - 2>();
          __syncwarp();  // the stage has landed, for all lanes; all lanes are done with the one before, whose place is next
          issue();
          const uint8_t* st = ring + stage * kStageBytes;
          stage = stage + 1 == S ? 0 : stage + 1;
#pragma unroll
          for (int p = 0; p < kChunkUnits / 4; ++p) {
            if (p >= pieces) break;
            uint32_t xf[NT][16];
            const int u = done + p * 4 + t < pn ? done + p * 4 + t : PU;  // behind the panel: zeros
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const uint4 w = *reinterpret_cast<const uint4*>(x_at(n * 8 + g, u, q));
                xf[n][q * 4] = w.x, xf[n][q * 4 + 1] = w.y, xf[n][q * 4 + 2] = w.z, xf[n][q * 4 + 3] = w.w;
              }
#pragma unroll
            for (int i = 0; i < 2; ++i) {  // the two tiles of the pair
              uint32_t w[2][4], sc[2][2];
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                const int r = i * 16 + half * 8 + g;
                const uint4 v = *reinterpret_cast<const uint4*>(st + r * 128 + (((p * 4 + t) ^ (r & 1) * 4) * 16));
                w[half][0] = v.x, w[half][1] = v.y, w[half][2] = v.z, w[half][3] = v.w;
                const uint32_t h = e4m3x2_to_h2(*reinterpret_cast<const uint16_t*>(st + 32 * 128 + r * 16 + (p * 4 + t) * 2));
                sc[half][0] = __byte_perm(h, h, 0x1010), sc[half][1] = __byte_perm(h, h, 0x3232);
              }
#pragma unroll
              for (int j = 0; j < 4; ++j) {  // 8 codes, two MMAs
                uint32_t cd[2][4];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                  e2m1x8_to_h2(w[half][j], cd[half]);
#pragma unroll
                  for (int e = 0; e < 4; ++e) cd[half][e] = h2_mul(cd[half][e], sc[half][j / 2]);
                }
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                  mma_16816(acc[pair * 2 + i][n], cd[0][0], cd[1][0], cd[0][1], cd[1][1], xf[n][j * 4], xf[n][j * 4 + 1]);
                  mma_16816(acc[pair * 2 + i][n], cd[0][2], cd[1][2], cd[0][3], cd[1][3], xf[n][j * 4 + 2], xf[n][j * 4 + 3]);
                }
              }
            }
          }
        }
      }
    }

    // ---- the warps' sums, then the cluster's: kJoin (tile, column tile) blocks at a time, one quad of a block a thread
    constexpr int kPasses = NT > kJoin ? NT / kJoin : 1, kN = NT / kPasses, kJoinTiles = kJoin / kN, kBlocks = kJoin;  // (many column tiles in turns)
    float inv[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) inv[n][0] = x_inv[warp][n * 8 + 2 * t], inv[n][1] = x_inv[warp][n * 8 + 2 * t + 1];
#pragma unroll
    for (int i0 = 0; i0 < TB; i0 += kJoinTiles) {
      if (i0 >= batch_tiles) break;
#pragma unroll
      for (int pass = 0; pass < kPasses; ++pass) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kJoinTiles; ++i)
#pragma unroll
          for (int n = 0; n < kN; ++n) {
            const int nn = pass * kN + n;
            const float(&v)[4] = acc[i0 + i][nn];
            join[(warp * kBlocks + i * kN + n) * 32 + lane] = make_float4(v[0] * inv[nn][0], v[1] * inv[nn][1], v[2] * inv[nn][0], v[3] * inv[nn][1]);
          }
        __syncthreads();
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
        if (tid < kBlocks * 32) {
#pragma unroll
          for (int w = 0; w < kWarps; ++w) {
            const float4 v = join[w * kBlocks * 32 + tid];
            s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
          }
        }
        bool mine = tid < kBlocks * 32;
        if (c > 1) {
          if (mine) cluster_sums[buffer][tid] = s;
          cluster.sync();
          mine = mine && tid / 32 % c == rank;  // a warp's quads to one of the CTAs
          if (mine) {
            s = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int r = 0; r < c; ++r) {
              const float4 v = *cluster.map_shared_rank(&cluster_sums[buffer][tid], r);
              s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
            }
          }
          buffer ^= 1;  // (written again two meetings later, when all have read it)
        }
        if (mine) {
          const int block = tid / 32, row = (tile + i0 + block / kN) * 16 + g, nn = pass * kN + block % kN;
          const float v[2][2] = {{s.x, s.y}, {s.z, s.w}};
#pragma unroll
          for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int j = 0; j < (kF32 ? 1 : 2); ++j) {
              const int n = row + half * 8, m = kF32 ? nn * 4 + t : nn * 8 + 2 * t + j;
              if (n >= a.N || n >= tile1 * 16 || m >= a.M) continue;
              const float sum = a.alpha * (kF32 ? v[half][0] + v[half][1] : v[half][j]);
              const long long at = m * a.ldy + n;
              store_y(a.y, a.y_type, at, a.accumulate ? load_y(a.y, a.y_type, at) + sum : sum);
            }
        }
      }
    }
  }
  cp_wait<0>();
  if (c > 1) cluster.sync();  // no CTA leaves while another reads its sums
}

// ---------------------------------------------------------------------------------------------- launch
DeviceInfo g_devices[kMaxDevices];
std::mutex g_mutex;
// Clusters of 1, 2, 4 and 8 CTAs that fit the device at a time, by 8-column tiles (1, 2, 4, 8).
int g_clusters[kMaxDevices][4][4];

template <typename TX, int NT, bool kRow16>
int init_one(int (*clusters)[4]) {
  auto* k = nvfp4_matvec_kernel<TX, NT, kRow16>;
  LB_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, mv_smem(NT)));
  const int row = NT == 1 ? 0 : NT == 2 ? 1 : NT == 4 ? 2 : 3;
  if (clusters[row][0] != 0) return LING_B200_OK;
  for (int i = 0; i < 4; ++i) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(1u << i), cfg.blockDim = dim3(kThreads), cfg.dynamicSmemBytes = mv_smem(NT);
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 1u << i, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
    cfg.attrs = at, cfg.numAttrs = 1;
    int n = 0;
    LB_CUDA(cudaOccupancyMaxActiveClusters(&n, k, &cfg));
    clusters[row][i] = std::max(n, 1);
  }
  return LING_B200_OK;
}
template <typename TX>
int init_type(int (*clusters)[4]) {
  if (const int r = init_one<TX, 1, true>(clusters)) return r;
  if (const int r = init_one<TX, 1, false>(clusters)) return r;
  if (const int r = init_one<TX, 2, true>(clusters)) return r;
  if (const int r = init_one<TX, 2, false>(clusters)) return r;
  if (const int r = init_one<TX, 4, true>(clusters)) return r;
  if (const int r = init_one<TX, 4, false>(clusters)) return r;
  if (sizeof(TX) < 4) return LING_B200_OK;
  if (const int r = init_one<TX, 8, true>(clusters)) return r;
  return init_one<TX, 8, false>(clusters);
}
int init_all(int device) {
  if (const int r = init_type<float>(g_clusters[device])) return r;
  if (const int r = init_type<__nv_bfloat16>(g_clusters[device])) return r;
  return init_type<__half>(g_clusters[device]);
}

// CTAs that share K: the cluster size with the least estimated time.  A warp's unit of a tile is 288 bytes of a stream of about 5.5
// bytes a nanosecond (52 ns); a meeting of the cluster's CTAs costs about 1.5 us, of a CTA's warps 0.5 us; activations that do
// not fit shared memory are converted again for every batch (about 1 us a panel).
int choose_cluster(const int* clusters, int N, int K, int nt) {
  const int tiles = ceil_div(N, 16), units = ceil_div(K, kUnit);
  double best = 0;
  int pick = 0;
  for (int i = 0; i < 4; ++i) {
    const int c = 1 << i, at_once = std::min(clusters[i], tiles), t = ceil_div(tiles, at_once), u = ceil_div(units, c * kWarps);
    const int batches = ceil_div(t, mv_tiles(nt)), panels = ceil_div(u, mv_panel(nt));
    const double cost = 52.0 * t * u + batches * (c > 1 ? 1500.0 : 500.0) + (panels > 1 ? 1000.0 * panels * batches : 0.0);
    if (i == 0 || cost < best) best = cost, pick = i;
  }
  return pick;
}

template <typename TX, int NT>
int matvec_launch(const MatvecArgs& a, int device, cudaStream_t s) {
  const int row = NT == 1 ? 0 : NT == 2 ? 1 : NT == 4 ? 2 : 3;
  const int i = choose_cluster(g_clusters[device][row], a.N, a.K, NT), c = 1 << i;
  const int clusters = std::min(g_clusters[device][row][i], ceil_div(a.N, 16));
  const bool row16 = a.K % 32 == 0 && aligned(a.values, 16);
  LB_CUDA(launch_kernel_cluster(row16 ? nvfp4_matvec_kernel<TX, NT, true> : nvfp4_matvec_kernel<TX, NT, false>, dim3(clusters * c), dim3(kThreads),
                                size_t(mv_smem(NT)), c, s, a));
  LB_LAUNCH("nvfp4_matvec_kernel");
  return LING_B200_OK;
}
template <typename TX>
int matvec_columns(const MatvecArgs& a, int device, cudaStream_t s) {
  const int cols = a.M * (sizeof(TX) == 4 ? 2 : 1);
  if (cols <= 8) return matvec_launch<TX, 1>(a, device, s);
  if (cols <= 16) return matvec_launch<TX, 2>(a, device, s);
  if (cols <= 32) return matvec_launch<TX, 4>(a, device, s);
  if constexpr (sizeof(TX) == 4) return matvec_launch<TX, 8>(a, device, s);
  return LING_B200_ERR_ARG;  // not reached: at most 32 rows
}

}  // namespace
}  // namespace lb

using namespace lb;

extern "C" int ling_b200_nvfp4_matvec(int device, const void* x, int x_type, long long ldx, int M, const uint8_t* values,
                                      const uint8_t* scales, float alpha, int N, int K, void* y, int y_type, long long ldy, int accumulate,
                                      void* stream) {
  if (!d4::type_ok(x_type) || !d4::type_ok(y_type)) {
    set_error("nvfp4_matvec: element types are LING_B200_F32, _BF16 and _F16");
    return LING_B200_ERR_ARG;
  }
  if (!x || !values || !scales || !y || M < 1 || M > 32 || N < 1 || K < 16 || K % 16 != 0 || ldx < K || ldy < N ||
      !d4::aligned(x, d4::type_size(x_type)) || !d4::aligned(y, d4::type_size(y_type)) || !d4::aligned(values, 8)) {
    set_error("nvfp4_matvec: bad argument (1 <= M <= 32, K a multiple of 16, ldx >= K, ldy >= N, values on an 8-byte boundary)");
    return LING_B200_ERR_ARG;
  }
  d4::DeviceGuard guard;
  int sms = 0;
  if (const int r = d4::enter_device(guard, device, g_devices, g_mutex, [device] { return init_all(device); }, &sms)) return r;
  MatvecArgs a{x, ldx, M, values, scales, alpha, N, K, y, ldy, y_type, accumulate, false};
  a.x_vec = d4::aligned(x, 16) && ldx * d4::type_size(x_type) % 16 == 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return x_type == LING_B200_F32 ? matvec_columns<float>(a, device, s)
         : x_type == LING_B200_BF16 ? matvec_columns<__nv_bfloat16>(a, device, s)
                                    : matvec_columns<__half>(a, device, s);
}
