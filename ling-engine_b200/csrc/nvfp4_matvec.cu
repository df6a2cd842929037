// nvfp4_matvec.cu -- a few rows of activations times an NVFP4 weight matrix, activations in their own type:
//   y[m][n] = alpha * sum_k x[m][k] * e2m1(values[n][k]) * e4m3(scales[n][k / 16])
// for one token to a draft tree's 32 rows.  A launch reads the weights once, N * K * 9 / 16 bytes: at these row counts that
// stream is the floor (the prefill chunk's GEMM in nvfp4.cu pays a 128-row tile and an activation quantizer instead).  Rows whose
// activations do not fit beside the others' (matvec_rows) are launches of their own.
//
//   tensor cores  mma.sync m16n8k16 in FP16 with fp32 sums: 16 weight rows are the MMA's M, 8 activation columns its N.  A thread
//                 builds its A fragments in registers from the codes as the matrix holds them: 32 neighbouring codes of a
//                 row (16 bytes, two scales), four to an MMA; the order of k is free as long as the activations follow it.  A
//                 weight is exact in FP16 (E2M1 x E4M3 has 6 significant bits).
//   activations   FP16 as they are; BF16 and fp32 times a power of two per row and CTA that brings the largest into FP16's top
//                 binade, fp32 as the sum of two FP16 columns (22 bits and more).  An element is off by at most 2^-39 of its row's
//                 largest, fp32 by 2^-23 of itself besides: under what the fp32 sum keeps as long as the largest elements have a
//                 part in it.  In a sum that the weights leave to elements 2^25 times smaller (theirs being 0), it shows: the
//                 price of one scale a row.  Converted once into shared memory, they serve every weight row of the CTA.
//   split         a cluster of 1, 2, 4 or 8 CTAs takes a share of the weight rows, its CTAs a share of K each; in a CTA the warps
//                 are groups with rows of their own, whose 1 to 8 warps share the CTA's K again.  Shared sums meet in shared
//                 memory and distributed shared memory: no workspace, one launch, an order of additions that depends on the
//                 shape alone.  Many rows want no meeting (head: a warp per row pair), few rows many hands.
//   loads         every warp streams 32 rows x 256 k (4.5 KB) at a time by cp.async through a private ring, across its rows;
//                 nothing waits for another warp between meetings.
// Measured, one BF16 row: 1024 x 5120 5.5 us; 5120 x 17408 22 us, 2.3 TB/s; 34816 x 5120 27 us, 3.8 TB/s; 248320 x 5120 155 us, 4.6 TB/s
// (6.5 TB/s is a plain copy).  34816 x 5120: 8 rows 32 us, 16 rows 44 us, 32 rows 94 us, 32 fp32 rows (two launches) 182 us.  No unit
// is full (head: DRAM 53 %, issue slots 50 %, tensor pipe 24 % busy; 16 rows: 28, 36 and 29 %): two warps a scheduler do not hide the
// latencies of MMAs and conversions, and where CTAs share K the meetings and unequal shares come on top.
#include <algorithm>

#include <cooperative_groups.h>

#include "decode4.cuh"

namespace lb {
namespace {
using namespace d4;

constexpr int kWarps = 8, kThreads = kWarps * 32;
constexpr int kUnit = 32;        // k of a unit: 16 bytes of a row
constexpr int kChunkUnits = 8;   // units of a stage
constexpr int kStageBytes = 32 * 128 + 32 * 32;  // 32 rows: codes; scales, as the 16-byte pieces they lie in

constexpr int kSumBlocks = 64;   // (tile, K part, column tile) sums of a CTA between two meetings
constexpr int kSmem = 225 * 1024;  // rings of 2 to 6 stages, sums, activations: as many stages as the rest leaves room for
constexpr int kMaxStages = 6;

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
  int parts, stages;       // warps that share a CTA's K: 1, 2, 4 or 8; stages of a warp's ring
  int tiles, more_tiles;   // tiles of a cluster; clusters that have one more
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
__device__ __forceinline__ void cp_wait_but(int n) {  // all groups but the last n
  switch (n) {
    case 0: cp_wait<0>(); break;
    case 1: cp_wait<1>(); break;
    case 2: cp_wait<2>(); break;
    case 3: cp_wait<3>(); break;
    default: cp_wait<4>(); break;
  }
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

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_arrive_wait() { cluster_arrive(), cluster_wait(); }

// The power of two that a row whose largest finite magnitude has these bits was multiplied by (1 / x_inv): 2^(14 - exponent).
__device__ __forceinline__ float x_inv(uint32_t top) { return __uint_as_float(uint32_t(max(int(top >> 23) - 14, 1)) << 23); }
__device__ __forceinline__ float x_mul(uint32_t top) { return 1.f / x_inv(top); }

// kRow16: rows of codes start on 16-byte boundaries (else on 8), rows of scales on 2-byte ones (else anywhere).
template <typename TX, int NT, bool kRow16>
__global__ void __launch_bounds__(kThreads, 1) nvfp4_matvec_kernel(MatvecArgs a) {
  pdl_sync();  // first statement: see common.cuh
  namespace cg = cooperative_groups;
  const int S = a.stages;
  constexpr bool kF32 = sizeof(TX) == 4, kScaled = !std::is_same<TX, __half>::value;
  constexpr int kCols = kF32 ? 2 : 1;  // columns of a row
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint32_t x_top[8 * NT];  // of a row's finite magnitudes the largest, as bits
  cg::cluster_group cluster = cg::this_cluster();
  const int c = int(cluster.num_blocks()), rank = int(cluster.block_rank()), cid = int(blockIdx.x / unsigned(c));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int parts = a.parts, lp = 31 - __clz(parts), lg = 3 - lp, part = warp & (parts - 1), group = warp >> lp;  // (powers of two)
  uint8_t* ring = smem + warp * (S * kStageBytes);
  const bool alone = c * parts == 1;  // a warp has all of K: it writes its sums itself
  float4* sums = reinterpret_cast<float4*>(smem + kWarps * S * kStageBytes);  // [tile][part][column tile][lane], added into part 0
  uint8_t* xs = smem + kWarps * S * kStageBytes + (alone ? 0 : kSumBlocks * 512);
  const uint32_t ring_u32 = static_cast<uint32_t>(__cvta_generic_to_shared(ring));

  // ---- this cluster's weight tiles, this CTA's and this warp's units of K
  const int units = (a.K + kUnit - 1) / kUnit, row_bytes = a.K / 2, scale_bytes = a.K / 16;
  const int tile0 = a.tiles * cid + min(cid, a.more_tiles), tile1 = tile0 + a.tiles + (cid < a.more_tiles ? 1 : 0);
  const int chunks = (units + kChunkUnits - 1) / kChunkUnits, h0 = chunks * rank / c, h1 = chunks * (rank + 1) / c;  // K is cut at whole chunks
  const int c0 = h0 * kChunkUnits, c1 = min(units, h1 * kChunkUnits);
  const int u0 = (h0 + ((h1 - h0) * part >> lp)) * kChunkUnits, u1 = min(units, (h0 + ((h1 - h0) * (part + 1) >> lp)) * kChunkUnits);
  const bool scales16 = ((reinterpret_cast<uintptr_t>(a.scales) | uintptr_t(scale_bytes)) & 15) == 0;  // a chunk's scales of a row are one piece
  // Batches of tiles between meetings, of which this warp's group has the pairs [first_pair, last_pair).
  const int batch = alone ? max(tile1 - tile0, 1) : max((kSumBlocks / NT >> lp) & ~1, 2);
  auto first_pair = [&](int tile, int who) { return ((min(batch, tile1 - tile) + 1) / 2 * who + (1 << lg) - 1) >> lg; };

  // ---- the activations, asked for first: unit u, 16-byte piece q of column n lies at piece (4 u + q) ^ (u / 2 & 1 | 2 (n & 1)).  Raw at
  // first: eight 16-bit elements where their FP16 will lie, of eight fp32 elements four where their upper parts will, four where
  // their lower ones.
  const int cols = a.M * kCols, x_units = max(c1 - c0, 0), x_stride = x_units * 64, x_pieces = x_units * 4, k0 = c0 * kUnit;
  auto x_at = [&](int n, int u, int q) { return xs + n * x_stride + (((u * 4 + q) ^ ((u >> 1 & 1) | (n & 1) << 1)) * 16); };
  if (tid < 8 * NT) x_top[tid] = 0;
#pragma unroll 1
  for (int m = 0, p = tid; m < a.M; p += kThreads) {
    while (p >= x_pieces) p -= x_pieces, ++m;  // piece p of row m
    if (m >= a.M) break;
    const int k = k0 + p * 8;
    const TX* src = static_cast<const TX*>(a.x) + m * a.ldx + k;
    constexpr int kPer = 16 / sizeof(TX);
#pragma unroll
    for (int j = 0; j < kCols; ++j) {
      uint8_t* to = x_at(m * kCols + j, p >> 2, p & 3);
      if (a.x_vec) {  // (K is a multiple of 16: a piece is there whole or not at all)
        cp16(static_cast<uint32_t>(__cvta_generic_to_shared(to)), k < a.K ? src + j * kPer : static_cast<const TX*>(a.x), k < a.K ? 16 : 0);
      } else {
#pragma unroll 1
        for (int e = 0; e < kPer; ++e) reinterpret_cast<TX*>(to)[e] = k < a.K ? src[j * kPer + e] : TX(0.f);
      }
    }
  }
  cp_commit();

  // ---- the loading side: batch by batch, pair of tiles by pair, chunk of 8 units by chunk
  int in_tile = tile0, in_pair = first_pair(tile0, group), in_last = first_pair(tile0, group + 1), in_unit = u0, put = 0;
  const int r = lane >> 3, cu = lane & 7;  // copied: row r (of four) and unit cu of a stage's 8
  auto issue = [&]() {
    if (u0 >= u1) in_tile = tile1;
    while (in_pair == in_last && in_tile < tile1) {
      in_tile += batch;
      if (in_tile < tile1) in_pair = first_pair(in_tile, group), in_last = first_pair(in_tile, group + 1);
    }
    if (in_tile < tile1) {
      const int n = min(kChunkUnits, u1 - in_unit);
      const int row0 = (in_tile + in_pair * 2) * 16, rows = min(a.N, tile1 * 16) - row0;  // rows that are there
      const uint32_t st = ring_u32 + put * kStageBytes;
      // codes: four rows an instruction; unit u of row r lies at u ^ 4 (r & 1)
      const uint8_t* src = a.values + size_t(row0 + r) * row_bytes + (in_unit + cu) * 16;
      const uint32_t dst = st + r * 128 + ((cu ^ (r & 1) * 4) * 16);
      if (kRow16 && rows >= 32 && n == kChunkUnits) {
#pragma unroll
        for (int i = 0; i < 8; ++i) cp16(dst + i * 512, src + size_t(i * 4) * row_bytes, 16);
      } else {
        const int left = cu < n ? min(row_bytes - (in_unit + cu) * 16, 16) : 0;
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
      }
      // scales: a row a lane, the one or two 16-byte pieces that hold at least one of its bytes (of pieces that reach beyond the array,
      // what lies in it)
      const int bytes = lane < rows ? min(scale_bytes - in_unit * 2, n * 2) : 0;
      const uintptr_t at = reinterpret_cast<uintptr_t>(a.scales) + size_t(row0 + (lane < rows ? lane : 0)) * scale_bytes + in_unit * 2;
      const uint8_t* w = reinterpret_cast<const uint8_t*>(at & ~uintptr_t(15));
      const uint32_t to = st + 32 * 128 + lane * 32;
      if (scales16) {
        cp16(to, w, bytes > 0 ? 16 : 0);
      } else {
        const long long left = a.scales + size_t(a.N) * scale_bytes - w;
        const bool two = bytes > 0 && int(at & 15) + bytes > 16;
        if (bytes > 0 && w < a.scales) {
          for (int i = int(at & 15); i < 16 && i < left; ++i) ring[put * kStageBytes + 32 * 128 + lane * 32 + i] = w[i];
        } else {
          cp16(to, w, bytes > 0 ? int(min(left, 16ll)) : 0);
        }
        cp16(to + 16, two ? w + 16 : w, two ? int(min(left - 16, 16ll)) : 0);
      }
      put = put + 1 == S ? 0 : put + 1;
      in_unit += n;
      if (in_unit == u1) in_unit = u0, ++in_pair;
    }
    cp_commit();
  };
#pragma unroll 1
  for (int i = 0; i < S - 1; ++i) issue();

  // ---- the activations to FP16, in place: a warp takes a row, or a part of it where there are few
  cp_wait_but(S - 1);
  __syncthreads();
  if constexpr (kScaled) {
    const int segments = a.M >= kWarps ? 1 : a.M == 1 ? kWarps : kWarps / a.M, per = (x_pieces + segments - 1) / segments;
#pragma unroll 1
    for (int i = warp; i < a.M * segments; i += kWarps) {
      const int m = i / segments, p0 = (i - m * segments) * per, p1 = min(x_pieces, p0 + per);
      uint32_t top = 0;
#pragma unroll 1
      for (int p = p0 + lane; p < p1; p += 32)
#pragma unroll
        for (int j = 0; j < kCols; ++j) {
          const uint4 w = *reinterpret_cast<const uint4*>(x_at(m * kCols + j, p >> 2, p & 3));
          const uint32_t e[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            if constexpr (kF32) {
              const uint32_t b = e[q] & 0x7fffffffu;
              top = b < 0x7f800000u ? max(top, b) : top;
            } else {
              const uint32_t b0 = e[q] << 16 & 0x7fffffffu, b1 = e[q] & 0x7fff0000u;
              top = b0 < 0x7f800000u ? max(top, b0) : top, top = b1 < 0x7f800000u ? max(top, b1) : top;
            }
          }
        }
      top = __reduce_max_sync(0xffffffffu, top);
      if (lane == 0) atomicMax(&x_top[m], top);
    }
    __syncthreads();
#pragma unroll 1
    for (int m = 0, p = tid; m < a.M; p += kThreads) {
      while (p >= x_pieces) p -= x_pieces, ++m;
      if (m >= a.M) break;
      const float mul = x_mul(x_top[m]);
      uint4* hi = reinterpret_cast<uint4*>(x_at(m * kCols, p >> 2, p & 3));
      const uint4 w = *hi;
      if constexpr (kF32) {
        uint4* lo = reinterpret_cast<uint4*>(x_at(m * kCols + 1, p >> 2, p & 3));
        const uint4 v = *lo;
        const uint32_t e[8] = {w.x, w.y, w.z, w.w, v.x, v.y, v.z, v.w};
        uint32_t h[4], l[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float e0 = __uint_as_float(e[2 * q]) * mul, e1 = __uint_as_float(e[2 * q + 1]) * mul;
          h[q] = h2(e0, e1);
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[q]));
          l[q] = h2(fabsf(e0) < INFINITY ? e0 - f.x : 0.f, fabsf(e1) < INFINITY ? e1 - f.y : 0.f);
        }
        *hi = make_uint4(h[0], h[1], h[2], h[3]), *lo = make_uint4(l[0], l[1], l[2], l[3]);
      } else {
        const uint32_t e[4] = {w.x, w.y, w.z, w.w};
        uint32_t h[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) h[q] = h2(__uint_as_float(e[q] << 16) * mul, __uint_as_float(e[q] & 0xffff0000u) * mul);
        *hi = make_uint4(h[0], h[1], h[2], h[3]);
      }
    }
    __syncthreads();
  }
  float inv[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int j = 0; j < 2; ++j) inv[n][j] = kScaled ? x_inv(x_top[(n * 8 + 2 * t + j) / kCols]) : 1.f;

  // Writes quad v of (tile, column tile): rows g and g + 8, columns 2t and 2t + 1.
  auto write_quad = [&](int tile, int nn, const float4& s) {
    const float v[2][2] = {{s.x, s.y}, {s.z, s.w}};
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int j = 0; j < (kF32 ? 1 : 2); ++j) {
        const int n = tile * 16 + g + half * 8, m = kF32 ? nn * 4 + t : nn * 8 + 2 * t + j;
        if (n >= a.N || m >= a.M) continue;
        const float sum = a.alpha * (kF32 ? v[half][0] + v[half][1] : v[half][j]);
        const long long at = m * a.ldy + n;
        store_y(a.y, a.y_type, at, a.accumulate ? load_y(a.y, a.y_type, at) + sum : sum);
      }
  };

  // this thread's columns (one that is not there is never written: any stands in); a chunk starts at a multiple of 8 units, so where
  // a piece lies in its unit depends on the thread alone
  const uint8_t* x_col[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) x_col[n] = xs + min(n * 8 + g, cols - 1) * x_stride;
  const int x_swizzle = t >> 1 | (g & 1) << 1;
  int stage = 0;
  bool read_pending = false;  // the other CTAs may still be reading this one's sums
  for (int tile = tile0; tile < tile1; tile += batch) {
    const int batch_tiles = min(batch, tile1 - tile), last_pair = first_pair(tile, group + 1);
    for (int pair = first_pair(tile, group); pair < last_pair; ++pair) {
      float total[2][NT][4] = {};
      for (int unit = u0; unit < u1; unit += kChunkUnits) {
        const int n_units = min(kChunkUnits, u1 - unit);
        cp_wait_but(S - 2);
        __syncwarp();  // the stage has landed, for all lanes; all lanes are done with the one before, whose place is next
        issue();
        const uint8_t* st = ring + stage * kStageBytes;
        stage = stage + 1 == S ? 0 : stage + 1;
        const uint8_t* row_s[2][2];  // scales of this thread's first unit, rows g and g + 8 of the two tiles
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int row = i * 16 + half * 8 + g;
            row_s[i][half] = st + 32 * 128 + row * 32 + t * 2;
            if (!scales16) row_s[i][half] += (uint32_t(reinterpret_cast<uintptr_t>(a.scales)) + uint32_t((tile + pair * 2) * 16 + row) * uint32_t(scale_bytes) + uint32_t(unit) * 2u) & 15u;
          }
        const uint8_t* row_w = st + g * 128 + t * 16;
        const int x_off = (unit - c0) * 64;
        float acc[2][NT][4] = {};  // of this chunk: an MMA cuts its sums off instead of rounding them, which a long chain would add up
        auto piece = [&](int p, bool here) {  // four units, this thread's being unit + 4 p + t; !here: it is not in the chunk
          uint32_t w[2][2][4], sc[2][2][2];  // codes; scales of the two groups
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const uint4 v = *reinterpret_cast<const uint4*>(row_w + (i * 16 + half * 8) * 128 + ((p ^ (g & 1)) * 64));
              w[i][half][0] = v.x, w[i][half][1] = v.y, w[i][half][2] = v.z, w[i][half][3] = v.w;
              const uint8_t* at_s = row_s[i][half] + p * 8;
              uint32_t two;
              if constexpr (kRow16) two = *reinterpret_cast<const uint16_t*>(at_s);
              else two = at_s[0] | (unit + p * 4 + t < a.K / kUnit ? uint32_t(at_s[1]) << 8 : 0u);  // (the last unit may be half of one)
              const uint32_t h = e4m3x2_to_h2(uint16_t(here ? two : 0u));
              sc[i][half][0] = __byte_perm(h, h, 0x1010), sc[i][half][1] = __byte_perm(h, h, 0x3232);
            }
#pragma unroll
          for (int j = 0; j < 4; ++j) {  // 8 codes of a row, two MMAs
            uint4 xf[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              xf[n] = *reinterpret_cast<const uint4*>(x_col[n] + (here ? x_off + p * 256 + t * 64 : 0) + ((j ^ x_swizzle) * 16));
              if (!here) xf[n] = make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              uint32_t cd[2][4];
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                e2m1x8_to_h2(w[i][half][j], cd[half]);
#pragma unroll
                for (int e = 0; e < 4; ++e) cd[half][e] = h2_mul(cd[half][e], sc[i][half][j / 2]);
              }
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                mma_16816(acc[i][n], cd[0][0], cd[1][0], cd[0][1], cd[1][1], xf[n].x, xf[n].y);
                mma_16816(acc[i][n], cd[0][2], cd[1][2], cd[0][3], cd[1][3], xf[n].z, xf[n].w);
              }
            }
          }
        };
        if (n_units == kChunkUnits) {
          piece(0, true), piece(1, true);
        } else {
#pragma unroll 1
          for (int p = 0; p * 4 < n_units; ++p) piece(p, p * 4 + t < n_units);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) total[i][n][j] += acc[i][n][j];
      }
      if (c > 1 && read_pending) cluster_wait(), read_pending = false;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const float(&v)[4] = total[i][n];
          const float4 s = make_float4(v[0] * inv[n][0], v[1] * inv[n][1], v[2] * inv[n][0], v[3] * inv[n][1]);
          const int at = pair * 2 + i;  // in the batch
          if (at >= batch_tiles) continue;
          if (alone) write_quad(tile + at, n, s);
          else sums[((at * parts + part) * NT + n) * 32 + lane] = s;
        }
    }
    if (alone) break;

    // ---- a meeting: the parts' sums into part 0's, the CTAs' at the one that writes them
    if (c > 1 && read_pending) cluster_wait(), read_pending = false;
    __syncthreads();
    if (parts > 1) {
#pragma unroll 1
      for (int i = tid; i < batch_tiles * NT * 32; i += kThreads) {
        float4* at = sums + size_t(i / (NT * 32)) * (parts * NT * 32) + i % (NT * 32);
        float4 s = *at;
#pragma unroll
        for (int p = 1; p < kWarps; ++p) {
          if (p >= parts) break;
          const float4 v = at[p * NT * 32];
          s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
        }
        if (c > 1) *at = s;
        else write_quad(tile + i / (NT * 32), i / 32 % NT, s);
      }
    }
    if (c > 1) {
      cluster_arrive_wait();
#pragma unroll 1
      for (int block = rank + warp * c; block < batch_tiles * NT; block += kWarps * c) {
        float4* at = sums + size_t(block / NT) * (parts * NT * 32) + block % NT * 32 + lane;
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int q = 0; q < c; ++q) {
          const float4 v = *cluster.map_shared_rank(at, q);
          s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
        }
        write_quad(tile + block / NT, block % NT, s);
      }
      cluster_arrive();  // this CTA has read the others' sums: waited for before they are written again
      read_pending = true;
    } else {
      __syncthreads();
    }
  }
  cp_wait<0>();
  if (c > 1 && read_pending) cluster_wait();  // no CTA leaves while another reads its sums
}

// ---------------------------------------------------------------------------------------------- launch
DeviceInfo g_devices[kMaxDevices];
std::mutex g_mutex;
int g_clusters[kMaxDevices][4];  // clusters of 1, 2, 4 and 8 CTAs that fit the device at a time

template <typename TX, int NT, bool kRow16>
int init_one(int* clusters) {
  auto* k = nvfp4_matvec_kernel<TX, NT, kRow16>;
  LB_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
  if (clusters[0] != 0) return LING_B200_OK;  // the same for all: one CTA a SM
  for (int i = 3; i >= 0; --i) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(1u << i), cfg.blockDim = dim3(kThreads), cfg.dynamicSmemBytes = kSmem;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 1u << i, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
    cfg.attrs = at, cfg.numAttrs = 1;
    int n = 0;
    LB_CUDA(cudaOccupancyMaxActiveClusters(&n, k, &cfg));
    clusters[i] = std::max(n, 1);
  }
  return LING_B200_OK;
}
template <typename TX>
int init_type(int* clusters) {
  if (const int r = init_one<TX, 1, true>(clusters)) return r;
  if (const int r = init_one<TX, 1, false>(clusters)) return r;
  if (const int r = init_one<TX, 2, true>(clusters)) return r;
  if (const int r = init_one<TX, 2, false>(clusters)) return r;
  if (const int r = init_one<TX, 4, true>(clusters)) return r;
  return init_one<TX, 4, false>(clusters);
}
int init_all(int device) {
  if (const int r = init_type<float>(g_clusters[device])) return r;
  if (const int r = init_type<__nv_bfloat16>(g_clusters[device])) return r;
  return init_type<__half>(g_clusters[device]);
}

// Whether `cols` columns of K activations fit a cluster of 8 CTAs beside the sums and the shortest rings: what every plan can fall back to.
bool fits(int K, int cols) {
  const long long chunks = ((long long)K + kUnit * kChunkUnits - 1) / (kUnit * kChunkUnits), cta_chunks = (chunks + 7) / 8;
  return cta_chunks * kChunkUnits * 64 * cols <= kSmem - kSumBlocks * 512 - 2 * kWarps * kStageBytes;
}

// CTAs and warps that share K: the split with the least estimated time.  A warp's stage takes its share of the SM's part of HBM (4736
// bytes at 5.5 a nanosecond), or the loaded latency of about 2 us over the stages in flight, or its instructions (about 700 ns and
// 150 a column tile beyond the first); a meeting costs about 0.7 us, of a cluster's CTAs 2 us.  false: `cols` columns of activations (in
// `nt` tiles of 8) fit no split.
struct Split {
  int c = 0, parts = 0, clusters = 0, stages = 0;
};
bool choose_split(const int* at_once, int N, int K, int nt, int cols, Split* out) {
  const int tiles = ceil_div(N, 16), chunks = ceil_div(K, kUnit * kChunkUnits);
  double best = 0;
  for (int i = 0; i < 4; ++i) {
    const int c = 1 << i, clusters = std::min(at_once[i], tiles), cta_chunks = ceil_div(chunks, c);
    if (i > 0 && chunks < c) continue;
    for (int parts = 1; parts <= kWarps; parts *= 2) {
      const int room = kSmem - cta_chunks * kChunkUnits * 64 * cols - (c * parts == 1 ? 0 : kSumBlocks * 512), stages = std::min(kMaxStages, room / (kWarps * kStageBytes));
      if (room < 0 || stages < 2) continue;
      const int groups = kWarps / parts, t = ceil_div(tiles, clusters), h = ceil_div(cta_chunks, parts);
      const int batch = c * parts == 1 ? t : std::max(kSumBlocks / (parts * nt) & ~1, 2);
      const double full = std::max({861.0, 2000.0 / (stages - 1), 700.0 + 150.0 * (nt - 1)});
      double cost = 0;
      for (int left = t; left > 0; left -= batch) {
        const int pairs = ceil_div(ceil_div(std::min(left, batch), 2), groups);
        cost += pairs * h * full + (c > 1 ? 2000.0 : parts > 1 ? 700.0 : 0.0);
      }
      if (!out->c || cost < best) best = cost, *out = Split{c, parts, clusters, stages};
    }
  }
  return out->c != 0;
}

template <typename TX, int NT>
int matvec_launch(MatvecArgs a, const Split& split, cudaStream_t s) {
  const bool row16 = a.K % 32 == 0 && aligned(a.values, 16) && aligned(a.scales, 2);
  a.parts = split.parts, a.stages = split.stages;
  a.tiles = ceil_div(a.N, 16) / split.clusters, a.more_tiles = ceil_div(a.N, 16) % split.clusters;
  LB_CUDA(launch_kernel_cluster(row16 ? nvfp4_matvec_kernel<TX, NT, true> : nvfp4_matvec_kernel<TX, NT, false>, dim3(split.clusters * split.c),
                                dim3(kThreads), size_t(kSmem), split.c, s, a));
  LB_LAUNCH("nvfp4_matvec_kernel");
  return LING_B200_OK;
}
// As many rows a launch as their activations fit beside the weights' rings, in 1, 2 or 4 tiles of 8 columns: at K = 5120 32 columns, at
// 17408 up to 25 at once, more as 16 and 16.
template <typename TX>
int matvec_rows(MatvecArgs a, int device, cudaStream_t s) {
  constexpr int kCols = sizeof(TX) == 4 ? 2 : 1;
  const TX* x = static_cast<const TX*>(a.x);
  for (int m = 0, rows; m < a.M; m += rows) {
    MatvecArgs b = a;
    Split split;
    int nt = 4, left = (a.M - m) * kCols;
    while (nt > 1 && left <= 4 * nt) nt /= 2;
    while (!choose_split(g_clusters[device], a.N, a.K, nt, std::min(left, 8 * nt), &split)) nt /= 2;  // (8 columns fit)
    rows = std::min(a.M - m, 8 * nt / kCols);
    b.x = x + m * a.ldx, b.M = rows, b.y = static_cast<uint8_t*>(a.y) + m * a.ldy * type_size(a.y_type);
    const int r = nt == 1 ? matvec_launch<TX, 1>(b, split, s) : nt == 2 ? matvec_launch<TX, 2>(b, split, s) : matvec_launch<TX, 4>(b, split, s);
    if (r) return r;
  }
  return LING_B200_OK;
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
  constexpr int kMaxN = 0x7fffffff - 31;  // (the kernel counts rows in pairs of 16-row tiles)
  if (!x || !values || !scales || !y || M < 1 || M > 32 || N < 1 || N > kMaxN || K < 16 || K % 16 != 0 || ldx < K || ldy < N ||
      !d4::aligned(x, d4::type_size(x_type)) || !d4::aligned(y, d4::type_size(y_type)) || !d4::aligned(values, 8)) {
    set_error("nvfp4_matvec: bad argument (1 <= M <= 32, K a multiple of 16, ldx >= K, ldy >= N, values on an 8-byte boundary)");
    return LING_B200_ERR_ARG;
  }
  if (!fits(K, std::min(8, M * (x_type == LING_B200_F32 ? 2 : 1)))) {
    set_error("nvfp4_matvec: K = " + std::to_string(K) + " is beyond the activations' shared memory");
    return LING_B200_ERR_UNSUPPORTED;
  }
  d4::DeviceGuard guard;
  int sms = 0;
  if (const int r = d4::enter_device(guard, device, g_devices, g_mutex, [device] { return init_all(device); }, &sms)) return r;
  MatvecArgs a{x, ldx, M, values, scales, alpha, N, K, y, ldy, y_type, accumulate, false, 1, 2, 0, 0};
  a.x_vec = d4::aligned(x, 16) && ldx * d4::type_size(x_type) % 16 == 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return x_type == LING_B200_F32 ? matvec_rows<float>(a, device, s)
         : x_type == LING_B200_BF16 ? matvec_rows<__nv_bfloat16>(a, device, s)
                                    : matvec_rows<__half>(a, device, s);
}
