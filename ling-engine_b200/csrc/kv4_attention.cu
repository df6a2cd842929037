// kv4_attention.cu -- attention over the paged NVFP4 KV cache (ling_b200_kv4_attention).
//
//   out[r][h] = sum_j p_j V_j / sum_j p_j,  p_j = exp(scale * q . K_j - m),  m = max_j scale * q . K_j,
// over the positions j that row r sees: [0, pos) of its sequence, and of the in-flight positions pos + i those its ancestor
// mask (or, without one, its index) admits.
#include <algorithm>

#include "decode4.cuh"

namespace lb {
namespace {
using namespace d4;

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kPShift = 8.f;  // probabilities are carried times 2^8 in FP16: clear of its subnormals down to 2^-22
constexpr int kStepKeys = 16;   // keys of one step of a warp: never crosses a page

struct AttnArgs {
  ling_b200_kv4 c;
  ling_b200_kv4_batch b;
  ling_b200_rows q, out;
  int q_heads;
  float scale;
  float* lse;
  int* err;
  unsigned* tickets;
  float* parts;
  bool q_vec;  // four elements of q start on a boundary of four elements
};

// ---------------------------------------------------------------------------------------------- few query rows
// The decode kernel: up to 8 query rows (row, head of the group) of one (sequence, kv head) against its context.  Bound by
// the cache's bytes, so everything else is kept off that stream's way:
//   tensor cores  S^T = K Q^T and O^T = V^T P^T by mma.sync m16n8k16: 16 keys (dims) are the MMA's M, the 8 query rows its N.
//                 A thread's A fragments are built in registers from the codes as the cache holds them: for S^T a thread takes one
//                 key's 4 neighbouring codes per MMA (the order of dims is free as long as Q's fragments follow it), for O^T
//                 the same byte of two neighbouring keys, nibbles merged so that one cvt gives (key, key + 1) of a dim.  P
//                 turns from an accumulator into a B fragment by movmatrix.  Values in FP16 are exact (E2M1 x E4M3 has 6
//                 significant bits); q goes to FP16 times a power of two of its row, which loses nothing that a sum in fp32 keeps.
//   loads         every warp streams its own 16-key steps by cp.async through a private ring of kStages; no block barriers
//                 inside a context.
//   balance       the steps of all (sequence, kv head, row tile) items lie end to end and are cut into equal ranges, one per
//                 CTA; an item that several CTAs share leaves partial results (O, m, l) and the last of them to arrive
//                 adds them in order, so a result does not depend on the order of arrival.
constexpr int kDecWarps = 8, kDecThreads = kDecWarps * 32, kDecRows = 8, kDecMaxCtas = 592;

__host__ __device__ constexpr int dec_stages(int D) { return D == 256 ? 3 : D == 128 ? 5 : 8; }
__host__ __device__ constexpr int dec_stage_bytes(int D) { return 18 * D; }  // 16 keys: codes 2 x 8 D, scales 2 x D
__host__ __device__ constexpr int dec_smem(int D) { return kDecWarps * dec_stages(D) * dec_stage_bytes(D); }
__host__ __device__ constexpr size_t dec_part_floats(int D) { return size_t(kDecRows) * D + 2 * kDecRows; }

template <int N>
__device__ __forceinline__ void cp_async(void* dst, const void* src) {
  const uint32_t a = static_cast<uint32_t>(__cvta_generic_to_shared(dst));
  if constexpr (N == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(a), "l"(src) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(a), "l"(src), "n"(N) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t movmatrix(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t h2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t h2_mul(uint32_t a, uint32_t b) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// B bytes of shared memory as 32-bit words.
template <int B>
__device__ __forceinline__ void lds(const uint8_t* p, uint32_t (&w)[B / 4]) {
  if constexpr (B == 16) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else if constexpr (B == 8) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x, w[1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

// What of the work lies where: an item is (sequence, kv head, tile of kDecRows query rows), `steps` 16-key steps long.
struct Item {
  int s, h, tile, steps;
  Kv4Seq sq;
};

template <typename T, int D>
__global__ void __launch_bounds__(kDecThreads, 1) kv4_decode_kernel(AttnArgs a) {
  pdl_sync();  // first statement: see common.cuh
  constexpr int S = dec_stages(D), KP = D == 256 ? 2 : 1, KB = D == 64 ? 8 : 16, VB = D / 16, SB = D / 16;
  constexpr int kK = 2 * KP * KB * 32, kV = 4 * VB * 32;  // bytes of a stage's K and V codes
  static_assert(kK == 8 * D && kV == 8 * D, "a stage holds 16 keys");
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ long long first[LING_B200_KV4_MAX_SEQS + 1];  // steps of the sequences before s
  __shared__ float ml[kDecWarps][2][kDecRows];
  __shared__ unsigned last;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int G = a.q_heads / a.c.kv_heads, H = a.c.kv_heads, T_page = a.c.page_tokens;

  // ---- the sequences' steps, end to end
  if (warp == 0) {
    long long sum = 0;
    for (int s0 = 0; s0 < a.b.seqs; s0 += 32) {
      const int s = s0 + lane;
      long long n = 0;
      if (s < a.b.seqs) {
        const Kv4Seq q = kv4_seq(a.c, a.b, s);
        if (!q.ok && blockIdx.x == 0) dev_fail(a.err, kDevBadBatch);
        if (q.ok && q.n > 0) n = (long long)((q.n * G + kDecRows - 1) / kDecRows) * H * ((q.pos + q.n + kStepKeys - 1) / kStepKeys);
      }
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, n, o);
        if (lane >= o) n += v;
      }
      if (s < a.b.seqs) first[s + 1] = sum + n;
      sum += __shfl_sync(0xffffffffu, n, 31);
    }
    if (lane == 0) first[0] = 0;
  }
  __syncthreads();
  const long long total = first[a.b.seqs];
  const long long quota = (total + gridDim.x - 1) / gridDim.x;
  long long at = quota * blockIdx.x;
  const long long end = min(total, at + quota);

  uint8_t* ring = smem + warp * (S * dec_stage_bytes(D));
  while (at < end) {
    // ---- the item that step `at` belongs to
    int lo = 0, hi = a.b.seqs;  // first[lo] <= at < first[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (first[mid] <= at) lo = mid; else hi = mid;
    }
    Item it;
    it.s = lo;
    it.sq = kv4_seq(a.c, a.b, lo);
    const int keys = it.sq.pos + it.sq.n, tiles = (it.sq.n * G + kDecRows - 1) / kDecRows;
    it.steps = (keys + kStepKeys - 1) / kStepKeys;
    const long long off = at - first[lo];
    const int which = int(off / it.steps), step0 = int(off % it.steps);
    it.h = which / tiles, it.tile = which % tiles;
    const int step1 = int(min((long long)it.steps, step0 + (end - at)));
    const long long item_first = at - step0;  // the item's steps are [item_first, item_first + steps)

    // ---- Q^T as B fragments: column g is query row f = tile * 8 + g, (row f / G, head f % G)
    uint32_t qb[D / 16][2];
    float inv;
    {
      const int f = it.tile * kDecRows + g;
      const bool real = f < it.sq.n * G;
      const T* src = static_cast<const T*>(a.q.p) + (it.sq.row0 + (real ? f / G : 0)) * a.q.row + (it.h * G + (real ? f % G : 0)) * a.q.head;
      float top = 0.f;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        const int d = D == 256 ? (kk / 8) * 128 + t * 32 + (kk % 8) * 4 : t * (D / 4) + kk * 4;
        T e[4];
        if (a.q_vec) {
          *reinterpret_cast<uint2*>(e) = *reinterpret_cast<const uint2*>(src + d);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) e[j] = src[d + j];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float v = fabsf(to_f32<T>(e[j]));
          top = v > top || v != v ? v : top;  // a NaN stays
        }
        qb[kk][0] = reinterpret_cast<uint32_t*>(e)[0], qb[kk][1] = reinterpret_cast<uint32_t*>(e)[1];
      }
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        const float v = __shfl_xor_sync(0xffffffffu, top, o);
        top = v > top || v != v ? v : top;
      }
      // the row times 2^(8 - exponent of its largest value): FP16 keeps 2^-25 of an element whose row reaches 2^8
      const int ex = int(__float_as_uint(top) >> 23 & 255u), field = min(max(262 - ex, 2), 252);
      const float mul = top == 0.f ? 1.f : top < INFINITY ? __uint_as_float(uint32_t(field) << 23) : NAN;
      inv = top > 0.f && top < INFINITY ? __uint_as_float(uint32_t(254 - field) << 23) : 1.f;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const T* e = reinterpret_cast<const T*>(&qb[kk][j]);
          qb[kk][j] = real ? h2(to_f32<T>(e[0]) * mul, to_f32<T>(e[1]) * mul) : 0u;
        }
    }
    // this thread's score columns are query rows 2t and 2t + 1
    const float to_log2 = a.scale * a.c.k_scale * kLog2e;
    float coef[2];
    uint32_t see[2];  // in-flight rows each sees, as a mask or (no masks) their number
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      coef[j] = to_log2 * __shfl_sync(0xffffffffu, inv, (2 * t + j) * 4);
      const int f = it.tile * kDecRows + 2 * t + j, i = f / G;
      see[j] = i >= it.sq.n ? 0u : a.b.anc ? a.b.anc[it.sq.row0 + i] : uint32_t(i + 1);
    }

    float o[D / 16][4] = {}, m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

    // ---- this warp's steps: step0 + warp, step0 + warp + 8, ...
    const int* table = a.c.tables + size_t(it.sq.slot) * a.c.max_pages;
    const int mine = (step1 - step0 - warp + kDecWarps - 1) / kDecWarps;
    int page_batch = 0;   // this lane's page of the current 32 steps
    uint32_t good = 0;    // of the steps on their way, youngest in bit 0: whether the page is one
    auto issue = [&](int n) {
      if (n < mine) {
        if ((n & 31) == 0) {
          const int st = step0 + warp + (n + lane) * kDecWarps;
          page_batch = n + lane < mine ? table[st * kStepKeys / T_page] : 0;
        }
        int page = __shfl_sync(0xffffffffu, page_batch, n & 31);
        const bool ok = page >= 1 && page <= a.c.pages;
        if (!ok) {
          if (lane == 0) dev_fail(a.err, kDevBadPage);
          page = 0;  // the reserved page: its keys are masked
        }
        good = good << 1 | (ok ? 1u : 0u);
        const int pos = (step0 + warp + n * kDecWarps) * kStepKeys;
        const size_t vec = kv4_vector(a.c, page, it.h, pos % T_page);
        uint8_t* st = ring + (n % S) * dec_stage_bytes(D);
        const uint8_t* k = a.c.k + vec * (D / 2) + g * (D / 2) + t * KB;
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int p = 0; p < KP; ++p) cp_async<KB>(st + ((half * KP + p) * 32 + lane) * KB, k + half * 8 * (D / 2) + p * 64);
        const uint8_t* v = a.c.v + vec * (D / 2) + 2 * t * (D / 2) + g * VB;
#pragma unroll
        for (int j = 0; j < 4; ++j) cp_async<VB>(st + kK + (j * 32 + lane) * VB, v + (j / 2 * 8 + j % 2) * (D / 2));
        const uint8_t* sc = (lane < 16 ? a.c.k_scales : a.c.v_scales) + vec * SB + (lane & 15) * SB;
        cp_async<SB>(st + kK + kV + lane * SB, sc);
      } else {
        good <<= 1;
      }
      cp_commit();
    };
#pragma unroll
    for (int n = 0; n < S - 1; ++n) issue(n);
    for (int n = 0; n < mine; ++n) {
      cp_wait<S - 2>();
      __syncwarp();  // step n has landed, for all lanes; all lanes are done with step n - 1, whose stage is next
      issue(n + S - 1);
      const uint8_t* st = ring + (n % S) * dec_stage_bytes(D);
      const uint8_t* ks = st + kK + kV;
      const uint8_t* vs = ks + D;
      const int pos0 = (step0 + warp + n * kDecWarps) * kStepKeys;
      const bool masked = !(good >> (S - 1) & 1u) || pos0 + kStepKeys > it.sq.pos;

      // scores
      float s[4] = {0.f, 0.f, 0.f, 0.f}, s2[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int p = 0; p < KP; ++p) {
        uint32_t w[2][KB / 4], sc[2][KB / 8];  // of keys g and g + 8: codes, scales by group as half2
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          lds<KB>(st + ((half * KP + p) * 32 + lane) * KB, w[half]);
          const uint8_t* at_s = ks + (half * 8 + g) * SB + (KB == 16 ? p * 8 + t * 2 : t);
          const uint32_t pair = KB == 16 ? *reinterpret_cast<const uint16_t*>(at_s) : *at_s;
          const uint32_t h = e4m3x2_to_h2(uint16_t(pair));
          sc[half][0] = __byte_perm(h, h, 0x1010);
          if constexpr (KB == 16) sc[half][1] = __byte_perm(h, h, 0x3232);
        }
#pragma unroll
        for (int i = 0; i < KB / 4; ++i) {  // word i: 8 codes, two MMAs
          uint32_t c[2][4];
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            e2m1x8_to_h2(w[half][i], c[half]);
#pragma unroll
            for (int j = 0; j < 4; ++j) c[half][j] = h2_mul(c[half][j], sc[half][i / 2]);
          }
          const int kk = p * (KB / 2) + i * 2;
          mma_16816(s, c[0][0], c[1][0], c[0][1], c[1][1], qb[kk][0], qb[kk][1]);
          mma_16816(s2, c[0][2], c[1][2], c[0][3], c[1][3], qb[kk + 1][0], qb[kk + 1][1]);
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) s[j] = (s[j] + s2[j]) * coef[j & 1];

      // V's scales: of this thread's key pairs (2t, 2t+1) and (2t+8, 2t+9), per group of its dims, as (key, key + 1)
      constexpr int VG = D == 256 ? 2 : 1;
      uint32_t vsc[2][VG];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint8_t* at_s = vs + (2 * t + j * 8) * SB + (D == 256 ? g * 2 : D == 128 ? g : g / 2);
        if constexpr (D == 256) {
          const uint32_t x = *reinterpret_cast<const uint16_t*>(at_s), y = *reinterpret_cast<const uint16_t*>(at_s + SB);
          vsc[j][0] = x & 0xffu | (y & 0xffu) << 8, vsc[j][1] = x >> 8 | y & 0xff00u;
        } else {
          vsc[j][0] = uint32_t(at_s[0]) | uint32_t(at_s[SB]) << 8;
        }
      }
      uint32_t poison = 0;  // of this thread's four (key, row): a visible key whose V is NaN
      if (masked) {
        // A V vector that is NaN must reach exactly the rows that see it: its scale is taken as 0 and its probability as NaN.
        uint32_t nan = 0;  // keys of this step
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int v = 0; v < VG; ++v)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if ((vsc[j][v] >> (8 * e) & 0x7fu) == 0x7fu) {
                nan |= 1u << (2 * t + j * 8 + e);
                vsc[j][v] &= e ? 0x00ffu : 0xff00u;
              }
        nan = __reduce_or_sync(0xffffffffu, nan);
        const bool page_ok = good >> (S - 1) & 1u;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int key = g + (j >> 1) * 8, pos = pos0 + key, i = pos - it.sq.pos;
          const uint32_t mask = see[j & 1];
          const bool visible = page_ok && pos < keys && (i < 0 || (a.b.anc ? (mask >> i & 1u) : i < int(mask)));
          if (!visible) s[j] = -INFINITY;
          else poison |= (nan >> key & 1u) << j;
        }
      }

      // running maximum and sum; rows are columns 2t, 2t + 1, keys lie across the lanes with the same t
      float mx[2] = {fmaxf(s[0], s[2]), fmaxf(s[1], s[3])};
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) mx[j] = fmaxf(mx[j], __shfl_xor_sync(0xffffffffu, mx[j], x));
        mx[j] = fmaxf(mx[j], m[j]);
      }
      if (__any_sync(0xffffffffu, mx[0] > m[0] || mx[1] > m[1])) {
        float keep[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          keep[j] = m[j] == -INFINITY ? 0.f : ex2(m[j] - mx[j]);
          l[j] *= keep[j];
          m[j] = mx[j];
        }
#pragma unroll
        for (int i = 0; i < D / 16; ++i) o[i][0] *= keep[0], o[i][2] *= keep[0], o[i][1] *= keep[1], o[i][3] *= keep[1];
      }
      float p[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) p[j] = ex2(s[j] - (m[j & 1] == -INFINITY ? 0.f : m[j & 1] - kPShift));
      l[0] += p[0] + p[2], l[1] += p[1] + p[3];
      if (poison) {
#pragma unroll
        for (int j = 0; j < 4; ++j) p[j] = poison >> j & 1u ? NAN : p[j];
      }
      const uint32_t b0 = movmatrix(h2(p[0], p[1])), b1 = movmatrix(h2(p[2], p[3]));

      // values
      uint32_t v[4][VB / 4], vh[2][VG];
#pragma unroll
      for (int j = 0; j < 4; ++j) lds<VB>(st + kK + (j * 32 + lane) * VB, v[j]);
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int x = 0; x < VG; ++x) vh[j][x] = e4m3x2_to_h2(uint16_t(vsc[j][x]));
#pragma unroll
      for (int i = 0; i < VB / 4; ++i) {  // word i: 8 dims, four MMAs' rows g (even dims) and g + 8 (odd dims)
        uint32_t even[2][4], odd[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint32_t x = v[2 * j][i], y = v[2 * j + 1][i];
          e2m1x8_to_h2(x & 0x0f0f0f0fu | (y & 0x0f0f0f0fu) << 4, even[j]);
          e2m1x8_to_h2(x >> 4 & 0x0f0f0f0fu | y & 0xf0f0f0f0u, odd[j]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t f = vh[j][VG == 2 ? i / 2 : 0];
            even[j][e] = h2_mul(even[j][e], f), odd[j][e] = h2_mul(odd[j][e], f);
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) mma_16816(o[i * 4 + e], even[0][e], odd[0][e], even[1][e], odd[1][e], b0, b1);
      }
    }
    cp_wait<0>();

    // ---- the warps' results meet in shared memory (each warp's own ring), raw: [D / 16][lane][4]
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) l[j] += __shfl_xor_sync(0xffffffffu, l[j], x);
    __syncwarp();
    float4* mine_o = reinterpret_cast<float4*>(ring);
#pragma unroll
    for (int i = 0; i < D / 16; ++i) mine_o[i * 32 + lane] = make_float4(o[i][0], o[i][1], o[i][2], o[i][3]);
    if (lane < 4) ml[warp][0][2 * lane] = m[0], ml[warp][0][2 * lane + 1] = m[1], ml[warp][1][2 * lane] = l[0], ml[warp][1][2 * lane + 1] = l[1];
    __syncthreads();
    const bool whole = step0 == 0 && step1 == it.steps;
    constexpr int kQuads = D / 16 * 32, kEach = (kQuads + kDecThreads - 1) / kDecThreads;
    float4 acc[kEach];
    float mm[2], ll[2];  // of this thread's rows 2t', 2t' + 1 (t' of the quad's lane: the same for all its quads)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int row = 2 * t + j;
      mm[j] = -INFINITY, ll[j] = 0.f;
#pragma unroll
      for (int w = 0; w < kDecWarps; ++w) mm[j] = fmaxf(mm[j], ml[w][0][row]);
    }
#pragma unroll
    for (int e = 0; e < kEach; ++e) acc[e] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kDecWarps; ++w) {
      float f[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float mw = ml[w][0][2 * t + j];
        f[j] = mw == -INFINITY ? (ml[w][1][2 * t + j] == 0.f ? 0.f : 1.f) : ex2(mw - mm[j]);
        ll[j] = fmaf(ml[w][1][2 * t + j], f[j], ll[j]);
      }
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        const int quad = tid + e * kDecThreads;
        if (quad < kQuads) {
          const float4 x = reinterpret_cast<const float4*>(smem + w * (S * dec_stage_bytes(D)))[quad];
          acc[e].x = fmaf(x.x, f[0], acc[e].x), acc[e].y = fmaf(x.y, f[1], acc[e].y);
          acc[e].z = fmaf(x.z, f[0], acc[e].z), acc[e].w = fmaf(x.w, f[1], acc[e].w);
        }
      }
    }
    bool write = whole;
    if (!whole) {
      // ---- a part of the item: left for the last of its CTAs.  A CTA has at most two parts: of the item it opens with (slot
      // 0) and of one that goes on behind it (slot 1), whose ticket is the CTA's own.
      const int cta0 = int(item_first / quota), cta1 = int((item_first + it.steps - 1) / quota);
      const bool head = int(blockIdx.x) == cta0;
      float* part = a.parts + (size_t(blockIdx.x) * 2 + (head ? 1 : 0)) * dec_part_floats(D);
#pragma unroll
      for (int e = 0; e < kEach; ++e)
        if (tid + e * kDecThreads < kQuads) reinterpret_cast<float4*>(part)[tid + e * kDecThreads] = acc[e];
      if (tid < 4) {
        float* pm = part + kDecRows * D;
        pm[2 * tid] = mm[0], pm[2 * tid + 1] = mm[1], pm[kDecRows + 2 * tid] = ll[0], pm[kDecRows + 2 * tid + 1] = ll[1];
      }
      __threadfence();
      __syncthreads();
      if (tid == 0) last = atomicInc(&a.tickets[cta0], unsigned(cta1 - cta0)) == unsigned(cta1 - cta0) ? 1u : 0u;
      __syncthreads();
      write = last != 0;
      if (write) {
        __threadfence();
        mm[0] = mm[1] = -INFINITY, ll[0] = ll[1] = 0.f;
        for (int c = cta0; c <= cta1; ++c) {
          const float* pm = a.parts + (size_t(c) * 2 + (c == cta0 ? 1 : 0)) * dec_part_floats(D) + kDecRows * D;
#pragma unroll
          for (int j = 0; j < 2; ++j) mm[j] = fmaxf(mm[j], __ldcg(pm + 2 * t + j));
        }
#pragma unroll
        for (int e = 0; e < kEach; ++e) acc[e] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int c = cta0; c <= cta1; ++c) {
          const float* pp = a.parts + (size_t(c) * 2 + (c == cta0 ? 1 : 0)) * dec_part_floats(D);
          const float* pm = pp + kDecRows * D;
          float f[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float mw = __ldcg(pm + 2 * t + j), lw = __ldcg(pm + kDecRows + 2 * t + j);
            f[j] = mw == -INFINITY ? (lw == 0.f ? 0.f : 1.f) : ex2(mw - mm[j]);
            ll[j] = fmaf(lw, f[j], ll[j]);
          }
#pragma unroll
          for (int e = 0; e < kEach; ++e) {
            const int quad = tid + e * kDecThreads;
            if (quad < kQuads) {
              const float4 x = __ldcg(reinterpret_cast<const float4*>(pp) + quad);
              acc[e].x = fmaf(x.x, f[0], acc[e].x), acc[e].y = fmaf(x.y, f[1], acc[e].y);
              acc[e].z = fmaf(x.z, f[0], acc[e].z), acc[e].w = fmaf(x.w, f[1], acc[e].w);
            }
          }
        }
      }
    }
    if (write) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int f = it.tile * kDecRows + 2 * t + j;
        if (f >= it.sq.n * G) continue;
        const int row = it.sq.row0 + f / G, head = it.h * G + f % G;
        const bool empty = mm[j] == -INFINITY && ll[j] == 0.f;
        const float scale = empty ? 0.f : a.c.v_scale / ll[j];
        T* to = static_cast<T*>(a.out.p) + row * a.out.row + head * a.out.head;
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
          const int quad = tid + e * kDecThreads;
          if (quad < kQuads) {
            const int d = (quad % 32 / 4) * (D / 8) + quad / 32 * 2;  // raw quad (i, lane): dims 2 i, 2 i + 1 of lane's chunk
            to[d] = from_f32<T>(empty ? 0.f : (j ? acc[e].y : acc[e].x) * scale);
            to[d + 1] = from_f32<T>(empty ? 0.f : (j ? acc[e].w : acc[e].z) * scale);
          }
        }
        if (a.lse && tid < 4) a.lse[size_t(row) * a.q_heads + head] = empty ? -INFINITY : (mm[j] + log2f(ll[j]) - kPShift) * kLn2;
      }
    }
    __syncthreads();  // the shared results are read: the rings are free
    at += step1 - step0;
  }
}

template <typename T, int D>
int decode_init() {
  LB_CUDA(cudaFuncSetAttribute(kv4_decode_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, dec_smem(D)));
  return LING_B200_OK;
}
template <typename T>
int decode_init_all() {
  if (const int r = decode_init<T, 64>()) return r;
  if (const int r = decode_init<T, 128>()) return r;
  return decode_init<T, 256>();
}
int attention_init() {
  if (const int r = decode_init_all<__nv_bfloat16>()) return r;
  return decode_init_all<__half>();
}
template <typename T>
int decode_launch(const AttnArgs& a, int sms, cudaStream_t s) {
  auto* k = a.c.head_dim == 64 ? kv4_decode_kernel<T, 64> : a.c.head_dim == 128 ? kv4_decode_kernel<T, 128> : kv4_decode_kernel<T, 256>;
  const int grid = std::min(sms, kDecMaxCtas);
  LB_CUDA(launch_kernel(k, dim3(grid), dim3(kDecThreads), size_t(dec_smem(a.c.head_dim)), s, a));
  LB_LAUNCH("kv4_decode_kernel");
  return LING_B200_OK;
}

DeviceInfo g_devices[kMaxDevices];
std::mutex g_mutex;

constexpr size_t kTicketBytes = size_t(kDecMaxCtas + 15) / 16 * 64;

bool heads_ok(const ling_b200_kv4* c, int q_heads, const char* who) {
  if (q_heads >= 1 && q_heads <= 1024 && q_heads % c->kv_heads == 0) return true;
  set_error(std::string(who) + ": q_heads must be a multiple of kv_heads, at most 1024");
  return false;
}

}  // namespace
}  // namespace lb

using namespace lb;
using namespace lb::d4;

extern "C" size_t ling_b200_kv4_attention_workspace(const ling_b200_kv4* cache, const ling_b200_kv4_batch* batch, int q_heads) {
  const char* who = "kv4_attention_workspace";
  if (!kv4_cache_ok(cache, who) || !kv4_batch_ok(cache, batch, who) || !heads_ok(cache, q_heads, who)) return 0;
  return kTicketBytes + size_t(kDecMaxCtas) * 2 * dec_part_floats(cache->head_dim) * 4;
}

extern "C" int ling_b200_kv4_attention(int device, const ling_b200_kv4* cache, const ling_b200_kv4_batch* batch, int type,
                                       const ling_b200_rows* q, int q_heads, float scale, const ling_b200_rows* out, float* lse,
                                       void* workspace, size_t workspace_bytes, int* err, void* stream) {
  const char* who = "kv4_attention";
  if (!kv4_cache_ok(cache, who) || !kv4_batch_ok(cache, batch, who) || !heads_ok(cache, q_heads, who)) return LING_B200_ERR_ARG;
  if (type != LING_B200_BF16 && type != LING_B200_F16) {
    set_error("kv4_attention: queries are LING_B200_BF16 or LING_B200_F16");
    return LING_B200_ERR_ARG;
  }
  if (!kv4_rows_ok(q, type, q_heads, cache->head_dim, who, "q") || !kv4_out_ok(out, type, batch->rows, q_heads, cache->head_dim, who, "out"))
    return LING_B200_ERR_ARG;
  if (!std::isfinite(scale) || !aligned(lse, 4) || !aligned(err, 4)) {
    set_error("kv4_attention: scale must be finite, lse and err aligned");
    return LING_B200_ERR_ARG;
  }
  const size_t need = ling_b200_kv4_attention_workspace(cache, batch, q_heads);
  if (!workspace || workspace_bytes < need || !aligned(workspace, 16)) {
    set_error("kv4_attention: a 16-byte aligned workspace of " + std::to_string(need) + " bytes expected");
    return LING_B200_ERR_ARG;
  }
  if (batch->rows == 0 || batch->max_rows == 0) return LING_B200_OK;
  DeviceGuard guard;
  int sms = 0;
  if (const int r = enter_device(guard, device, g_devices, g_mutex, attention_init, &sms)) return r;
  AttnArgs a{*cache, *batch, *q, *out, q_heads, scale, lse, err, static_cast<unsigned*>(workspace),
             reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kTicketBytes), false};
  a.q_vec = aligned(q->p, 8) && q->row % 4 == 0 && q->head % 4 == 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return type == LING_B200_BF16 ? decode_launch<__nv_bfloat16>(a, sms, s) : decode_launch<__half>(a, sms, s);
}
