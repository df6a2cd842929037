// kv4_attention.cu -- attention over the paged NVFP4 KV cache (ling_b200_kv4_attention).
//
//   out[r][h] = sum_j p_j V_j / sum_j p_j,  p_j = exp(scale * q . K_j - m),  m = max_j scale * q . K_j,
// over the positions j that row r sees: [0, pos) of its sequence, and of the in-flight positions pos + i those its ancestor
// mask (or, without one, its index) admits.
#include <algorithm>

#include "decode4.cuh"
#include "tc.cuh"

namespace lb {
namespace {
using namespace d4;

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// A tensor core cuts its fp32 sums off instead of rounding them, so a long chain of MMAs drifts towards 0: by 6e-9 of the sum a position,
// measured (4e-3 over 2^19 positions).  The value product's chains end after these many positions (2.5e-5, in the tile kernel, which
// waits for its MMAs there, 5e-5) and are added in fp32.
constexpr int kChainKeys = 4096, kTileChainKeys = 8192;
constexpr float kPShift = 8.f;  // probabilities are carried times 2^8 in FP16: clear of its subnormals down to 2^-22

struct Join;
struct AttnArgs {
  ling_b200_kv4 c;
  ling_b200_kv4_batch b;
  ling_b200_rows q, out;
  int q_heads;
  float scale;
  float* lse;
  int* err;
  Join* joins;
  float* parts;
  float* totals;  // sums of the chains that have ended (kChainKeys), where contexts are longer than one
  bool q_vec, out_vec;  // rows of q, of out start on 16-byte boundaries
};

// ---------------------------------------------------------------------------------------------- few query rows
// The decode kernel: up to 8 query rows (row, head of the group) of one (sequence, kv head) against its context.  Bound by
// the cache's bytes, so everything else is kept off that stream's way:
//   tensor cores  S^T = K Q^T and O^T = V^T P^T by mma.sync m16n8k16: 16 keys (dims) are the MMA's M, the 8 query rows its N.
//                 A thread's A fragments are built in registers from the codes as the cache holds them: for S^T a thread takes one
//                 key's 4 neighbouring codes per MMA (the order of dims is free as long as Q's fragments follow it), for O^T
//                 the same byte of two neighbouring keys, nibbles merged so that one cvt gives (key, key + 1) of a dim.  P
//                 turns from an accumulator into a B fragment by movmatrix.  Values in FP16 are exact (E2M1 x E4M3 has 6
//                 significant bits); q goes to FP16 times a power of two of its row: an element is off by at most 2^-33 of the
//                 row's largest, under what a sum in fp32 keeps as long as the largest meet keys that are not 0.
//   loads         every warp streams its own steps (4.5 KB: 16, 32 or 64 keys) by cp.async through a private ring; the ring runs
//                 on across the items of a CTA, and nothing inside an item waits for another warp.
//   balance       the steps of all (sequence, kv head, row tile) items lie end to end and are cut into equal ranges, one per
//                 worker: a CTA, whose warps take its steps in turn and add their results in shared memory, or (kSolo) a warp on
//                 its own, which meets nobody.  An item that several workers share leaves partial results (O, m, l), which a
//                 second kernel, launched dependent so that its start overlaps the first one's end, adds in order.
// Measured, both kernels: one token over 128k positions (24 query heads on 4 kv heads of 256) 48.5 us, 3.1 TB/s of cache read; 64 tokens
// over 1k to 8k positions (32 on 8 of 128) 102 us, 3.5 TB/s, over up to 64k (24 on 4 of 256) 648 us, 3.9 TB/s (6.5 TB/s is a plain copy).
// No unit is full there (issue slots 40 to 48 % busy, DRAM 39 to 43 %, tensor pipe 18 to 21 %): two warps a scheduler wait for their own
// conversions and MMAs.  8k positions 15 us: a launch, the plan, one ring's latency, the meeting, the join.
constexpr int kDecRows = 8, kDecMaxCtas = 160;
constexpr int kDecWarps = 8, kDecThreads = kDecWarps * 32, kDecMaxWorkers = kDecMaxCtas * kDecWarps;
// Items from which warps work alone.  Measured, meeting / alone, 4 kv heads: 48 items of 8k positions 31 / 36 us, 64 items 41 / 41,
// 80 items 46 / 43, 256 items 108 / 95; of 1k positions 48 items 23 / 19, 64 items 18 / 20, 256 items 51 / 36.
constexpr int kSoloItems = 74;
constexpr float kLazy = 7.f;  // a score may exceed the running reference by this (log2) before the sums are scaled anew

__host__ __device__ constexpr int dec_stages(int D) { return D == 256 ? 4 : 5; }
__host__ __device__ constexpr int dec_sub(int D) { return 256 / D; }       // 16-key blocks of a step
__host__ __device__ constexpr int dec_block_bytes(int D) { return 18 * D; }  // 16 keys: codes 2 x 8 D, scales 2 x D
__host__ __device__ constexpr int dec_stage_bytes(int D) { return dec_sub(D) * dec_block_bytes(D); }
__host__ __device__ constexpr int dec_q_stride(int D) { return 2 * D + 16; }  // bytes of a query row in shared memory (padded against bank conflicts)
__host__ __device__ constexpr int dec_q_bytes(int D) { return kDecRows * dec_q_stride(D); }
__host__ __device__ constexpr int dec_sum_bytes(int D) { return 32 * D; }   // a warp's O, raw: [D / 16][lane][4] floats
__host__ __device__ constexpr int dec_smem(int D) {
  return kDecWarps * dec_stages(D) * dec_stage_bytes(D) + kDecWarps / 2 * dec_sum_bytes(D) + dec_stages(D) * dec_q_bytes(D);
}
__host__ __device__ constexpr size_t dec_part_floats(int D) { return size_t(kDecRows) * D + 2 * kDecRows; }

// An item that goes on behind the CTA it starts in: what the join needs of it.  parts = 0: none.
struct Join {
  int parts, row0, rows, h, tile, pad[3];
};

// N bytes from src + SRC to the shared address dst + DST (the offsets ride in the instruction).
template <int N, int DST, int SRC>
__device__ __forceinline__ void cp_async(uint32_t dst, const void* src) {
  if constexpr (N == 16) asm volatile("cp.async.cg.shared.global [%0 + %2], [%1 + %3], 16;" ::"r"(dst), "l"(src), "n"(DST), "n"(SRC) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0 + %2], [%1 + %3], %4;" ::"r"(dst), "l"(src), "n"(DST), "n"(SRC), "n"(N) : "memory");
}
// One 16-key block into a stage, by whole 512-byte lines of the cache: k, v and sc are the block's bytes from this lane's 16 (its
// share of the scales) on.  Where a line lands is arranged so that the fragments are read without bank conflicts:
//   K  key k, 16-byte chunk c:  D = 256: k * 128 + (c ^ 4 (k & 1)) * 16;  else as in the cache
//   V  D = 256: key k, chunk c: k * 128 + (c ^ 2 t) * 16;  else the keys 2t + (j & 1) + 8 (j >> 1) in the order (j, t), D = 128 with chunk c
//      at c ^ 2 (t >> 1)
struct BlockDst {
  uint32_t k, v, v2, sc;  // offsets of this lane in a stage (v2: V's second and fourth line, D = 256)
};
template <int D>
__device__ __forceinline__ BlockDst block_dst(int lane) {
  BlockDst d;
  const int r = lane >> 3, c = lane & 7, r4 = lane >> 2, c4 = lane & 3, r2 = lane >> 1, c2 = lane & 1;
  if constexpr (D == 256) {
    d.k = r * 128 + ((c ^ (r & 1) * 4) * 16);
    d.v = r * 128 + ((c ^ (r >> 1) * 2) * 16), d.v2 = r * 128 + ((c ^ (4 + (r >> 1) * 2)) * 16);
  } else if constexpr (D == 128) {
    d.k = lane * 16;
    d.v = (r4 & 1) * 256 + (r4 >> 1) * 64 + ((c4 ^ (r4 >> 2) * 2) * 16), d.v2 = d.v;
  } else {
    d.k = lane * 16;
    d.v = ((r2 >> 3) * 2 + (r2 & 1)) * 128 + (r2 >> 1 & 3) * 32 + c2 * 16, d.v2 = d.v;
  }
  d.sc = lane * (D / 16);
  return d;
}
template <int D>
__device__ __forceinline__ void cp_block(uint32_t stage, const BlockDst& d, const uint8_t* k, const uint8_t* v, const uint8_t* sc) {
  cp_async<16, 0, 0>(stage + d.k, k);
  if constexpr (D >= 128) cp_async<16, 512, 512>(stage + d.k, k);
  if constexpr (D == 256) cp_async<16, 1024, 1024>(stage + d.k, k), cp_async<16, 1536, 1536>(stage + d.k, k);
  cp_async<16, 8 * D, 0>(stage + d.v, v);
  if constexpr (D >= 128) cp_async<16, 8 * D + 512, 512>(stage + d.v2, v);
  if constexpr (D == 256) cp_async<16, 8 * D + 1024, 1024>(stage + d.v, v), cp_async<16, 8 * D + 1536, 1536>(stage + d.v2, v);
  cp_async<D / 16, 16 * D, 0>(stage + d.sc, sc);
}
// Where this thread (g, t) finds piece p of key half * 8 + g, and its dims of V's key 2t + (j & 1) + 8 (j >> 1).
template <int D>
__device__ __forceinline__ int k_offset(int g, int t, int half, int p) {
  if constexpr (D == 256) return (half * 8 + g) * 128 + (((p * 4 + t) ^ (g & 1) * 4) * 16);
  return (half * 8 + g) * (D / 2) + t * (D / 8);
}
template <int D>
__device__ __forceinline__ int v_offset(int g, int t, int j) {
  if constexpr (D == 256) return (2 * t + (j & 1) + (j >> 1) * 8) * 128 + ((g ^ 2 * t) * 16);
  if constexpr (D == 128) return (j * 4 + t) * 64 + (((g >> 1) ^ (t >> 1) * 2) * 16) + (g & 1) * 8;
  return j * 128 + t * 32 + g * 4;
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
__device__ __forceinline__ uint32_t movmatrix(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
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
// Two fp32 operations an instruction.
__device__ __forceinline__ uint64_t f2_pack(float lo, float hi) { return uint64_t(__float_as_uint(hi)) << 32 | __float_as_uint(lo); }
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float f2_lo(uint64_t a) { return __uint_as_float(uint32_t(a)); }
__device__ __forceinline__ float f2_hi(uint64_t a) { return __uint_as_float(uint32_t(a >> 32)); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// What a row's raw scores are worth as powers of two; never 0 (a scale of 0, or a product below fp32): a masked score is -inf.
__device__ __forceinline__ float score_coef(const AttnArgs& a, float q_inv) { return fmaxf(fabsf(a.scale) * a.c.k_scale * kLog2e * q_inv, 0x1p-126f); }
// What a partial result (reference m, sum l) counts for under the common reference: one without a visible key has l = 0, one whose
// scores were all NaN has l = NaN and no m.
__device__ __forceinline__ float part_weight(float m, float l, float common) { return m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : ex2(m - common); }
// What a chain that ended under the reference `then` counts for under `now` (-inf both: no visible key yet, or NaN alone).
__device__ __forceinline__ float chain_weight(float then, float now) { return then == now ? 1.f : ex2(then - now); }
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

// Writes quad `quad` of an item's result: of the raw order [D / 16][lane][4], entry (i, lane) holds dims 2 i and 2 i + 1 of the
// lane's D / 8 dims for query rows 2t and 2t + 1, as (row 2t, row 2t+1) of the first, then of the second dim.
template <typename T, int D>
__device__ __forceinline__ void store_quad(const AttnArgs& a, int row0, int n, int h, int tile, int quad, const float4& acc, const float (&mm)[2], const float (&ll)[2]) {
  const int G = a.q_heads / a.c.kv_heads, lane = quad % 32, t = lane & 3, d = lane / 4 * (D / 8) + quad / 32 * 2;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int f = tile * kDecRows + 2 * t + j;
    if (f >= n * G) continue;
    const int row = row0 + f / G, head = h * G + f % G;
    const bool empty = mm[j] == -INFINITY && ll[j] == 0.f;
    const float scale = empty ? 0.f : a.c.v_scale / ll[j];
    T* to = static_cast<T*>(a.out.p) + row * a.out.row + head * a.out.head + d;
    to[0] = from_f32<T>(empty ? 0.f : (j ? acc.y : acc.x) * scale);
    to[1] = from_f32<T>(empty ? 0.f : (j ? acc.w : acc.z) * scale);
    if (a.lse && quad < 4) a.lse[size_t(row) * a.q_heads + head] = empty ? -INFINITY : (mm[j] + log2f(ll[j]) - kPShift) * kLn2;
  }
}

template <typename T, int D, bool kSolo>
__global__ void __launch_bounds__(kDecThreads, 1) kv4_decode_kernel(AttnArgs a) {
  pdl_sync();  // first statement: see common.cuh
  constexpr int S = dec_stages(D), U = dec_sub(D), kKeys = 16 * U, kHalf = kDecWarps / 2;
  constexpr int KP = D == 256 ? 2 : 1, KB = D == 64 ? 8 : 16, VB = D / 16, SB = D / 16;
  constexpr int kK = 8 * D, kV = 8 * D;  // bytes of a block's K and V codes
  constexpr int kStride = kSolo ? 1 : kDecWarps, kMinSteps = kSolo ? 4 : kDecWarps;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int first[LING_B200_KV4_MAX_SEQS + 1], steps_of[LING_B200_KV4_MAX_SEQS];  // steps of the sequences before s; of an item of s
  __shared__ float ml[kDecWarps][2][kDecRows];
  __shared__ int quota_sh;    // steps of a worker
  __shared__ bool round_sh;   // whether an item takes whole ranges
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int workers = int(gridDim.x) * (kSolo ? kDecWarps : 1), me = kSolo ? int(blockIdx.x) * kDecWarps + warp : int(blockIdx.x);
  const int turn = kSolo ? 0 : warp;  // the worker's steps this warp takes: turn, turn + kStride, ..
  const int G = a.q_heads / a.c.kv_heads, H = a.c.kv_heads, lp = 31 - __clz(a.c.page_tokens);
  uint8_t* ring = smem + warp * (S * dec_stage_bytes(D));
  uint8_t* sums = smem + kDecWarps * S * dec_stage_bytes(D);
  uint8_t* q_raw = sums + kHalf * dec_sum_bytes(D);
  const uint32_t ring_u32 = static_cast<uint32_t>(__cvta_generic_to_shared(ring));

  // ---- the items' steps, end to end, and a range of them for every worker (warp 0 counts)
  if (warp == 0) {
    int sum = 0, items = 0;
    bool down = false;
    for (int s = lane; s < a.b.seqs; s += 32) {
      const Kv4Seq q = kv4_seq(a.c, a.b, s);
      if (!q.ok && blockIdx.x == 0) dev_fail(a.err, kDevBadBatch);
      down |= q.n < 0;
      const int mine = q.ok && q.n > 0 ? (q.n * G + kDecRows - 1) / kDecRows * H : 0;
      steps_of[s] = mine > 0 ? (q.pos + q.n + kKeys - 1) / kKeys : 0;
      first[s + 1] = mine;
      sum += mine * steps_of[s], items += mine;
    }
    sum = __reduce_add_sync(0xffffffffu, sum), items = __reduce_add_sync(0xffffffffu, items);
    if (__any_sync(0xffffffffu, down)) {  // row0 descends: sequences may share rows, none of them is done
      for (int s = lane; s < a.b.seqs; s += 32) first[s + 1] = 0, steps_of[s] = 0;
      sum = items = 0;
    }
    // no range is shorter than kMinSteps (a step for every warp of a CTA), unless the contexts themselves are
    int quota = max(max((sum + workers - 1) / workers, min(kMinSteps, sum / max(items, 1))), 1);
    const bool round = 4 * items <= workers;
    if (round) {
      // Several workers to an item: it takes whole ranges, so that no worker pays for two items (at most an eighth of them is lost to
      // rounding).  The shortest range that suffices:
      auto ranges = [&](int q) {
        int n = 0;
        for (int s = lane; s < a.b.seqs; s += 32) n += first[s + 1] * ((steps_of[s] + q - 1) / q);
        return __reduce_add_sync(0xffffffffu, n);
      };
      int lo = quota - 1, hi = quota;
      while (ranges(hi) > workers) lo = hi, hi *= 2;
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (ranges(mid) > workers) lo = mid; else hi = mid;
      }
      quota = hi;
    }
    sum = 0;
    for (int s0 = 0; s0 < a.b.seqs; s0 += 32) {
      const int s = s0 + lane;
      int n = s < a.b.seqs ? first[s + 1] * (round ? (steps_of[s] + quota - 1) / quota * quota : steps_of[s]) : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, n, o);
        if (lane >= o) n += v;
      }
      if (s < a.b.seqs) first[s + 1] = sum + n;
      sum += __shfl_sync(0xffffffffu, n, 31);
    }
    if (lane == 0) first[0] = 0, quota_sh = quota, round_sh = round;
  }
  __syncthreads();
  const int total = first[a.b.seqs], quota = quota_sh;
  const bool round = round_sh;
  const int begin = min(total, quota * me), end = min(total, begin + quota);
  if (kSolo ? lane == 0 : tid == 0) a.joins[me].parts = 0;
  if (begin >= end) return;

  // The part of an item that starts at step `at` of this worker's range: first[seq] <= at < first[seq + 1].
  struct Part {
    Kv4Seq sq;
    int keys, steps, step0, step1, next, h, tile, mine;  // mine: this warp's steps, step0 + turn and on by kStride
  };
  auto part_at = [&](int at) {
    int seq = 0, hi = a.b.seqs;
    while (hi - seq > 1) {
      const int mid = (seq + hi) / 2;
      if (first[mid] <= at) seq = mid; else hi = mid;
    }
    Part p;
    p.sq = kv4_seq(a.c, a.b, seq);
    p.keys = p.sq.pos + p.sq.n;
    p.steps = steps_of[seq];
    const int len = round ? (p.steps + quota - 1) / quota * quota : p.steps;
    const int tiles = (p.sq.n * G + kDecRows - 1) / kDecRows, which = (at - first[seq]) / len;
    p.step0 = (at - first[seq]) - which * len;
    p.step1 = min(p.steps, p.step0 + (end - at));
    p.next = round ? end : at + (p.step1 - p.step0);
    p.h = which / tiles, p.tile = which - p.h * tiles;
    p.mine = max(0, (p.step1 - p.step0 - turn + kStride - 1) / kStride);
    return p;
  };

  // ---- the loading side: runs S - 1 steps ahead of the computing side, across items
  const BlockDst dst = block_dst<D>(lane);
  const uint8_t* k_lane = a.c.k + lane * 16;
  const uint8_t* v_lane = a.c.v + lane * 16;
  const uint8_t* s_lane = (lane < 16 ? a.c.k_scales : a.c.v_scales) + (lane & 15) * SB;
  int in_at = begin, in_part = 0;             // the next item part to load from, and its number among the worker's
  int in_n = 0, in_mine = 0, in_pos = 0, in_keys = 0, in_h = 0;  // of the current one: this warp's steps, first position, ..
  const int* in_table = nullptr;
  int put = 0;          // the ring's next stage to fill
  uint32_t block_of = 0, block_ok = 0;  // of the current 32 blocks: this lane's, among the cache's blocks of 16 tokens; whether the pages are ones
  uint32_t good = 0;    // of the steps on their way, U bits each, youngest lowest: whether the blocks' pages are ones
  auto issue = [&]() {
    while (in_n == in_mine && in_at < end) {
      const Part p = part_at(in_at);
      in_at = p.next;
      in_n = 0, in_mine = p.mine, in_pos = (p.step0 + turn) * kKeys, in_keys = p.keys, in_h = p.h;
      in_table = a.c.tables + size_t(p.sq.slot) * a.c.max_pages;
      // the query rows, row f = tile * 8 + r being (row f / G, head f % G): into shared memory as they are, or (kSolo) on their way to L2
      if (kSolo || warp == 0) {
        uint8_t* to = q_raw + in_part % S * dec_q_bytes(D);
        for (int i = lane; i < kDecRows * (D / 8); i += 32) {
          const int r = i / (D / 8), f = p.tile * kDecRows + r;
          if (f >= p.sq.n * G) break;
          const T* src = static_cast<const T*>(a.q.p) + (p.sq.row0 + f / G) * a.q.row + (p.h * G + f % G) * a.q.head + i % (D / 8) * 8;
          uint8_t* dst = to + r * dec_q_stride(D) + i % (D / 8) * 16;
          if constexpr (kSolo) {
            asm volatile("prefetch.global.L2 [%0];" ::"l"(src));
          } else if (a.q_vec) {
            cp_async<16, 0, 0>(static_cast<uint32_t>(__cvta_generic_to_shared(dst)), src);
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) reinterpret_cast<T*>(dst)[j] = src[j];
          }
        }
      }
      ++in_part;
    }
    if (in_n < in_mine) {
      if ((in_n * U & 31) == 0) {  // the next 32 blocks: a lane looks one up
        const int pos = in_pos + (in_n + lane / U) * (kStride * kKeys) + lane % U * 16;
        const bool there = in_n + lane / U < in_mine && pos < in_keys;
        const int page = there ? in_table[pos >> lp] : 0;
        const bool ok = page >= 1 && page <= a.c.pages;
        if (there && !ok) dev_fail(a.err, kDevBadPage);
        block_ok = __ballot_sync(0xffffffffu, ok);  // the others are masked later; the reserved page stands in
        block_of = ((uint32_t(ok ? page : 0) * H + in_h) << (lp - 4)) + ((pos & ((1 << lp) - 1)) >> 4);
      }
      uint32_t st = ring_u32 + put * dec_stage_bytes(D);
      put = put + 1 == S ? 0 : put + 1;
      good = good << U | (block_ok >> (in_n * U & 31) & ((1u << U) - 1u));
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t block = __shfl_sync(0xffffffffu, block_of, (in_n * U + u) & 31);
        cp_block<D>(st, dst, k_lane + size_t(block) * (8 * D), v_lane + size_t(block) * (8 * D), s_lane + size_t(block) * D);
        st += dec_block_bytes(D);
      }
      ++in_n;
    } else {
      good <<= U;
    }
    cp_commit();
  };
#pragma unroll
  for (int n = 0; n < S - 1; ++n) issue();

  // ---- the computing side, item part by item part
  int stage = 0;
  for (int at = begin, number = 0; at < end; ++number) {
    const Part p = part_at(at);
    const int step0 = p.step0, step1 = p.step1, steps = p.steps, keys = p.keys, tile = p.tile, h = p.h, mine = p.mine;
    const Kv4Seq sq = p.sq;
    if constexpr (!kSolo) {
      cp_wait<S - 2>();  // warp 0: the query rows travel with its first step of the part
      __syncthreads();
    }

    // Q^T as B fragments in FP16 (column g is query row tile * 8 + g), each row times 2^(8 - exponent of its largest value): FP16
    // keeps 2^-25 of an element whose row reaches 2^8.  A row with a value that is not finite becomes NaN, as its softmax would.
    uint32_t qb[D / 16][2];
    float inv;
    {
      const int q_f = tile * kDecRows + g;
      const bool real = q_f < sq.n * G;
      const uint8_t* row = q_raw + number % S * dec_q_bytes(D) + g * dec_q_stride(D);
      if constexpr (kSolo) row = reinterpret_cast<const uint8_t*>(static_cast<const T*>(a.q.p) + (sq.row0 + (real ? q_f / G : 0)) * a.q.row + (h * G + (real ? q_f % G : 0)) * a.q.head);
      uint32_t top2 = 0;  // largest magnitudes of the pairs' halves: the bits of values of one sign order as integers, NaN highest
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        const uint8_t* four = row + 2 * (D == 256 ? (kk / 8) * 128 + t * 32 + (kk % 8) * 4 : t * (D / 4) + kk * 4);
        uint2 w;
        if (!kSolo || a.q_vec) {
          w = *reinterpret_cast<const uint2*>(four);
        } else {
          const uint16_t* e = reinterpret_cast<const uint16_t*>(four);
          w = make_uint2(e[0] | uint32_t(e[1]) << 16, e[2] | uint32_t(e[3]) << 16);
        }
        qb[kk][0] = w.x, qb[kk][1] = w.y;
        top2 = __vmaxu2(top2, __vmaxu2(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu));
      }
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) top2 = __vmaxu2(top2, __shfl_xor_sync(0xffffffffu, top2, o));
      const uint16_t top_bits = uint16_t(max(top2 & 0xffffu, top2 >> 16));
      const float top = to_f32<T>(*reinterpret_cast<const T*>(&top_bits));
      const int ex = int(__float_as_uint(top) >> 23 & 255u), field = min(max(262 - ex, 2), 252);
      const float sign = a.scale < 0.f ? -1.f : 1.f;  // the queries carry the scale's sign
      const float mul = sign * (top == 0.f ? 1.f : top < INFINITY ? __uint_as_float(uint32_t(field) << 23) : NAN);
      inv = top > 0.f && top < INFINITY && real ? __uint_as_float(uint32_t(254 - field) << 23) : 1.f;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const T* e = reinterpret_cast<const T*>(&qb[kk][j]);
          qb[kk][j] = real ? h2(to_f32<T>(e[0]) * mul, to_f32<T>(e[1]) * mul) : 0u;
        }
    }
    // this thread's score columns are query rows 2t and 2t + 1
    float coef[2];
    uint32_t see[2];  // in-flight rows each sees, as a mask or (no masks) their number
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      coef[j] = score_coef(a, __shfl_sync(0xffffffffu, inv, (2 * t + j) * 4));
      const int i = (tile * kDecRows + 2 * t + j) / G;
      see[j] = i >= sq.n ? 0u : a.b.anc ? a.b.anc[sq.row0 + i] : uint32_t(i + 1);
    }

    float o[D / 16][4] = {}, m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    constexpr int kChain = kChainKeys / kKeys;  // steps of a chain
    float then[2] = {-INFINITY, -INFINITY};     // reference of the chains that have ended
    float4* totals = reinterpret_cast<float4*>(a.totals + (size_t(blockIdx.x) * kDecWarps + warp) * (kDecRows * D)) + lane;
    auto add_totals = [&] {
      const float w[2] = {chain_weight(then[0], m[0]), chain_weight(then[1], m[1])};
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        const float4 x = totals[i * 32];
        o[i][0] = fmaf(x.x, w[0], o[i][0]), o[i][1] = fmaf(x.y, w[1], o[i][1]), o[i][2] = fmaf(x.z, w[0], o[i][2]), o[i][3] = fmaf(x.w, w[1], o[i][3]);
      }
    };
    for (int chain = 0; chain < mine; chain += kChain) {
      if (chain > 0) {
        if (chain > kChain) add_totals();
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          totals[i * 32] = make_float4(o[i][0], o[i][1], o[i][2], o[i][3]);
          o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        }
        then[0] = m[0], then[1] = m[1];
      }
      const int chain_end = min(mine, chain + kChain);
      for (int n = chain; n < chain_end; ++n) {
        cp_wait<S - 2>();
        __syncwarp();  // the step has landed, for all lanes; all lanes are done with the one before, whose stage is next
        issue();
        const uint8_t* st = ring + stage * dec_stage_bytes(D);
        stage = stage + 1 == S ? 0 : stage + 1;
        const int pos0 = (step0 + turn + n * kStride) * kKeys;
        const uint32_t ok_bits = good >> (S - 1) * U & ((1u << U) - 1u);  // block u in bit u
        const bool masked = ok_bits != (1u << U) - 1u || pos0 + kKeys > sq.pos;

        // scores
        float s[U][4];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const uint8_t* kc = st + u * dec_block_bytes(D);
          const uint8_t* ks = kc + kK + kV;
          float s2[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int j = 0; j < 4; ++j) s[u][j] = 0.f;
#pragma unroll
          for (int p = 0; p < KP; ++p) {
            uint32_t w[2][KB / 4], sc[2][KB / 8];  // of keys g and g + 8: codes, scales by group as half2
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              lds<KB>(kc + k_offset<D>(g, t, half, p), w[half]);
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
              mma_16816(s[u], c[0][0], c[1][0], c[0][1], c[1][1], qb[kk][0], qb[kk][1]);
              mma_16816(U == 1 ? s2 : s[u], c[0][2], c[1][2], c[0][3], c[1][3], qb[kk + 1][0], qb[kk + 1][1]);  // (two chains where one block is all there is)
            }
          }
          if constexpr (U == 1) {
#pragma unroll
            for (int j = 0; j < 4; ++j) s[u][j] += s2[j];
          }
        }

        // V's scales: of this thread's key pairs (2t, 2t+1) and (2t+8, 2t+9), per group of its dims, as (key, key + 1)
        constexpr int VG = D == 256 ? 2 : 1;
        uint32_t vsc[U][2][VG], poison = 0;  // poison: of this thread's (block, key, row): a visible key whose V is NaN
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint8_t* at_s = st + u * dec_block_bytes(D) + kK + kV + D + (2 * t + j * 8) * SB + (D == 256 ? g * 2 : D == 128 ? g : g / 2);
            if constexpr (D == 256) {
              const uint32_t x = *reinterpret_cast<const uint16_t*>(at_s), y = *reinterpret_cast<const uint16_t*>(at_s + SB);
              vsc[u][j][0] = __byte_perm(x, y, 0x0040) & 0xffffu, vsc[u][j][1] = __byte_perm(x, y, 0x0051) & 0xffffu;
            } else {
              vsc[u][j][0] = uint32_t(at_s[0]) | uint32_t(at_s[SB]) << 8;
            }
          }
        uint32_t vw[U][4][VB / 4];  // (asked for ahead of the softmax)
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int j = 0; j < 4; ++j) lds<VB>(st + u * dec_block_bytes(D) + kK + v_offset<D>(g, t, j), vw[u][j]);
        if (masked) {
          // A V vector that is NaN must reach exactly the rows that see it: its scale is taken as 0 and its probability as NaN.
#pragma unroll
          for (int u = 0; u < U; ++u) {
            uint32_t nan = 0;  // keys of this block
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int v = 0; v < VG; ++v)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                  if ((vsc[u][j][v] >> (8 * e) & 0x7fu) == 0x7fu) {
                    nan |= 1u << (2 * t + j * 8 + e);
                    vsc[u][j][v] &= e ? 0x00ffu : 0xff00u;
                  }
            nan = __reduce_or_sync(0xffffffffu, nan);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int key = g + (j >> 1) * 8, pos = pos0 + u * 16 + key, i = pos - sq.pos;
              const uint32_t mask = see[j & 1];
              const bool visible = (ok_bits >> u & 1u) && pos < keys && (i < 0 || (a.b.anc ? (mask >> i & 1u) : i < int(mask)));
              if (!visible) s[u][j] = -INFINITY;
              else poison |= (nan >> key & 1u) << (u * 4 + j);
            }
          }
        }

        // Scores are s * coef, coef >= 0.  The sums are kept relative to a reference m of each row, not its maximum: as long as no score exceeds it by 2^kLazy,
        // P (times 2^8) stays inside FP16 and nothing is exchanged or scaled.  Rows are columns 2t, 2t + 1; keys lie across the
        // lanes with the same t.
        float mx[2] = {fmaxf(s[0][0], s[0][2]), fmaxf(s[0][1], s[0][3])};
#pragma unroll
        for (int u = 1; u < U; ++u) mx[0] = fmaxf(mx[0], fmaxf(s[u][0], s[u][2])), mx[1] = fmaxf(mx[1], fmaxf(s[u][1], s[u][3]));
        if (__any_sync(0xffffffffu, fmaf(mx[0], coef[0], -m[0]) > kLazy || fmaf(mx[1], coef[1], -m[1]) > kLazy)) {
          float keep[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) mx[j] = fmaxf(mx[j], __shfl_xor_sync(0xffffffffu, mx[j], x));
            mx[j] = fmaxf(mx[j] * coef[j], m[j]);
            keep[j] = m[j] == -INFINITY ? 0.f : ex2(m[j] - mx[j]);
            l[j] *= keep[j];
            m[j] = mx[j];
          }
#pragma unroll
          for (int i = 0; i < D / 16; ++i) o[i][0] *= keep[0], o[i][2] *= keep[0], o[i][1] *= keep[1], o[i][3] *= keep[1];
        }
        const float base[2] = {m[0] == -INFINITY ? 0.f : m[0] - kPShift, m[1] == -INFINITY ? 0.f : m[1] - kPShift};
#pragma unroll
        for (int u = 0; u < U; ++u) {
          float p[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) p[j] = ex2(fmaf(s[u][j], coef[j & 1], -base[j & 1]));
          l[0] += p[0] + p[2], l[1] += p[1] + p[3];
          if (poison) {
#pragma unroll
            for (int j = 0; j < 4; ++j) p[j] = poison >> (u * 4 + j) & 1u ? NAN : p[j];
          }
          const uint32_t b0 = movmatrix(h2(p[0], p[1])), b1 = movmatrix(h2(p[2], p[3]));
          uint32_t vh[2][VG];
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int x = 0; x < VG; ++x) vh[j][x] = e4m3x2_to_h2(uint16_t(vsc[u][j][x]));
#pragma unroll
          for (int i = 0; i < VB / 4; ++i) {  // word i: 8 dims, four MMAs' rows g (even dims) and g + 8 (odd dims)
            uint32_t even[2][4], odd[2][4];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const uint32_t x = vw[u][2 * j][i], y = vw[u][2 * j + 1][i];
              e2m1x8_to_h2(x & 0x0f0f0f0fu | (y << 4 & 0xf0f0f0f0u), even[j]);
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
      }
    }
    if (mine > kChain) add_totals();
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) l[j] += __shfl_xor_sync(0xffffffffu, l[j], x);
    const bool whole = step0 == 0 && step1 == steps;
    const int first_of = (at - step0) / quota, last_of = (at - step0 + steps - 1) / quota;  // the workers that share the item
    // A worker has at most two parts of shared items: of the one it opens with (slot 0), of one that goes on behind it (slot 1).
    float* part = a.parts + (size_t(me) * 2 + (me == first_of ? 1 : 0)) * dec_part_floats(D);
    const Join join{last_of - first_of + 1, sq.row0, sq.n, h, tile, {0, 0, 0}};
    at = p.next;
    if constexpr (kSolo) {
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        const float4 acc = make_float4(o[i][0], o[i][1], o[i][2], o[i][3]);
        if (whole) store_quad<T, D>(a, sq.row0, sq.n, h, tile, i * 32 + lane, acc, m, l);
        else reinterpret_cast<float4*>(part)[i * 32 + lane] = acc;
      }
      if (!whole) {
        float* pm = part + kDecRows * D;
        if (lane < 4) pm[2 * lane] = m[0], pm[2 * lane + 1] = m[1], pm[kDecRows + 2 * lane] = l[0], pm[kDecRows + 2 * lane + 1] = l[1];
        if (lane == 0 && me == first_of) a.joins[me] = join;
      }
      continue;
    }

    // ---- the warps' results meet: the upper half's in shared memory, added to the lower half's, those added by all threads
    if (lane < 4) ml[warp][0][2 * lane] = m[0], ml[warp][0][2 * lane + 1] = m[1], ml[warp][1][2 * lane] = l[0], ml[warp][1][2 * lane + 1] = l[1];
    float4* mine_o = reinterpret_cast<float4*>(sums + warp % kHalf * dec_sum_bytes(D)) + lane;
    if (warp >= kHalf) {
#pragma unroll
      for (int i = 0; i < D / 16; ++i) mine_o[i * 32] = make_float4(o[i][0], o[i][1], o[i][2], o[i][3]);
    }
    __syncthreads();
    float mm[2], ll[2], own[2], other[2];  // of rows 2t, 2t + 1: common reference and sum, weights of this warp and its partner
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float mw[kDecWarps], lw[kDecWarps];
      mm[j] = -INFINITY, ll[j] = 0.f;
#pragma unroll
      for (int w = 0; w < kDecWarps; ++w) mw[w] = ml[w][0][2 * t + j], lw[w] = ml[w][1][2 * t + j], mm[j] = fmaxf(mm[j], mw[w]);
#pragma unroll
      for (int w = 0; w < kDecWarps; ++w) ll[j] = fmaf(lw[w], part_weight(mw[w], lw[w], mm[j]), ll[j]);
      own[j] = part_weight(m[j], l[j], mm[j]);
      const int w = (warp + kHalf) % kDecWarps;
      other[j] = part_weight(ml[w][0][2 * t + j], ml[w][1][2 * t + j], mm[j]);
    }
    if (warp < kHalf) {
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        const float4 x = mine_o[i * 32];
        mine_o[i * 32] = make_float4(fmaf(o[i][0], own[0], x.x * other[0]), fmaf(o[i][1], own[1], x.y * other[1]),
                                     fmaf(o[i][2], own[0], x.z * other[0]), fmaf(o[i][3], own[1], x.w * other[1]));
      }
    }
    __syncthreads();
    constexpr int kQuads = D / 16 * 32;
#pragma unroll
    for (int quad = tid; quad < kQuads; quad += kDecThreads) {
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kHalf; ++w) {
        const float4 x = reinterpret_cast<const float4*>(sums + w * dec_sum_bytes(D))[quad];
        acc.x += x.x, acc.y += x.y, acc.z += x.z, acc.w += x.w;
      }
      if (whole) store_quad<T, D>(a, sq.row0, sq.n, h, tile, quad, acc, mm, ll);
      else reinterpret_cast<float4*>(part)[quad] = acc;
    }
    if (!whole) {
      if (tid < 4) {
        float* pm = part + kDecRows * D;
        pm[2 * tid] = mm[0], pm[2 * tid + 1] = mm[1], pm[kDecRows + 2 * tid] = ll[0], pm[kDecRows + 2 * tid + 1] = ll[1];
      }
      if (tid == 0 && me == first_of) a.joins[me] = join;
    }
    // (the next part's opening barrier keeps its results off these sums)
  }
  cp_wait<0>();
}

// The partial results of the items that workers of the decode kernel shared: block (w, piece) adds kJoinThreads / kSplit quads of
// the item that starts with worker w and goes on behind it, kSplit threads a quad.
constexpr int kJoinThreads = 256, kJoinParts = 160;  // parts whose weights are held at a time
template <typename T, int D, int kSplit>
__global__ void __launch_bounds__(kJoinThreads) kv4_join_kernel(AttnArgs a) {
  pdl_sync();  // first statement: see common.cuh
  constexpr int kEach = kJoinThreads / kSplit, kQuads = 2 * D;
  __shared__ float pml[kJoinParts][2][kDecRows], red[2][kJoinThreads / 32][kDecRows];
  __shared__ float4 sums[kSplit][kEach];
  const int w0 = blockIdx.x, tid = threadIdx.x, lane = tid & 31, t = lane & 3, row = tid & 7, group = tid / kEach, quad = blockIdx.y * kEach + tid % kEach;
  const Join join = a.joins[w0];
  if (join.parts == 0) return;
  const int n = join.parts;
  auto part_of = [&](int i) { return a.parts + (size_t(w0 + i) * 2 + (i == 0 ? 1 : 0)) * dec_part_floats(D); };
  constexpr int kFly = 10;  // parts of a thread in flight
  float4 x[kFly];
  auto fetch = [&](int i0) {
#pragma unroll
    for (int i = 0; i < kFly; ++i)
      if (i0 + i * kSplit < n && quad < kQuads) x[i] = reinterpret_cast<const float4*>(part_of(i0 + i * kSplit))[quad];
  };
  fetch(group);
  auto reduce = [&](float v, int what) {  // over the threads with the same row: lanes, then warps through shared memory
    float u = __shfl_xor_sync(0xffffffffu, v, 8);
    v = what ? v + u : fmaxf(v, u);
    u = __shfl_xor_sync(0xffffffffu, v, 16);
    v = what ? v + u : fmaxf(v, u);
    if (lane < 8) red[what][tid >> 5][row] = v;
  };
  // the rows' common reference; a thread per (part, row)
  float top = -INFINITY;
  for (int i = tid >> 3; i < n; i += kJoinThreads / 8) {
    const float* pm = part_of(i) + kDecRows * D + row;
    const float m = pm[0];
    if (i < kJoinParts) pml[i][0][row] = m, pml[i][1][row] = pm[kDecRows];
    top = fmaxf(top, m);
  }
  reduce(top, 0);
  __syncthreads();
  top = -INFINITY;
#pragma unroll
  for (int w = 0; w < kJoinThreads / 32; ++w) top = fmaxf(top, red[0][w][row]);
  float sum = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int base = 0; base < n; base += kJoinParts) {
    const int m = min(n - base, kJoinParts);
    for (int i = tid >> 3; i < m; i += kJoinThreads / 8) {  // weights, in the place of the references
      const float* pm = part_of(base + i) + kDecRows * D + row;
      const float pmax = base ? pm[0] : pml[i][0][row], l = base ? pm[kDecRows] : pml[i][1][row], w = part_weight(pmax, l, top);
      sum = fmaf(l, w, sum);
      pml[i][0][row] = w;
    }
    __syncthreads();
    for (int i0 = group; i0 < m; i0 += kFly * kSplit) {
      if (base + i0 != group) fetch(base + i0);
#pragma unroll
      for (int i = 0; i < kFly; ++i) {
        const int p = i0 + i * kSplit;
        if (p >= m) break;
        const float f0 = pml[p][0][2 * t], f1 = pml[p][0][2 * t + 1];
        acc.x = fmaf(x[i].x, f0, acc.x), acc.y = fmaf(x[i].y, f1, acc.y), acc.z = fmaf(x[i].z, f0, acc.z), acc.w = fmaf(x[i].w, f1, acc.w);
      }
    }
    __syncthreads();
  }
  reduce(sum, 1);
  if constexpr (kSplit > 1) sums[group][tid % kEach] = acc;
  __syncthreads();
  if (group > 0 || quad >= kQuads) return;
  float mm[2], ll[2] = {0.f, 0.f};
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    mm[j] = -INFINITY;
#pragma unroll
    for (int w = 0; w < kJoinThreads / 32; ++w) mm[j] = fmaxf(mm[j], red[0][w][2 * t + j]), ll[j] += red[1][w][2 * t + j];
  }
#pragma unroll
  for (int i = 1; i < kSplit; ++i) {
    const float4 y = sums[i][tid];
    acc.x += y.x, acc.y += y.y, acc.z += y.z, acc.w += y.w;
  }
  store_quad<T, D>(a, join.row0, join.rows, join.h, join.tile, quad, acc, mm, ll);
}

// ---------------------------------------------------------------------------------------------- many query rows
// The tile kernel: 128 query rows of one (sequence, kv head) against its keys, 128 at a time, on tcgen05.mma kind::f16 with the
// accumulators in TMEM.  Roles:
//   warps 8..15  turn a tile's codes into FP16 operands in 128B-swizzled shared memory, keys as rows: K as the score product's
//                K-major B operand, V, in the same layout, as the value product's MN-major one (no transposition).  K(t+1) comes
//                before V(t), so that S(t+1) = Q K(t+1)^T runs under the softmax of tile t.  Loads run ahead in registers.
//   warp 16      one thread issues the MMAs: S(t+1), double in TMEM, then O += P(t) V(t).
//   warps 0..7   a thread half a row (its TMEM lane, 64 of the tile's keys): maximum, probabilities to FP16 in TMEM, in the place of
//                the scores, as the value product's A operand; sum.  O is scaled in TMEM only when a score exceeds the row's
//                reference by 2^kLazy, so that a tile's softmax need not wait for the tile before.
// Measured (24 query heads on 4 kv heads of 256): 4096 rows behind 4096 positions 758 us, 816 TFLOP/s (1644 is a library GEMM's rate), 5100
// cycles a tile; the MMAs are 2048 of them (tensor pipe 40 % busy).  Operands are read once by the MMAs and written once by the
// converting warps (D = 256: 192 KB and 128 KB a tile, 2560 cycles at 128 bytes; L1 and shared memory 79 % busy with that and the codes'
// loads), and K and V have one buffer each, so that conversions and MMAs take turns.  4 trees of 20 rows behind up to 8k positions 48 us,
// of which nearly 20 go into a CTA's first keys, its queries' conversion and its last rows.  A ring of pieces for K and V, with
// or without warps of their own for each, was slower (840 and 909 us).
// Every wait is bounded; one that runs out is recorded and the CTA leaves with its TMEM freed.
constexpr int kTileRows = 128, kTileKeys = 128, kTileWarps = 17, kTileThreads = kTileWarps * 32, kTileWorkers = 256, kTileMarks = 8;
constexpr int kMmaWarp = 16, kTileChain = kTileChainKeys / kTileKeys;  // tiles of a chain of value products
template <int D>
struct TileSmem {
  static constexpr int kOperand = 256 * D;  // 128 rows of D halves: [D / 64][128][128 B]
  static constexpr int kBytes = 3 * kOperand + 2 * 2 * kTileRows * 4 + 1024;
};
__host__ __device__ constexpr size_t tile_part_floats(int D) { return size_t(kTileRows) * D + 2 * kTileRows; }

// Shared-memory descriptor of an MN-major operand under the 128B swizzle: rows are k, 128 bytes (64 elements of mn) each; eight rows are
// 1024 bytes apart (stride offset), blocks of 64 mn `lead` bytes (leading offset).
__device__ __forceinline__ uint64_t desc_mn_sw128(uint32_t addr, uint32_t lead) {
  return uint64_t((addr & 0x3FFFFu) >> 4) | uint64_t(lead >> 4) << 16 | uint64_t(1024 >> 4) << 32 | uint64_t(1) << 46 | uint64_t(2) << 61;
}

// The eight softmax warps meet: whether all of them are well.
__device__ __forceinline__ bool meet_all(bool ok) {
  uint32_t all;
  asm volatile(
      "{\n"
      ".reg .pred p, q;\n"
      "setp.ne.b32 p, %1, 0;\n"
      "barrier.red.and.pred q, 1, 256, p;\n"
      "selp.b32 %0, 1, 0, q;\n"
      "}\n"
      : "=r"(all)
      : "r"(uint32_t(ok))
      : "memory");
  return all != 0;
}
// By a block: whether row0 descends somewhere, so that sequences may share rows (a barrier of its threads).
__device__ __forceinline__ bool row0_descends(const ling_b200_kv4_batch& b) {
  bool down = false;
  for (int s = threadIdx.x; s < b.seqs; s += blockDim.x) down |= b.row0[s + 1] < b.row0[s];
  return __syncthreads_or(down) != 0;
}
// D += A B with A in TMEM: lane = row, a column two neighbouring k.
__device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
      "}\n" ::"r"(tmem_d), "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

template <typename T, int D>
__global__ void __launch_bounds__(kTileThreads, 1) kv4_tile_kernel(AttnArgs a, int splits) {
  pdl_sync();  // first statement: see common.cuh
  using namespace tc;
  constexpr int kOperand = TileSmem<D>::kOperand, kBlocks = D / 64, kUnits = D / 64;  // 32-dim units of a key a worker converts per tile
  constexpr uint32_t kOcol = 2 * kTileKeys;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* qs = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* ks = qs + kOperand;
  uint8_t* vs = ks + kOperand;
  __shared__ uint64_t k_full, v_full, qk_done[2], p_full[2], pv_done[2];  // (by tile parity: a wait knows a phase's parity only, and every one must be waited for in turn)
  __shared__ uint32_t tmem_slot, bad_keys[kTileMarks][4], nan_keys[kTileMarks][4];  // by tile: keys on bad pages; (masked tiles) keys whose V is NaN
  __shared__ float q_inv[kTileRows];
  float(*row_max)[2][kTileRows] = reinterpret_cast<float(*)[2][kTileRows]>(vs + kOperand);  // [tile parity][half]; at the end the sums
  __shared__ int where[2];
  __shared__ volatile int failed;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int G = a.q_heads / a.c.kv_heads, H = a.c.kv_heads, h = blockIdx.y, lp = 31 - __clz(a.c.page_tokens);

  // ---- which 128 query rows: the long contexts' (later tiles) first
  const int index = int(gridDim.x) - 1 - int(blockIdx.x);
  if (warp == 0) {
    int before = 0, found = -1, found_tile = 0;
    for (int s0 = 0; s0 < a.b.seqs && found < 0; s0 += 32) {
      const int s = s0 + lane;
      int n = 0;
      if (s < a.b.seqs) {
        const Kv4Seq q = kv4_seq(a.c, a.b, s);
        if (!q.ok && blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0) dev_fail(a.err, kDevBadBatch);
        n = q.ok ? (q.n * G + kTileRows - 1) / kTileRows : 0;
      }
      int end = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, end, o);
        if (lane >= o) end += v;
      }
      end += before;
      const unsigned mine = __ballot_sync(0xffffffffu, index >= end - n && index < end);
      if (mine) {
        found = s0 + __ffs(mine) - 1;
        found_tile = index - __shfl_sync(0xffffffffu, end - n, __ffs(mine) - 1);
      }
      before = __shfl_sync(0xffffffffu, end, 31);
    }
    if (lane == 0) where[0] = found, where[1] = found_tile;
  }
  if (tid == 0) {
    mbar_init(&k_full, kTileWorkers / 32);
    mbar_init(&v_full, kTileWorkers / 32);
    mbar_init(&qk_done[0], 1);
    mbar_init(&qk_done[1], 1);
    mbar_init(&p_full[0], 8);
    mbar_init(&p_full[1], 8);
    mbar_init(&pv_done[0], 1);
    mbar_init(&pv_done[1], 1);
    failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (tid < kTileMarks * 4) (&bad_keys[0][0])[tid] = 0, (&nan_keys[0][0])[tid] = 0;
  if (row0_descends(a.b)) {  // (the barrier that the lines above and below need) none of the sequences is done
    if (tid == 0 && blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0) dev_fail(a.err, kDevBadBatch);
    return;
  }
  if (where[0] < 0) return;
  const Kv4Seq sq = kv4_seq(a.c, a.b, where[0]);
  const int f0 = where[1] * kTileRows, R = sq.n * G;  // this block's query rows f0 .. f0 + 127 of R: row f is (row f / G, head f % G)
  const int last_i = min(f0 + kTileRows, R) - 1;
  const int keys = a.b.anc ? sq.pos + sq.n : sq.pos + last_i / G + 1;             // no row sees further
  const int all_see = a.b.anc ? sq.pos : sq.pos + f0 / G + 1;                     // every row sees at least these
  const int tiles = (keys + kTileKeys - 1) / kTileKeys;
  const int t0 = int((long long)tiles * blockIdx.z / splits), nt = int((long long)tiles * (blockIdx.z + 1) / splits) - t0;
  auto partial = [&] { return a.parts + ((size_t(index) * H + h) * splits + blockIdx.z) * tile_part_floats(D); };  // (splits > 1, or nt > kTileChain)
  if (nt == 0) {  // (more splits than tiles)
    if (tid < kTileRows) partial()[kTileRows * D + tid] = -INFINITY, partial()[kTileRows * D + kTileRows + tid] = 0.f;
    return;
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    tc_fence_before();
  }
  // ---- Q to FP16, each row times 2^(8 - exponent of its largest value) and the scale's sign (a row with a value that is not finite
  // becomes NaN): D / 8 lanes a row
  {
    constexpr int kLanes = D / 8, kRowsAtOnce = 32 / kLanes, kFly = 4;
    const int sub = lane / kLanes, piece = lane % kLanes;
    for (int r0 = warp * kRowsAtOnce * kFly; r0 < kTileRows; r0 += kTileWarps * kRowsAtOnce * kFly) {
      uint4 w[kFly];
      const T* src[kFly];
#pragma unroll
      for (int i = 0; i < kFly; ++i) {  // (rows past the last read the last one's, so that all loads are under way together)
        const int f = min(f0 + r0 + i * kRowsAtOnce + sub, R - 1);
        src[i] = static_cast<const T*>(a.q.p) + (sq.row0 + f / G) * a.q.row + (h * G + f % G) * a.q.head + piece * 8;
      }
      if (a.q_vec) {
#pragma unroll
        for (int i = 0; i < kFly; ++i) w[i] = *reinterpret_cast<const uint4*>(src[i]);
      } else {
#pragma unroll
        for (int i = 0; i < kFly; ++i) {
          const uint16_t* e = reinterpret_cast<const uint16_t*>(src[i]);
          w[i] = make_uint4(e[0] | uint32_t(e[1]) << 16, e[2] | uint32_t(e[3]) << 16, e[4] | uint32_t(e[5]) << 16, e[6] | uint32_t(e[7]) << 16);
        }
      }
#pragma unroll
      for (int i = 0; i < kFly; ++i) {
        const int r = r0 + i * kRowsAtOnce + sub;
        if (f0 + r >= R) w[i] = make_uint4(0, 0, 0, 0);
        uint32_t top2 = __vmaxu2(__vmaxu2(w[i].x & 0x7fff7fffu, w[i].y & 0x7fff7fffu), __vmaxu2(w[i].z & 0x7fff7fffu, w[i].w & 0x7fff7fffu));
#pragma unroll
        for (int o = 1; o < kLanes; o <<= 1) top2 = __vmaxu2(top2, __shfl_xor_sync(0xffffffffu, top2, o));
        const uint16_t bits = uint16_t(max(top2 & 0xffffu, top2 >> 16));
        const float top = to_f32<T>(*reinterpret_cast<const T*>(&bits));
        const int field = min(max(262 - int(__float_as_uint(top) >> 23 & 255u), 2), 252);
        const float mul = (a.scale < 0.f ? -1.f : 1.f) * (top == 0.f ? 1.f : top < INFINITY ? __uint_as_float(uint32_t(field) << 23) : NAN);
        const uint32_t e[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
        uint32_t o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const T* two = reinterpret_cast<const T*>(&e[j]);
          o[j] = h2(to_f32<T>(two[0]) * mul, to_f32<T>(two[1]) * mul);
        }
        if (r < kTileRows) {
          *reinterpret_cast<uint4*>(qs + (piece >> 3) * (kTileRows * 128) + sw128_offset(r, piece & 7)) = make_uint4(o[0], o[1], o[2], o[3]);
          if (piece == 0) q_inv[r] = top > 0.f && top < INFINITY ? __uint_as_float(uint32_t(254 - field) << 23) : 1.f;
        }
      }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  auto wait = [&](uint64_t* bar, int n, int code) {  // the n-th completion (n < 0: none to wait for); false: give up
    if (n < 0 || mbar_wait(bar, uint32_t(n) & 1u, &failed)) return true;
    dev_fail(a.err, code);
    failed = 1;
    return false;
  };

  if (warp == kMmaWarp) {
    // ---------------------------------------------------------------- the MMAs
    if (lane == 0) {
      constexpr uint32_t kIdescS = umma_idesc_f16(kTileKeys), kIdescO = umma_idesc_f16(D) | 1u << 16;  // (bit 16: B is MN-major)
      auto scores = [&](int t) {
        if (!wait(&k_full, t, kDevWaitFull)) return false;
        tc_fence_after();
#pragma unroll
        for (int b = 0; b < kBlocks; ++b)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_f16(tmem + uint32_t(t & 1) * kTileKeys, umma_desc_sw128(smem_u32(qs + b * (kTileRows * 128))) + uint64_t(k * 2),
                     umma_desc_sw128(smem_u32(ks + b * (kTileKeys * 128))) + uint64_t(k * 2), kIdescS, (b | k) ? 1u : 0u);
        umma_commit(&qk_done[t & 1]);
        return true;
      };
      bool ok = scores(0);
      for (int t = 0; t < nt && ok; ++t) {
        if (t + 1 < nt) ok = scores(t + 1);
        ok = ok && wait(&p_full[t & 1], t >> 1, kDevWaitFull) && wait(&v_full, t, kDevWaitFull);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int k = 0; k < kTileKeys / 16; ++k)
          umma_f16_ts(tmem + kOcol, tmem + uint32_t(t & 1) * kTileKeys + uint32_t((k >> 2) * 64 + (k & 3) * 8),
                      desc_mn_sw128(smem_u32(vs + k * 16 * 128), kTileKeys * 128), kIdescO, (t % kTileChain | k) ? 1u : 0u);
        umma_commit(&pv_done[t & 1]);
      }
    }
    __syncwarp();
  } else if (warp >= 8) {
    // ---------------------------------------------------------------- the operands
    // a worker's units of 32 dims: eight neighbouring lanes take eight keys (their stores hit eight different chunks)
    constexpr int kPer = D / 32, kKeyStep = kTileWorkers / kPer;
    const int w = tid - 256, unit = (w >> 3) % kPer, key0 = (w >> 3) / kPer * 8 + (w & 7);  // keys key0, key0 + kKeyStep, ..
    const int* table = a.c.tables + size_t(sq.slot) * a.c.max_pages;
    // Of a tile's units: where their vectors are (kNone: no key, kBad: no page), as indices among the cache's vectors.
    constexpr uint32_t kNone = 0xffffffffu, kBad = 0xfffffffeu;
    struct Codes {
      uint4 c[kUnits];
      uint16_t s[kUnits];
    };
    auto look_up = [&](int t, int (&page)[kUnits]) {
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        const int pos = (t0 + t) * kTileKeys + key0 + u * kKeyStep;
        page[u] = t < nt && pos < keys ? table[pos >> lp] : -1;
      }
    };
    auto locate = [&](int t, const int (&page)[kUnits], uint32_t (&vec)[kUnits]) {
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        const int pos = (t0 + t) * kTileKeys + key0 + u * kKeyStep;
        vec[u] = (((uint32_t(page[u]) * H + h) << lp) + (pos & ((1 << lp) - 1)));
        if (page[u] < 1 || page[u] > a.c.pages) vec[u] = t < nt && pos < keys ? kBad : kNone;
      }
    };
    const uint8_t *k_unit = a.c.k + unit * 16, *v_unit = a.c.v + unit * 16, *ks_unit = a.c.k_scales + unit * 2, *vs_unit = a.c.v_scales + unit * 2;
    auto ask = [&](const uint8_t* codes, const uint8_t* scales, const uint32_t (&vec)[kUnits], Codes& x) {
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        x.c[u] = make_uint4(0, 0, 0, 0), x.s[u] = 0;
        if (vec[u] < kBad) {
          x.c[u] = *reinterpret_cast<const uint4*>(codes + size_t(vec[u]) * (D / 2));
          x.s[u] = *reinterpret_cast<const uint16_t*>(scales + size_t(vec[u]) * (D / 16));
        }
      }
    };
    uint32_t chunk_at[4];  // where the unit's four 16-byte chunks lie (the keys of a thread differ by multiples of 8: the swizzle is one)
#pragma unroll
    for (int i = 0; i < 4; ++i) chunk_at[i] = (unit >> 1) * (kTileKeys * 128) + sw128_offset(key0, (unit & 1) * 4 + i);
    auto convert = [&](uint8_t* to, const Codes& x) {
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        const uint32_t sc = e4m3x2_to_h2(x.s[u]), s0 = __byte_perm(sc, sc, 0x1010), s1 = __byte_perm(sc, sc, 0x3232);
        const uint32_t cw[4] = {x.c[u].x, x.c[u].y, x.c[u].z, x.c[u].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t v[4];
          e2m1x8_to_h2(cw[i], v);
          const uint32_t sx = i < 2 ? s0 : s1;
          *reinterpret_cast<uint4*>(to + chunk_at[i] + u * (kKeyStep * 128)) = make_uint4(h2_mul(v[0], sx), h2_mul(v[1], sx), h2_mul(v[2], sx), h2_mul(v[3], sx));
        }
      }
    };
    auto publish = [&](uint64_t* bar) {
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    auto mark_bad = [&](int t, const uint32_t (&vec)[kUnits]) {
#pragma unroll
      for (int u = 0; u < kUnits; ++u)
        if (vec[u] == kBad && unit == 0) {
          const int key = key0 + u * kKeyStep;
          dev_fail(a.err, kDevBadPage);
          atomicOr(&bad_keys[t % kTileMarks][key >> 5], 1u << (key & 31));
        }
    };
    Codes kc, vc;
    int page[kUnits];                              // of tile t + 2
    uint32_t vec[kUnits], vec1[kUnits], vec2[kUnits];  // of tiles t, t + 1, t + 2
    look_up(0, page);
    locate(0, page, vec);
    look_up(1, page);
    ask(k_unit, ks_unit, vec, kc);
    mark_bad(0, vec);
    locate(1, page, vec1);
    look_up(2, page);
    convert(ks, kc);
    publish(&k_full);
    ask(k_unit, ks_unit, vec1, kc);
    bool ok = true;
    for (int t = 0; t < nt && ok; ++t) {
      ask(v_unit, vs_unit, vec, vc);
      if (w < 4) bad_keys[(t + 3) % kTileMarks][w] = 0, nan_keys[(t + 3) % kTileMarks][w] = 0;  // (last used five tiles ago)
      if (t + 1 < nt) {  // K(t + 1), where K(t) was
        ok = __all_sync(0xffffffffu, wait(&qk_done[t & 1], t >> 1, kDevWaitEmpty));  // (a warp gives up as one)
        if (!ok) break;
        mark_bad(t + 1, vec1);
        convert(ks, kc);
        publish(&k_full);
      }
      locate(t + 2, page, vec2);
      look_up(t + 3, page);
      ask(k_unit, ks_unit, vec2, kc);
      if ((t0 + t + 1) * kTileKeys > all_see) {  // a masked tile: NaN must not meet the zero probabilities of rows that do not see it
#pragma unroll
        for (int u = 0; u < kUnits; ++u)
          if ((vc.s[u] & 0x7f) == 0x7f || (vc.s[u] & 0x7f00) == 0x7f00) {
            const int key = key0 + u * kKeyStep;
            atomicOr(&nan_keys[t % kTileMarks][key >> 5], 1u << (key & 31));
            vc.s[u] = 0;
          }
      }
      ok = __all_sync(0xffffffffu, t == 0 || wait(&pv_done[(t - 1) & 1], (t - 1) >> 1, kDevWaitEmpty));  // V(t), where V(t - 1) was
      if (!ok) break;
      convert(vs, vc);
      publish(&v_full);
#pragma unroll
      for (int u = 0; u < kUnits; ++u) vec[u] = vec1[u], vec1[u] = vec2[u];
    }
  } else {
    // ---------------------------------------------------------------- the softmax
    const int r = tid & (kTileRows - 1), half = tid >> 7, f = f0 + r, i_row = f / G;  // row r, keys half * 64 .. + 64 of a tile
    const bool real = f < R;
    const float coef = score_coef(a, q_inv[r]);
    const uint32_t see = real && a.b.anc ? a.b.anc[sq.row0 + i_row] : 0u;
    const int limit = real ? sq.pos + i_row + 1 : 0;  // (no masks) positions this row sees
    const uint32_t lane_addr = tmem + (uint32_t((warp & 3) * 32) << 16);
    float m = -INFINITY, l = 0.f, then = -INFINITY;  // then: reference of the chains that have ended
    // 32 dims (from 32 c on) of this row's total of the ended chains, where its partial result will lie, times w, added to x
    auto add_total = [&](int c, float w, uint32_t (&x)[32]) {
      const float* total = partial();
#pragma unroll
      for (int j = 0; j < 32; j += 4) {
        const float4 y = *reinterpret_cast<const float4*>(total + (size_t(c * 8 + j / 4) * kTileRows + r) * 4);
        x[j] = __float_as_uint(fmaf(y.x, w, __uint_as_float(x[j]))), x[j + 1] = __float_as_uint(fmaf(y.y, w, __uint_as_float(x[j + 1])));
        x[j + 2] = __float_as_uint(fmaf(y.z, w, __uint_as_float(x[j + 2]))), x[j + 3] = __float_as_uint(fmaf(y.w, w, __uint_as_float(x[j + 3])));
      }
    };
    bool ok = true;
    for (int t = 0; t < nt; ++t) {
      ok = ok && wait(&qk_done[t & 1], t >> 1, kDevWaitTmemFull);
      ok = ok && (t < 2 || wait(&pv_done[t & 1], (t - 2) >> 1, kDevWaitTmemFull));  // (done long since: the scores were asked for after it)
      tc_fence_after();
      const uint32_t s_addr = lane_addr + uint32_t(t & 1) * kTileKeys + half * 64;
      const int base_pos = (t0 + t) * kTileKeys + half * 64;
      uint32_t bad = 0;
#pragma unroll
      for (int c = 0; c < 4; ++c) bad |= bad_keys[t % kTileMarks][c];
      const bool masked = (t0 + t + 1) * kTileKeys > all_see || bad;
      uint32_t vis[2] = {0xffffffffu, 0xffffffffu};  // which of its 64 keys this row sees
      if (masked) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int p0 = base_pos + c * 32;
          if (a.b.anc) {  // the context, then the row's ancestors
            const int ctx = sq.pos - p0;  // keys of the context among them
            const uint32_t mine = sq.n >= 32 ? see : see & ((1u << sq.n) - 1u);
            vis[c] = ctx >= 32 ? 0xffffffffu : ctx >= 0 ? (1u << ctx) - 1u | mine << ctx : ctx > -32 ? mine >> -ctx : 0u;
          } else {
            const int n = limit - p0;
            vis[c] = n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u;
          }
          vis[c] &= ~bad_keys[t % kTileMarks][half * 2 + c];
        }
      }
      float mx = -INFINITY;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t v[32];
        tmem_ld32(s_addr + c * 32, v);
        tmem_ld_wait();
        if (masked) {
#pragma unroll
          for (int j = 0; j < 32; ++j) mx = fmaxf(mx, vis[c] >> j & 1u ? __uint_as_float(v[j]) : -INFINITY);
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) mx = fmaxf(mx, __uint_as_float(v[j]));
        }
      }
      row_max[t & 1][half][r] = mx;
      ok = meet_all(ok);  // the other half's maximum; and all eight warps go on, or none
      if (!ok) break;
      mx = fmaxf(mx, row_max[t & 1][half ^ 1][r]);
      if (masked) ok = (t == 0 || wait(&pv_done[(t - 1) & 1], (t - 1) >> 1, kDevWaitTmemFull)) && wait(&v_full, t, kDevWaitFull);  // the marks of V's NaN
      if (t % kTileChain == 0 && t > 0) {  // a chain ends
        ok = ok && wait(&pv_done[(t - 1) & 1], (t - 1) >> 1, kDevWaitTmemFull);  // O is complete
        tc_fence_after();
        const float w = chain_weight(then, m);
#pragma unroll 1
        for (int c = half * (D / 64); c < (half + 1) * (D / 64); ++c) {
          uint32_t x[32];
          tmem_ld32(lane_addr + kOcol + c * 32, x);
          tmem_ld_wait();
          if (t > kTileChain) add_total(c, w, x);
          float* total = partial();
#pragma unroll
          for (int j = 0; j < 32; j += 4)
            *reinterpret_cast<uint4*>(total + (size_t(c * 8 + j / 4) * kTileRows + r) * 4) = make_uint4(x[j], x[j + 1], x[j + 2], x[j + 3]);
        }
        then = m;
      }
      const float top = mx * coef;  // (-inf where nothing is seen)
      const bool grow = top > m + kLazy;
      if (__any_sync(0xffffffffu, grow)) {
        const float m_new = grow ? top : m, keep = m == -INFINITY ? 0.f : ex2(m - m_new);
        l *= keep, m = m_new;
        if (t % kTileChain != 0) {  // (where a chain starts, O is written anew)
          ok = ok && wait(&pv_done[(t - 1) & 1], (t - 1) >> 1, kDevWaitTmemFull);  // O is complete
          tc_fence_after();
#pragma unroll 1
          for (int c = half * (D / 64); c < (half + 1) * (D / 64); ++c) {
            uint32_t x[32];
            tmem_ld32(lane_addr + kOcol + c * 32, x);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; ++j) x[j] = __float_as_uint(__uint_as_float(x[j]) * keep);
            tmem_st32(lane_addr + kOcol + c * 32, x);
          }
          tmem_st_wait();
        }
      }
      const float base = m == -INFINITY ? 0.f : m - kPShift;
      uint64_t l2[2] = {0, 0};
      uint32_t pk[32];  // 64 probabilities
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t v[32];
        tmem_ld32(s_addr + c * 32, v);
        tmem_ld_wait();
        float p[32];
        const uint64_t coef2 = f2_pack(coef, coef), base2 = f2_pack(-base, -base);
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
          const uint64_t s2 = f2_fma(f2_pack(__uint_as_float(v[j]), __uint_as_float(v[j + 1])), coef2, base2);
          p[j] = ex2(f2_lo(s2)), p[j + 1] = ex2(f2_hi(s2));
        }
        if (masked) {
#pragma unroll
          for (int j = 0; j < 32; ++j) p[j] = vis[c] >> j & 1u ? p[j] : 0.f;
        }
#pragma unroll
        for (int j = 0; j < 32; j += 4) l2[j / 4 & 1] = f2_add(l2[j / 4 & 1], f2_add(f2_pack(p[j], p[j + 1]), f2_pack(p[j + 2], p[j + 3])));
        if (masked) {
          const uint32_t nan = nan_keys[t % kTileMarks][half * 2 + c] & vis[c];
          if (nan) {
#pragma unroll
            for (int j = 0; j < 32; ++j) p[j] = nan >> j & 1u ? NAN : p[j];
          }
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) pk[c * 16 + j] = h2(p[2 * j], p[2 * j + 1]);
      }
      tmem_st32(s_addr, pk);  // where this thread's first 32 scores were: it has read them all
      tmem_st_wait();
      l += (f2_lo(l2[0]) + f2_hi(l2[0])) + (f2_lo(l2[1]) + f2_hi(l2[1]));
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[t & 1]);
    }
    // ---- the result, half of the dims a thread
    row_max[nt & 1][half][r] = l;
    ok = meet_all(ok);
    l = row_max[nt & 1][0][r] + row_max[nt & 1][1][r];
    if (__all_sync(0xffffffffu, ok && wait(&pv_done[(nt - 1) & 1], (nt - 1) >> 1, kDevWaitTmemFull))) {
      tc_fence_after();
      float* part = partial();
      const bool empty = m == -INFINITY && l == 0.f;
      const float scale = empty ? 0.f : a.c.v_scale / l;
      const int row = sq.row0 + (real ? i_row : 0), head = h * G + (real ? f % G : 0);
      T* to = static_cast<T*>(a.out.p) + row * a.out.row + head * a.out.head;
      // O by rows is what a thread holds; the operands' memory, which no MMA reads any more, turns it for whole lines
      constexpr int kStage = D + 16;  // bytes of half a row, padded against bank conflicts
      uint8_t* stage = ks + warp * (32 * kStage);
#pragma unroll 1
      for (int c = half * (D / 64); c < (half + 1) * (D / 64); ++c) {
        uint32_t x[32];
        tmem_ld32(lane_addr + kOcol + c * 32, x);
        tmem_ld_wait();
        if (nt > kTileChain) add_total(c, chain_weight(then, m), x);
        if (splits > 1) {  // [dims / 4][row][4]
#pragma unroll
          for (int j = 0; j < 32; j += 4)
            *reinterpret_cast<uint4*>(part + (size_t(c * 8 + j / 4) * kTileRows + r) * 4) = make_uint4(x[j], x[j + 1], x[j + 2], x[j + 3]);
        } else if (a.out_vec) {
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            T e[8];
#pragma unroll
            for (int y = 0; y < 8; ++y) e[y] = from_f32<T>(empty ? 0.f : __uint_as_float(x[j + y]) * scale);
            *reinterpret_cast<uint4*>(stage + lane * kStage + (c - half * (D / 64)) * 64 + j * 2) = *reinterpret_cast<const uint4*>(e);
          }
        } else if (real) {
#pragma unroll
          for (int j = 0; j < 32; ++j) to[c * 32 + j] = from_f32<T>(empty ? 0.f : __uint_as_float(x[j]) * scale);
        }
      }
      if (splits == 1 && a.out_vec) {
        __syncwarp();
        constexpr int kLanes = D / 16, kAtOnce = 32 / kLanes;  // lanes of half a row
        T* out = static_cast<T*>(a.out.p) + half * (D / 2);
        for (int i = lane / kLanes; i < 32; i += kAtOnce) {
          const int fi = f0 + (warp & 3) * 32 + i;
          if (fi >= R) break;
          T* dst = out + (sq.row0 + fi / G) * a.out.row + (h * G + fi % G) * a.out.head;
          reinterpret_cast<uint4*>(dst)[lane % kLanes] = *reinterpret_cast<const uint4*>(stage + i * kStage + lane % kLanes * 16);
        }
      }
      if (half == 0) {
        if (splits > 1) part[kTileRows * D + r] = m, part[kTileRows * D + kTileRows + r] = l;
        else if (real && a.lse) a.lse[size_t(row) * a.q_heads + head] = empty ? -INFINITY : (m + log2f(l) - kPShift) * kLn2;
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

// The splits' partial results of the tile kernel: a warp a query row, in the order of the splits.
template <typename T, int D>
__global__ void __launch_bounds__(256) kv4_tile_join_kernel(AttnArgs a, int splits) {
  pdl_sync();  // first statement: see common.cuh
  __shared__ int at[8];  // of the block's rows: tile * kTileRows + row of the tile; -1: none
  const int tid = threadIdx.x, lane = tid & 31, G = a.q_heads / a.c.kv_heads, H = a.c.kv_heads, h = blockIdx.y;
  // ---- a warp a row (packed row * G + head of the group): the sequence and its first tile
  {
    const int r = blockIdx.x * 8 + (tid >> 5), row = r / G;
    int before = 0, seq = -1, tile0 = 0;
    for (int s0 = 0; s0 < a.b.seqs && seq < 0; s0 += 32) {
      const int s = s0 + lane;
      Kv4Seq q{0, 0, 0, 0, false};
      if (s < a.b.seqs) q = kv4_seq(a.c, a.b, s);
      const int n = q.ok ? (q.n * G + kTileRows - 1) / kTileRows : 0;
      int end = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, end, o);
        if (lane >= o) end += v;
      }
      end += before;
      const unsigned mine = __ballot_sync(0xffffffffu, q.ok && row >= q.row0 && row < q.row0 + q.n);
      if (mine) {
        seq = s0 + __ffs(mine) - 1;
        tile0 = __shfl_sync(0xffffffffu, end - n, __ffs(mine) - 1);
      }
      before = __shfl_sync(0xffffffffu, end, 31);
    }
    int f = 0;
    if (seq >= 0) f = (row - a.b.row0[seq]) * G + r % G;
    if (lane == 0) at[tid >> 5] = seq >= 0 ? (tile0 + f / kTileRows) * kTileRows + f % kTileRows : -1;
  }
  if (row0_descends(a.b)) return;  // (the barrier before `at` is read)
  // ---- a thread four dims of a row: eight neighbouring rows' are 128 bytes of a partial result
  const int mine = at[tid & 7], r = blockIdx.x * 8 + (tid & 7), in = mine & (kTileRows - 1);
  if (mine < 0) return;
  const float* parts = a.parts + (size_t(mine / kTileRows) * H + h) * splits * tile_part_floats(D);
  float mm = -INFINITY;
  for (int s = 0; s < splits; ++s) mm = fmaxf(mm, parts[s * tile_part_floats(D) + kTileRows * D + in]);
  constexpr int kEach = D == 256 ? 2 : 1;
  const int quad = tid >> 3;
  if (quad >= D / 4) return;
  float l = 0.f;
  float4 o[kEach] = {};
#pragma unroll 4
  for (int s = 0; s < splits; ++s) {
    const float* p = parts + s * tile_part_floats(D);
    const float pm = p[kTileRows * D + in], ps = p[kTileRows * D + kTileRows + in], w = part_weight(pm, ps, mm);
    if (pm == -INFINITY && ps == 0.f) continue;  // (a split without keys has written no O; one whose weight is 0 may hold a NaN)
    l = fmaf(ps, w, l);
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const float4 x = *reinterpret_cast<const float4*>(p + (size_t(quad + j * 32) * kTileRows + in) * 4);
      o[j].x = fmaf(x.x, w, o[j].x), o[j].y = fmaf(x.y, w, o[j].y), o[j].z = fmaf(x.z, w, o[j].z), o[j].w = fmaf(x.w, w, o[j].w);
    }
  }
  const bool empty = mm == -INFINITY && l == 0.f;
  const int row = r / G, head = h * G + r % G;
  T* to = static_cast<T*>(a.out.p) + row * a.out.row + head * a.out.head;
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const float x[4] = {o[j].x, o[j].y, o[j].z, o[j].w};
    T e[4];
#pragma unroll
    for (int y = 0; y < 4; ++y) e[y] = from_f32<T>(empty ? 0.f : x[y] / l * a.c.v_scale);
    T* dst = to + (quad + j * 32) * 4;
    if (a.out_vec) {
      *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(e);
    } else {
#pragma unroll
      for (int y = 0; y < 4; ++y) dst[y] = e[y];
    }
  }
  if (a.lse && quad == 0) a.lse[size_t(row) * a.q_heads + head] = empty ? -INFINITY : (mm + log2f(l) - kPShift) * kLn2;
}

template <typename T, int D>
int decode_init() {
  LB_CUDA(cudaFuncSetAttribute(kv4_decode_kernel<T, D, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, dec_smem(D)));
  LB_CUDA(cudaFuncSetAttribute(kv4_tile_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, TileSmem<D>::kBytes));
  LB_CUDA(cudaFuncSetAttribute(kv4_decode_kernel<T, D, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, dec_smem(D)));
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
template <typename T, int D>
int decode_launch_t(const AttnArgs& a, bool solo, int sms, cudaStream_t s) {
  const int grid = std::min(sms, kDecMaxCtas);
  LB_CUDA(launch_kernel(solo ? kv4_decode_kernel<T, D, true> : kv4_decode_kernel<T, D, false>, dim3(grid), dim3(kDecThreads), size_t(dec_smem(D)), s, a));
  LB_LAUNCH("kv4_decode_kernel");
  // of a CTA's parts there may be many to an item: four threads a quad; of a warp's there are few
  if (solo) LB_CUDA(launch_dependent(kv4_join_kernel<T, D, 1>, dim3(grid * kDecWarps, ceil_div(2 * D, kJoinThreads)), dim3(kJoinThreads), size_t(0), s, a));
  else LB_CUDA(launch_dependent(kv4_join_kernel<T, D, 4>, dim3(grid, D / 32), dim3(kJoinThreads), size_t(0), s, a));
  LB_LAUNCH("kv4_join_kernel");
  return LING_B200_OK;
}
// Whether warps work alone: with many (sequence, kv head, row tile) items the CTAs' meetings at every item's end cost more than
// the partial results of single warps.
bool decode_solo(const ling_b200_kv4& c, const ling_b200_kv4_batch& b, int q_heads) {
  const long long tiles = ((long long)b.max_rows * (q_heads / c.kv_heads) + kDecRows - 1) / kDecRows;
  return tiles * c.kv_heads * b.seqs >= kSoloItems;
}
template <typename T>
int decode_launch(const AttnArgs& a, int sms, cudaStream_t s) {
  const bool solo = decode_solo(a.c, a.b, a.q_heads);
  return a.c.head_dim == 64    ? decode_launch_t<T, 64>(a, solo, sms, s)
         : a.c.head_dim == 128 ? decode_launch_t<T, 128>(a, solo, sms, s)
                               : decode_launch_t<T, 256>(a, solo, sms, s);
}

// How a batch with up to these rows and positions runs.  Up to kDecodeRows query rows of a kv head the decode kernel reads the cache once
// per 8 of them; beyond, the tile kernel once per 128, contexts split over CTAs where the row tiles alone do not fill the device.
// Measured, decode / tile kernel, 6 heads a kv head: 24 query rows over 128k positions 113 / 120 us, 30 rows 145 / 121; over 8k 19 / 32 and
// 22 / 33; 64 sequences of up to 8k, 3 rows each on average, 228 / 326.  A split is worth kTileSplitKeys positions: 16 rows over 2k
// positions 27.5 us (256: 26.8, 1024: 38.4), over 8k 34.3 (41.1, 42.0), from 60k on the same.
constexpr int kDecodeRows = 24, kTileCtas = 148, kTileSplitKeys = 512;  // CTAs wanted; positions that a split is worth
struct Plan {
  bool tile = false, solo = false;
  int row_tiles = 0, splits = 1;
};
Plan make_plan(const ling_b200_kv4& c, const ling_b200_kv4_batch& b, int q_heads) {
  Plan p;
  const int G = q_heads / c.kv_heads;
  p.tile = (long long)b.max_rows * G > kDecodeRows;
  if (!p.tile) {
    p.solo = decode_solo(c, b, q_heads);
    return p;
  }
  const long long most = (long long)b.seqs * (((long long)b.max_rows * G + kTileRows - 1) / kTileRows), packed = (long long)b.rows * G / kTileRows + b.seqs;
  p.row_tiles = int(std::min(most, packed));
  p.splits = int(std::max(1ll, std::min<long long>(kTileCtas / ((long long)p.row_tiles * c.kv_heads), (b.max_context + kTileSplitKeys - 1) / kTileSplitKeys)));
  return p;
}
template <typename T, int D>
int tile_launch_t(const AttnArgs& a, const Plan& p, cudaStream_t s) {
  LB_CUDA(launch_kernel(kv4_tile_kernel<T, D>, dim3(p.row_tiles, a.c.kv_heads, p.splits), dim3(kTileThreads), size_t(TileSmem<D>::kBytes), s, a, p.splits));
  LB_LAUNCH("kv4_tile_kernel");
  if (p.splits > 1) {
    LB_CUDA(launch_dependent(kv4_tile_join_kernel<T, D>, dim3(ceil_div(a.b.rows * (a.q_heads / a.c.kv_heads), 8), a.c.kv_heads), dim3(256), size_t(0), s, a, p.splits));
    LB_LAUNCH("kv4_tile_join_kernel");
  }
  return LING_B200_OK;
}
template <typename T>
int attention_launch(const AttnArgs& a, int sms, cudaStream_t s) {
  const Plan p = make_plan(a.c, a.b, a.q_heads);
  if (!p.tile) return decode_launch<T>(a, sms, s);
  return a.c.head_dim == 64 ? tile_launch_t<T, 64>(a, p, s) : a.c.head_dim == 128 ? tile_launch_t<T, 128>(a, p, s) : tile_launch_t<T, 256>(a, p, s);
}

DeviceInfo g_devices[kMaxDevices];
std::mutex g_mutex;

constexpr size_t kJoinBytes = kDecMaxWorkers * sizeof(Join);
// Floats of partial results (the tile kernel's ended chains are added up in their place), and of the totals of the decode kernel's ended
// chains behind them.
size_t part_floats(const Plan& p, const ling_b200_kv4& c, const ling_b200_kv4_batch& b) {
  if (p.tile) return p.splits > 1 || b.max_context > kTileChainKeys ? size_t(p.row_tiles) * c.kv_heads * p.splits * tile_part_floats(c.head_dim) : 0;
  return size_t(p.solo ? kDecMaxWorkers : kDecMaxCtas) * 2 * dec_part_floats(c.head_dim);
}
size_t total_floats(const Plan& p, const ling_b200_kv4& c, const ling_b200_kv4_batch& b) {
  if (p.tile) return 0;
  return b.max_context > (p.solo ? 1 : kDecWarps) * kChainKeys ? size_t(kDecMaxCtas) * kDecWarps * kDecRows * c.head_dim : 0;  // (a warp's longest share)
}

bool heads_ok(const ling_b200_kv4* c, const ling_b200_kv4_batch* b, int q_heads, const char* who) {
  if (q_heads < 1 || q_heads > 1024 || q_heads % c->kv_heads != 0) {
    set_error(std::string(who) + ": q_heads must be a multiple of kv_heads, at most 1024");
    return false;
  }
  if ((long long)b->rows * (q_heads / c->kv_heads) > 0x7fffffffll - kTileRows) {  // (the kernels count query rows of a kv head in 32 bits)
    set_error(std::string(who) + ": rows x (q_heads / kv_heads) is 2^31 - 128 or more");
    return false;
  }
  return true;
}

}  // namespace
}  // namespace lb

using namespace lb;
using namespace lb::d4;

extern "C" size_t ling_b200_kv4_attention_workspace(const ling_b200_kv4* cache, const ling_b200_kv4_batch* batch, int q_heads) {
  const char* who = "kv4_attention_workspace";
  if (!kv4_cache_ok(cache, who) || !kv4_batch_ok(cache, batch, who) || !heads_ok(cache, batch, q_heads, who)) return 0;
  const Plan p = make_plan(*cache, *batch, q_heads);
  return kJoinBytes + (part_floats(p, *cache, *batch) + total_floats(p, *cache, *batch)) * 4;
}

extern "C" int ling_b200_kv4_attention(int device, const ling_b200_kv4* cache, const ling_b200_kv4_batch* batch, int type,
                                       const ling_b200_rows* q, int q_heads, float scale, const ling_b200_rows* out, float* lse,
                                       void* workspace, size_t workspace_bytes, int* err, void* stream) {
  const char* who = "kv4_attention";
  if (!kv4_cache_ok(cache, who) || !kv4_batch_ok(cache, batch, who) || !heads_ok(cache, batch, q_heads, who)) return LING_B200_ERR_ARG;
  if (type != LING_B200_BF16 && type != LING_B200_F16) {
    set_error("kv4_attention: queries are LING_B200_BF16 or LING_B200_F16");
    return LING_B200_ERR_ARG;
  }
  if (batch->rows == 0) return LING_B200_OK;  // (arrays without rows may have no address)
  if (!kv4_rows_ok(q, type, q_heads, cache->head_dim, who, "q") || !kv4_out_ok(out, type, batch->rows, q_heads, cache->head_dim, who, "out"))
    return LING_B200_ERR_ARG;
  if (!std::isfinite(scale) || !aligned(lse, 4) || !aligned(err, 4)) {
    set_error("kv4_attention: scale must be finite, lse and err aligned");
    return LING_B200_ERR_ARG;
  }
  const long long tiles = ((long long)batch->max_rows * (q_heads / cache->kv_heads) + kDecRows - 1) / kDecRows * cache->kv_heads;
  if (!make_plan(*cache, *batch, q_heads).tile && tiles * batch->seqs > (1ll << 30) / (batch->max_context / 16 + 1)) {
    set_error("kv4_attention: the batch's bounds (seqs x max_rows x max_context) are beyond 2^30 steps of the kernel");
    return LING_B200_ERR_UNSUPPORTED;
  }
  const size_t need = ling_b200_kv4_attention_workspace(cache, batch, q_heads);
  if (!workspace || workspace_bytes < need || !aligned(workspace, 16)) {
    set_error("kv4_attention: a 16-byte aligned workspace of " + std::to_string(need) + " bytes expected");
    return LING_B200_ERR_ARG;
  }
  DeviceGuard guard;
  int sms = 0;
  if (const int r = enter_device(guard, device, g_devices, g_mutex, attention_init, &sms)) return r;
  AttnArgs a{*cache, *batch, *q, *out, q_heads, scale, lse, err, static_cast<Join*>(workspace),
             reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kJoinBytes), nullptr, rows_vec(*q, type), rows_vec(*out, type)};
  a.totals = a.parts + part_floats(make_plan(*cache, *batch, q_heads), *cache, *batch);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return type == LING_B200_BF16 ? attention_launch<__nv_bfloat16>(a, sms, s) : attention_launch<__half>(a, sms, s);
}
