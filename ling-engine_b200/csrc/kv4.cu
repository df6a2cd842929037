// kv4.cu -- writing and reading a paged NVFP4 KV cache: ling_b200_kv4_append, ling_b200_kv4_read.
//
// append, of a vector x of head_dim values (a key after its rotation, a value as it is), per group g of 16 dims:
//   s = E4M3(clamp(max |x| / 6, 2^-9, 448)),  code = the E2M1 value nearest x / s, halfway to the smaller magnitude.
// x / s lies above a border b exactly when |x| > b * s, and b * s (3 + 4 significant bits) is exact in fp32, so the codes are
// found by comparisons alone.  A key's rotation, and its largest value over 6, are carried in double and brought to fp32 by rounding to
// odd (the last bit set when anything was cut off), which keeps every comparison with a value of fewer bits what it is for the exact
// number: neither codes nor scales depend on how fp32 would have rounded the rotation.  Where nothing turns, the quotient of an
// fp32 value and 6 needs no such care: beside a middle of two E4M3 values it lies at least two thirds of an fp32 step from it.  Queries
// need no such care and turn in fp32.
#include <algorithm>
#include <cfloat>

#include "decode4.cuh"

namespace lb {
namespace d4 {

bool kv4_cache_ok(const ling_b200_kv4* c, const char* who) {
  auto no = [&](const char* why) {
    set_error(std::string(who) + ": " + why);
    return false;
  };
  if (!c || !c->k || !c->v || !c->k_scales || !c->v_scales || !c->tables) return no("null cache pointer");
  if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->k_scales, 16) || !aligned(c->v_scales, 16) || !aligned(c->tables, 4))
    return no("the cache's arrays must start on 16-byte boundaries");
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return no("head_dim must be 64, 128 or 256");
  if (c->page_tokens != 16 && c->page_tokens != 32 && c->page_tokens != 64 && c->page_tokens != 128)
    return no("page_tokens must be 16, 32, 64 or 128");
  if (c->kv_heads < 1 || c->kv_heads > 1024 || c->pages < 1 || c->slots < 1 || c->max_pages < 1 ||
      c->max_pages > (1 << 30) / c->page_tokens)
    return no("a cache size out of range");
  if ((long long)c->pages >= (1ll << 32) / ((long long)c->kv_heads * c->page_tokens) - 1)  // (the kernels' vector indices have 32 bits)
    return no("the cache holds 2^32 vectors or more");
  for (float s : {c->k_scale, c->v_scale}) {
    int e = 0;
    if (!(s >= 0x1p-30f && s <= 0x1p30f) || std::frexp(s, &e) != 0.5f) return no("k_scale and v_scale must be powers of two in [2^-30, 2^30]");
  }
  return true;
}

bool kv4_batch_ok(const ling_b200_kv4* c, const ling_b200_kv4_batch* b, const char* who) {
  auto no = [&](const char* why) {
    set_error(std::string(who) + ": " + why);
    return false;
  };
  if (!b || !b->row0 || !b->slot || !b->pos) return no("null batch pointer");
  if (!aligned(b->row0, 4) || !aligned(b->slot, 4) || !aligned(b->pos, 4) || !aligned(b->rope_pos, 4) || !aligned(b->anc, 4))
    return no("a batch array is not aligned");
  if (b->seqs < 1 || b->seqs > LING_B200_KV4_MAX_SEQS) return no("seqs out of range");
  if (b->rows < 0 || b->rows > (1 << 24) || b->max_rows < 0 || b->max_rows > b->rows) return no("rows or max_rows out of range");
  if (b->anc && b->max_rows > LING_B200_MAX_TREE_ROWS) return no("ancestor masks hold 32 rows of a sequence");
  if (b->max_context < b->max_rows || (long long)b->max_context > (long long)c->max_pages * c->page_tokens)
    return no("max_context is below max_rows or beyond the page tables");
  return true;
}

bool kv4_rows_ok(const ling_b200_rows* r, int type, int heads, int dim, const char* who, const char* what) {
  if (!r || !r->p || !aligned(r->p, type_size(type)) || r->head < dim || r->row < dim) {
    set_error(std::string(who) + ": bad rows (" + what + "): a pointer aligned to its type and strides of at least head_dim expected");
    return false;
  }
  return true;
}

bool kv4_out_ok(const ling_b200_rows* r, int type, int rows, int heads, int dim, const char* who, const char* what) {
  if (!kv4_rows_ok(r, type, heads, dim, who, what)) return false;
  const bool apart = r->head <= r->row ? r->row >= (heads - 1) * r->head + dim : r->head >= (rows - 1) * r->row + dim;
  if (!apart) set_error(std::string(who) + ": the rows of " + what + " overlap");
  return apart;
}

}  // namespace d4
namespace {
using namespace d4;

constexpr int kThreads = 256;

// fp32 with the last bit set when d is not an fp32 value (rounding to odd).
__device__ __forceinline__ float round_to_odd(double d) {
  const float f = __double2float_rz(d);
  return double(f) == d ? f : __uint_as_float(__float_as_uint(f) | 1u);
}

// Eight codes of x[0..8) under the scale s, the first in the low nibble.
__device__ __forceinline__ uint32_t e2m1_codes(const float* x, float s) {
  const float b0 = 0.25f * s, b1 = 0.75f * s, b2 = 1.25f * s, b3 = 1.75f * s, b4 = 2.5f * s, b5 = 3.5f * s, b6 = 5.f * s;
  uint32_t w = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float a = fabsf(x[j]);
    const bool hi = a > b3;                         // codes 4..7 or 0..3
    const bool mid = a > (hi ? b5 : b1);
    const bool lo = a > (hi ? (mid ? b6 : b4) : (mid ? b2 : b0));
    w |= ((hi ? 4u : 0u) | (mid ? 2u : 0u) | (lo ? 1u : 0u) | (__float_as_uint(x[j]) >> 31 << 3)) << (4 * j);
  }
  return w;
}

struct AppendArgs {
  ling_b200_kv4 c;
  ling_b200_kv4_batch b;
  ling_b200_rows k, v, q, q_out;
  int q_heads, rot;
  double theta;
  int* err;
};

// Where a packed row's vectors go: what a warp finds for the rest of the block.
struct RowAt {
  int pos, rope, page;  // page 0: nothing is done for this row
};
constexpr int kChunk = kThreads / 32;  // rows of a block at most

// By one warp of a call: sequences outside the batch's bounds are recorded, whether one of the packed rows is theirs or not (one that
// starts behind the rows has none here; where row0 descends one has fewer than none).
__device__ __forceinline__ void record_bad_seqs(const ling_b200_kv4& c, const ling_b200_kv4_batch& b, int* err) {
  for (int s = threadIdx.x & 31; s < b.seqs; s += 32)
    if (!kv4_seq(c, b, s).ok) dev_fail(err, kDevBadBatch);
}
// By warp: row r's place.  The error of a row whose page is out of bounds is recorded here.
__device__ __forceinline__ RowAt row_at(const ling_b200_kv4& c, const ling_b200_kv4_batch& b, int r, int* err) {
  RowAt at{0, 0, 0};
  const int s = kv4_find_seq(b.row0, b.seqs, r);
  if (s < 0) return at;  // padding behind the last sequence, or a batch against the rules
  const Kv4Seq q = kv4_seq(c, b, s);
  at.pos = q.pos + r - q.row0;
  if (q.ok) {
    at.page = c.tables[size_t(q.slot) * c.max_pages + at.pos / c.page_tokens];
    at.rope = b.rope_pos ? b.rope_pos[r] : at.pos;
  }
  if (at.page < 1 || at.page > c.pages) {
    if ((threadIdx.x & 31) == 0 && q.ok) dev_fail(err, kDevBadPage);
    at.page = 0;
  }
  return at;
}

// u / per and the rest for u < 2^18 and per <= 256, without a division (u times the reciprocal's error stays below 2^32).
struct Split {
  int per;
  uint32_t inv;
  __device__ explicit Split(int p) : per(p), inv(p > 1 ? 0xffffffffu / uint32_t(p) + 1u : 0u) {}
  __device__ int head(int u) const { return per > 1 ? int(__umulhi(uint32_t(u), inv)) : u; }
};

// A block takes `chunk` packed rows (1 to 8: rows_per_block): a warp per row finds its place, the rows' angles are shared out over
// the threads, then a thread takes a group of 16 dims of one K or V vector at a time (the groups of a vector are neighbouring lanes
// of one warp), then 16 pairs of dims of a query that turn together, then 16 bytes of the queries' dims that do not turn.  What a
// warp executes is of one kind: a query's turning dims beside its resting ones, lane by lane, cost three times the instructions.
// Bound by L1 and shared memory at many rows (76 % busy: the angles in double and fp32 beside the rows; issue slots 54 %, DRAM 27 %; the
// rows are read once, the queries written once, 9 / 16 byte a value goes to the cache), by the chain row0 -> slot -> page -> store
// and a cosine in double at few.  Measured: 8192 rows of 32 + 2 x 8 heads of 128 dims, all turning, BF16: 57 us, 3.2 TB/s; 64 rows of
// 24 + 2 x 4 heads of 256, 64 turning: 5 us.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) kv4_append_kernel(AppendArgs a, int chunk) {
  pdl_sync();  // first statement: see common.cuh
  __shared__ double2 turn[kChunk][128];  // cos, sin of a row's angles
  __shared__ float2 turn32[kChunk][128];
  __shared__ double freq[128];
  __shared__ RowAt rows[kChunk];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, r0 = blockIdx.x * chunk, n = min(chunk, a.b.rows - r0);
  const int D = a.c.head_dim, groups = D / 16, lg = 31 - __clz(groups), lp = 31 - __clz(a.c.page_tokens), half = a.rot / 2;
  if (warp < n) {
    const RowAt at = row_at(a.c, a.b, r0 + warp, a.err);
    if (lane == 0) rows[warp] = at;
  }
  if (blockIdx.x == 0 && warp == kChunk - 1) record_bad_seqs(a.c, a.b, a.err);
  if (tid < half) freq[tid] = pow(a.theta, -2.0 * tid / a.rot);
  __syncthreads();
  for (int t = tid; t < n * half; t += kThreads) {
    const int i = t / half, j = t - i * half;
    double sn, cs;
    sincos(double(rows[i].rope) * freq[j], &sn, &cs);
    turn[i][j] = make_double2(cs, sn), turn32[i][j] = make_float2(float(cs), float(sn));
  }
  __syncthreads();
  const int n_kv = a.c.kv_heads << lg;
  const double inv64 = 1.0 / double(a.c.k_scale);
  const float k_inv = 1.f / a.c.k_scale, v_inv = 1.f / a.c.v_scale;  // (powers of two: exact)
  const bool whole = half % 16 == 0;  // a group's dims turn all in one way or not at all
  // ---- K and V into the cache
  for (int t = tid; t - lane < n * 2 * n_kv; t += kThreads) {  // whole warps: the lanes of a warp exchange below
    const int row = t / (2 * n_kv), u_all = t - row * (2 * n_kv);
    const bool live = row < n && rows[row].page != 0, is_v = u_all >= n_kv;
    const int u = is_v ? u_all - n_kv : u_all, head = u >> lg, g = u & (groups - 1), r = r0 + row;
    const ling_b200_rows& src = is_v ? a.v : a.k;
    const T* vec = static_cast<const T*>(src.p) + r * src.row + head * src.head;
    float x[16] = {};
    bool bad = false;
    float amax6 = 0.f;  // max |x| / 6
    if (live) {
      load16<T, VEC>(vec + g * 16, x);
      if (!is_v && g * 16 < a.rot) {
        double top = 0.0;
        auto turned = [&](int j, double z) {
          bad |= !(fabs(z) <= double(FLT_MAX));
          top = fmax(top, fabs(z));
          x[j] = round_to_odd(z);
        };
        if (whole) {
          const bool low = g * 16 < half;
          const int at = low ? g * 16 : g * 16 - half;
          float o[16];  // the dims these turn with
          load16<T, VEC>(vec + (low ? g * 16 + half : at), o);
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const double2 cs = turn[row][at + j];
            const double sn = low ? -cs.y : cs.y;
            turned(j, (double(x[j]) * cs.x + double(o[j]) * sn) * inv64);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const int d = g * 16 + j;
            if (d >= a.rot) {
              turned(j, double(x[j]) * inv64);
              continue;
            }
            const bool low = d < half;
            const double2 cs = turn[row][low ? d : d - half];
            const double o = double(to_f32<T>(vec[low ? d + half : d - half]));
            turned(j, (double(x[j]) * cs.x + o * (low ? -cs.y : cs.y)) * inv64);
          }
        }
        amax6 = round_to_odd(top / 6.0);  // (E4M3 keeps four bits of it: what fp32 cuts off must not make a middle of two)
      } else {
        const float inv = is_v ? v_inv : k_inv;
        float top = 0.f;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          x[j] *= inv;
          bad |= !isfinite(x[j]);
          top = fmaxf(top, fabsf(x[j]));
        }
        amax6 = __fdiv_rn(top, 6.f);
      }
    }
    // a vector with a value that is not finite is NaN whole
    const unsigned any = __ballot_sync(0xffffffffu, bad) >> (lane >> lg << lg) & ((1u << groups) - 1u);
    if (!live) continue;
    const size_t at = kv4_vector(a.c, rows[row].page, head, rows[row].pos & ((1 << lp) - 1));
    uint8_t code = to_e4m3(fminf(fmaxf(amax6, 0x1p-9f), 448.f));
    const float sc = from_e4m3(code);
    uint2 w = make_uint2(e2m1_codes(x, sc), e2m1_codes(x + 8, sc));
    if (any) w = make_uint2(0, 0), code = 0x7f;
    reinterpret_cast<uint2*>((is_v ? a.c.v : a.c.k) + at * (D / 2))[g] = w;
    (is_v ? a.c.v_scales : a.c.k_scales)[at * groups + g] = code;
  }
  if (a.q_heads == 0) return;
  // ---- the queries' turning dims: a thread has both dims of its pairs, so q_out may be q
  const T* q = static_cast<const T*>(a.q.p);
  T* q_out = static_cast<T*>(a.q_out.p);
  const Split pairs((half + 15) / 16);
  for (int t = tid, per = a.q_heads * pairs.per; t < n * per; t += kThreads) {
    const int row = t / per, u = t - row * per, head = pairs.head(u), i0 = (u - head * pairs.per) * 16;
    if (rows[row].page == 0) continue;
    const T* from = q + (r0 + row) * a.q.row + head * a.q.head + i0;
    T* to = q_out + (r0 + row) * a.q_out.row + head * a.q_out.head + i0;
    if (whole) {
      float x[16], o[16];
      load16<T, VEC>(from, x);
      load16<T, VEC>(from + half, o);
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float2 cs = turn32[row][i0 + j];
        const float y = x[j] * cs.x - o[j] * cs.y;
        o[j] = x[j] * cs.y + o[j] * cs.x, x[j] = y;
      }
      store16<T, VEC>(to, x);
      store16<T, VEC>(to + half, o);
    } else {
      for (int j = 0; j < 16 && i0 + j < half; ++j) {
        const float2 cs = turn32[row][i0 + j];
        const float x = to_f32<T>(from[j]), o = to_f32<T>(from[j + half]);
        to[j] = from_f32<T>(x * cs.x - o * cs.y), to[j + half] = from_f32<T>(x * cs.y + o * cs.x);
      }
    }
  }
  // ---- and those that do not turn, where q_out is not q
  if (a.rot == D || (a.q.p == a.q_out.p && a.q.row == a.q_out.row && a.q.head == a.q_out.head)) return;
  if (VEC && whole) {
    constexpr int kPer = 16 / sizeof(T), kFly = 4;
    const Split pieces((D - a.rot) / kPer);
    const int per = a.q_heads * pieces.per;
    for (int t0 = tid; t0 < n * per; t0 += kThreads * kFly) {
      uint4 w[kFly];
      T* to[kFly];
#pragma unroll
      for (int f = 0; f < kFly; ++f) {
        const int t = t0 + f * kThreads, row = t / per, u = t - row * per, head = pieces.head(u), d = a.rot + (u - head * pieces.per) * kPer;
        to[f] = nullptr;
        if (t < n * per && rows[row].page != 0) {
          w[f] = *reinterpret_cast<const uint4*>(q + (r0 + row) * a.q.row + head * a.q.head + d);
          to[f] = q_out + (r0 + row) * a.q_out.row + head * a.q_out.head + d;
        }
      }
#pragma unroll
      for (int f = 0; f < kFly; ++f)
        if (to[f]) *reinterpret_cast<uint4*>(to[f]) = w[f];
    }
  } else {
    const Split rest(D - a.rot);
    for (int t = tid, per = a.q_heads * rest.per; t < n * per; t += kThreads) {
      const int row = t / per, u = t - row * per, head = rest.head(u), d = a.rot + u - head * rest.per;
      if (rows[row].page != 0) q_out[(r0 + row) * a.q_out.row + head * a.q_out.head + d] = q[(r0 + row) * a.q.row + head * a.q.head + d];
    }
  }
}

struct ReadArgs {
  ling_b200_kv4 c;
  ling_b200_kv4_batch b;
  ling_b200_rows k, v;
  int* err;
};

// As the append, the other way: a thread per group of 16 dims, read, decoded and stored.  8192 rows of 8 heads of 128 dims to BF16: 14 us,
// 3 TB/s; the loads wait for the lookups and one another (issue slots 61 %, L1 48 % busy), 1024 blocks are 1.7 waves.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) kv4_read_kernel(ReadArgs a, int chunk) {
  pdl_sync();  // first statement: see common.cuh
  __shared__ RowAt rows[kChunk];
  const int tid = threadIdx.x, warp = tid >> 5, r0 = blockIdx.x * chunk, n = min(chunk, a.b.rows - r0);
  const int D = a.c.head_dim, groups = D / 16, lg = 31 - __clz(groups), lp = 31 - __clz(a.c.page_tokens), n_kv = a.c.kv_heads << lg;
  if (warp < n) {
    const RowAt at = row_at(a.c, a.b, r0 + warp, a.err);
    if ((tid & 31) == 0) rows[warp] = at;
  }
  if (blockIdx.x == 0 && warp == kChunk - 1) record_bad_seqs(a.c, a.b, a.err);
  __syncthreads();
  int i = 0, left = tid;
  for (; left >= 2 * n_kv; left -= 2 * n_kv) ++i;
  while (i < n) {
    const int row = i, u_all = left;
    for (left += kThreads; left >= 2 * n_kv; left -= 2 * n_kv) ++i;
    const bool is_v = u_all >= n_kv;
    const int u = is_v ? u_all - n_kv : u_all, head = u >> lg, g = u & (groups - 1);
    const ling_b200_rows& to = is_v ? a.v : a.k;
    if (!to.p || rows[row].page == 0) continue;
    const size_t at = kv4_vector(a.c, rows[row].page, head, rows[row].pos & ((1 << lp) - 1));
    float x[16];
    decode16(reinterpret_cast<const uint2*>((is_v ? a.c.v : a.c.k) + at * (D / 2))[g],
             from_e4m3((is_v ? a.c.v_scales : a.c.k_scales)[at * groups + g]) * (is_v ? a.c.v_scale : a.c.k_scale), x);
    store16<T, VEC>(static_cast<T*>(to.p) + (r0 + row) * to.row + head * to.head + g * 16, x);
  }
}

// Rows of a block: one while the SMs are not filled (a row's chain of lookups is what a small batch takes), eight when they are
// filled many times over (the frequencies and the lookups' latency are then shared by eight rows).  Append and read of 8192 rows: at
// most 8 rows a block 71 us, 4 71, 2 78, 1 99.
inline int rows_per_block(int rows, int sms) { return std::min(kChunk, std::max(1, rows / (4 * sms))); }

DeviceInfo g_devices[kMaxDevices];
std::mutex g_mutex;

template <typename T>
int append_launch(const AppendArgs& a, bool vec, int sms, cudaStream_t s) {
  const int chunk = rows_per_block(a.b.rows, sms);
  LB_CUDA(launch_kernel(vec ? kv4_append_kernel<T, true> : kv4_append_kernel<T, false>, dim3((a.b.rows + chunk - 1) / chunk), dim3(kThreads), size_t(0), s, a, chunk));
  LB_LAUNCH("kv4_append_kernel");
  return LING_B200_OK;
}
template <typename T>
int read_launch(const ReadArgs& a, bool vec, int sms, cudaStream_t s) {
  const int chunk = rows_per_block(a.b.rows, sms);
  LB_CUDA(launch_kernel(vec ? kv4_read_kernel<T, true> : kv4_read_kernel<T, false>, dim3((a.b.rows + chunk - 1) / chunk), dim3(kThreads), size_t(0), s, a, chunk));
  LB_LAUNCH("kv4_read_kernel");
  return LING_B200_OK;
}

}  // namespace
}  // namespace lb

using namespace lb;
using namespace lb::d4;

extern "C" int ling_b200_kv4_append(int device, const ling_b200_kv4* cache, const ling_b200_kv4_batch* batch, int type,
                                    const ling_b200_rows* k, const ling_b200_rows* v, const ling_b200_rows* q, int q_heads,
                                    const ling_b200_rows* q_out, int rotary_dim, double theta, int* err, void* stream) {
  const char* who = "kv4_append";
  if (!kv4_cache_ok(cache, who) || !kv4_batch_ok(cache, batch, who)) return LING_B200_ERR_ARG;
  if (!type_ok(type)) {
    set_error("kv4_append: element types are LING_B200_F32, _BF16 and _F16");
    return LING_B200_ERR_ARG;
  }
  if (batch->rows == 0) return LING_B200_OK;  // (arrays without rows may have no address)
  const int D = cache->head_dim;
  if (!kv4_rows_ok(k, type, cache->kv_heads, D, who, "k") || !kv4_rows_ok(v, type, cache->kv_heads, D, who, "v")) return LING_B200_ERR_ARG;
  if (!q != !q_out || (q && (q_heads < 1 || q_heads > 1024 || !kv4_rows_ok(q, type, q_heads, D, who, "q") || !kv4_out_ok(q_out, type, batch->rows, q_heads, D, who, "q_out")))) {
    if (!q != !q_out || q_heads < 1 || q_heads > 1024) set_error("kv4_append: q and q_out come together, with 1 to 1024 heads");
    return LING_B200_ERR_ARG;
  }
  if (rotary_dim < 0 || rotary_dim > D || rotary_dim % 2 != 0 || !(theta > 0.0) || !std::isfinite(theta) || !aligned(err, 4)) {
    set_error("kv4_append: rotary_dim must be even and at most head_dim, theta positive and finite");
    return LING_B200_ERR_ARG;
  }
  DeviceGuard guard;
  int sms = 0;
  if (const int r = enter_device(guard, device, g_devices, g_mutex, [] { return LING_B200_OK; }, &sms)) return r;
  AppendArgs a{*cache, *batch, *k, *v, {nullptr, 0, 0}, {nullptr, 0, 0}, 0, rotary_dim, theta, err};
  bool vec = rows_vec(*k, type) && rows_vec(*v, type) && (rotary_dim / 2 % 16 != 0 || rotary_dim / 2 * type_size(type) % 16 == 0);
  if (q) a.q = *q, a.q_out = *q_out, a.q_heads = q_heads, vec = vec && rows_vec(*q, type) && rows_vec(*q_out, type);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return type == LING_B200_F32 ? append_launch<float>(a, vec, sms, s) : type == LING_B200_BF16 ? append_launch<__nv_bfloat16>(a, vec, sms, s) : append_launch<__half>(a, vec, sms, s);
}

extern "C" int ling_b200_kv4_read(int device, const ling_b200_kv4* cache, const ling_b200_kv4_batch* batch, int type, const ling_b200_rows* k,
                                  const ling_b200_rows* v, int* err, void* stream) {
  const char* who = "kv4_read";
  if (!kv4_cache_ok(cache, who) || !kv4_batch_ok(cache, batch, who)) return LING_B200_ERR_ARG;
  if (!type_ok(type) || (!k && !v) || !aligned(err, 4)) {
    set_error("kv4_read: a type and k or v expected");
    return LING_B200_ERR_ARG;
  }
  if (batch->rows == 0) return LING_B200_OK;
  if ((k && !kv4_out_ok(k, type, batch->rows, cache->kv_heads, cache->head_dim, who, "k")) ||
      (v && !kv4_out_ok(v, type, batch->rows, cache->kv_heads, cache->head_dim, who, "v")))
    return LING_B200_ERR_ARG;
  DeviceGuard guard;
  int sms = 0;
  if (const int r = enter_device(guard, device, g_devices, g_mutex, [] { return LING_B200_OK; }, &sms)) return r;
  const ReadArgs a{*cache, *batch, k ? *k : ling_b200_rows{nullptr, 0, 0}, v ? *v : ling_b200_rows{nullptr, 0, 0}, err};
  const bool vec = (!k || rows_vec(*k, type)) && (!v || rows_vec(*v, type));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return type == LING_B200_F32 ? read_launch<float>(a, vec, sms, s) : type == LING_B200_BF16 ? read_launch<__nv_bfloat16>(a, vec, sms, s) : read_launch<__half>(a, vec, sms, s);
}
