// kv4_attention.cu -- attention over the paged NVFP4 KV cache (ling_b200_kv4_attention).
//
//   out[r][h] = sum_j p_j V_j / sum_j p_j,  p_j = exp(scale * q . K_j - m),  m = max_j scale * q . K_j,
// over the positions j that row r sees: [0, pos) of its sequence, and of the in-flight positions pos + i those its ancestor
// mask (or, without one, its index) admits.
#include "decode4.cuh"

namespace lb {
namespace {
using namespace d4;

constexpr int kThreads = 128;

struct AttnArgs {
  ling_b200_kv4 c;
  ling_b200_kv4_batch b;
  ling_b200_rows q, out;
  int q_heads;
  float scale;
  float* lse;
  int* err;
};

// A block per (row, query head): 128 keys at a time, a thread a key for the scores, then a thread two dims for the values,
// with the running maximum and sum of the softmax in fp32.
template <typename T>
__global__ void __launch_bounds__(kThreads) kv4_attention_simple_kernel(AttnArgs a) {
  pdl_sync();  // first statement: see common.cuh
  __shared__ float qs[256], red[32], ps[kThreads];
  __shared__ int pages[kThreads];
  const int r = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, D = a.c.head_dim, groups = D / 16, T_page = a.c.page_tokens;
  const int s = kv4_find_seq(a.b.row0, a.b.seqs, r);
  if (s < 0) return;
  const Kv4Seq sq = kv4_seq(a.c, a.b, s);
  if (!sq.ok) {
    if (tid == 0) dev_fail(a.err, kDevBadBatch);
    return;
  }
  const int i = r - sq.row0, kvh = h / (a.q_heads / a.c.kv_heads), keys = sq.pos + sq.n;
  const uint32_t see = a.b.anc ? a.b.anc[r] : i < 31 ? (2u << i) - 1u : 0xffffffffu;
  for (int d = tid; d < D; d += kThreads) qs[d] = to_f32<T>(static_cast<const T*>(a.q.p)[r * a.q.row + h * a.q.head + d]);
  float m = -INFINITY, l = 0.f, o[2] = {0.f, 0.f};
  for (int k0 = 0; k0 < keys; k0 += kThreads) {
    const int pos = k0 + tid, j = pos - sq.pos;
    bool visible = pos < keys && (j < 0 || (a.b.anc ? (see >> j & 1u) : j <= i));
    int page = 0;
    if (visible) {
      page = a.c.tables[size_t(sq.slot) * a.c.max_pages + pos / T_page];
      if (page < 1 || page > a.c.pages) {
        dev_fail(a.err, kDevBadPage);
        visible = false;
      }
    }
    __syncthreads();  // the previous tile is done with ps and pages; qs is written
    float sc = -INFINITY;
    if (visible) {
      const size_t at = kv4_vector(a.c, page, kvh, pos % T_page);
      float dot = 0.f;
      for (int g = 0; g < groups; ++g) {
        float x[16];
        decode16(reinterpret_cast<const uint2*>(a.c.k + at * (D / 2))[g], from_e4m3(a.c.k_scales[at * groups + g]), x);
#pragma unroll
        for (int e = 0; e < 16; ++e) dot = fmaf(x[e], qs[g * 16 + e], dot);
      }
      sc = dot * (a.scale * a.c.k_scale);
    }
    float top = warp_max(sc);
    // a score that is not a number must stay one: fmaxf drops it, the sums below do not
    if ((tid & 31) == 0) red[tid >> 5] = top;
    __syncthreads();
    const float m_new = fmaxf(fmaxf(m, fmaxf(red[0], red[1])), fmaxf(red[2], red[3]));
    const float keep = m == -INFINITY ? 0.f : expf(m - m_new);
    const float p = !visible ? 0.f : m_new == -INFINITY ? (sc == sc ? 0.f : sc) : expf(sc - m_new);
    ps[tid] = p, pages[tid] = visible ? page : 0;
    const float sum = block_sum(p, red);
    __syncthreads();
    l = l * keep + sum;
    o[0] *= keep, o[1] *= keep;
    m = m_new;
    for (int k = 0; k < min(kThreads, keys - k0); ++k) {
      if (pages[k] == 0) continue;
      const size_t at = kv4_vector(a.c, pages[k], kvh, (k0 + k) % T_page);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int d = tid * 2 + e;
        if (d < D) {
          const uint32_t byte = a.c.v[at * (D / 2) + d / 2];
          o[e] = fmaf(ps[k], from_e2m1(d & 1 ? byte >> 4 : byte & 15u) * from_e4m3(a.c.v_scales[at * groups + d / 16]), o[e]);
        }
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int d = tid * 2 + e;
    const bool empty = m == -INFINITY && l == 0.f;
    if (d < D) static_cast<T*>(a.out.p)[r * a.out.row + h * a.out.head + d] = from_f32<T>(empty ? 0.f : o[e] / l * a.c.v_scale);
    if (d == 0 && a.lse) a.lse[size_t(r) * a.q_heads + h] = empty ? -INFINITY : m + logf(l);
  }
}

DeviceInfo g_devices[kMaxDevices];
std::mutex g_mutex;

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
  return 16;
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
  if (const int r = enter_device(guard, device, g_devices, g_mutex, [] { return LING_B200_OK; }, &sms)) return r;
  const AttnArgs a{*cache, *batch, *q, *out, q_heads, scale, lse, err};
  LB_CUDA(launch_kernel(type == LING_B200_BF16 ? kv4_attention_simple_kernel<__nv_bfloat16> : kv4_attention_simple_kernel<__half>,
                        dim3(batch->rows, q_heads), dim3(kThreads), size_t(0), static_cast<cudaStream_t>(stream), a));
  LB_LAUNCH("kv4_attention_simple_kernel");
  return LING_B200_OK;
}
