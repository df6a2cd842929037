// nvfp4_matvec.cu -- a few rows of activations times an NVFP4 weight matrix, activations in their own type:
//   y[m][n] = alpha * sum_k x[m][k] * e2m1(values[n][k]) * e4m3(scales[n][k / 16])
// for one token to a draft tree's 32 rows.  The weights are read once, N * K * 9 / 16 bytes: at these row counts that
// stream is the floor (the prefill chunk's GEMM in nvfp4.cu pays a 128-row tile and an activation quantizer instead).
#include "decode4.cuh"

namespace lb {
namespace {
using namespace d4;

constexpr int kRowBlock = 4;  // activation rows a warp carries at a time

__device__ __forceinline__ uint2 load8(const uint8_t* p, bool vec) {
  if (vec) return *reinterpret_cast<const uint2*>(p);
  uint2 w{0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) w.x |= uint32_t(p[i]) << (8 * i), w.y |= uint32_t(p[4 + i]) << (8 * i);
  return w;
}

// A warp per output column n: its lanes take groups of 16 k in turn, the lanes' sums meet in a fixed tree.
template <typename TX, typename TY>
__global__ void __launch_bounds__(256)
    matvec_simple_kernel(const TX* __restrict__ x, long long ldx, int M, const uint8_t* __restrict__ values,
                         const uint8_t* __restrict__ scales, float alpha, int N, int K, TY* y, long long ldy, int accumulate, bool vec) {
  pdl_sync();  // first statement: see common.cuh
  const int n = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31, groups = K / 16;
  if (n >= N) return;
  const uint8_t* w = values + size_t(n) * (K / 2);
  const uint8_t* ws = scales + size_t(n) * groups;
  for (int m0 = 0; m0 < M; m0 += kRowBlock) {
    float acc[kRowBlock] = {};
    for (int g = lane; g < groups; g += 32) {
      float wv[16];
      decode16(load8(w + size_t(g) * 8, vec), from_e4m3(ws[g]), wv);
#pragma unroll
      for (int i = 0; i < kRowBlock; ++i) {
        if (m0 + i >= M) break;
        const TX* row = x + (m0 + i) * ldx + size_t(g) * 16;
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[i] = fmaf(to_f32<TX>(row[j]), wv[j], acc[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < kRowBlock; ++i) {
      const float v = warp_sum(acc[i]);
      if (lane == 0 && m0 + i < M) {
        TY* to = y + (m0 + i) * ldy + n;
        *to = from_f32<TY>(accumulate ? to_f32<TY>(*to) + alpha * v : alpha * v);
      }
    }
  }
}

template <typename TX, typename TY>
int matvec_launch(const void* x, long long ldx, int M, const uint8_t* values, const uint8_t* scales, float alpha, int N, int K, void* y,
                  long long ldy, int accumulate, cudaStream_t s) {
  const bool vec = aligned(values, 8);  // a row is K / 2 bytes, a multiple of 8
  LB_CUDA(launch_kernel(matvec_simple_kernel<TX, TY>, dim3(ceil_div(N, 8)), dim3(256), size_t(0), s, static_cast<const TX*>(x), ldx, M, values,
                        scales, alpha, N, K, static_cast<TY*>(y), ldy, accumulate, vec));
  LB_LAUNCH("matvec_simple_kernel");
  return LING_B200_OK;
}

DeviceInfo g_devices[kMaxDevices];
std::mutex g_mutex;

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
      !d4::aligned(x, d4::type_size(x_type)) || !d4::aligned(y, d4::type_size(y_type))) {
    set_error("nvfp4_matvec: bad argument (1 <= M <= 32, K a multiple of 16, ldx >= K, ldy >= N)");
    return LING_B200_ERR_ARG;
  }
  d4::DeviceGuard guard;
  int sms = 0;
  if (const int r = d4::enter_device(guard, device, g_devices, g_mutex, [] { return LING_B200_OK; }, &sms)) return r;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
#define LB_MV(TX, TY) matvec_launch<TX, TY>(x, ldx, M, values, scales, alpha, N, K, y, ldy, accumulate, s)
#define LB_MV_Y(TX) (y_type == LING_B200_F32 ? LB_MV(TX, float) : y_type == LING_B200_BF16 ? LB_MV(TX, __nv_bfloat16) : LB_MV(TX, __half))
  return x_type == LING_B200_F32 ? LB_MV_Y(float) : x_type == LING_B200_BF16 ? LB_MV_Y(__nv_bfloat16) : LB_MV_Y(__half);
#undef LB_MV_Y
#undef LB_MV
}
