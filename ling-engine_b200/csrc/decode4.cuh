// decode4.cuh -- what the operators of a decode layer in 4 bits share (nvfp4_matvec.cu, kv4.cu, kv4_attention.cu): element
// types, the device guard of the entry points that take device pointers, NVFP4 decoding, the packed batch's lookups.
#pragma once

#include <cmath>
#include <mutex>

#include "../../include/ling_b200.h"
#include "common.cuh"

namespace lb {
namespace d4 {

constexpr int kDevBadBatch = 8;  // a packed batch outside its bounds: rows, slot, position or token of a sequence

// ---------------------------------------------------------------------------------------------- element types
template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

inline int type_size(int type) { return type == LING_B200_F32 ? 4 : 2; }
inline bool type_ok(int type) { return type == LING_B200_F32 || type == LING_B200_BF16 || type == LING_B200_F16; }
inline bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// 16 consecutive elements as floats; VEC: their address is a multiple of 16 bytes.
template <typename T, bool VEC>
__device__ __forceinline__ void load16(const T* p, float (&x)[16]) {
  if constexpr (VEC) {
    constexpr int kPer = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < 16 / kPer; ++i) {
      const uint4 w = reinterpret_cast<const uint4*>(p)[i];
      const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
      for (int j = 0; j < kPer; ++j) x[i * kPer + j] = to_f32<T>(e[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j) x[j] = to_f32<T>(p[j]);
  }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store16(T* p, const float (&x)[16]) {
  if constexpr (VEC) {
    constexpr int kPer = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < 16 / kPer; ++i) {
      uint4 w;
      T* e = reinterpret_cast<T*>(&w);
#pragma unroll
      for (int j = 0; j < kPer; ++j) e[j] = from_f32<T>(x[i * kPer + j]);
      reinterpret_cast<uint4*>(p)[i] = w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j) p[j] = from_f32<T>(x[j]);
  }
}

// ---------------------------------------------------------------------------------------------- NVFP4
// Two codes of a byte (the first in the low nibble) as two halves, exactly.
__device__ __forceinline__ uint32_t e2m1x2_to_h2(uint32_t byte) {
  uint32_t r;
  asm("{\n .reg .b8 b;\n mov.b16 {b, _}, %1;\n cvt.rn.f16x2.e2m1x2 %0, b;\n}" : "=r"(r) : "h"(uint16_t(byte)));
  return r;
}
// Eight codes of a word as four pairs of halves, exactly (half the rate of an fp32 operation on B200, a third of what shifts and masks cost).
__device__ __forceinline__ void e2m1x8_to_h2(uint32_t w, uint32_t (&h)[4]) {
  asm("{\n .reg .b8 a, b, c, d;\n mov.b32 {a, b, c, d}, %4;\n cvt.rn.f16x2.e2m1x2 %0, a;\n cvt.rn.f16x2.e2m1x2 %1, b;\n"
      " cvt.rn.f16x2.e2m1x2 %2, c;\n cvt.rn.f16x2.e2m1x2 %3, d;\n}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
}
// The 16 codes of 8 bytes times one scale.
__device__ __forceinline__ void decode16(const uint2& w, float scale, float (&x)[16]) {
  const uint32_t part[2] = {w.x, w.y};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t h = e2m1x2_to_h2((part[i >> 2] >> (8 * (i & 3))) & 0xffu);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    x[2 * i] = f.x * scale, x[2 * i + 1] = f.y * scale;
  }
}

// ---------------------------------------------------------------------------------------------- entry points
// The library's device for the length of a call; the caller's current device is put back.
class DeviceGuard {
 public:
  DeviceGuard() = default;
  ~DeviceGuard() {
    if (back_ >= 0) cudaSetDevice(back_);
  }
  int enter(int device) {
    int now = -1;
    LB_CUDA(cudaGetDevice(&now));
    if (now != device) {
      LB_CUDA(cudaSetDevice(device));
      back_ = now;
    }
    return LING_B200_OK;
  }

 private:
  int back_ = -1;
};

// A kernel that continues the one launched just before it on the stream: always as a programmatic dependent launch, so that its
// start overlaps that kernel's end (both wait for their predecessor in pdl_sync before they touch memory).
template <typename... KArgs, typename... Args>
inline cudaError_t launch_dependent(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid, cfg.blockDim = block, cfg.dynamicSmemBytes = smem, cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at, cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, KArgs(std::forward<Args>(args))...);
}

struct DeviceInfo {
  int sms = 0;  // 0: not looked at yet
};
constexpr int kMaxDevices = 64;

// Enters `device` and, on its first use, checks that it is a B200 and runs `init` (kernel attributes) for it.
template <typename F>
inline int enter_device(DeviceGuard& guard, int device, DeviceInfo (&infos)[kMaxDevices], std::mutex& m, F init, int* sms) {
  if (device < 0 || device >= kMaxDevices) {
    set_error("device ordinal out of range");
    return LING_B200_ERR_ARG;
  }
  if (const int r = guard.enter(device)) return r;
  std::lock_guard<std::mutex> lock(m);
  DeviceInfo& d = infos[device];
  if (d.sms == 0) {
    int major = 0, n = 0;
    LB_CUDA(cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device));
    if (major != 10) {
      set_error("this library is built for sm_100a (B200) only");
      return LING_B200_ERR_UNSUPPORTED;
    }
    LB_CUDA(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device));
    if (const int r = init()) return r;
    d.sms = n;
  }
  *sms = d.sms;
  return LING_B200_OK;
}

// ---------------------------------------------------------------------------------------------- the cache and the batch
bool kv4_cache_ok(const ling_b200_kv4* c, const char* who);
bool kv4_batch_ok(const ling_b200_kv4* c, const ling_b200_kv4_batch* b, const char* who);
bool kv4_rows_ok(const ling_b200_rows* r, int type, int heads, int dim, const char* who, const char* what);
bool kv4_out_ok(const ling_b200_rows* r, int type, int rows, int heads, int dim, const char* who, const char* what);  // and no two rows overlap
// Whether every 16-element piece of a strided row tensor starts on a 16-byte boundary.
inline bool rows_vec(const ling_b200_rows& r, int type) {
  const int per = 16 / type_size(type);
  return aligned(r.p, 16) && r.row % per == 0 && r.head % per == 0;
}

// Position `tok` of page `page`, kv head h: its index among the cache's (page, head, token) vectors.
__device__ __forceinline__ size_t kv4_vector(const ling_b200_kv4& c, int page, int h, int tok) {
  return (size_t(page) * c.kv_heads + h) * c.page_tokens + tok;
}
// The sequence of packed row r (all lanes of a warp together, any number of sequences), or -1: none has it, or row0 descends, so that it
// could lie in several, or be counted to one that does not hold it.
__device__ __forceinline__ int kv4_find_seq(const int* __restrict__ row0, int seqs, int r) {
  int n = 0;  // sequences that end at or before r
  bool down = false;
  for (int s = 0; s < seqs; s += 32) {
    const int i = s + int(threadIdx.x & 31), begin = i < seqs ? row0[i] : 0, end = i < seqs ? row0[i + 1] : 0;
    n += __popc(__ballot_sync(0xffffffffu, i < seqs && end <= r));
    down |= end < begin;
  }
  return !__any_sync(0xffffffffu, down) && n < seqs && row0[n] <= r ? n : -1;
}
struct Kv4Seq {
  int row0, n, slot, pos;
  bool ok;  // inside the batch's and the cache's bounds
};
__device__ __forceinline__ Kv4Seq kv4_seq(const ling_b200_kv4& c, const ling_b200_kv4_batch& b, int s) {
  Kv4Seq q{b.row0[s], 0, b.slot[s], b.pos[s], false};
  q.n = b.row0[s + 1] - q.row0;
  q.ok = q.row0 >= 0 && q.n >= 0 && q.n <= b.max_rows && q.row0 <= b.rows - q.n && q.slot >= 0 && q.slot < c.slots && q.pos >= 0 &&
         q.pos <= b.max_context - q.n;
  return q;
}

}  // namespace d4
}  // namespace lb
