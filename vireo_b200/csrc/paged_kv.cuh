// What the paged key-value sources share: the handle behind gguf_kv, the
// types of activations and cache, and the conversions between them and fp32.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <mutex>

#include "gguf_kv.h"
#include "vireo_internal.h"
#include "vireo_ptx.cuh"

namespace vireo {

enum KvType : uint32_t { KV_F32 = 0, KV_F16 = 1, KV_BF16 = 30 };
inline int kv_type_size(uint32_t t) { return t == KV_F32 ? 4 : 2; }

constexpr int kKvMaxHalf = 128;  // rotation pairs of the largest head
// revolutions per position of each rotation pair, base^(-2j / dim) / (2 pi);
// a kernel parameter, so that a handle needs no device memory
struct KvFreq {
  double rev[kKvMaxHalf];
};

// launches on the library's device whatever the calling thread's current one
// is, and puts the thread's device back
struct DeviceGuard {
  int old = -1;
  int status = VIREO_OK;
  explicit DeviceGuard(int device) {
    int cur = -1;
    if ((status = cuda_status(cudaGetDevice(&cur))) || cur == device) return;
    if (!(status = cuda_status(cudaSetDevice(device)))) old = cur;
  }
  ~DeviceGuard() {
    if (old >= 0) cudaSetDevice(old);
  }
};

inline bool kv_aligned(const void* p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }
// a row stride of `row` elements of `el` bytes or more, in whole 16 bytes
inline bool kv_stride_ok(int64_t stride, int64_t row, int el) {
  return stride >= row && stride <= (INT64_MAX >> 6) && (stride * el) % 16 == 0;
}

VDEV float to_f(float v) { return v; }
VDEV float to_f(__half v) { return __half2float(v); }
VDEV float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
VDEV T from_f(float v);
template <>
VDEV float from_f<float>(float v) { return v; }
template <>
VDEV __half from_f<__half>(float v) { return __float2half_rn(v); }
template <>
VDEV __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// N consecutive values between memory and fp32 registers, in accesses of at
// most 16 bytes (p aligned to min(16, N * sizeof(T)) bytes)
template <int N, class T>
VDEV void load_f(const T* p, float (&o)[N]) {
  constexpr int B = N * (int)sizeof(T);
  static_assert(B % 4 == 0, "whole words");
  uint32_t w[B / 4];
  if constexpr (B >= 16) {
#pragma unroll
    for (int i = 0; i < B / 16; i++)
      *reinterpret_cast<uint4*>(w + 4 * i) = *(reinterpret_cast<const uint4*>(p) + i);
  } else if constexpr (B == 8) {
    *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(p);
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
  const T* t = reinterpret_cast<const T*>(w);
#pragma unroll
  for (int i = 0; i < N; i++) o[i] = to_f(t[i]);
}
template <int N, class T>
VDEV void store_f(T* p, const float (&v)[N]) {
  constexpr int B = N * (int)sizeof(T);
  uint32_t w[B / 4];
  T* t = reinterpret_cast<T*>(w);
#pragma unroll
  for (int i = 0; i < N; i++) t[i] = from_f<T>(v[i]);
  if constexpr (B >= 16) {
#pragma unroll
    for (int i = 0; i < B / 16; i++)
      *(reinterpret_cast<uint4*>(p) + i) = *reinterpret_cast<const uint4*>(w + 4 * i);
  } else if constexpr (B == 8) {
    *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(w);
  } else {
    *reinterpret_cast<uint32_t*>(p) = w[0];
  }
}

// Pairs of fp32 values in one register pair: each half is rounded as the
// scalar operation is.
typedef unsigned long long f2;
VDEV f2 f2_make(float a, float b) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
VDEV void f2_get(f2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
VDEV f2 f2_mul(f2 a, f2 b) {
  f2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
VDEV f2 f2_add(f2 a, f2 b) {
  f2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
VDEV f2 f2_fma(f2 a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
// four values, 16-byte aligned
VDEV void load4(const float* p, f2* o) {
  const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(p);
  o[0] = v.x;
  o[1] = v.y;
}

}  // namespace vireo

struct gguf_kv {
  gguf_kv_desc d;
  int ps_shift;
  vireo::KvFreq freq;
  // tensor maps of the two pools, made at the first attention call
  std::mutex mu;
  bool maps_ok = false;
  int per_sm = 0;  // attention CTAs an SM holds
  CUtensorMap map_k, map_v;
};
