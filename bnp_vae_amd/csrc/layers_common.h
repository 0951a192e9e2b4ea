// What the layer operators (leaf_routes.hip, dense.hip) share: element types, 16-byte accesses, sums over the lanes of
// a row, the device guard of their entry points.
#pragma once

#include <algorithm>
#include <atomic>

#include "common.h"

namespace bnpvi {

constexpr int kTopMax = 8;              // choices per frame that top_leaves keeps in registers
constexpr int kSortMaxLeaves = 16384;   // two rows of counters of the sort fit the LDS

typedef __bf16 bf16_t;
typedef _Float16 f16_t;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_anywhere __attribute__((ext_vector_type(4), aligned(2)));      // global loads take any address
typedef uint32_t u32_anywhere __attribute__((aligned(2)));

inline int dtype_bytes(int dtype) { return dtype == BNPVI_F32 ? 4 : dtype == BNPVI_BF16 || dtype == BNPVI_F16 ? 2 : 0; }

// The entry points leave the caller's current device as they found it.
class OnDevice {
 public:
  explicit OnDevice(int device) {
    st_ = hipGetDevice(&before_);
    if (st_ == hipSuccess && before_ != device) {
      st_ = hipSetDevice(device);
      moved_ = st_ == hipSuccess;
    }
  }
  ~OnDevice() {
    if (moved_) (void)hipSetDevice(before_);
  }
  hipError_t status() const { return st_; }

 private:
  int before_ = 0;
  bool moved_ = false;
  hipError_t st_ = hipSuccess;
};

// Lets a kernel use the whole LDS on a device, once per device (any thread, any order).
class LdsLimit {
 public:
  hipError_t raise(const void* kernel, int device) {
    const uint64_t bit = uint64_t(1) << (device & 63);
    if (done_.load(std::memory_order_acquire) & bit) return hipSuccess;
    hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, kMaxLdsBytes);
    if (e == hipSuccess) done_.fetch_or(bit, std::memory_order_release);
    return e;
  }

 private:
  std::atomic<uint64_t> done_{0};
};

// E elements of T -- 16 bytes at any address, or one element -- as fp32; and back with one rounding to nearest even.
template <typename T, int E>
__device__ __forceinline__ void load_piece(const T* p, float (&v)[E]) {
  if constexpr (E == 1) {
    v[0] = (float)*p;
  } else {
    union {
      u32x4_anywhere u;
      T t[E];
    } q;
    q.u = *reinterpret_cast<const u32x4_anywhere*>(p);
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = (float)q.t[e];
  }
}
template <typename T, int E>
__device__ __forceinline__ void store_piece(T* p, const float (&v)[E]) {
  if constexpr (E == 1) {
    *p = (T)v[0];
  } else {
    union {
      u32x4_anywhere u;
      T t[E];
    } q;
#pragma unroll
    for (int e = 0; e < E; ++e) q.t[e] = (T)v[e];
    *reinterpret_cast<u32x4_anywhere*>(p) = q.u;
  }
}

// E elements anywhere in memory, the first `inside` of them (the others are 0, or not written).  Global loads and stores
// of 16 bytes take any address.
template <typename T, int E>
__device__ __forceinline__ void load_any(const T* p, int inside, float (&v)[E]) {
  union {
    u32x4_anywhere u[E * sizeof(T) / 16];
    T t[E];
  } q;
  if (inside >= E) {
#pragma unroll
    for (int i = 0; i < (int)(E * sizeof(T) / 16); ++i) q.u[i] = reinterpret_cast<const u32x4_anywhere*>(p)[i];
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = (float)q.t[e];
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = e < inside ? (float)p[e] : 0.f;
  }
}
// STREAM: past the caches' reuse order, for results as large as the caches that are written once
template <bool STREAM, typename T, int E>
__device__ __forceinline__ void store_any(T* p, int inside, const float (&v)[E]) {
  union {
    u32x4_anywhere u[E * sizeof(T) / 16];
    T t[E];
  } q;
#pragma unroll
  for (int e = 0; e < E; ++e) q.t[e] = (T)v[e];
  if (inside >= E) {
#pragma unroll
    for (int i = 0; i < (int)(E * sizeof(T) / 16); ++i) {
      if (STREAM)
        __builtin_nontemporal_store(q.u[i], reinterpret_cast<u32x4_anywhere*>(p) + i);
      else
        reinterpret_cast<u32x4_anywhere*>(p)[i] = q.u[i];
    }
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (e < inside) p[e] = q.t[e];
  }
}

// The value another lane of the same 16 holds (data-parallel primitive `CTRL`); all lanes take part.
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, false));
}
template <int CTRL>
__device__ __forceinline__ int dpp(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xf, 0xf, false);
}

// All-reduce over groups of G lanes (8, 16 or 64): pairs, quads, the two quads of eight (mirror), the two eights of
// sixteen (mirror) -- each step pairs a lane with one whose part is disjoint -- then across the rows of sixteen.
template <int G, typename V, typename Op>
__device__ __forceinline__ V lanes_reduce(V v, Op op) {
  v = op(v, dpp<0xB1>(v));
  v = op(v, dpp<0x4E>(v));
  v = op(v, dpp<0x141>(v));
  if (G >= 16) v = op(v, dpp<0x140>(v));
  if (G >= 32) v = op(v, __shfl_xor(v, 16));
  if (G >= 64) v = op(v, __shfl_xor(v, 32));
  return v;
}
template <int G>
__device__ __forceinline__ float lanes_max(float v) {
  return lanes_reduce<G>(v, [](float a, float b) { return a > b ? a : b; });
}
template <int G>
__device__ __forceinline__ int lanes_min(int v) {
  return lanes_reduce<G>(v, [](int a, int b) { return a < b ? a : b; });
}

}  // namespace bnpvi
