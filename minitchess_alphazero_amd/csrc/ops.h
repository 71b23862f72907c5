// Pieces shared by the learner operators (mtaz_muon.hip, mtaz_logits.hip): their error entry, element
// types, and the choice of device around a call.
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/mtaz.h"

namespace mtaz {

// sets mtaz_last_error() to "what: why" and returns code (mtaz_host.cpp)
int ops_error(int code, const char* what, const char* why);

// The calling thread's current device becomes `device` for the scope, and what it was afterwards.
struct DeviceScope {
  int before = -1;
  hipError_t status;
  explicit DeviceScope(int device) {
    status = hipGetDevice(&before);
    if (status == hipSuccess && before != device) status = hipSetDevice(device);
    if (before == device) before = -1;
  }
  ~DeviceScope() {
    if (before >= 0) (void)hipSetDevice(before);
  }
};

// One element of type MTAZ_F32 / MTAZ_F16 / MTAZ_BF16 in memory; arithmetic is in float, a store rounds
// to nearest even.
template <int DT> struct Elem;
template <> struct Elem<MTAZ_F32> {
  typedef float T;
  static __device__ __forceinline__ float get(float x) { return x; }
  static __device__ __forceinline__ float put(float x) { return x; }
};
template <> struct Elem<MTAZ_F16> {
  typedef _Float16 T;
  static __device__ __forceinline__ float get(_Float16 x) { return (float)x; }
  static __device__ __forceinline__ _Float16 put(float x) { return (_Float16)x; }
};
template <> struct Elem<MTAZ_BF16> {
  typedef __bf16 T;
  static __device__ __forceinline__ float get(__bf16 x) { return (float)x; }
  static __device__ __forceinline__ __bf16 put(float x) { return (__bf16)x; }
};
constexpr int elem_size(int dtype) { return dtype == MTAZ_F32 ? 4 : 2; }

// N consecutive elements at any address an element may have (the global memory path takes wide
// accesses at element alignment)
template <typename T, int N> struct __attribute__((packed, aligned(sizeof(T)))) Pack {
  T v[N];
};

}  // namespace mtaz
