// Statistics of one 16-byte column of a page of keys, shared by the kernels that build and refresh them.
//
// Arithmetic (mirrored by the CPU oracle): rows of a page in storage order;
// mean = (((x0+x1)+x2)+...)/n; var = ((d0*d0+d1*d1)+...)/n with d = x - mean and
// separately rounded products and sums; std = max(sqrt(var), 1e-6); one rounding
// to the storage dtype at the end.
#pragma once

#include "ekv_common.cuh"

namespace ekv {

template <typename T>
struct ColumnStats {
  static constexpr int EPL = ElemTraits<T>::EPL;
  float mn[EPL], mx[EPL], sum[EPL], mean[EPL], sq[EPL];
  __device__ __forceinline__ void begin() {
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      mn[j] = INFINITY;
      mx[j] = -INFINITY;
      sum[j] = 0.f;
    }
  }
  __device__ __forceinline__ void first_pass(const uint4& raw) {
    float x[EPL];
    unpack<T>(raw, x);
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      mn[j] = fminf(mn[j], x[j]);
      mx[j] = fmaxf(mx[j], x[j]);
      sum[j] = __fadd_rn(sum[j], x[j]);
    }
  }
  __device__ __forceinline__ void middle(float n) {
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      mean[j] = __fdiv_rn(sum[j], n);
      sq[j] = 0.f;
    }
  }
  __device__ __forceinline__ void second_pass(const uint4& raw) {
    float x[EPL];
    unpack<T>(raw, x);
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      const float d = __fsub_rn(x[j], mean[j]);
      sq[j] = __fadd_rn(sq[j], __fmul_rn(d, d));
    }
  }
  __device__ __forceinline__ void finish(float n, T* o_min, T* o_max, T* o_mean, T* o_std) {
    float sd[EPL];
#pragma unroll
    for (int j = 0; j < EPL; ++j) sd[j] = fmaxf(__fsqrt_rn(__fdiv_rn(sq[j], n)), 1e-6f);
    *reinterpret_cast<uint4*>(o_min) = pack<T>(mn);
    *reinterpret_cast<uint4*>(o_max) = pack<T>(mx);
    *reinterpret_cast<uint4*>(o_mean) = pack<T>(mean);
    *reinterpret_cast<uint4*>(o_std) = pack<T>(sd);
  }
};

}  // namespace ekv
