// What the kernels of 4-bit weights share: W[n, k] = scales[k / group, n] * (code[n, k] - 8).  Codes are bytes [n_out, padded / 2] (low nibble = even
// column, padded = n_in rounded up to a whole group; what the padding holds has no effect), scales fp32 [padded / group, n_out], group = a power of two >= 32.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace bf {

struct W4 {
  const uint8_t* codes;
  const float* scales;
  int n_out, n_in, group_log2;
  __host__ __device__ int groups() const { return (n_in + (1 << group_log2) - 1) >> group_log2; }
  __host__ __device__ long long pitch() const { return ((long long)groups() << group_log2) / 2; }
};

__device__ __forceinline__ float load_any(const void* p, int type, long long i) {
  if (type == BF_TYPE_F32) return static_cast<const float*>(p)[i];
  if (type == BF_TYPE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store_any(void* p, int type, long long i, float v) {
  if (type == BF_TYPE_F32) static_cast<float*>(p)[i] = v;
  else if (type == BF_TYPE_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16(v);
  else static_cast<__half*>(p)[i] = __float2half(v);
}

// Codes in bits 0-3 and 16-19 of `w`, minus 8, as two bfloat16: 0x4300 | code is 128 + code, since 128 has its last mantissa bit at 1 (building a float from an integer's bits so is common practice).  ("And, or" is one instruction where one of the two constants is
// in a register, which the compiler does not do by itself: the integer pipe, 64 lanes a clock, is what these kernels fill first.)
__device__ __forceinline__ uint32_t weights_of(uint32_t w) {
  uint32_t v;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(v) : "r"(w), "r"(0x000f000fu), "r"(0x43004300u));
  const __nv_bfloat162 off = __halves2bfloat162(__ushort_as_bfloat16(0x4308), __ushort_as_bfloat16(0x4308));
  const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), off);
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ void put16(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// y = x W^T + bias, or with `b` the bounds of it over boxes.
struct W4LinearArgs {
  W4 w;
  const void* a;      // x, or the first input of an interval
  const float* b;     // the second input of an interval
  const void* bias;
  void* y;            // y, or lower bounds
  float* y2;          // upper bounds
  int type, bias_type, mode, relu_in, M;
};
// z = a W, or with `b` the gradients of the bounds' inputs.
struct W4RowsArgs {
  W4 w;
  const void* a;   // rows, or gradients of lower bounds
  const float* b;  // gradients of upper bounds
  void* z;
  float* z2;
  int type, M;
};
int launch_w4_linear(const W4LinearArgs& p, cudaStream_t stream);
int launch_w4_rows(const W4RowsArgs& p, cudaStream_t stream);
// The same for many rows, with a workspace of w4_many_bytes; whether they are the faster ones.
long long w4_many_bytes(int M, int sum, int type);
bool w4_many_pays(int M, int n_in, int n_out, int group, int type, bool forward, bool pair);
int launch_w4_linear_many(const W4LinearArgs& p, void* workspace, cudaStream_t stream);
int launch_w4_rows_many(const W4RowsArgs& p, void* workspace, cudaStream_t stream);

}  // namespace bf
