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
