// Linear layers whose weights are held in 4 bits: W[n, k] = scales[k / group, n] * (code[n, k] - 8).
// Codes are bytes [n_out, padded / 2] (low nibble = even column, padded = n_in rounded up to a whole group; what the padding holds has
// no effect), scales fp32 [padded / group, n_out], group = a power of two >= 32.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include "common.cuh"

namespace bf {
namespace {

struct W4 {
  const uint8_t* codes;
  const float* scales;
  int n_out, n_in, group_log2;
  __host__ __device__ int groups() const { return (n_in + (1 << group_log2) - 1) >> group_log2; }
  __host__ __device__ long long pitch() const { return ((long long)groups() << group_log2) / 2; }
};

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half(v); }

__device__ __forceinline__ float load_any(const void* p, int type, long long i) {
  if (type == BF_TYPE_F32) return static_cast<const float*>(p)[i];
  if (type == BF_TYPE_BF16) return to_f32(static_cast<const __nv_bfloat16*>(p)[i]);
  return to_f32(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store_any(void* p, int type, long long i, float v) {
  if (type == BF_TYPE_F32) static_cast<float*>(p)[i] = v;
  else if (type == BF_TYPE_BF16) static_cast<__nv_bfloat16*>(p)[i] = from_f32<__nv_bfloat16>(v);
  else static_cast<__half*>(p)[i] = from_f32<__half>(v);
}

// ---- quantisation ----------------------------------------------------------------
// A warp per (row, group): largest magnitude, scale = that times 1/7 (as a 32-bit number), codes = round(w / scale) + 8.  The largest is taken over bit patterns, whose
// order is that of the magnitudes with infinities and NaN above: a group that holds one has it as its scale and is NaN throughout.
__global__ void __launch_bounds__(256) w4_quantise_kernel(const void* W, int type, uint8_t* codes, float* scales, W4 w) {
  const int G = 1 << w.group_log2, lane = threadIdx.x & 31;
  const int groups = w.groups();
  const long long units = (long long)w.n_out * groups, stride = (long long)gridDim.x * 8;
  for (long long u = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); u < units; u += stride) {
    const long long n = u / groups;
    const int g = (int)(u - n * groups);
    uint32_t top = 0;
    for (int j = lane; j < G; j += 32) {
      const int k = g * G + j;
      if (k < w.n_in) top = max(top, __float_as_uint(load_any(W, type, n * w.n_in + k)) & 0x7fffffffu);
    }
    top = __reduce_max_sync(0xffffffffu, top);
    const float scale = __fmul_rn(__uint_as_float(top), 1.f / 7.f);
    if (lane == 0) scales[(long long)g * w.n_out + n] = scale;
    uint8_t* out = codes + n * w.pitch() + (long long)g * (G / 2);
    for (int j = lane; j < G / 2; j += 32) {
      int q[2];
      for (int h = 0; h < 2; ++h) {
        const int k = g * G + 2 * j + h;
        const float v = k < w.n_in ? load_any(W, type, n * w.n_in + k) : 0.f;
        q[h] = (scale > 0.f && scale < INFINITY) ? min(7, max(-7, __float2int_rn(__fdiv_rn(v, scale)))) : 0;
      }
      out[j] = (uint8_t)((q[0] + 8) | ((q[1] + 8) << 4));
    }
  }
}

__global__ void __launch_bounds__(256) w4_unpack_kernel(W4 w, int8_t* integers, float* dense) {
  const long long total = (long long)w.n_out * w.n_in;
  for (long long i = blockIdx.x * 256LL + threadIdx.x; i < total; i += gridDim.x * 256LL) {
    const long long n = i / w.n_in;
    const int k = (int)(i - n * w.n_in);
    const int q = ((w.codes[n * w.pitch() + k / 2] >> (4 * (k & 1))) & 15) - 8;
    if (integers) integers[i] = (int8_t)q;
    else dense[i] = w.scales[(long long)(k >> w.group_log2) * w.n_out + n] * (float)q;
  }
}

// ---- products ----------------------------------------------------------------------
struct LinearArgs {
  W4 w;
  const void* a;      // x, or the first input of an interval
  const float* b;     // the second input of an interval
  const void* bias;
  void* y;            // y, or lower bounds
  float* y2;          // upper bounds
  int type, bias_type, mode, relu_in, M;
};

__device__ __forceinline__ void centre_radius(float a, float b, int mode, int relu_in, float& c, float& r) {
  if (mode == BF_IN_LOWER_UPPER) {
    if (relu_in) { a = fmaxf(a, 0.f); b = fmaxf(b, 0.f); }
    c = 0.5f * (a + b);
    r = 0.5f * (b - a);
  } else {
    c = a;
    r = b;
  }
}

// A warp per output and row; lanes walk the words of eight codes.
template <bool INTERVAL>
__global__ void __launch_bounds__(256) w4_forward_kernel(LinearArgs p) {
  const W4 w = p.w;
  const long long unit = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const long long m = unit / w.n_out;
  const int n = (int)(unit - m * w.n_out), lane = threadIdx.x & 31;
  if (m >= p.M) return;
  const uint8_t* row = w.codes + n * w.pitch();
  float c = 0.f, r = 0.f;
  for (int k = lane; k < w.n_in; k += 32) {
    const int q = ((row[k / 2] >> (4 * (k & 1))) & 15) - 8;
    const float s = w.scales[(long long)(k >> w.group_log2) * w.n_out + n] * (float)q;
    const long long at = m * w.n_in + k;
    if (INTERVAL) {
      float xc, xr;
      centre_radius(static_cast<const float*>(p.a)[at], p.b[at], p.mode, p.relu_in, xc, xr);
      c = fmaf(s, xc, c);
      r = fmaf(fabsf(s), xr, r);
    } else {
      c = fmaf(s, load_any(p.a, p.type, at), c);
    }
  }
  for (int o = 16; o > 0; o >>= 1) {
    c += __shfl_xor_sync(0xffffffffu, c, o);
    r += __shfl_xor_sync(0xffffffffu, r, o);
  }
  if (lane == 0) {
    if (p.bias) c += load_any(p.bias, p.bias_type, n);
    const long long at = m * w.n_out + n;
    if (INTERVAL) {
      static_cast<float*>(p.y)[at] = c - r;
      p.y2[at] = c + r;
    } else {
      store_any(p.y, p.type, at, c);
    }
  }
}

struct RowsArgs {
  W4 w;
  const void* a;   // rows, or gradients of lower bounds
  const float* b;  // gradients of upper bounds
  void* z;
  float* z2;
  int type, M;
};

// A thread per input feature and row.
template <bool INTERVAL>
__global__ void __launch_bounds__(256) w4_rows_kernel(RowsArgs p) {
  const W4 w = p.w;
  const long long unit = blockIdx.x * 256LL + threadIdx.x;
  const long long m = unit / w.n_in;
  const int k = (int)(unit - m * w.n_in);
  if (m >= p.M) return;
  const float* scale = w.scales + (long long)(k >> w.group_log2) * w.n_out;
  const uint8_t* code = w.codes + k / 2;
  float c = 0.f, r = 0.f;
  for (int n = 0; n < w.n_out; ++n) {
    const int q = ((code[n * w.pitch()] >> (4 * (k & 1))) & 15) - 8;
    const float s = scale[n] * (float)q;
    const long long at = m * w.n_out + n;
    if (INTERVAL) {
      const float lo = static_cast<const float*>(p.a)[at], up = p.b[at];
      c = fmaf(s, lo + up, c);
      r = fmaf(fabsf(s), up - lo, r);
    } else {
      c = fmaf(s, load_any(p.a, p.type, at), c);
    }
  }
  const long long at = m * w.n_in + k;
  if (INTERVAL) {
    static_cast<float*>(p.z)[at] = 0.5f * (c - r);
    p.z2[at] = 0.5f * (c + r);
  } else {
    store_any(p.z, p.type, at, c);
  }
}

// ---- sums beside the products ------------------------------------------------------------
// d[m] (+)= A[m, :] . bias: a warp per row.
__global__ void __launch_bounds__(256) rows_dot_kernel(const float* A, const float* bias, float* d, int accumulate, int M, int n) {
  const int m = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (m >= M) return;
  float s = 0.f;
  for (int j = lane; j < n; j += 32) s = fmaf(A[(long long)m * n + j], bias[j], s);
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) d[m] = accumulate ? d[m] + s : s;
}

// out[j] = sum over rows of A[:, j], rows in order.
__global__ void __launch_bounds__(256) column_sums_kernel(const void* A, int type, void* out, int out_type, int M, int n) {
  const int j = blockIdx.x * 256 + threadIdx.x;
  if (j >= n) return;
  float s = 0.f;
  for (int m = 0; m < M; ++m) s += load_any(A, type, (long long)m * n + j);
  store_any(out, out_type, j, s);
}

bool type_ok(int t) { return t == BF_TYPE_F32 || t == BF_TYPE_BF16 || t == BF_TYPE_F16; }

int make_w4(W4& w, const char* who, const void* codes, const void* scales, int n_out, int n_in, int group) {
  BF_REQUIRE(codes && scales, BF_E_INVALID, "%s: null weight", who);
  BF_REQUIRE(n_out > 0 && n_in > 0 && n_in <= 1 << 30, BF_E_INVALID, "%s: bad sizes %d x %d", who, n_out, n_in);
  BF_REQUIRE(group >= 32 && group <= 1 << 20 && (group & (group - 1)) == 0, BF_E_INVALID, "%s: group %d is not a power of two from 32 to 2^20", who, group);
  BF_REQUIRE((reinterpret_cast<uintptr_t>(codes) & 15u) == 0 && (reinterpret_cast<uintptr_t>(scales) & 3u) == 0, BF_E_INVALID,
             "%s: codes must lie on a 16-byte boundary", who);
  w.codes = static_cast<const uint8_t*>(codes);
  w.scales = static_cast<const float*>(scales);
  w.n_out = n_out;
  w.n_in = n_in;
  w.group_log2 = 0;
  while ((1 << w.group_log2) < group) ++w.group_log2;
  return BF_OK;
}

int blocks_for(long long units, int per_block) {
  const long long b = (units + per_block - 1) / per_block, cap = 148LL * 32;
  return (int)(b < cap ? b : cap);
}

}  // namespace
}  // namespace bf

extern "C" int bf_w4_quantise(const void* W, int type, uint8_t* codes, float* scales, int n_out, int n_in, int group, bf_stream_t stream) {
  bf::W4 w;
  const int rc = bf::make_w4(w, "bf_w4_quantise", codes, scales, n_out, n_in, group);
  if (rc != BF_OK) return rc;
  BF_REQUIRE(W && bf::type_ok(type), BF_E_INVALID, "bf_w4_quantise: null weight or unknown type %d", type);
  bf::w4_quantise_kernel<<<bf::blocks_for((long long)n_out * w.groups(), 8), 256, 0, bf::as_stream(stream)>>>(W, type, codes, scales, w);
  BF_CHECK_LAUNCH("w4_quantise_kernel");
  return BF_OK;
}

extern "C" int bf_w4_integers(const uint8_t* codes, int8_t* out, int n_out, int n_in, int group, bf_stream_t stream) {
  bf::W4 w;
  const int rc = bf::make_w4(w, "bf_w4_integers", codes, codes, n_out, n_in, group);
  if (rc != BF_OK) return rc;
  BF_REQUIRE(out, BF_E_INVALID, "bf_w4_integers: null output");
  bf::w4_unpack_kernel<<<bf::blocks_for((long long)n_out * n_in, 256), 256, 0, bf::as_stream(stream)>>>(w, out, nullptr);
  BF_CHECK_LAUNCH("w4_unpack_kernel");
  return BF_OK;
}

extern "C" int bf_w4_dense(const uint8_t* codes, const float* scales, float* out, int n_out, int n_in, int group, bf_stream_t stream) {
  bf::W4 w;
  const int rc = bf::make_w4(w, "bf_w4_dense", codes, scales, n_out, n_in, group);
  if (rc != BF_OK) return rc;
  BF_REQUIRE(out, BF_E_INVALID, "bf_w4_dense: null output");
  bf::w4_unpack_kernel<<<bf::blocks_for((long long)n_out * n_in, 256), 256, 0, bf::as_stream(stream)>>>(w, nullptr, out);
  BF_CHECK_LAUNCH("w4_unpack_kernel");
  return BF_OK;
}

extern "C" int bf_w4_linear(const void* x, int type, const uint8_t* codes, const float* scales, const void* bias, int bias_type, void* y, int M, int n_in,
                            int n_out, int group, bf_stream_t stream) {
  bf::LinearArgs p = {};
  const int rc = bf::make_w4(p.w, "bf_w4_linear", codes, scales, n_out, n_in, group);
  if (rc != BF_OK) return rc;
  BF_REQUIRE(x && y && M > 0 && bf::type_ok(type) && (!bias || bf::type_ok(bias_type)), BF_E_INVALID, "bf_w4_linear: null tensor, no rows or unknown type");
  p.a = x;
  p.bias = bias;
  p.y = y;
  p.type = type;
  p.bias_type = bias_type;
  p.M = M;
  bf::w4_forward_kernel<false><<<bf::ceil_div((long long)M * n_out, 8), 256, 0, bf::as_stream(stream)>>>(p);
  BF_CHECK_LAUNCH("w4_forward_kernel");
  return BF_OK;
}

extern "C" int bf_w4_interval(const float* in_a, const float* in_b, int in_mode, int relu_in, const uint8_t* codes, const float* scales, const float* bias,
                              float* out_l, float* out_u, int M, int n_in, int n_out, int group, bf_stream_t stream) {
  bf::LinearArgs p = {};
  const int rc = bf::make_w4(p.w, "bf_w4_interval", codes, scales, n_out, n_in, group);
  if (rc != BF_OK) return rc;
  BF_REQUIRE(in_a && in_b && out_l && out_u && M > 0, BF_E_INVALID, "bf_w4_interval: null tensor or no rows");
  BF_REQUIRE(in_mode == BF_IN_LOWER_UPPER || (in_mode == BF_IN_MID_RAD && !relu_in), BF_E_INVALID, "bf_w4_interval: bad input mode %d", in_mode);
  p.a = in_a;
  p.b = in_b;
  p.bias = bias;
  p.y = out_l;
  p.y2 = out_u;
  p.mode = in_mode;
  p.relu_in = relu_in;
  p.M = M;
  bf::w4_forward_kernel<true><<<bf::ceil_div((long long)M * n_out, 8), 256, 0, bf::as_stream(stream)>>>(p);
  BF_CHECK_LAUNCH("w4_forward_kernel");
  return BF_OK;
}

extern "C" int bf_w4_rows(const void* a, int type, const uint8_t* codes, const float* scales, void* z, int M, int n_in, int n_out, int group,
                          bf_stream_t stream) {
  bf::RowsArgs p = {};
  const int rc = bf::make_w4(p.w, "bf_w4_rows", codes, scales, n_out, n_in, group);
  if (rc != BF_OK) return rc;
  BF_REQUIRE(a && z && M > 0 && bf::type_ok(type), BF_E_INVALID, "bf_w4_rows: null tensor, no rows or unknown type");
  p.a = a;
  p.z = z;
  p.type = type;
  p.M = M;
  bf::w4_rows_kernel<false><<<bf::ceil_div((long long)M * n_in, 256), 256, 0, bf::as_stream(stream)>>>(p);
  BF_CHECK_LAUNCH("w4_rows_kernel");
  return BF_OK;
}

extern "C" int bf_w4_interval_grad(const float* grad_l, const float* grad_u, const uint8_t* codes, const float* scales, float* z_l, float* z_u, int M,
                                   int n_in, int n_out, int group, bf_stream_t stream) {
  bf::RowsArgs p = {};
  const int rc = bf::make_w4(p.w, "bf_w4_interval_grad", codes, scales, n_out, n_in, group);
  if (rc != BF_OK) return rc;
  BF_REQUIRE(grad_l && grad_u && z_l && z_u && M > 0, BF_E_INVALID, "bf_w4_interval_grad: null tensor or no rows");
  p.a = grad_l;
  p.b = grad_u;
  p.z = z_l;
  p.z2 = z_u;
  p.M = M;
  bf::w4_rows_kernel<true><<<bf::ceil_div((long long)M * n_in, 256), 256, 0, bf::as_stream(stream)>>>(p);
  BF_CHECK_LAUNCH("w4_rows_kernel");
  return BF_OK;
}

extern "C" int bf_rows_dot(const float* A, const float* bias, float* d, int accumulate, int M, int n, bf_stream_t stream) {
  BF_REQUIRE(A && bias && d && M > 0 && n > 0, BF_E_INVALID, "bf_rows_dot: null tensor or bad sizes");
  bf::rows_dot_kernel<<<bf::ceil_div(M, 8), 256, 0, bf::as_stream(stream)>>>(A, bias, d, accumulate, M, n);
  BF_CHECK_LAUNCH("rows_dot_kernel");
  return BF_OK;
}

extern "C" int bf_column_sums(const void* A, int type, void* out, int out_type, int M, int n, bf_stream_t stream) {
  BF_REQUIRE(A && out && M > 0 && n > 0 && bf::type_ok(type) && bf::type_ok(out_type), BF_E_INVALID, "bf_column_sums: null tensor, bad sizes or type");
  bf::column_sums_kernel<<<bf::ceil_div(n, 256), 256, 0, bf::as_stream(stream)>>>(A, type, out, out_type, M, n);
  BF_CHECK_LAUNCH("column_sums_kernel");
  return BF_OK;
}
