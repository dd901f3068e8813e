// Linear layers whose weights are held in 4 bits (weights4.cuh): quantisation, unpacking, the sums beside the products, and the C entries.
#include <math.h>

#include "weights4.cuh"

namespace bf {
namespace {

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
  bf::W4LinearArgs p = {};
  const int rc = bf::make_w4(p.w, "bf_w4_linear", codes, scales, n_out, n_in, group);
  if (rc != BF_OK) return rc;
  BF_REQUIRE(x && y && M > 0 && bf::type_ok(type) && (!bias || bf::type_ok(bias_type)), BF_E_INVALID, "bf_w4_linear: null tensor, no rows or unknown type");
  p.a = x;
  p.bias = bias;
  p.y = y;
  p.type = type;
  p.bias_type = bias_type;
  p.M = M;
  return bf::launch_w4_linear(p, bf::as_stream(stream));
}

extern "C" int bf_w4_interval(const float* in_a, const float* in_b, int in_mode, int relu_in, const uint8_t* codes, const float* scales, const float* bias,
                              float* out_l, float* out_u, int M, int n_in, int n_out, int group, bf_stream_t stream) {
  bf::W4LinearArgs p = {};
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
  return bf::launch_w4_linear(p, bf::as_stream(stream));
}

extern "C" int bf_w4_rows(const void* a, int type, const uint8_t* codes, const float* scales, void* z, int M, int n_in, int n_out, int group,
                          bf_stream_t stream) {
  bf::W4RowsArgs p = {};
  const int rc = bf::make_w4(p.w, "bf_w4_rows", codes, scales, n_out, n_in, group);
  if (rc != BF_OK) return rc;
  BF_REQUIRE(a && z && M > 0 && bf::type_ok(type), BF_E_INVALID, "bf_w4_rows: null tensor, no rows or unknown type");
  p.a = a;
  p.z = z;
  p.type = type;
  p.M = M;
  return bf::launch_w4_rows(p, bf::as_stream(stream));
}

extern "C" int bf_w4_interval_grad(const float* grad_l, const float* grad_u, const uint8_t* codes, const float* scales, float* z_l, float* z_u, int M,
                                   int n_in, int n_out, int group, bf_stream_t stream) {
  bf::W4RowsArgs p = {};
  const int rc = bf::make_w4(p.w, "bf_w4_interval_grad", codes, scales, n_out, n_in, group);
  if (rc != BF_OK) return rc;
  BF_REQUIRE(grad_l && grad_u && z_l && z_u && M > 0, BF_E_INVALID, "bf_w4_interval_grad: null tensor or no rows");
  p.a = grad_l;
  p.b = grad_u;
  p.z = z_l;
  p.z2 = z_u;
  p.M = M;
  return bf::launch_w4_rows(p, bf::as_stream(stream));
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
