// Linear layers whose weights are held in 4 bits (weights4.cuh): quantisation, unpacking, the sums beside the products, and the C entries.
#include <math.h>

#include <algorithm>

#include "weights4.cuh"

namespace bf {
namespace {

// ---- quantisation ----------------------------------------------------------------
__device__ __forceinline__ void load_eight(const void* p, int type, long long at, int left, bool wide, float (&v)[8]) {
  if (!wide || left < 8) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < left ? load_any(p, type, at + j) : 0.f;
  } else if (type == BF_TYPE_F32) {
    const float4 x = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + at), y = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + at + 4);
    v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
    v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
  } else {
    const uint4 x = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + at);
    const uint32_t q[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = type == BF_TYPE_BF16 ? __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&q[j])) : __half22float2(*reinterpret_cast<const __half2*>(&q[j]));
      v[2 * j] = f.x;
      v[2 * j + 1] = f.y;
    }
  }
}
// Bit pattern of the largest magnitude, that of a NaN where one is among them.
__device__ __forceinline__ uint32_t largest(const float (&v)[8]) {
  float top = fabsf(v[0]);
#pragma unroll
  for (int j = 1; j < 8; ++j) asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(fabsf(v[j])));
  return __float_as_uint(top) & 0x7fffffffu;
}
// 1 / x to the nearest, for normal x with a normal reciprocal: the approximation is within one unit in the last place, and Newton's step in two multiply-adds rounds
// correctly from there (Markstein 1990, who excepts a mantissa of ones; all 2^23 mantissas were compared with the division here, that one among them).
__device__ __forceinline__ float reciprocal(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return fmaf(fmaf(-x, y, 1.f), y, y);
}
// Eight codes.  The quotient is the rounded one of a division by definition: with the rounded reciprocal, a product and the remainder that it leaves give it exactly
// (Markstein 1990).  Adding 1.5 * 2^23 rounds to a whole number and leaves it, + 8, in the last bits, which are collected with products: what the
// constants' own bits come to is taken off at the end.  (16-bit weights lie on a lattice, halves of a code are frequent among them: no branch for those.)
__device__ __forceinline__ uint32_t codes_of(const float (&v)[8], float scale) {
  uint32_t word = 0;
  if (scale > 1e-30f && scale < 1e30f) {
    const float inverse = reciprocal(scale);
    float c[8];
#pragma unroll
    for (int j = 0; j < 8; j += 2)  // two numbers an instruction: product, remainder, correction, rounding
      asm("{\n\t.reg .b64 v, i, s, m, n, r;\n\t"
          "mov.b64 v, {%2, %3};\n\tmov.b64 i, {%4, %4};\n\tmov.b64 s, {%5, %5};\n\tmov.b64 m, {%6, %6};\n\t"
          "mul.rn.f32x2 n, v, i;\n\t"
          "fma.rn.f32x2 r, n, s, v;\n\t"
          "fma.rn.f32x2 n, r, i, n;\n\t"
          "add.rn.f32x2 n, n, m;\n\t"
          "mov.b64 {%0, %1}, n;\n\t}"
          : "=f"(c[j]), "=f"(c[j + 1])
          : "f"(v[j]), "f"(v[j + 1]), "f"(inverse), "f"(-scale), "f"(12582912.f + 8.f));
#pragma unroll
    for (int j = 7; j >= 0; --j) word = word * 16u + __float_as_uint(c[j]);
    return word - 0x4B400000u * 0x11111111u;
  }
  if (!(scale > 0.f && scale < INFINITY)) return 0x88888888u;  // zeros, or a group that its scale makes NaN
#pragma unroll
  for (int j = 7; j >= 0; --j) word = word * 16u + (uint32_t)(__float2int_rn(fminf(fmaxf(rintf(__fdiv_rn(v[j], scale)), -7.f), 7.f)) + 8);
  return word;
}

// Largest magnitude of a group, scale = that times 1/7 (as a 32-bit number), codes = round(w / scale) + 8.  The largest is taken over bit patterns, whose order
// is that of the magnitudes with infinities and NaN above: a group that holds one has it as its scale and is NaN throughout.
// A thread takes eight neighbours; as many lanes as a group of up to 256 needs share its largest (groups do not straddle warps).
// A warp's turn is 1024 columns of a row, all on their way before the first are worked on.
// 8192 x 8192 in bf16: 41 us, 4.2 TB/s (44 with one number an instruction in the quotients); issue slots are 66% busy, the integer ALU 41%, 27 warps an SM wait on one another
// (a maximum of three numbers an instruction changed nothing).
template <typename T> struct Raw { uint4 q; };
template <> struct Raw<float> { uint4 q, r; };
__device__ __forceinline__ void numbers(const Raw<float>& w, float (&v)[8]) {
  const uint32_t q[8] = {w.q.x, w.q.y, w.q.z, w.q.w, w.r.x, w.r.y, w.r.z, w.r.w};
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(q[j]);
}
__device__ __forceinline__ void numbers(const Raw<__nv_bfloat16>& w, float (&v)[8]) {
  const uint32_t q[4] = {w.q.x, w.q.y, w.q.z, w.q.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[2 * j] = __uint_as_float(q[j] << 16);
    v[2 * j + 1] = __uint_as_float(q[j] & 0xffff0000u);
  }
}
__device__ __forceinline__ void numbers(const Raw<__half>& w, float (&v)[8]) {
  const uint32_t q[4] = {w.q.x, w.q.y, w.q.z, w.q.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&q[j]));
    v[2 * j] = f.x;
    v[2 * j + 1] = f.y;
  }
}
template <typename T, int LANES>
__global__ void __launch_bounds__(256) w4_quantise_kernel(const T* W, int type, uint8_t* codes, float* scales, W4 w) {
  constexpr int AHEAD = 4;
  const int padded = w.groups() << w.group_log2, lane8 = (threadIdx.x & 31) * 8;
  const unsigned per_row = (unsigned)(padded + 1023) >> 10;
  const long long turns = (long long)w.n_out * per_row, stride = (long long)gridDim.x * 8;
  const bool wide = w.n_in % 8 == 0 && (reinterpret_cast<uintptr_t>(W) & 15) == 0;
  for (long long turn = blockIdx.x * 8LL + (threadIdx.x >> 5); turn < turns; turn += stride) {
    const long long n = per_row == 1 ? turn : turns < (1LL << 32) ? (long long)((unsigned)turn / per_row) : turn / per_row;
    const int k0 = (int)(turn - n * per_row) * 1024 + lane8;
    const T* from = W + n * w.n_in + k0;
    uint32_t* out = reinterpret_cast<uint32_t*>(codes + (n * padded + k0) / 2);
    float* to = scales + (long long)(k0 >> w.group_log2) * w.n_out + n;
    const bool whole = wide && k0 - lane8 + 256 * AHEAD <= w.n_in;
    Raw<T> raw[AHEAD];
    if (whole) {
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) raw[i] = *reinterpret_cast<const Raw<T>*>(from + 256 * i);
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      if (k0 - lane8 + 256 * i >= padded) break;  // (for the whole warp: the lanes of a group meet in the shuffles)
      float v[8];
      if (whole) numbers(raw[i], v);
      else load_eight(W, type, n * w.n_in + k0 + 256 * i, w.n_in - k0 - 256 * i, wide, v);
      uint32_t top = largest(v);
#pragma unroll
      for (int o = LANES >> 1; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float scale = __fmul_rn(__uint_as_float(top), 1.f / 7.f);
      if (k0 + 256 * i < padded) {
        out[32 * i] = codes_of(v, scale);
        if ((threadIdx.x & (LANES - 1)) == 0) to[(long long)((256 * i) >> w.group_log2) * w.n_out] = scale;
      }
    }
  }
}
template <typename T>
void quantise(const T* W, int type, uint8_t* codes, float* scales, const W4& w, int blocks, cudaStream_t stream) {
  if (w.group_log2 == 5) w4_quantise_kernel<T, 4><<<blocks, 256, 0, stream>>>(W, type, codes, scales, w);
  else if (w.group_log2 == 6) w4_quantise_kernel<T, 8><<<blocks, 256, 0, stream>>>(W, type, codes, scales, w);
  else if (w.group_log2 == 7) w4_quantise_kernel<T, 16><<<blocks, 256, 0, stream>>>(W, type, codes, scales, w);
  else w4_quantise_kernel<T, 32><<<blocks, 256, 0, stream>>>(W, type, codes, scales, w);
}
// Groups over 256: a warp each, which reads it twice.
__global__ void __launch_bounds__(256) w4_quantise_long_kernel(const void* W, int type, uint8_t* codes, float* scales, W4 w) {
  const int G = 1 << w.group_log2, lane = threadIdx.x & 31, groups = w.groups();
  const long long units = (long long)w.n_out * groups, stride = (long long)gridDim.x * 8;
  const bool wide = w.n_in % 8 == 0 && (reinterpret_cast<uintptr_t>(W) & 15) == 0;
  for (long long u = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); u < units; u += stride) {
    const long long n = u / groups;
    const int g = (int)(u - n * groups);
    uint32_t top = 0;
    float v[8];
    for (int j = lane * 8; j < G; j += 256) {
      load_eight(W, type, n * w.n_in + g * G + j, w.n_in - g * G - j, wide, v);
      top = max(top, largest(v));
    }
    const float scale = __fmul_rn(__uint_as_float(__reduce_max_sync(0xffffffffu, top)), 1.f / 7.f);
    if (lane == 0) scales[(long long)g * w.n_out + n] = scale;
    uint32_t* out = reinterpret_cast<uint32_t*>(codes + n * w.pitch() + (long long)g * (G / 2));
    for (int j = lane * 8; j < G; j += 256) {
      load_eight(W, type, n * w.n_in + g * G + j, w.n_in - g * G - j, wide, v);
      out[j / 8] = codes_of(v, scale);
    }
  }
}

// A word's codes - 8 as eight 8-bit numbers: a byte c of 0..15 to c - 8, where (128 + c - 8) with its highest bit turned borrows nothing from its neighbour.
__device__ __forceinline__ uint2 integers_of(uint32_t word) {
  const uint32_t lo = (((word & 0x0f0f0f0fu) | 0x80808080u) - 0x08080808u) ^ 0x80808080u;
  const uint32_t hi = ((((word >> 4) & 0x0f0f0f0fu) | 0x80808080u) - 0x08080808u) ^ 0x80808080u;
  return make_uint2(__byte_perm(lo, hi, 0x5140), __byte_perm(lo, hi, 0x7362));
}
// code - 8 in 8 bits: PER columns a thread, 16 where rows are whole multiples of that (8192 x 8192: 17 us, 5.9 TB/s; 24 with 8 columns).
template <int PER>
__global__ void __launch_bounds__(256) w4_integers_kernel(W4 w, int8_t* integers) {
  const unsigned per_row = (unsigned)(w.n_in + PER - 1) / PER;
  const long long units = (long long)w.n_out * per_row, pitch = w.pitch();
  for (long long u = blockIdx.x * 256LL + threadIdx.x; u < units; u += gridDim.x * 256LL) {
    const long long n = units < (1LL << 32) ? (long long)((unsigned)u / per_row) : u / per_row;
    const int k = (int)(u - n * per_row) * PER;
    int8_t* to = integers + n * w.n_in + k;
    if (PER == 16) {
      const uint2 words = *reinterpret_cast<const uint2*>(w.codes + n * pitch + k / 2), a = integers_of(words.x), b = integers_of(words.y);
      *reinterpret_cast<uint4*>(to) = make_uint4(a.x, a.y, b.x, b.y);
    } else {
      const uint2 q = integers_of(*reinterpret_cast<const uint32_t*>(w.codes + n * pitch + k / 2));
      const int left = min(8, w.n_in - k);
      for (int j = 0; j < left; ++j) to[j] = (int8_t)((j < 4 ? q.x : q.y) >> (8 * (j & 3)));
    }
  }
}
// The weight in 32 bits: eight columns a thread (8192 x 8192: 59 us, 5.1 TB/s).
__global__ void __launch_bounds__(256) w4_dense_kernel(W4 w, float* dense) {
  const unsigned per_row = (unsigned)((w.n_in + 7) >> 3);
  const long long units = (long long)w.n_out * per_row, pitch = w.pitch();
  const bool wide = w.n_in % 4 == 0 && (reinterpret_cast<uintptr_t>(dense) & 15) == 0;
  for (long long u = blockIdx.x * 256LL + threadIdx.x; u < units; u += gridDim.x * 256LL) {
    const long long n = units < (1LL << 32) ? (long long)((unsigned)u / per_row) : u / per_row;
    const int k = (int)(u - n * per_row) * 8, left = min(8, w.n_in - k);
    const uint2 q = integers_of(*reinterpret_cast<const uint32_t*>(w.codes + n * pitch + k / 2));
    const float scale = w.scales[(long long)(k >> w.group_log2) * w.n_out + n];
    float* to = dense + n * w.n_in + k;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = scale * (float)(int8_t)((j < 4 ? q.x : q.y) >> (8 * (j & 3)));
    if (wide && left == 8) {
      reinterpret_cast<float4*>(to)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4*>(to)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < left) to[j] = v[j];
    }
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

// out[j] = sum over rows of A[:, j].  Many rows: a warp for every eighth, eight on their way at a time; the warps' sums in order (4096 rows of 8192 bf16: 14 us).
__global__ void __launch_bounds__(256) column_sums_many_kernel(const void* A, int type, void* out, int out_type, int M, int n) {
  __shared__ float part[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, j = blockIdx.x * 32 + lane;
  float s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) s[i] = 0.f;
  if (j < n) {
    int m = warp;
    for (; m + 56 < M; m += 64) {
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] += load_any(A, type, (long long)(m + 8 * i) * n + j);
    }
    for (; m < M; m += 8) s[0] += load_any(A, type, (long long)m * n + j);
  }
  part[warp][lane] = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
  __syncthreads();
  if (warp == 0 && j < n) {
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) v += part[i][lane];
    store_any(out, out_type, j, v);
  }
}
// Few rows, in order.
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
  BF_REQUIRE(n_out > 0 && n_in > 0 && n_in <= 1 << 30 && n_out <= 1 << 30, BF_E_INVALID, "%s: bad sizes %d x %d", who, n_out, n_in);
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
  const long long b = (units + per_block - 1) / per_block, cap = 148LL * 256;
  return (int)(b < cap ? b : cap);
}

}  // namespace
}  // namespace bf

extern "C" int bf_w4_quantise(const void* W, int type, uint8_t* codes, float* scales, int n_out, int n_in, int group, bf_stream_t stream) {
  bf::W4 w;
  const int rc = bf::make_w4(w, "bf_w4_quantise", codes, scales, n_out, n_in, group);
  if (rc != BF_OK) return rc;
  BF_REQUIRE(W && bf::type_ok(type), BF_E_INVALID, "bf_w4_quantise: null weight or unknown type %d", type);
  const long long turns = (long long)n_out * ((((long long)w.groups() << w.group_log2) + 1023) / 1024);
  if (w.group_log2 > 8) bf::w4_quantise_long_kernel<<<bf::blocks_for((long long)n_out * w.groups(), 8), 256, 0, bf::as_stream(stream)>>>(W, type, codes, scales, w);
  else if (type == BF_TYPE_F32) bf::quantise(static_cast<const float*>(W), type, codes, scales, w, bf::blocks_for(turns, 8), bf::as_stream(stream));
  else if (type == BF_TYPE_BF16) bf::quantise(static_cast<const __nv_bfloat16*>(W), type, codes, scales, w, bf::blocks_for(turns, 8), bf::as_stream(stream));
  else bf::quantise(static_cast<const __half*>(W), type, codes, scales, w, bf::blocks_for(turns, 8), bf::as_stream(stream));
  BF_CHECK_LAUNCH("w4_quantise_kernel");
  return BF_OK;
}

extern "C" int bf_w4_integers(const uint8_t* codes, int8_t* out, int n_out, int n_in, int group, bf_stream_t stream) {
  bf::W4 w;
  const int rc = bf::make_w4(w, "bf_w4_integers", codes, codes, n_out, n_in, group);
  if (rc != BF_OK) return rc;
  BF_REQUIRE(out, BF_E_INVALID, "bf_w4_integers: null output");
  // (a grid of 32 blocks an SM: 8192 x 8192 24 us, 44 with a block for each 2048 columns)
  if (n_in % 16 == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0)
    bf::w4_integers_kernel<16><<<std::min(bf::blocks_for((long long)n_in / 16 * n_out, 256), 148 * 32), 256, 0, bf::as_stream(stream)>>>(w, out);
  else bf::w4_integers_kernel<8><<<std::min(bf::blocks_for(((long long)n_in + 7) / 8 * n_out, 256), 148 * 32), 256, 0, bf::as_stream(stream)>>>(w, out);
  BF_CHECK_LAUNCH("w4_integers_kernel");
  return BF_OK;
}

extern "C" int bf_w4_dense(const uint8_t* codes, const float* scales, float* out, int n_out, int n_in, int group, bf_stream_t stream) {
  bf::W4 w;
  const int rc = bf::make_w4(w, "bf_w4_dense", codes, scales, n_out, n_in, group);
  if (rc != BF_OK) return rc;
  BF_REQUIRE(out, BF_E_INVALID, "bf_w4_dense: null output");
  bf::w4_dense_kernel<<<bf::blocks_for(((long long)n_in + 7) / 8 * n_out, 256), 256, 0, bf::as_stream(stream)>>>(w, out);
  BF_CHECK_LAUNCH("w4_dense_kernel");
  return BF_OK;
}

// A product's arguments, checked.
namespace bf {
namespace {
int linear_args(W4LinearArgs& p, const char* who, const void* x, int type, const uint8_t* codes, const float* scales, const void* bias, int bias_type, void* y, int M, int n_in,
                int n_out, int group) {
  const int rc = make_w4(p.w, who, codes, scales, n_out, n_in, group);
  if (rc != BF_OK) return rc;
  BF_REQUIRE(x && y && M > 0 && type_ok(type) && (!bias || type_ok(bias_type)), BF_E_INVALID, "%s: null tensor, no rows or unknown type", who);
  p.a = x;
  p.bias = bias;
  p.y = y;
  p.type = type;
  p.bias_type = bias_type;
  p.M = M;
  return BF_OK;
}
int interval_args(W4LinearArgs& p, const char* who, const float* in_a, const float* in_b, int in_mode, int relu_in, const uint8_t* codes, const float* scales, const float* bias,
                  float* out_l, float* out_u, int M, int n_in, int n_out, int group) {
  const int rc = make_w4(p.w, who, codes, scales, n_out, n_in, group);
  if (rc != BF_OK) return rc;
  BF_REQUIRE(in_a && in_b && out_l && out_u && M > 0, BF_E_INVALID, "%s: null tensor or no rows", who);
  BF_REQUIRE(in_mode == BF_IN_LOWER_UPPER || (in_mode == BF_IN_MID_RAD && !relu_in), BF_E_INVALID, "%s: bad input mode %d", who, in_mode);
  p.a = in_a;
  p.b = in_b;
  p.bias = bias;
  p.y = out_l;
  p.y2 = out_u;
  p.mode = in_mode;
  p.relu_in = relu_in;
  p.M = M;
  return BF_OK;
}
int rows_args(W4RowsArgs& p, const char* who, const void* a, const float* b, int type, const uint8_t* codes, const float* scales, void* z, float* z2, int M, int n_in, int n_out,
              int group) {
  const int rc = make_w4(p.w, who, codes, scales, n_out, n_in, group);
  if (rc != BF_OK) return rc;
  BF_REQUIRE(a && z && (z2 == nullptr) == (b == nullptr) && M > 0 && type_ok(type), BF_E_INVALID, "%s: null tensor, no rows or unknown type", who);
  p.a = a;
  p.b = b;
  p.z = z;
  p.z2 = z2;
  p.type = type;
  p.M = M;
  return BF_OK;
}
int check_workspace(const char* who, const void* workspace) {
  BF_REQUIRE(workspace && (reinterpret_cast<uintptr_t>(workspace) & 127u) == 0, BF_E_INVALID, "%s: a workspace on a 128-byte boundary is wanted", who);
  return BF_OK;
}
}  // namespace
}  // namespace bf

extern "C" long long bf_w4_workspace_bytes(int M, int n_sum, int type) {
  return M > 0 && n_sum > 0 && n_sum <= 1 << 30 && bf::type_ok(type) ? bf::w4_many_bytes(M, n_sum, type) : 0;
}

extern "C" int bf_w4_many_pays(int M, int n_in, int n_out, int group, int type, int backward, int pair) {
  if (M <= 0 || n_in <= 0 || n_out <= 0 || n_in > 1 << 30 || n_out > 1 << 30 || !bf::type_ok(type)) return 0;
  return bf::w4_many_pays(M, n_in, n_out, group, type, backward == 0, pair != 0) ? 1 : 0;
}

extern "C" int bf_w4_linear(const void* x, int type, const uint8_t* codes, const float* scales, const void* bias, int bias_type, void* y, int M, int n_in,
                            int n_out, int group, bf_stream_t stream) {
  bf::W4LinearArgs p = {};
  const int rc = bf::linear_args(p, "bf_w4_linear", x, type, codes, scales, bias, bias_type, y, M, n_in, n_out, group);
  return rc != BF_OK ? rc : bf::launch_w4_linear(p, bf::as_stream(stream));
}
extern "C" int bf_w4_linear_many(const void* x, int type, const uint8_t* codes, const float* scales, const void* bias, int bias_type, void* y, int M, int n_in,
                                 int n_out, int group, void* workspace, bf_stream_t stream) {
  bf::W4LinearArgs p = {};
  int rc = bf::linear_args(p, "bf_w4_linear_many", x, type, codes, scales, bias, bias_type, y, M, n_in, n_out, group);
  if (rc == BF_OK) rc = bf::check_workspace("bf_w4_linear_many", workspace);
  return rc != BF_OK ? rc : bf::launch_w4_linear_many(p, workspace, bf::as_stream(stream));
}

extern "C" int bf_w4_interval(const float* in_a, const float* in_b, int in_mode, int relu_in, const uint8_t* codes, const float* scales, const float* bias,
                              float* out_l, float* out_u, int M, int n_in, int n_out, int group, bf_stream_t stream) {
  bf::W4LinearArgs p = {};
  const int rc = bf::interval_args(p, "bf_w4_interval", in_a, in_b, in_mode, relu_in, codes, scales, bias, out_l, out_u, M, n_in, n_out, group);
  return rc != BF_OK ? rc : bf::launch_w4_linear(p, bf::as_stream(stream));
}
extern "C" int bf_w4_interval_many(const float* in_a, const float* in_b, int in_mode, int relu_in, const uint8_t* codes, const float* scales, const float* bias,
                                   float* out_l, float* out_u, int M, int n_in, int n_out, int group, void* workspace, bf_stream_t stream) {
  bf::W4LinearArgs p = {};
  int rc = bf::interval_args(p, "bf_w4_interval_many", in_a, in_b, in_mode, relu_in, codes, scales, bias, out_l, out_u, M, n_in, n_out, group);
  if (rc == BF_OK) rc = bf::check_workspace("bf_w4_interval_many", workspace);
  return rc != BF_OK ? rc : bf::launch_w4_linear_many(p, workspace, bf::as_stream(stream));
}

extern "C" int bf_w4_rows(const void* a, int type, const uint8_t* codes, const float* scales, void* z, int M, int n_in, int n_out, int group,
                          bf_stream_t stream) {
  bf::W4RowsArgs p = {};
  const int rc = bf::rows_args(p, "bf_w4_rows", a, nullptr, type, codes, scales, z, nullptr, M, n_in, n_out, group);
  return rc != BF_OK ? rc : bf::launch_w4_rows(p, bf::as_stream(stream));
}
extern "C" int bf_w4_rows_many(const void* a, int type, const uint8_t* codes, const float* scales, void* z, int M, int n_in, int n_out, int group, void* workspace,
                               bf_stream_t stream) {
  bf::W4RowsArgs p = {};
  int rc = bf::rows_args(p, "bf_w4_rows_many", a, nullptr, type, codes, scales, z, nullptr, M, n_in, n_out, group);
  if (rc == BF_OK) rc = bf::check_workspace("bf_w4_rows_many", workspace);
  return rc != BF_OK ? rc : bf::launch_w4_rows_many(p, workspace, bf::as_stream(stream));
}

extern "C" int bf_w4_interval_grad(const float* grad_l, const float* grad_u, const uint8_t* codes, const float* scales, float* z_l, float* z_u, int M,
                                   int n_in, int n_out, int group, bf_stream_t stream) {
  bf::W4RowsArgs p = {};
  BF_REQUIRE(grad_u && z_u, BF_E_INVALID, "bf_w4_interval_grad: null tensor");
  const int rc = bf::rows_args(p, "bf_w4_interval_grad", grad_l, grad_u, BF_TYPE_F32, codes, scales, z_l, z_u, M, n_in, n_out, group);
  return rc != BF_OK ? rc : bf::launch_w4_rows(p, bf::as_stream(stream));
}
extern "C" int bf_w4_interval_grad_many(const float* grad_l, const float* grad_u, const uint8_t* codes, const float* scales, float* z_l, float* z_u, int M,
                                        int n_in, int n_out, int group, void* workspace, bf_stream_t stream) {
  bf::W4RowsArgs p = {};
  BF_REQUIRE(grad_u && z_u, BF_E_INVALID, "bf_w4_interval_grad_many: null tensor");
  int rc = bf::rows_args(p, "bf_w4_interval_grad_many", grad_l, grad_u, BF_TYPE_F32, codes, scales, z_l, z_u, M, n_in, n_out, group);
  if (rc == BF_OK) rc = bf::check_workspace("bf_w4_interval_grad_many", workspace);
  return rc != BF_OK ? rc : bf::launch_w4_rows_many(p, workspace, bf::as_stream(stream));
}

extern "C" int bf_w4_linear_grad(const void* grad, int type, const uint8_t* codes, const float* scales, void* grad_x, void* grad_bias, int bias_type, int M,
                                 int n_in, int n_out, int group, bf_stream_t stream) {
  if (grad_x) {
    const int rc = bf_w4_rows(grad, type, codes, scales, grad_x, M, n_in, n_out, group, stream);
    if (rc != BF_OK) return rc;
  }
  return grad_bias ? bf_column_sums(grad, type, grad_bias, bias_type, M, n_out, stream) : BF_OK;
}

extern "C" int bf_rows_dot(const float* A, const float* bias, float* d, int accumulate, int M, int n, bf_stream_t stream) {
  BF_REQUIRE(A && bias && d && M > 0 && n > 0, BF_E_INVALID, "bf_rows_dot: null tensor or bad sizes");
  bf::rows_dot_kernel<<<bf::ceil_div(M, 8), 256, 0, bf::as_stream(stream)>>>(A, bias, d, accumulate, M, n);
  BF_CHECK_LAUNCH("rows_dot_kernel");
  return BF_OK;
}

extern "C" int bf_column_sums(const void* A, int type, void* out, int out_type, int M, int n, bf_stream_t stream) {
  BF_REQUIRE(A && out && M > 0 && n > 0 && bf::type_ok(type) && bf::type_ok(out_type), BF_E_INVALID, "bf_column_sums: null tensor, bad sizes or type");
  if (M > 64) bf::column_sums_many_kernel<<<bf::ceil_div(n, 32), 256, 0, bf::as_stream(stream)>>>(A, type, out, out_type, M, n);
  else bf::column_sums_kernel<<<bf::ceil_div(n, 256), 256, 0, bf::as_stream(stream)>>>(A, type, out, out_type, M, n);
  BF_CHECK_LAUNCH("column_sums_kernel");
  return BF_OK;
}
