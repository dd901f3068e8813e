// AdamW over many tensors in one launch, moments in 32 bits or in 8.
//
//   m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2;  p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// All arithmetic is in 32 bits; p is rounded once when it is stored.  Every product and sum of a moment is rounded by itself, so that the
// moments are defined bit for bit.
//
// Moments in 8 bits: 256 neighbours share an exponent e, that of their largest magnitude (one more where its mantissa is above 1.875 and
// could be rounded up).  A code holds exponent and mantissa as one number, counted from a power of two below e:
//   m: sign, 7 bits = 4 exponent + 3 mantissa bits above 2^(e - 15);  v: 8 bits = 5 + 3 above 2^(e - 31);  zero is the code 0
// (e is the biased exponent of the 32-bit format, kept as a byte; 255 marks a block that held an infinity or a NaN, and all of it is NaN).
// A step moves v by a thousandth, the codes are an eighth apart: rounded to the nearest they would never move.  The 20 bits that a code drops
// are rounded up in proportion to what they hold instead, by a hash of the element's place and the step, so that the mean of many steps
// is that of the 32-bit moments.  Magnitudes of m below the codes' range become zero; those of v become the smallest code,
// never zero, for a second moment of zero beside a first moment that is not would make a step of m / eps.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include "common.cuh"

namespace bf {
namespace {

constexpr int BLOCK = 256;         // elements that share an exponent: one warp's work at a time
constexpr int CHUNK = 8 * BLOCK;   // elements of a thread block's turn

struct AdamEntry {
  void* p;
  const void* g;
  long long n;      // elements
  long long first;  // where the tensor's moments begin in the flat buffers (a multiple of BLOCK)
  float lr, decay;  // decay = 1 - lr * weight_decay
  unsigned chunk0;  // number of the tensor's first chunk
};
template <int CAP>
struct AdamTable {
  AdamEntry e[CAP];
  int count;
  unsigned chunks;
};
struct AdamCommon {
  void *m, *v;
  uint8_t *me, *ve;
  float b1, c1, b2, c2, eps;
  double beta1, beta2;
  double* state;  // b1^t, b2^t, t, blocks that are done
  const float* grad_scale;
  int last;
};

template <typename T> struct Four;
template <> struct Four<float> { using type = float4; };
template <> struct Four<__nv_bfloat16> { using type = uint2; };
template <> struct Four<__half> { using type = uint2; };
__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ void put(float& d, float v) { d = v; }
__device__ __forceinline__ void put(__nv_bfloat16& d, float v) { d = __float2bfloat16(v); }
__device__ __forceinline__ void put(__half& d, float v) { d = __float2half(v); }

// A lane's eight elements of a block: four at 4 * lane, four at 128 + 4 * lane.
template <typename T>
__device__ __forceinline__ void load8(const T* p, int lane, int left, bool wide, float (&x)[8]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int at = h * 128 + lane * 4;
    if (wide && at + 4 <= left) {
      typename Four<T>::type q = *reinterpret_cast<const typename Four<T>::type*>(p + at);
      const T* t = reinterpret_cast<const T*>(&q);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[4 * h + i] = to_f(t[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[4 * h + i] = at + i < left ? to_f(p[at + i]) : 0.f;
    }
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, int lane, int left, bool wide, const float (&x)[8]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int at = h * 128 + lane * 4;
    T t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) put(t[i], x[4 * h + i]);
    if (wide && at + 4 <= left) {
      typename Four<T>::type q;
      memcpy(&q, t, sizeof q);
      *reinterpret_cast<typename Four<T>::type*>(p + at) = q;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (at + i < left) p[at + i] = t[i];
    }
  }
}

// ---- 8-bit moments -----------------------------------------------------------------
constexpr int M_FIELDS = 15, V_FIELDS = 31;  // powers of two below the block's exponent

__device__ __forceinline__ uint32_t rounding_noise(uint32_t place, uint32_t step) {
  uint32_t x = place ^ (step * 0x9E3779B1u);
  x = (x ^ (x >> 16)) * 0x9BC84D59u;
  x = (x ^ (x >> 15)) * 0x7641A5C5u;
  return x ^ (x >> 16);
}
template <int FIELDS>
__device__ __forceinline__ float decode(uint32_t code, int e) {
  if (e == 255) return __int_as_float(0x7fffffff);
  return code == 0 ? 0.f : __uint_as_float((code + ((uint32_t)(e - FIELDS) << 3)) << 20);
}
// `top`: bit pattern of the block's largest magnitude.
template <int FIELDS>
__device__ __forceinline__ int shared_exponent(uint32_t top) {
  if (top >= 0x7f800000u) return 255;
  return min(254, max(FIELDS + 1, (int)((top + 0xfffffu) >> 23)));
}
template <int FIELDS>
__device__ __forceinline__ uint32_t encode(float magnitude, uint32_t noise20, int e) {
  const int rel = (int)((__float_as_uint(magnitude) + noise20) >> 20) - ((e - FIELDS) << 3);
  return (uint32_t)min(8 * FIELDS + 7, max(0, rel));
}

template <typename P, typename G, bool EIGHT, int CAP>
__global__ void __launch_bounds__(256) adamw_kernel(const __grid_constant__ AdamTable<CAP> tab, const AdamCommon c) {
  __shared__ float sh_rate, sh_root, sh_scale;
  __shared__ uint32_t sh_step;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    const double q1 = c.state[0] * c.beta1, q2 = c.state[1] * c.beta2;
    sh_rate = (float)(1.0 / (1.0 - q1));
    sh_root = (float)(1.0 / sqrt(1.0 - q2));
    sh_step = (uint32_t)(c.state[2] + 1.0);
    sh_scale = c.grad_scale ? *c.grad_scale : 1.f;
  }
  __syncthreads();
  const float rate = sh_rate, root = sh_root, scale = sh_scale;
  const uint32_t step = sh_step;
  int t = 0;
  for (unsigned chunk = blockIdx.x; chunk < tab.chunks; chunk += gridDim.x) {
    if (t + 1 < tab.count && chunk >= tab.e[t + 1].chunk0) {  // the last tensor that begins at or before this chunk
      int lo = t + 1, hi = tab.count;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (chunk >= tab.e[mid].chunk0) lo = mid;
        else hi = mid;
      }
      t = lo;
    }
    const AdamEntry& e = tab.e[t];
    const long long at = (long long)(chunk - e.chunk0) * CHUNK + warp * BLOCK;
    if (at >= e.n) continue;
    const int left = (int)min((long long)BLOCK, e.n - at);
    P* p = static_cast<P*>(e.p) + at;
    const G* g = static_cast<const G*>(e.g) + at;
    const bool wide_p = (reinterpret_cast<uintptr_t>(e.p) & (4 * sizeof(P) - 1)) == 0, wide_g = (reinterpret_cast<uintptr_t>(e.g) & (4 * sizeof(G) - 1)) == 0;
    const long long slot = e.first + at;
    float pv[8], gv[8], m[8], v[8];
    load8(p, lane, left, wide_p, pv);
    load8(g, lane, left, wide_g, gv);
    if (EIGHT) {
      const int me = c.me[slot / BLOCK], ve = c.ve[slot / BLOCK];
      const uint8_t *m8 = static_cast<const uint8_t*>(c.m) + slot, *v8 = static_cast<const uint8_t*>(c.v) + slot;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t mw = *reinterpret_cast<const uint32_t*>(m8 + h * 128 + lane * 4), vw = *reinterpret_cast<const uint32_t*>(v8 + h * 128 + lane * 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t mc = (mw >> (8 * i)) & 255u, vc = (vw >> (8 * i)) & 255u;
          const float size = decode<M_FIELDS>(mc & 127u, me);
          m[4 * h + i] = (mc & 128u) ? -size : size;
          v[4 * h + i] = decode<V_FIELDS>(vc, ve);
        }
      }
    } else {
      load8(static_cast<const float*>(c.m) + slot, lane, BLOCK, true, m);
      load8(static_cast<const float*>(c.v) + slot, lane, BLOCK, true, v);
    }
    const float rate_lr = -e.lr * rate, decay = e.decay;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float gi = __fmul_rn(gv[i], scale);
      m[i] = __fadd_rn(__fmul_rn(c.b1, m[i]), __fmul_rn(c.c1, gi));
      v[i] = __fadd_rn(__fmul_rn(c.b2, v[i]), __fmul_rn(__fmul_rn(c.c2, gi), gi));
      pv[i] = fmaf(rate_lr, m[i] / fmaf(sqrtf(v[i]), root, c.eps), pv[i] * decay);
    }
    store8(p, lane, left, wide_p, pv);
    if (EIGHT) {
      uint32_t mt = 0, vt = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        mt = max(mt, __float_as_uint(m[i]) & 0x7fffffffu);
        vt = max(vt, __float_as_uint(v[i]) & 0x7fffffffu);
      }
      mt = __reduce_max_sync(0xffffffffu, mt);
      vt = __reduce_max_sync(0xffffffffu, vt);
      const int me = shared_exponent<M_FIELDS>(mt), ve = shared_exponent<V_FIELDS>(vt);
      uint8_t *m8 = static_cast<uint8_t*>(c.m) + slot, *v8 = static_cast<uint8_t*>(c.v) + slot;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t mw = 0, vw = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float mi = m[4 * h + i], vi = v[4 * h + i];
          const uint32_t noise = rounding_noise((uint32_t)(slot + h * 128 + lane * 4 + i), step);
          const uint32_t mc = encode<M_FIELDS>(fabsf(mi), noise & 0xfffffu, me);
          uint32_t vc = encode<V_FIELDS>(vi, noise >> 12, ve);
          if (vi > 0.f && vc == 0) vc = 1;
          mw |= (mc | (mc != 0 && mi < 0.f ? 128u : 0u)) << (8 * i);
          vw |= vc << (8 * i);
        }
        *reinterpret_cast<uint32_t*>(m8 + h * 128 + lane * 4) = mw;
        *reinterpret_cast<uint32_t*>(v8 + h * 128 + lane * 4) = vw;
      }
      if (lane == 0) {
        c.me[slot / BLOCK] = (uint8_t)me;
        c.ve[slot / BLOCK] = (uint8_t)ve;
      }
    } else {
      store8(static_cast<float*>(c.m) + slot, lane, BLOCK, true, m);
      store8(static_cast<float*>(c.v) + slot, lane, BLOCK, true, v);
    }
  }
  // The step's last launch counts it: every block has read the count when it arrives here, the last to arrive moves it on.
  if (c.last && threadIdx.x == 0) {
    unsigned long long* done = reinterpret_cast<unsigned long long*>(c.state + 3);
    __threadfence();
    if (atomicAdd(done, 1ULL) == gridDim.x - 1) {
      c.state[0] *= c.beta1;
      c.state[1] *= c.beta2;
      c.state[2] += 1.0;
      *done = 0;
    }
  }
}

// The values that 8-bit moments stand for, in bfloat16 (which holds them exactly: 8 exponent bits, 3 of 7 mantissa bits).
__global__ void __launch_bounds__(256) adamw_moments_kernel(const uint8_t* m8, const uint8_t* v8, const uint8_t* me, const uint8_t* ve, __nv_bfloat16* m,
                                                            __nv_bfloat16* v, long long n) {
  for (long long i = (blockIdx.x * 256LL + threadIdx.x) * 4; i < n; i += gridDim.x * 1024LL) {
    const uint32_t mw = *reinterpret_cast<const uint32_t*>(m8 + i), vw = *reinterpret_cast<const uint32_t*>(v8 + i);
    const int em = me[i / BLOCK], ev = ve[i / BLOCK];
    float a[4], b[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t mc = (mw >> (8 * j)) & 255u;
      const float size = decode<M_FIELDS>(mc & 127u, em);
      a[j] = (mc & 128u) ? -size : size;
      b[j] = decode<V_FIELDS>((vw >> (8 * j)) & 255u, ev);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      m[i + j] = __float2bfloat16(a[j]);
      v[i + j] = __float2bfloat16(b[j]);
    }
  }
}

template <typename P, typename G, bool EIGHT, int CAP>
int launch(const bf_adamw_tensor* t, int count, const AdamCommon& c, cudaStream_t stream) {
  AdamTable<CAP> tab;
  unsigned long long chunks = 0;
  for (int i = 0; i < count; ++i) {
    tab.e[i] = {t[i].p, t[i].g, t[i].n, t[i].first, t[i].lr, (float)(1.0 - (double)t[i].lr * (double)t[i].weight_decay), (unsigned)chunks};
    chunks += (unsigned long long)((t[i].n + CHUNK - 1) / CHUNK);
  }
  BF_REQUIRE(chunks < (1ULL << 31), BF_E_UNSUPPORTED, "bf_adamw_step: more than 2^42 elements in one launch");
  tab.count = count;
  tab.chunks = (unsigned)chunks;
  const int cap = 148 * 8, grid = chunks == 0 ? 1 : chunks < (unsigned)cap ? (int)chunks : cap;
  adamw_kernel<P, G, EIGHT, CAP><<<grid, 256, 0, stream>>>(tab, c);
  BF_CHECK_LAUNCH("adamw_kernel");
  return BF_OK;
}

template <typename P, typename G, bool EIGHT>
int launch_all(const bf_adamw_tensor* t, int count, AdamCommon c, cudaStream_t stream) {
  constexpr int MOST = 512;  // entries of 48 bytes in the 32 KB that a launch can carry
  const int last = c.last;
  int first = 0;
  do {
    const int here = count - first < MOST ? count - first : MOST;
    c.last = last && first + here == count;
    const int rc = here <= 16 ? launch<P, G, EIGHT, 16>(t + first, here, c, stream) : here <= 64 ? launch<P, G, EIGHT, 64>(t + first, here, c, stream)
                                                                                       : launch<P, G, EIGHT, MOST>(t + first, here, c, stream);
    if (rc != BF_OK) return rc;
    first += here;
  } while (first < count);
  return BF_OK;
}

template <bool EIGHT>
int by_type(const bf_adamw_tensor* t, int count, int pt, int gt, const AdamCommon& c, cudaStream_t s) {
  if (pt == BF_TYPE_F32 && gt == BF_TYPE_F32) return launch_all<float, float, EIGHT>(t, count, c, s);
  if (pt == BF_TYPE_F32 && gt == BF_TYPE_BF16) return launch_all<float, __nv_bfloat16, EIGHT>(t, count, c, s);
  if (pt == BF_TYPE_F32 && gt == BF_TYPE_F16) return launch_all<float, __half, EIGHT>(t, count, c, s);
  if (pt == BF_TYPE_BF16 && gt == BF_TYPE_BF16) return launch_all<__nv_bfloat16, __nv_bfloat16, EIGHT>(t, count, c, s);
  if (pt == BF_TYPE_F16 && gt == BF_TYPE_F16) return launch_all<__half, __half, EIGHT>(t, count, c, s);
  set_error("bf_adamw_step: parameters of type %d with gradients of type %d", pt, gt);
  return BF_E_UNSUPPORTED;
}

}  // namespace
}  // namespace bf

extern "C" int bf_adamw_step(const bf_adamw_tensor* tensors, int count, int p_type, int g_type, int state_bits, void* m, void* v, uint8_t* m_exponent,
                             uint8_t* v_exponent, double beta1, double beta2, float eps, const float* grad_scale, double* state, int last,
                             bf_stream_t stream) {
  BF_REQUIRE(count >= 0 && (tensors || count == 0) && m && v && state, BF_E_INVALID, "bf_adamw_step: null tensor or bad count");
  BF_REQUIRE(state_bits == 32 || (state_bits == 8 && m_exponent && v_exponent), BF_E_INVALID, "bf_adamw_step: state_bits is 32, or 8 with exponents");
  BF_REQUIRE(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0 && eps >= 0.f, BF_E_INVALID, "bf_adamw_step: bad options");
  BF_REQUIRE(((reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(v)) & 15u) == 0, BF_E_INVALID, "bf_adamw_step: moments must lie on 16-byte boundaries");
  for (int i = 0; i < count; ++i)
    BF_REQUIRE(tensors[i].n >= 0 && tensors[i].first >= 0 && tensors[i].first % bf::BLOCK == 0 && ((tensors[i].p && tensors[i].g) || tensors[i].n == 0), BF_E_INVALID,
               "bf_adamw_step: tensor %d is null, of negative size, or its moments do not begin at a whole block", i);
  const bf::AdamCommon c = {m, v, m_exponent, v_exponent, (float)beta1, (float)(1.0 - beta1), (float)beta2, (float)(1.0 - beta2), eps, beta1, beta2, state,
                            grad_scale, last};
  return state_bits == 8 ? bf::by_type<true>(tensors, count, p_type, g_type, c, bf::as_stream(stream))
                         : bf::by_type<false>(tensors, count, p_type, g_type, c, bf::as_stream(stream));
}

extern "C" int bf_adamw_moments(const uint8_t* m, const uint8_t* v, const uint8_t* m_exponent, const uint8_t* v_exponent, void* m_out, void* v_out,
                                long long n, bf_stream_t stream) {
  BF_REQUIRE(m && v && m_exponent && v_exponent && m_out && v_out && n > 0 && n % bf::BLOCK == 0, BF_E_INVALID, "bf_adamw_moments: null tensor or no whole blocks");
  const long long blocks = (n + 1023) / 1024;
  bf::adamw_moments_kernel<<<(int)(blocks < 148 * 16 ? blocks : 148 * 16), 256, 0, bf::as_stream(stream)>>>(
      m, v, m_exponent, v_exponent, static_cast<__nv_bfloat16*>(m_out), static_cast<__nv_bfloat16*>(v_out), n);
  BF_CHECK_LAUNCH("adamw_moments_kernel");
  return BF_OK;
}
