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

constexpr int STARTS = 256;

struct AdamEntry {
  void* p;
  const void* g;
  long long n;      // elements
  long long first;  // where the tensor's moments begin in the flat buffers (a multiple of BLOCK)
  float lr, decay;  // decay = 1 - lr * weight_decay
  unsigned chunk0;  // number of the tensor's first chunk
  int wide;         // p and g lie on boundaries of four elements
};
template <int CAP>
struct AdamTable {
  AdamEntry e[CAP];
  int count;
  unsigned chunks;
  int shift;             // chunk >> shift < STARTS
  uint16_t start[STARTS];  // the tensor that the first chunk of that many belongs to: a search is a step or two from there
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

// A lane's eight elements of a block, four at 4 * lane and four at 128 + 4 * lane, as they lie in memory.
template <typename T> struct Eight { using Four = uint2; Four q[2]; };
template <> struct Eight<float> { using Four = uint4; Four q[2]; };

// `whole`: all of them are there, on a boundary of four.
template <typename T>
__device__ __forceinline__ Eight<T> load8(const T* p, int lane, int left, bool whole) {
  Eight<T> r;
  if (whole) {
    r.q[0] = *reinterpret_cast<const typename Eight<T>::Four*>(p + lane * 4);
    r.q[1] = *reinterpret_cast<const typename Eight<T>::Four*>(p + 128 + lane * 4);
  } else {
    for (int h = 0; h < 2; ++h) {
      T t[4];
      for (int i = 0; i < 4; ++i) t[i] = h * 128 + lane * 4 + i < left ? p[h * 128 + lane * 4 + i] : T(0.f);
      memcpy(&r.q[h], t, sizeof t);
    }
  }
  return r;
}
template <typename T>
__device__ __forceinline__ void store8(T* p, int lane, int left, bool whole, const Eight<T>& r) {
  if (whole) {
    *reinterpret_cast<typename Eight<T>::Four*>(p + lane * 4) = r.q[0];
    *reinterpret_cast<typename Eight<T>::Four*>(p + 128 + lane * 4) = r.q[1];
  } else {
    for (int h = 0; h < 2; ++h) {
      T t[4];
      memcpy(t, &r.q[h], sizeof t);
      for (int i = 0; i < 4; ++i)
        if (h * 128 + lane * 4 + i < left) p[h * 128 + lane * 4 + i] = t[i];
    }
  }
}
__device__ __forceinline__ void numbers(const Eight<float>& r, float (&x)[8]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    x[4 * h] = __uint_as_float(r.q[h].x);
    x[4 * h + 1] = __uint_as_float(r.q[h].y);
    x[4 * h + 2] = __uint_as_float(r.q[h].z);
    x[4 * h + 3] = __uint_as_float(r.q[h].w);
  }
}
__device__ __forceinline__ void numbers(const Eight<__nv_bfloat16>& r, float (&x)[8]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    x[4 * h] = __uint_as_float(r.q[h].x * 65536u);
    x[4 * h + 1] = __uint_as_float(r.q[h].x & 0xffff0000u);
    x[4 * h + 2] = __uint_as_float(r.q[h].y * 65536u);
    x[4 * h + 3] = __uint_as_float(r.q[h].y & 0xffff0000u);
  }
}
__device__ __forceinline__ void numbers(const Eight<__half>& r, float (&x)[8]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&r.q[h].x)), b = __half22float2(*reinterpret_cast<const __half2*>(&r.q[h].y));
    x[4 * h] = a.x;
    x[4 * h + 1] = a.y;
    x[4 * h + 2] = b.x;
    x[4 * h + 3] = b.y;
  }
}
__device__ __forceinline__ uint32_t two(__nv_bfloat16*, float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t two(__half*, float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <typename T>
__device__ __forceinline__ Eight<T> rounded(const float (&x)[8]) {
  Eight<T> r;
#pragma unroll
  for (int h = 0; h < 2; ++h) r.q[h] = make_uint2(two(static_cast<T*>(nullptr), x[4 * h], x[4 * h + 1]), two(static_cast<T*>(nullptr), x[4 * h + 2], x[4 * h + 3]));
  return r;
}
template <>
__device__ __forceinline__ Eight<float> rounded<float>(const float (&x)[8]) {
  Eight<float> r;
#pragma unroll
  for (int h = 0; h < 2; ++h)
    r.q[h] = make_uint4(__float_as_uint(x[4 * h]), __float_as_uint(x[4 * h + 1]), __float_as_uint(x[4 * h + 2]), __float_as_uint(x[4 * h + 3]));
  return r;
}

// ---- 8-bit moments -----------------------------------------------------------------
// Integer work is what the 8-bit step is short of (64 lanes a clock, half of what FP32 has): codes are kept where a byte permutation finds them, shifts to the left
// are multiplications (which run beside it), and signs and zeros are dealt with for four codes at a time.
constexpr int M_FIELDS = 15, V_FIELDS = 31;  // powers of two below the block's exponent

// The 32 random bits of the four elements at `place` (a multiple of four, so that the first mixing is the same for them but for the last two bits).  Shifts and products with odd
// constants, arbitrary ones: what is asked of them is that roundings up and down balance over elements and steps, to which a test of the moments' means holds them.
__device__ __forceinline__ void rounding_noise(uint32_t place, uint32_t key, uint32_t (&noise)[4]) {
  const uint32_t first = place ^ key, mixed = first ^ (first >> 16);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t x = (mixed ^ (uint32_t)i) * 0x9BC84D59u;
    x = (x ^ (x >> 15)) * 0x7641A5C5u;
    noise[i] = x ^ (x >> 16);
  }
}
// The four numbers of `word`; a code is added to the bit pattern of the power of two below its range.
template <int FIELDS, bool SIGNED>
__device__ __forceinline__ void decode4(uint32_t word, int exponent, float* x) {
  const uint32_t base = (uint32_t)(exponent - FIELDS) << 23, codes = SIGNED ? word & 0x7f7f7f7fu : word;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t c = __byte_perm(codes, 0, 0x4044 | (i << 8));  // the code in bits 16-23
    const uint32_t bits = (c * 16 + base) * min(c, 1u);
    x[i] = __uint_as_float(SIGNED ? bits | ((word << (24 - 8 * i)) & 0x80000000u) : bits);
  }
}
// `top`: bit pattern of the block's largest magnitude.
template <int FIELDS>
__device__ __forceinline__ int shared_exponent(uint32_t top) {
  if (top >= 0x7f800000u) return 255;
  return min(254, max(FIELDS + 1, (int)((top + 0xfffffu) >> 23)));
}
// Four codes: magnitude and 20 bits of noise, counted from the power of two below the range; the code is what is above bit 20.  Nothing is above the largest
// code, as the exponent is chosen; `below`: something may be below the smallest.
template <int FIELDS, bool SIGNED>
__device__ __forceinline__ uint32_t encode4(const float* x, const uint32_t (&noise20)[4], int exponent, bool below) {
  const uint32_t base = (uint32_t)(exponent - FIELDS) << 23;
  uint32_t d[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t bits = __float_as_uint(x[i]);
    d[i] = (SIGNED ? bits & 0x7fffffffu : bits) + noise20[i] - base;
  }
  if (below) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int least = SIGNED || x[i] == 0.f ? 0 : 1 << 20;  // a second moment that is not zero keeps a code that is not
      d[i] = (uint32_t)max((int)d[i], least);
    }
  }
  uint32_t word = __byte_perm(__byte_perm(d[0] * 16, d[1] * 16, 0x0073), __byte_perm(d[2] * 16, d[3] * 16, 0x0073), 0x5410);
  if (SIGNED) {
    const uint32_t signs = __byte_perm(__byte_perm(__float_as_uint(x[0]), __float_as_uint(x[1]), 0x0073), __byte_perm(__float_as_uint(x[2]), __float_as_uint(x[3]), 0x0073), 0x5410);
    word |= (word + 0x7f7f7f7fu) & signs & 0x80808080u;  // zero has no sign
  }
  return word;
}
// Where the largest exponent is cut (254), magnitudes above the largest code are cut to it.
template <int FIELDS>
__device__ __forceinline__ void cut(float (&x)[8]) {
  const float most = __uint_as_float(((uint32_t)(254 - FIELDS) << 23) + ((8u * FIELDS + 7u) << 20));
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = copysignf(fminf(fabsf(x[i]), most), x[i]);
}

// With 8-bit moments root and quotient are the approximations, good to 2^-22: the moments themselves are rounded to an eighth (64 million bf16 parameters 176 us, 207 with the
// rounded ones).  With 32-bit moments they are rounded to the nearest (fp32 with bf16 gradients 246.9 -> 247.7 us, bf16 throughout 210.6 -> 214.1).  Numbers below the normal range
// count as zero in the approximations: a root below 2^-63, times the correction 1 / sqrt(1 - b2^t), which is below 2^-22 of an eps from LEAST_EPS times that correction on.
constexpr float LEAST_EPS = 4.6e-13f;
__device__ __forceinline__ float quotient(float m, float v, float root, float eps) {
  float s, q;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(v));
  asm("div.approx.ftz.f32 %0, %1, %2;" : "=f"(q) : "f"(m), "f"(fmaf(s, root, eps)));
  return q;
}

// A warp's work of a turn: where it lies, and for 8-bit moments all that it reads, fetched a turn ahead.
template <typename P, typename G>
struct Turn {
  P* to;
  long long slot;
  int entry, left;  // left <= 0: nothing to do
  bool whole;
  Eight<P> p;
  Eight<G> g;
  uint32_t m[2], v[2];
  int me, ve;
};

// Bounds and measurements (B200, 64 million parameters in 40 tensors).  32-bit moments: memory; fp32 parameters with bf16 gradients 248 us, 6.7 TB/s, the rate of a plain
// copy; all in fp32 265 us.  8-bit moments of bf16 parameters: 176 us, 3.6 TB/s, the integer ALU is 68% and the issue slots 74% busy; of fp32
// parameters 194 to 208 us.  (A thread block's chunks lie a grid apart: with them side by side it took 272 us against 172.)
template <typename P, typename G, bool EIGHT, int CAP>
__global__ void __launch_bounds__(256, EIGHT ? 3 : 4) adamw_kernel(const __grid_constant__ AdamTable<CAP> tab, const AdamCommon c) {
  __shared__ float sh_rate, sh_root, sh_scale;
  __shared__ uint32_t sh_key;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto locate = [&](unsigned chunk, Turn<P, G>& w) {
    int near = tab.start[chunk >> tab.shift];
    while (near + 1 < tab.count && chunk >= tab.e[near + 1].chunk0) ++near;  // the last tensor that begins at or before this chunk
    const AdamEntry& e = tab.e[near];
    const long long at = (long long)(chunk - e.chunk0) * CHUNK + warp * BLOCK;
    w.entry = near;
    w.to = static_cast<P*>(e.p) + at;
    w.slot = e.first + at;
    w.left = (int)min((long long)BLOCK, e.n - at);
    w.whole = w.left == BLOCK && e.wide != 0;
    return static_cast<const G*>(e.g) + at;
  };
  auto fetch = [&](Turn<P, G>& w, const G* from) {
    w.p = load8(static_cast<const P*>(w.to), lane, w.left, w.whole);
    w.g = load8(from, lane, w.left, w.whole);
    if (EIGHT) {
      const unsigned at = (unsigned)lane;
      w.me = c.me[w.slot / BLOCK];
      w.ve = c.ve[w.slot / BLOCK];
      const uint32_t *m = reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(c.m) + w.slot), *v = reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(c.v) + w.slot);
      w.m[0] = m[at];
      w.m[1] = m[at + 32];
      w.v[0] = v[at];
      w.v[1] = v[at + 32];
    }
  };
  unsigned chunk = blockIdx.x;
  Turn<P, G> now;
  now.left = 0;
  if (chunk < tab.chunks) {
    const G* from = locate(chunk, now);
    if (EIGHT && now.left > 0) fetch(now, from);
  }
  if (threadIdx.x == 0) {
    const double q1 = c.state[0] * c.beta1, q2 = c.state[1] * c.beta2;
    sh_rate = (float)(1.0 / (1.0 - q1));
    sh_root = (float)(1.0 / sqrt(1.0 - q2));
    sh_key = (uint32_t)(c.state[2] + 1.0) * 0x9E3779B1u;
    sh_scale = c.grad_scale ? *c.grad_scale : 1.f;
  }
  __syncthreads();
  const float rate = sh_rate, root = sh_root, scale = sh_scale;
  const uint32_t key = sh_key;
  while (chunk < tab.chunks) {
    Turn<P, G> then;
    then.left = 0;
    chunk += gridDim.x;
    if (chunk < tab.chunks) {
      const G* from = locate(chunk, then);
      if (EIGHT && then.left > 0) fetch(then, from);
    }
    if (now.left > 0) {
      const AdamEntry& e = tab.e[now.entry];
      float p[8], g[8], m[8], v[8];
      if (EIGHT) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          decode4<M_FIELDS, true>(now.m[h], now.me, m + 4 * h);
          decode4<V_FIELDS, false>(now.v[h], now.ve, v + 4 * h);
        }
        if (max(now.me, now.ve) == 255) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (now.me == 255) m[i] = __int_as_float(0x7fffffff);
            if (now.ve == 255) v[i] = __int_as_float(0x7fffffff);
          }
        }
      } else {
        fetch(now, static_cast<const G*>(e.g) + (now.to - static_cast<P*>(e.p)));
        numbers(load8(static_cast<const float*>(c.m) + now.slot, lane, BLOCK, true), m);
        numbers(load8(static_cast<const float*>(c.v) + now.slot, lane, BLOCK, true), v);
      }
      numbers(now.p, p);
      numbers(now.g, g);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float gi = __fmul_rn(g[i], scale);
        m[i] = __fadd_rn(__fmul_rn(c.b1, m[i]), __fmul_rn(c.c1, gi));
        v[i] = __fadd_rn(__fmul_rn(c.b2, v[i]), __fmul_rn(__fmul_rn(c.c2, gi), gi));
      }
      const float step = -e.lr * rate, decay = e.decay;
      if (EIGHT && c.eps > LEAST_EPS * root) {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = fmaf(step, quotient(m[i], v[i], root, c.eps), p[i] * decay);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = fmaf(step, __fdiv_rn(m[i], fmaf(__fsqrt_rn(v[i]), root, c.eps)), p[i] * decay);
      }
      store8(now.to, lane, now.left, now.whole, rounded<P>(p));
      if (EIGHT) {
        uint32_t mt = 0, vt = 0, ml = 0xffffffffu, vl = 0xffffffffu;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t mi = __float_as_uint(m[i]) & 0x7fffffffu, vi = __float_as_uint(v[i]) & 0x7fffffffu;
          mt = max(mt, mi);
          vt = max(vt, vi);
          ml = min(ml, mi);
          vl = min(vl, vi);
        }
        mt = __reduce_max_sync(0xffffffffu, mt);
        vt = __reduce_max_sync(0xffffffffu, vt);
        const int me = shared_exponent<M_FIELDS>(mt), ve = shared_exponent<V_FIELDS>(vt);
        if (max(me, ve) >= 254) {
          cut<M_FIELDS>(m);
          cut<V_FIELDS>(v);
        }
        const bool below = ml < (uint32_t)(me - M_FIELDS) << 23 || vl < ((uint32_t)(ve - V_FIELDS) << 23) + (1u << 20);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t noise[4], low[4], high[4];
          rounding_noise((uint32_t)now.slot + h * 128 + lane * 4, key, noise);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            low[i] = noise[i] & 0xfffffu;
            high[i] = noise[i] >> 12;
          }
          reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(c.m) + now.slot)[h * 32 + lane] = encode4<M_FIELDS, true>(m + 4 * h, low, me, below);
          reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(c.v) + now.slot)[h * 32 + lane] = encode4<V_FIELDS, false>(v + 4 * h, high, ve, below);
        }
        if (lane == 0) {
          c.me[now.slot / BLOCK] = (uint8_t)me;
          c.ve[now.slot / BLOCK] = (uint8_t)ve;
        }
      } else {
        store8(static_cast<float*>(c.m) + now.slot, lane, BLOCK, true, rounded<float>(m));
        store8(static_cast<float*>(c.v) + now.slot, lane, BLOCK, true, rounded<float>(v));
      }
    }
    now = then;
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

// The values that 8-bit moments stand for, in bfloat16 (which holds them exactly: 8 exponent bits, 3 of 7 mantissa bits).  64 million: 60 us, 6.4 TB/s.
__global__ void __launch_bounds__(256) adamw_moments_kernel(const uint8_t* m8, const uint8_t* v8, const uint8_t* me, const uint8_t* ve, __nv_bfloat16* m,
                                                            __nv_bfloat16* v, long long n) {
  for (long long i = (blockIdx.x * 256LL + threadIdx.x) * 8; i < n; i += gridDim.x * 2048LL) {
    float a[8], b[8];
    const int em = me[i / BLOCK], ev = ve[i / BLOCK];
    const uint2 mw = *reinterpret_cast<const uint2*>(m8 + i), vw = *reinterpret_cast<const uint2*>(v8 + i);
    decode4<M_FIELDS, true>(mw.x, em, a);
    decode4<M_FIELDS, true>(mw.y, em, a + 4);
    decode4<V_FIELDS, false>(vw.x, ev, b);
    decode4<V_FIELDS, false>(vw.y, ev, b + 4);
    if (max(em, ev) == 255) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (em == 255) a[j] = __int_as_float(0x7fffffff);
        if (ev == 255) b[j] = __int_as_float(0x7fffffff);
      }
    }
    __nv_bfloat16* const none = nullptr;
    *reinterpret_cast<uint4*>(m + i) = make_uint4(two(none, a[0], a[1]), two(none, a[2], a[3]), two(none, a[4], a[5]), two(none, a[6], a[7]));
    *reinterpret_cast<uint4*>(v + i) = make_uint4(two(none, b[0], b[1]), two(none, b[2], b[3]), two(none, b[4], b[5]), two(none, b[6], b[7]));
  }
}

template <typename P, typename G, bool EIGHT, int CAP>
int launch(const bf_adamw_tensor* t, int count, const AdamCommon& c, cudaStream_t stream) {
  AdamTable<CAP> tab;
  unsigned long long chunks = 0;
  for (int i = 0; i < count; ++i) {
    tab.e[i] = {t[i].p, t[i].g, t[i].n, t[i].first, t[i].lr, (float)(1.0 - (double)t[i].lr * (double)t[i].weight_decay), (unsigned)chunks,
                ((reinterpret_cast<uintptr_t>(t[i].p) & (4 * sizeof(P) - 1)) | (reinterpret_cast<uintptr_t>(t[i].g) & (4 * sizeof(G) - 1))) == 0};
    chunks += (unsigned long long)((t[i].n + CHUNK - 1) / CHUNK);
  }
  BF_REQUIRE(chunks < (1ULL << 31), BF_E_UNSUPPORTED, "bf_adamw_step: more than 2^42 elements in one launch");
  tab.count = count;
  tab.chunks = (unsigned)chunks;
  tab.shift = 0;
  while ((chunks >> tab.shift) >= STARTS) ++tab.shift;
  for (int i = 0, k = 0; i < STARTS; ++i) {
    while (k + 1 < count && tab.e[k + 1].chunk0 <= ((unsigned long long)i << tab.shift)) ++k;
    tab.start[i] = (uint16_t)k;
  }
  // Many more blocks than the chip holds: where each takes as many turns as any other, those of an SM come to their loads together and the memory waits with the
  // arithmetic (64 million parameters: 4 and 3 blocks an SM in one wave 279 and 212 us, 64 and 24 of them 246 and 174).  But four turns at least for the 8-bit
  // ones, whose first fetch nothing hides (3.3 million: 17.8 us with one turn each, 14.3 with four).
  const unsigned most = 148 * (EIGHT ? 24 : 64), least = 148 * (EIGHT ? 3 : 4), count_of = (unsigned)chunks;
  const int grid = (int)(count_of == 0 ? 1u : count_of <= least ? count_of : EIGHT ? (count_of / 4 < least ? least : count_of / 4 < most ? count_of / 4 : most)
                                                                                   : (count_of < most ? count_of : most));
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
  BF_REQUIRE(((reinterpret_cast<uintptr_t>(m_out) | reinterpret_cast<uintptr_t>(v_out)) & 15u) == 0 && ((reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(v)) & 7u) == 0,
             BF_E_INVALID, "bf_adamw_moments: moments must lie on 8-byte boundaries, the results on 16-byte ones");
  const long long blocks = (n + 2047) / 2048;
  bf::adamw_moments_kernel<<<(int)(blocks < 148 * 64 ? blocks : 148 * 64), 256, 0, bf::as_stream(stream)>>>(
      m, v, m_exponent, v_exponent, static_cast<__nv_bfloat16*>(m_out), static_cast<__nv_bfloat16*>(v_out), n);
  BF_CHECK_LAUNCH("adamw_moments_kernel");
  return BF_OK;
}
