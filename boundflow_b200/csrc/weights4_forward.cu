// y = x W^T + bias for few rows x and 4-bit weights, and the bounds of it over boxes (W c -/+ |W| r); weights4_mma.cuh says how.
#include <math.h>

#include "weights4_mma.cuh"

namespace bf {
namespace {

constexpr int SHARED_OF_TWO = 112 * 1024;  // shared memory of a block where two share an SM
constexpr int X_MOST = 120 * 1024;   // and what a block alone on an SM has left of its 227 KB beside the ring and 32 KB of sums

__device__ __forceinline__ void centre_radius(float a, float b, int mode, int relu_in, float& c, float& r) {
  if (mode == BF_IN_LOWER_UPPER) {
    // (a comparison with a NaN is false: it stays)
    if (relu_in) { a = a < 0.f ? 0.f : a; b = b < 0.f ? 0.f : b; }
    c = 0.5f * (a + b);
    r = 0.5f * (b - a);
  } else {
    c = a;
    r = b;
  }
}

// Eight neighbours of a row, as they lie in memory.
template <int P> struct Eight { uint4 q; };  // (16-bit numbers)
template <> struct Eight<3> { uint4 q, r; };
template <int P>
__device__ __forceinline__ Eight<P> load8(const void* base, long long at, int left, bool wide) {
  Eight<P> e;
  if (P == 3) {
    const float* p = static_cast<const float*>(base) + at;
    if (wide && left >= 8) return *reinterpret_cast<const Eight<P>*>(p);
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < left ? p[j] : 0.f;
    memcpy(&e, v, sizeof e);
  } else {
    const uint16_t* p = static_cast<const uint16_t*>(base) + at;
    if (wide && left >= 8) return *reinterpret_cast<const Eight<P>*>(p);
    uint16_t v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < left ? p[j] : 0;
    memcpy(&e, v, sizeof e);
  }
  return e;
}

// Digits (P = DIGITS): up to four 16-bit rows as whole numbers of four 8-bit digits, counted in 2^(e - 156) with e the biased exponent of the largest of the row's
// columns that share a scale (128 of them at most).  A bfloat16 number is held exactly down to 2^-22 of that largest, a half down to 2^-19.  The codes
// turn into 8-bit numbers, 16 (code - 8), with three operations a word instead of eleven, the integer instruction takes twice as many columns, and its sums are
// exact; a factor for each column brings them back.  What the digits leave of smaller numbers counts where the weights beside the larger ones are zero: where a block meets
// such a number, `add_rest` multiplies what is left as bfloat16 parts, and infinities and NaN, of which the digits hold nothing: each meets its own weight.
constexpr int DIGITS = 4;

// The exponent that digits are counted from (below 2^-97 the unit stays), by the largest magnitude; the least exponent whose numbers the digits hold whole.
__device__ __forceinline__ int digits_exponent(float top) { return max((int)(__float_as_uint(top) >> 23), 30); }
__device__ __forceinline__ int whole_from(int exponent, int type) {
  return type == BF_TYPE_BF16 ? exponent - 22 : exponent > 132 ? exponent - 19 : 0;  // (halves are multiples of 2^-24)
}
__device__ __forceinline__ void eight_numbers(const uint4& q, int type, float (&v)[8]) {
  const uint32_t q4[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = type == BF_TYPE_BF16 ? make_float2(__uint_as_float(q4[j] << 16), __uint_as_float(q4[j] & 0xffff0000u)) : __half22float2(*reinterpret_cast<const __half2*>(&q4[j]));
    v[2 * j] = f.x;
    v[2 * j + 1] = f.y;
  }
}
// Largest magnitude, NaN where one is among them.
__device__ __forceinline__ float largest_of(const float (&v)[8]) {
  float top = 0.f;
#pragma unroll
  for (int j = 0; j < 8; j += 2) asm("max.NaN.abs.f32 %0, %0, %1, %2;" : "+f"(top) : "f"(v[j]), "f"(v[j + 1]));
  return top;
}
__device__ __forceinline__ void finite_only(float (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = fabsf(v[j]) < INFINITY ? v[j] : 0.f;
}
__device__ __forceinline__ float largest_of(float a, float b) {
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(b));
  return a;
}

// Parts of the rows' columns [from, to) * 128 in shared memory: [step of 32 columns][product][part, tile][column][4 lanes][8 columns of the step], the 8 in the
// order 0 4 1 5 2 6 3 7 that `weights_of` gives the codes of a word in (digits: 0 2 4 6 1 3 5 7).  Eight columns of a row are a thread's turn, AHEAD of them are on their way at a time.
template <int P, bool PACKED, int NT, bool DUAL>
struct Stager {
  static constexpr int SETS = DUAL ? 2 : 1, AHEAD = P == 1 || P == DIGITS ? 4 : DUAL ? 1 : 2;
  Eight<P> raw[AHEAD][SETS];
  int rows[AHEAD], pieces[AHEAD];
  int item, items, piece, row, per_row;
  bool rest = false;  // digits: some number was not held whole

  __device__ __forceinline__ void begin(int from, int to, int M) {
    per_row = (to - from) * (CHUNK / 8);
    items = per_row * M;
    item = piece = threadIdx.x;
    row = 0;
  }
  __device__ __forceinline__ void fetch(const W4LinearArgs& p, int from, int m0, bool wide) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      rows[i] = -1;
      if (item < items) {
        while (piece >= per_row) { piece -= per_row; ++row; }
        const int k = from * CHUNK + piece * 8;
        const long long at = (long long)(m0 + row) * p.w.n_in + k;
        raw[i][0] = load8<P>(p.a, at, p.w.n_in - k, wide);
        if (DUAL) raw[i][SETS - 1] = load8<P>(p.b, at, p.w.n_in - k, wide);
        rows[i] = row;
        pieces[i] = piece;
      }
      item += blockDim.x;
      piece += blockDim.x;
    }
  }
  // Digits of eight columns: their word holds the four, byte by byte (balanced, -128 to 127); a transposition of bytes gives each digit's word of four columns.
  __device__ __forceinline__ void put_digits(const Eight<P>& e, int type, int lanes, int row, int piece, int step_bytes, uint32_t xs, uint32_t factors) {
    float v[8];
    eight_numbers(e.q, type, v);
    float top = largest_of(v);
    const uint32_t half = 0xffffu << (threadIdx.x & 16);  // the 16 lanes of a chunk's columns; `lanes` of them share a scale
    for (int o = lanes >> 1; o > 0; o >>= 1) top = largest_of(top, __shfl_xor_sync(half, top, o));
    if (!(top < INFINITY)) {  // (the lanes that share a scale come here together)
      rest = true;
      finite_only(v);
      top = largest_of(v);
      const uint32_t group = ((1u << lanes) - 1u) << (threadIdx.x & 31 & -lanes);
      for (int o = lanes >> 1; o > 0; o >>= 1) top = largest_of(top, __shfl_xor_sync(group, top, o));
    }
    const int exponent = digits_exponent(top);
    uint32_t least = 0xffffffffu;  // twice the smallest magnitude's bits, less one: zero counts as the largest
#pragma unroll
    for (int j = 0; j < 8; ++j) least = min(least, 2u * __float_as_uint(v[j]) - 1u);
    rest |= least < 0xfffffffeu && (int)(least >> 24) < whole_from(exponent, type);
    uint32_t z[8];
    const float scale = __uint_as_float((uint32_t)(283 - exponent) << 23);
#pragma unroll
    for (int j = 0; j < 8; ++j) z[j] = ((uint32_t)__float2int_rn(v[j] * scale) + 0x00808080u) ^ 0x00808080u;
    const uint32_t to = xs + (piece >> 2) * step_bytes + (row * 4 * 4 + (piece & 3)) * 8;
    uint32_t o[2][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t a = __byte_perm(z[h], z[h + 2], 0x5140), b = __byte_perm(z[h], z[h + 2], 0x7362);
      const uint32_t c = __byte_perm(z[h + 4], z[h + 6], 0x5140), d = __byte_perm(z[h + 4], z[h + 6], 0x7362);
      o[h][0] = __byte_perm(a, c, 0x5410);
      o[h][1] = __byte_perm(a, c, 0x7632);
      o[h][2] = __byte_perm(b, d, 0x5410);
      o[h][3] = __byte_perm(b, d, 0x7632);
    }
#pragma unroll
    for (int d = 0; d < 4; ++d) asm volatile("st.shared.v2.b32 [%0], {%1,%2};" ::"r"(to + d * 32), "r"(o[0][d]), "r"(o[1][d]) : "memory");
    if ((piece & (lanes - 1)) == 0) {  // 2^(e - 156) / 16 and the digits' places
      float f[4];
#pragma unroll
      for (int d = 0; d < 4; ++d) f[d] = ldexpf(1.f, exponent - 160 + 8 * d);
      asm volatile("st.shared.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(factors + (piece / lanes * NT * 8 + row * 4) * 4), "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]) : "memory");
    }
  }
  __device__ __forceinline__ void put(const W4LinearArgs& p, int cv, int step_bytes, int set_bytes, uint32_t xs, uint32_t factors) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      if (rows[i] < 0) break;
      if constexpr (P == DIGITS) put_digits(raw[i][0], p.type, 4 << min(p.w.group_log2 - 5, 2), rows[i], pieces[i], step_bytes, xs, factors);
      else put_parts(i, p, cv, step_bytes, set_bytes, xs);
    }
  }
  __device__ __forceinline__ void put_parts(int i, const W4LinearArgs& p, int cv, int step_bytes, int set_bytes, uint32_t xs) {
    {
      uint32_t o[SETS][P][4];
      if constexpr (P == 1) {
        const uint4 v = raw[i][0].q;
        o[0][0][0] = __byte_perm(v.x, v.z, 0x5410);
        o[0][0][1] = __byte_perm(v.x, v.z, 0x7632);
        o[0][0][2] = __byte_perm(v.y, v.w, 0x5410);
        o[0][0][3] = __byte_perm(v.y, v.w, 0x7632);
      } else {
        float v[SETS][8];
        if (P == 2) {
          const uint32_t q4[4] = {raw[i][0].q.x, raw[i][0].q.y, raw[i][0].q.z, raw[i][0].q.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&q4[j]));
            v[0][2 * j] = f.x;
            v[0][2 * j + 1] = f.y;
          }
        } else {
#pragma unroll
          for (int s = 0; s < SETS; ++s) memcpy(v[s], &raw[i][s], 32);
          if (DUAL) {
#pragma unroll
            for (int j = 0; j < 8; ++j) centre_radius(v[0][j], v[SETS - 1][j], p.mode, p.relu_in, v[0][j], v[SETS - 1][j]);
          }
        }
#pragma unroll
        for (int s = 0; s < SETS; ++s)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t q[P];
            two_numbers_checked<P>(v[s][j], v[s][j + 4], q);
#pragma unroll
            for (int n = 0; n < P; ++n) o[s][n][j] = q[n];
          }
      }
      const uint32_t dst = xs + (pieces[i] >> 2) * step_bytes + (pieces[i] & 3) * 16;
#pragma unroll
      for (int n = 0; n < P; ++n) {
        const int j = PACKED ? rows[i] * P + n : n * NT * cv + rows[i];  // column, counted through the tiles
        const uint32_t to = dst + j * 64;
#pragma unroll
        for (int s = 0; s < SETS; ++s) put16(to + s * set_bytes, o[s][n][0], o[s][n][1], o[s][n][2], o[s][n][3]);
      }
    }
  }
};

// What the digits leave of the rows in the warp's chunks: at most 8 bits of a bfloat16 number, 11 of a half, so that one or two bfloat16 parts hold it.  It goes in the column of the
// row's first digit, on top of the sums of that column, which the warp has laid down at `sums`.  Everything is read again where it lies: this is for the few calls whose numbers lie
// far apart (in the loop over the chunks the mere branch took one row through 16384 x 16384 from 30 to 34 us).
template <int NT, int F>
__device__ __forceinline__ void add_rest(const W4LinearArgs& p, int first, int end, int by, int n0, bool wide, uint32_t sums) {
  const W4& w = p.w;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const long long pitch = w.pitch();
  for (int c = first; c < end; c += by) {
#pragma unroll 1
    for (int j = 0; j < NT; ++j) {
      const int m = 2 * j + (g >> 2);
      const bool mine = (g & 3) == 0 && m < p.M;
      Eight<1> raw[4];
#pragma unroll
      for (int step = 0; step < 4; ++step) {
        const int k = c * CHUNK + step * 32 + t * 8;
        raw[step].q = make_uint4(0, 0, 0, 0);
        if (mine) raw[step] = load8<1>(p.a, (long long)m * w.n_in + k, w.n_in - k, wide);
      }
      float top[4];
#pragma unroll
      for (int step = 0; step < 4; ++step) {
        float v[8];
        eight_numbers(raw[step].q, p.type, v);
        finite_only(v);
        top[step] = largest_of(v);
        top[step] = largest_of(top[step], __shfl_xor_sync(0xffffffffu, top[step], 1));
        top[step] = largest_of(top[step], __shfl_xor_sync(0xffffffffu, top[step], 2));
        if (step % F > 0) top[step] = largest_of(top[step], top[step - 1]);  // (complete at a group's last step)
      }
      float acc[2][4];
#pragma unroll
      for (int step = 0; step < 4; ++step) {
        const int exponent = digits_exponent(top[step / F * F + F - 1]), k = c * CHUNK + step * 32 + t * 8;
        const float unit = __uint_as_float((uint32_t)(exponent - 29) << 23), per_unit = __uint_as_float((uint32_t)(283 - exponent) << 23);
        float left[8];
        eight_numbers(raw[step].q, p.type, left);
        bool some = false;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (fabsf(left[i]) < INFINITY) left[i] -= rintf(left[i] * per_unit) * unit;
          some |= left[i] != 0.f;
        }
        if (step % F == 0) {
#pragma unroll
          for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[r][i] = 0.f;
        }
        if (__any_sync(0xffffffffu, some)) {
          uint32_t parts[2][4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t q[2];
            two_numbers_checked<2>(left[i], left[i + 4], q);
            parts[0][i] = q[0];
            parts[1][i] = q[1];
          }
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            uint32_t word[2];
#pragma unroll
            for (int i = 0; i < 2; ++i)
              word[i] = k / 2 < pitch ? *reinterpret_cast<const uint32_t*>(w.codes + (long long)min(n0 + r * 16 + g + 8 * i, w.n_out - 1) * pitch + k / 2) : 0u;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t a[4] = {weights_of(word[0] >> (8 * h)), weights_of(word[1] >> (8 * h)), weights_of(word[0] >> (8 * h + 4)), weights_of(word[1] >> (8 * h + 4))};
              mma(acc[r], a[0], a[1], a[2], a[3], parts[0][2 * h], parts[0][2 * h + 1]);
              mma(acc[r], a[0], a[1], a[2], a[3], parts[1][2 * h], parts[1][2 * h + 1]);
            }
          }
        }
        if (step % F == F - 1) {
          const float* scales = w.scales + (long long)min((c * CHUNK + step * 32) >> w.group_log2, w.groups() - 1) * w.n_out;
#pragma unroll
          for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int row = r * 16 + g + (i >> 1) * 8;
              const uint32_t at = sums + ((j * 8 + 2 * t + (i & 1)) * 36 + row) * 4;
              if (acc[r][i] != 0.f)
                asm volatile("st.shared.f32 [%0], %1;" ::"r"(at), "f"(fmaf(scales[min(n0 + row, w.n_out - 1)], acc[r][i], __uint_as_float(lds32(at)))) : "memory");
            }
        }
      }
    }
  }
  __syncwarp();
}

// P parts of a row, side by side in the columns of NT tiles (PACKED) or an instruction each for NT tiles of 8 rows; DUAL: W c and |W| r; F: steps of 32 columns
// that share a scale (1, 2, or 4 and more).
//
// Bounds and measurements (B200, back to back on inputs larger than the L2 cache's share).  One bf16 row through 16384 x 16384: 31.7 us, 4.5 TB/s of codes, scales and
// rows (69% of a plain copy; 123 to 182 us where digits leave a rest in every group); issue slots are at 55%, DRAM at 52%, and a launch of nothing but clusters costs 3 to 4 us of it.  Boxes of 4 through 8192 x 8192: 25 us,
// 1.5 TB/s; two products of three parts keep the tensor cores 35% busy, the rest is waits of 16 warps an SM (128 registers each).  16 bf16 rows
// through 8192 x 4096: 12.3 us.  Rings of 2 and 4 stages, three blocks an SM, and columns split twice or four times as finely were slower or equal.
template <int P, bool PACKED, int NT, bool DUAL, int F>
__global__ void __launch_bounds__(THREADS, (PACKED ? 1 : P) * NT * (DUAL ? 2 : 1) > 6 ? 1 : 2) w4_forward_kernel(const W4LinearArgs p, const Split sp) {
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr int Q = (PACKED ? 1 : P) * NT, SETS = DUAL ? 2 : 1, COUNT = PACKED ? P : 1;
  const W4 w = p.w;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int kw = warp & (sp.kw - 1), rw = warp >> sp.kw_log2;
  const int rank = blockIdx.x & (sp.cluster - 1);
  const int n0 = ((blockIdx.x >> sp.cluster_log2) * sp.rw + rw) * TILE_N;
  const int m0 = blockIdx.y * sp.tile_m, M = min(sp.tile_m, p.M - m0);
  const int cv = NT > 1 ? 8 : M * COUNT;  // columns of a tile that are held
  const int chunks = (w.n_in + CHUNK - 1) / CHUNK, share = (chunks + sp.cluster - 1) >> sp.cluster_log2;
  const int first = min(rank * share, chunks), end = min(first + share, chunks);
  const int warps = sp.kw * sp.rw;
  const uint32_t inbox = smem_of(smem), ring = inbox + sp.inbox + warp * (STAGES * STAGE_BYTES), xs = inbox + sp.inbox + warps * (STAGES * STAGE_BYTES);
  const int set_bytes = Q * cv * (P == DIGITS ? 32 : 64), step_bytes = SETS * set_bytes;
  const uint32_t factors = xs + min(sp.per_phase, share) * 4 * step_bytes;  // (digits only)
  const bool wide = w.n_in % (P == 3 ? 4 : 8) == 0 && (((uintptr_t)p.a | (uintptr_t)p.b) & 15) == 0;
  Stager<P, PACKED, NT, DUAL> stager;
  int to = min(first + sp.per_phase, end);
  stager.begin(first, to, M);
  stager.fetch(p, first, m0, wide);  // before the codes: behind a ring of them in every warp these would wait for the memory's first microsecond
  if (sp.cluster > 1) cluster_arrive();  // (before the sums go out all blocks of the cluster have to be there)

  const int groups = w.groups();
  const int pitch = (int)w.pitch();
  const int rows = max(0, min(TILE_N, w.n_out - n0));
  const uint8_t* codes = w.codes + (lane >> 2 < rows ? (long long)(n0 + (lane >> 2)) * pitch + (lane & 3) * 16 : 0);
  float tot[SETS][2][NT][4];
#pragma unroll
  for (int s = 0; s < SETS; ++s)
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) tot[s][r][j][i] = 0.f;

  int next = first + kw;  // the chunk that is copied next
  auto load_next = [&](uint32_t at) {
    if (next < end) {
      load_codes(at, codes + next * (CHUNK / 2), codes, 8LL * pitch, rows, pitch - next * (CHUNK / 2), lane);
      load_scales(at, w, groups, n0, next, lane);
    }
    copies_begin();
    next += sp.kw;
  };
  load_next(ring);  // one stage; the others when the rows are in place (issuing them takes as long as the memory takes to answer)
  int slot = 0;
  for (int from = first; from < end; from = to, to = min(from + sp.per_phase, end)) {
    if (from != first) {
      __syncthreads();
      stager.begin(from, to, M);
      stager.fetch(p, from, m0, wide);
    }
    while (true) {
      stager.put(p, cv, step_bytes, set_bytes, xs, factors);
      if (stager.item - threadIdx.x >= stager.items) break;
      stager.fetch(p, from, m0, wide);
    }
    if (from == first) {
#pragma unroll
      for (int s = 1; s < STAGES - 1; ++s) load_next(ring + s * STAGE_BYTES);
    }
    __syncthreads();
    for (int c = from + kw; c < to; c += sp.kw) {
      copies_wait<STAGES - 2>();
      __syncwarp();
      load_next(ring + (slot == 0 ? STAGES - 1 : slot - 1) * STAGE_BYTES);  // into the slot that was read last
      const uint32_t st = ring + slot * STAGE_BYTES + g * ROW_BYTES + t * 4;
      slot = slot == STAGES - 1 ? 0 : slot + 1;
      const uint32_t sc = st - g * (ROW_BYTES - 4) - t * 4 + TILE_N * ROW_BYTES;
      const int held = min(g, cv - 1);  // columns that are not held repeat the last
      if constexpr (P == DIGITS) {
        const uint32_t xb = xs + (c - from) * 4 * step_bytes + (held * 4 + t) * 8;
        int acc[2][NT][4];
#pragma unroll
        for (int step = 0; step < 4; ++step) {
          if (step % F == 0) {  // (1.5 * 2^23 as a bit pattern: a whole number added to it is that number added to 1.5 * 2^23)
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
              for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[r][j][i] = 0x4B400000;
          }
          uint32_t b[NT][2];
#pragma unroll
          for (int j = 0; j < NT; ++j)
            asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(b[j][0]), "=r"(b[j][1]) : "r"(xb + step * step_bytes + j * cv * 32) : "memory");
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const uint32_t w0 = lds32(st + r * 16 * ROW_BYTES + step * 16), w1 = lds32(st + (r * 16 + 8) * ROW_BYTES + step * 16);
            const uint32_t a0 = digits_of(w0 * 16u), a1 = digits_of(w1 * 16u), a2 = digits_of(w0), a3 = digits_of(w1);
#pragma unroll
            for (int j = 0; j < NT; ++j) mma_digits(acc[r][j], a0, a1, a2, a3, b[j][0], b[j][1]);
          }
          if (step % F == F - 1) {  // the group ends here
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const uint32_t at = sc + (step / F) * TILE_N * 4 + r * 64;
              const float s0 = __uint_as_float(lds32(at)), s1 = __uint_as_float(lds32(at + 32));
#pragma unroll
              for (int j = 0; j < NT; ++j) {
                float f[2];
                asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(f[0]), "=f"(f[1]) : "r"(factors + (((c - from) * (4 / F) + step / F) * NT * 8 + j * 8 + 2 * t) * 4) : "memory");
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  tot[0][r][j][i] = fmaf((__int_as_float(acc[r][j][i]) - 12582912.f) * f[i & 1], i < 2 ? s0 : s1, tot[0][r][j][i]);
              }
            }
          }
        }
      } else {
      const uint32_t xb = xs + (c - from) * 4 * step_bytes + (held * 4 + t) * 16;
      float acc[SETS][2][NT][4];
#pragma unroll
      for (int step = 0; step < 4; ++step) {
        uint32_t b[SETS][Q][4];
#pragma unroll
        for (int s = 0; s < SETS; ++s)
#pragma unroll
          for (int q = 0; q < Q; ++q)
            asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                         : "=r"(b[s][q][0]), "=r"(b[s][q][1]), "=r"(b[s][q][2]), "=r"(b[s][q][3])
                         : "r"(xb + step * step_bytes + s * set_bytes + q * cv * 64)
                         : "memory");
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint32_t w0 = lds32(st + r * 16 * ROW_BYTES + step * 16), w1 = lds32(st + (r * 16 + 8) * ROW_BYTES + step * 16);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t a[4] = {weights_of(w0 >> (8 * h)), weights_of(w1 >> (8 * h)), weights_of(w0 >> (8 * h + 4)), weights_of(w1 >> (8 * h + 4))};
#pragma unroll
            for (int q = 0; q < Q; ++q) {
              if (step % F == 0 && h == 0 && q < NT) mma_anew(acc[0][r][q % NT], a[0], a[1], a[2], a[3], b[0][q][2 * h], b[0][q][2 * h + 1]);
              else mma(acc[0][r][q % NT], a[0], a[1], a[2], a[3], b[0][q][2 * h], b[0][q][2 * h + 1]);
            }
            if (DUAL) {
#pragma unroll
              for (int i = 0; i < 4; ++i) a[i] &= 0x7fff7fffu;
#pragma unroll
              for (int q = 0; q < Q; ++q) {
                if (step % F == 0 && h == 0 && q < NT) mma_anew(acc[SETS - 1][r][q % NT], a[0], a[1], a[2], a[3], b[SETS - 1][q][2 * h], b[SETS - 1][q][2 * h + 1]);
                else mma(acc[SETS - 1][r][q % NT], a[0], a[1], a[2], a[3], b[SETS - 1][q][2 * h], b[SETS - 1][q][2 * h + 1]);
              }
            }
          }
        }
        if (step % F == F - 1) {  // the group ends here
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const uint32_t at = sc + (step / F) * TILE_N * 4 + r * 64;
            const float s0 = __uint_as_float(lds32(at)), s1 = __uint_as_float(lds32(at + 32));
#pragma unroll
            for (int s = 0; s < SETS; ++s) {
              const float f0 = s == 0 ? s0 : fabsf(s0), f1 = s == 0 ? s1 : fabsf(s1);
#pragma unroll
              for (int j = 0; j < NT; ++j) {
                tot[s][r][j][0] = fmaf(f0, acc[s][r][j][0], tot[s][r][j][0]);
                tot[s][r][j][1] = fmaf(f0, acc[s][r][j][1], tot[s][r][j][1]);
                tot[s][r][j][2] = fmaf(f1, acc[s][r][j][2], tot[s][r][j][2]);
                tot[s][r][j][3] = fmaf(f1, acc[s][r][j][3], tot[s][r][j][3]);
              }
            }
          }
        }
      }
      }
    }
  }
  // A warp puts its sums beside its ring, a row to a lane, adds a row's parts, and sends them to the block of the cluster that finishes the row (each takes as many
  // rows of every tile): [product, row of the inputs][warp of the columns][row].  The sums over the columns are taken there, in a fixed order.
  const int sources = sp.cluster * sp.kw, each_log2 = 5 - sp.cluster_log2, mine = sp.rw << each_log2;
  copies_wait<0>();
  __syncwarp();
#pragma unroll
  for (int s = 0; s < SETS; ++s)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          asm volatile("st.shared.f32 [%0], %1;" ::"r"(ring + (((s * NT + j) * 8 + 2 * t + (i & 1)) * 36 + r * 16 + g + (i >> 1) * 8) * 4), "f"(tot[s][r][j][i]) : "memory");
  __syncwarp();
  if constexpr (P == DIGITS) {
    if (__syncthreads_or(stager.rest)) add_rest<NT, F>(p, first + kw, end, sp.kw, n0, wide, ring);
  }
  if (sp.cluster > 1) cluster_wait();
  {
    const int owner = lane >> each_log2;
    uint32_t at = inbox + ((rank * sp.kw + kw) * mine + (rw << each_log2) + lane - (owner << each_log2)) * 4;
    if (sp.cluster > 1) at = cluster_address(at, owner);
#pragma unroll
    for (int s = 0; s < SETS; ++s)
      for (int m = 0; m < M; ++m) {
        const uint32_t from = ring + ((s * NT * 8 + m * COUNT) * 36 + lane) * 4;
        float v = __uint_as_float(lds32(from));
#pragma unroll
        for (int n = 1; n < COUNT; ++n) v += __uint_as_float(lds32(from + n * 36 * 4));
        cluster_store(at + (s * M + m) * sources * mine * 4, v, sp.cluster > 1);
      }
  }
  if (sp.cluster > 1) cluster_barrier();
  else __syncthreads();
  const float* box = reinterpret_cast<const float*>(smem);
  for (int i = threadIdx.x; i < mine * M; i += blockDim.x) {
    const int m = __umulhi(i, sp.mine_inverse), row = i - m * mine;  // i / mine
    const int tile = row >> each_log2, n = ((blockIdx.x >> sp.cluster_log2) * sp.rw + tile) * TILE_N + (rank << each_log2) + row - (tile << each_log2);
    if (n >= w.n_out) continue;
    float sum[2];
#pragma unroll
    for (int s = 0; s < SETS; ++s) {
      const float* at = box + (s * M + m) * sources * mine + row;
      float v[4] = {0.f, 0.f, 0.f, 0.f};
      int k = 0;
      for (; k + 4 <= sources; k += 4, at += 4 * mine) {
#pragma unroll
        for (int x = 0; x < 4; ++x) v[x] += at[x * mine];
      }
      for (; k < sources; ++k, at += mine) v[0] += *at;
      sum[s] = (v[0] + v[1]) + (v[2] + v[3]);
    }
    const float c = sum[0] + (p.bias ? load_any(p.bias, p.bias_type, n) : 0.f);
    const long long at = (long long)(m0 + m) * w.n_out + n;
    if (DUAL) {
      static_cast<float*>(p.y)[at] = c - sum[1];
      p.y2[at] = c + sum[1];
    } else {
      store_any(p.y, p.type, at, c);
    }
  }
}

template <int P, bool PACKED, int NT, bool DUAL>
int forward(const W4LinearArgs& p, Split sp, int tiles_m, cudaStream_t stream) {
  static SmemOptIn table[3];
  constexpr int Q = (PACKED ? 1 : P) * NT, SETS = DUAL ? 2 : 1, COUNT = PACKED ? P : 1;
  const int tiles_n = ceil_div(p.w.n_out, TILE_N), chunks = ceil_div(p.w.n_in, CHUNK);
  const int cv = NT > 1 ? 8 : sp.tile_m * COUNT;
  const int chunk_bytes = P == DIGITS ? 4 * NT * cv * 32 + 4 * NT * 32 : 4 * SETS * Q * cv * 64;
  // 16 warps an SM: the columns are split as often as that takes.  Over a cluster while a block's part of the rows is long (every block makes
  // parts of what it reads, 4096 elements take about a microsecond), else over the warps of a block.
  const long long units = (long long)tiles_n * tiles_m;
  int split = power_below((int)std::max<long long>(1, std::min<long long>(chunks, (16LL * SMS) / units)));
  if (split < chunks && 2 * split * units <= 16LL * SMS) split *= 2;
  sp.cluster = 1;
  while (sp.cluster < 8 && sp.cluster < split && (long long)sp.tile_m * p.w.n_in / sp.cluster > 4096) sp.cluster *= 2;
  sp.kw = std::min(WARPS, split / sp.cluster);
  while (sp.kw * chunk_bytes > X_MOST) sp.kw /= 2;  // the warps of a block take a chunk each
  sp.cluster = std::min(8, std::max(sp.cluster, split / sp.kw));
  sp.kw_log2 = log2_of(sp.kw);
  sp.cluster_log2 = log2_of(sp.cluster);
  sp.rw = WARPS / sp.kw;
  const int mine = sp.rw * TILE_N / sp.cluster;
  sp.mine_inverse = mine == 1 ? 0xffffffffu : (unsigned)((0x100000000ULL + mine - 1) / mine);
  const int share = ceil_div(chunks, sp.cluster);
  sp.inbox = ceil_div((long long)sp.kw * SETS * sp.tile_m * TILE_N * sp.rw * 4, 128) * 128;
  const int room = SHARED_OF_TWO - sp.inbox - RING_BYTES;  // for the parts of the rows, with two blocks on an SM
  sp.per_phase = std::max(sp.kw, room / chunk_bytes / sp.kw * sp.kw);
  const int smem = sp.inbox + RING_BYTES + std::min(sp.per_phase, share) * chunk_bytes;
  const long long blocks = (long long)ceil_div(tiles_n, sp.rw) * sp.cluster;
  if (p.w.group_log2 == 5)
    return launch_clustered(w4_forward_kernel<P, PACKED, NT, DUAL, 1>, "w4_forward_kernel", table[0], p, sp, blocks, tiles_m, THREADS, smem, stream);
  if (p.w.group_log2 == 6)
    return launch_clustered(w4_forward_kernel<P, PACKED, NT, DUAL, 2>, "w4_forward_kernel", table[1], p, sp, blocks, tiles_m, THREADS, smem, stream);
  return launch_clustered(w4_forward_kernel<P, PACKED, NT, DUAL, 4>, "w4_forward_kernel", table[2], p, sp, blocks, tiles_m, THREADS, smem, stream);
}

}  // namespace

int launch_w4_linear(const W4LinearArgs& all, cudaStream_t stream) {
  Split sp = {};
  const bool dual = all.b != nullptr;
  const bool digits = all.type != BF_TYPE_F32 && all.M <= 4;
  const int parts = digits ? DIGITS : all.type == BF_TYPE_F32 ? 3 : all.type == BF_TYPE_F16 ? 2 : 1;
  const int side = all.M * parts;  // columns that the rows' parts fill side by side: fewer instructions up to two tiles
  // (9 and 10 rows in three parts: 4 tiles side by side, 6 otherwise)
  sp.packed = side <= 8 || (side <= 16 && parts > 1) || (side > 24 && side <= 32 && parts == 3 && !dual);
  const int nt = sp.packed ? (side <= 8 ? 1 : side <= 16 ? 2 : 4) : all.M <= 8 ? 1 : 2;
  sp.tile_m = sp.packed ? all.M : std::min(all.M, 8 * nt);
  const long long tiles = ceil_div(all.M, sp.tile_m);
  for (long long first = 0; first < tiles; first += MOST_TILES) {
    const int here = (int)std::min<long long>(MOST_TILES, tiles - first);
    W4LinearArgs p = all;
    const long long skip = first * sp.tile_m, size = all.type == BF_TYPE_F32 ? 4 : 2;
    p.M = (int)std::min<long long>(all.M - skip, (long long)here * sp.tile_m);
    p.a = static_cast<const char*>(all.a) + skip * all.w.n_in * size;
    p.b = dual ? all.b + skip * all.w.n_in : nullptr;
    p.y = static_cast<char*>(all.y) + skip * all.w.n_out * size;
    p.y2 = dual ? all.y2 + skip * all.w.n_out : nullptr;
    int rc;
    if (dual)
      rc = sp.packed ? (nt == 1 ? forward<3, true, 1, true>(p, sp, here, stream) : forward<3, true, 2, true>(p, sp, here, stream))
                     : (nt == 1 ? forward<3, false, 1, true>(p, sp, here, stream) : forward<3, false, 2, true>(p, sp, here, stream));
    else if (digits) rc = nt == 1 ? forward<DIGITS, true, 1, false>(p, sp, here, stream) : forward<DIGITS, true, 2, false>(p, sp, here, stream);
    else if (parts == 3)
      rc = sp.packed ? (nt == 1 ? forward<3, true, 1, false>(p, sp, here, stream) : nt == 2 ? forward<3, true, 2, false>(p, sp, here, stream)
                                                                                            : forward<3, true, 4, false>(p, sp, here, stream))
                     : (nt == 1 ? forward<3, false, 1, false>(p, sp, here, stream) : forward<3, false, 2, false>(p, sp, here, stream));
    else if (parts == 2)
      rc = !sp.packed ? forward<2, false, 2, false>(p, sp, here, stream) : nt == 1 ? forward<2, true, 1, false>(p, sp, here, stream) : forward<2, true, 2, false>(p, sp, here, stream);
    else rc = nt == 1 ? forward<1, true, 1, false>(p, sp, here, stream) : forward<1, false, 2, false>(p, sp, here, stream);
    if (rc != BF_OK) return rc;
  }
  return BF_OK;
}

}  // namespace bf
