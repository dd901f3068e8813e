// y = x W^T + bias for few rows x and 4-bit weights, and the bounds of it over boxes (W c -/+ |W| r); weights4_mma.cuh says how.
#include "weights4_mma.cuh"

namespace bf {
namespace {

constexpr int X_BYTES = 40 * 1024;   // parts of the rows: with the ring, two blocks share an SM
constexpr int X_MOST = 150 * 1024;   // and what a block alone on an SM has left of its 227 KB

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

__device__ __forceinline__ void load8(const float* p, int left, bool wide, float (&v)[8]) {
  if (wide && left >= 8) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < left ? p[j] : 0.f;
  }
}
// Eight 16-bit numbers as four words.
__device__ __forceinline__ uint4 load8(const uint16_t* p, int left, bool wide) {
  if (wide && left >= 8) return *reinterpret_cast<const uint4*>(p);
  uint32_t v[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = (2 * j < left ? p[2 * j] : 0) | ((uint32_t)(2 * j + 1 < left ? p[2 * j + 1] : 0) << 16);
  return make_uint4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void put16(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// Parts of the rows' columns [from, to) * 128 in shared memory: [step of 32 columns][product][part, tile][column][4 lanes][8 columns of the step], the 8 in the
// order 0 4 1 5 2 6 3 7 that `weights_of` gives the codes of a word in.  Eight columns of a row are a thread's turn.
template <int P, int NT, bool DUAL>
__device__ __forceinline__ void stage_rows(const W4LinearArgs& p, int packed, int from, int to, int m0, int M, int cv, int step_bytes, int set_bytes, uint32_t xs) {
  constexpr int SETS = DUAL ? 2 : 1;
  const int blocks = (to - from) * (CHUNK / 8), n_in = p.w.n_in;
  const int per = P == 3 ? 4 : 8;  // elements of a 16-byte piece
  const bool wide = n_in % per == 0 && (((uintptr_t)p.a | (uintptr_t)p.b) & 15) == 0;
  int m = 0, blk = threadIdx.x;
  while (blk >= blocks) { blk -= blocks; ++m; }
  while (m < M) {
    const int k = from * CHUNK + blk * 8, left = n_in - k;
    const long long at = (long long)(m0 + m) * n_in + k;
    uint32_t o[SETS][P][4];
    if (P == 1) {
      const uint4 v = load8(static_cast<const uint16_t*>(p.a) + at, left, wide);
      o[0][0][0] = __byte_perm(v.x, v.z, 0x5410);
      o[0][0][1] = __byte_perm(v.x, v.z, 0x7632);
      o[0][0][2] = __byte_perm(v.y, v.w, 0x5410);
      o[0][0][3] = __byte_perm(v.y, v.w, 0x7632);
    } else {
      float v[SETS][8];
      if (P == 2) {
        const uint4 q = load8(static_cast<const uint16_t*>(p.a) + at, left, wide);
        const uint32_t q4[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&q4[j]));
          v[0][2 * j] = f.x;
          v[0][2 * j + 1] = f.y;
        }
      } else {
        load8(static_cast<const float*>(p.a) + at, left, wide, v[0]);
        if (DUAL) {
          load8(p.b + at, left, wide, v[SETS - 1]);
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
          for (int i = 0; i < P; ++i) o[s][i][j] = q[i];
        }
    }
    const uint32_t dst = xs + (blk >> 2) * step_bytes + (blk & 3) * 16;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int j = packed ? m * P + i : i * NT * 8 + m;  // column, counted through the tiles
      const uint32_t to_q = dst + ((j >> 3) * cv + (j & 7)) * 64;
#pragma unroll
      for (int s = 0; s < SETS; ++s) put16(to_q + s * set_bytes, o[s][i][0], o[s][i][1], o[s][i][2], o[s][i][3]);
    }
    blk += THREADS;
    while (blk >= blocks) { blk -= blocks; ++m; }
  }
}

// PARTS instructions for NT tiles of 8 columns; DUAL: W c and |W| r; F: steps of 32 columns that share a scale (1, 2, or 4 and more).
template <int PARTS, int NT, bool DUAL, int F>
__global__ void __launch_bounds__(THREADS, PARTS * NT * (DUAL ? 2 : 1) > 6 ? 1 : 2) w4_forward_kernel(const W4LinearArgs p, const Split sp) {
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr int Q = PARTS * NT, SETS = DUAL ? 2 : 1;
  const W4 w = p.w;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int kw = warp % sp.kw, rw = warp / sp.kw, rows_cta = TILE_N * (WARPS / sp.kw);
  const int rank = blockIdx.x % sp.cluster;
  const int nb = (blockIdx.x / sp.cluster) * rows_cta, n0 = nb + rw * TILE_N;
  const int m0 = blockIdx.y * sp.tile_m, M = min(sp.tile_m, p.M - m0);
  const int parts = p.type == BF_TYPE_F32 ? 3 : p.type == BF_TYPE_F16 ? 2 : 1;
  const int cv = NT > 1 ? 8 : sp.packed ? M * parts : M;  // columns of a tile that are held
  const int chunks = (w.n_in + CHUNK - 1) / CHUNK, share = (chunks + sp.cluster - 1) / sp.cluster;
  const int first = min(rank * share, chunks), end = min(first + share, chunks);
  const int groups = w.groups();
  const int pitch = (int)w.pitch();
  const uint32_t ring = smem_of(smem) + warp * (STAGES * STAGE_BYTES), xs = smem_of(smem) + RING_BYTES;
  const int set_bytes = Q * cv * 64, step_bytes = SETS * set_bytes;
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
  auto load_next = [&](uint32_t to) {
    if (next < end) {
      load_codes(to, codes + next * (CHUNK / 2), 8LL * pitch, rows, pitch - next * (CHUNK / 2), lane);
      load_scales(to, w, groups, n0, next, lane);
    }
    copies_begin();
    next += sp.kw;
  };
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) load_next(ring + s * STAGE_BYTES);
  int slot = 0;
  for (int from = first; from < end; from += sp.per_phase) {
    const int to = min(from + sp.per_phase, end);
    if (from != first) __syncthreads();
    if (parts == 3) stage_rows<3, NT, DUAL>(p, sp.packed, from, to, m0, M, cv, step_bytes, set_bytes, xs);
    if (!DUAL && parts == 2) stage_rows<2, NT, false>(p, sp.packed, from, to, m0, M, cv, step_bytes, set_bytes, xs);
    if (!DUAL && parts == 1) stage_rows<1, NT, false>(p, sp.packed, from, to, m0, M, cv, step_bytes, set_bytes, xs);
    __syncthreads();
    for (int c = from + kw; c < to; c += sp.kw) {
      copies_wait<STAGES - 2>();
      __syncwarp();
      load_next(ring + (slot == 0 ? STAGES - 1 : slot - 1) * STAGE_BYTES);  // into the slot that was read last
      const uint32_t st = ring + slot * STAGE_BYTES + g * ROW_BYTES + t * 4;
      slot = slot == STAGES - 1 ? 0 : slot + 1;
      const uint32_t sc = st - g * (ROW_BYTES - 4) - t * 4 + TILE_N * ROW_BYTES;
      const uint32_t xb = xs + (c - from) * 4 * step_bytes + (min(g, cv - 1) * 4 + t) * 16;  // columns that are not held repeat the last
      float acc[SETS][2][NT][4];
#pragma unroll
      for (int step = 0; step < 4; ++step) {
        if (step % F == 0) {
#pragma unroll
          for (int s = 0; s < SETS; ++s)
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
              for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[s][r][j][i] = 0.f;
        }
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
            for (int q = 0; q < Q; ++q) mma(acc[0][r][q % NT], a[0], a[1], a[2], a[3], b[0][q][2 * h], b[0][q][2 * h + 1]);
            if (DUAL) {
#pragma unroll
              for (int i = 0; i < 4; ++i) a[i] &= 0x7fff7fffu;
#pragma unroll
              for (int q = 0; q < Q; ++q) mma(acc[SETS - 1][r][q % NT], a[0], a[1], a[2], a[3], b[SETS - 1][q][2 * h], b[SETS - 1][q][2 * h + 1]);
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
  // Sums over the warps that split the columns, then over the blocks that did, each in order.
  constexpr int CC = SETS * NT * 8;
  float* red = reinterpret_cast<float*>(smem);  // [kw][CC][rows of the block and a pad]
  const int line = rows_cta + 4;
  copies_wait<0>();
  __syncthreads();
#pragma unroll
  for (int s = 0; s < SETS; ++s)
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          red[(kw * CC + (s * NT + j) * 8 + 2 * t + (i & 1)) * line + rw * TILE_N + r * 16 + g + (i >> 1) * 8] = tot[s][r][j][i];
  __syncthreads();
  const int count = sp.packed ? parts : 1;
  float* own = red + sp.kw * CC * line;  // [product][row of the tile][rows of the block]
  for (int i = threadIdx.x; i < SETS * M * rows_cta; i += THREADS) {
    const int row = i % rows_cta, j = i / rows_cta, s = DUAL && j >= M ? 1 : 0, m = j - s * M;
    const float* at = red + (s * NT * 8 + m * count) * line + row;
    float v = 0.f;
    for (int k = 0; k < sp.kw; ++k)
      for (int part = 0; part < count; ++part) v += at[(k * CC + part) * line];
    own[i] = v;
  }
  if (sp.cluster > 1) cluster_barrier();
  else __syncthreads();
  const int mine = rows_cta / sp.cluster;  // rows of the block that this one finishes
  for (int i = threadIdx.x; i < mine * M; i += THREADS) {
    const int m = i / mine, row = rank * mine + i - m * mine, n = nb + row;
    if (n >= w.n_out) continue;
    float sum[2];
#pragma unroll
    for (int s = 0; s < SETS; ++s) sum[s] = cluster_sum(own + (s * M + m) * rows_cta + row, sp.cluster);
    const float c = sum[0] + (p.bias ? load_any(p.bias, p.bias_type, n) : 0.f);
    const long long at = (long long)(m0 + m) * w.n_out + n;
    if (DUAL) {
      static_cast<float*>(p.y)[at] = c - sum[1];
      p.y2[at] = c + sum[1];
    } else {
      store_any(p.y, p.type, at, c);
    }
  }
  if (sp.cluster > 1) cluster_barrier();  // the others may still read this block's sums
}

template <int PARTS, int NT, bool DUAL>
int forward(const W4LinearArgs& p, Split sp, int tiles_m, cudaStream_t stream) {
  static SmemOptIn table[3];
  const int tiles_n = ceil_div(p.w.n_out, TILE_N), chunks = ceil_div(p.w.n_in, CHUNK);
  const int parts = p.type == BF_TYPE_F32 ? 3 : p.type == BF_TYPE_F16 ? 2 : 1;
  const int cv = NT > 1 ? 8 : sp.packed ? sp.tile_m * parts : sp.tile_m;
  const int chunk_bytes = 4 * (DUAL ? 2 : 1) * PARTS * NT * cv * 64;
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
  const int share = ceil_div(chunks, sp.cluster);
  sp.per_phase = std::max(sp.kw, X_BYTES / chunk_bytes / sp.kw * sp.kw);
  const int x_bytes = std::min(sp.per_phase, share) * chunk_bytes;
  const long long blocks = (long long)ceil_div(p.w.n_out, TILE_N * (WARPS / sp.kw)) * sp.cluster;
  const int smem = RING_BYTES + x_bytes;
  if (p.w.group_log2 == 5) return launch_clustered(w4_forward_kernel<PARTS, NT, DUAL, 1>, "w4_forward_kernel", table[0], p, sp, blocks, tiles_m, smem, stream);
  if (p.w.group_log2 == 6) return launch_clustered(w4_forward_kernel<PARTS, NT, DUAL, 2>, "w4_forward_kernel", table[1], p, sp, blocks, tiles_m, smem, stream);
  return launch_clustered(w4_forward_kernel<PARTS, NT, DUAL, 4>, "w4_forward_kernel", table[2], p, sp, blocks, tiles_m, smem, stream);
}

}  // namespace

int launch_w4_linear(const W4LinearArgs& all, cudaStream_t stream) {
  Split sp = {};
  const bool dual = all.b != nullptr;
  const int parts = all.type == BF_TYPE_F32 ? 3 : all.type == BF_TYPE_F16 ? 2 : 1;
  const int side = all.M * parts;  // columns that the rows' parts fill side by side: fewer instructions up to two tiles
  sp.packed = side <= 8 || (side <= 16 && parts > 1);
  const int nt = sp.packed ? (side <= 8 ? 1 : 2) : all.M <= 8 ? 1 : 2;
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
      rc = sp.packed ? (nt == 1 ? forward<1, 1, true>(p, sp, here, stream) : forward<1, 2, true>(p, sp, here, stream))
                     : nt == 1 ? forward<3, 1, true>(p, sp, here, stream) : forward<3, 2, true>(p, sp, here, stream);
    else if (sp.packed || parts == 1) rc = nt == 1 ? forward<1, 1, false>(p, sp, here, stream) : forward<1, 2, false>(p, sp, here, stream);
    else if (parts == 2) rc = forward<2, 2, false>(p, sp, here, stream);
    else rc = nt == 1 ? forward<3, 1, false>(p, sp, here, stream) : forward<3, 2, false>(p, sp, here, stream);
    if (rc != BF_OK) return rc;
  }
  return BF_OK;
}

}  // namespace bf
