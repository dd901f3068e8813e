// Products of few rows with 4-bit weights, on the warp-level tensor-core instruction (m16n8k16, bfloat16 in, fp32 sums).
//
// The codes are what has to be read: half a byte a weight, so that at 6.5 TB/s 13 thousand million weights a millisecond pass and a
// multiplication in FP32 registers (convert, scale, multiply-add for every row) would bound the kernel instead.  A code minus 8 is exact in bfloat16:
// `weights_of` makes two of them from a word with three operations, and the rows go in as sums of bfloat16 parts, which hold a
// 32-bit number exactly (8 + 8 + 8 bits), a 16-bit one in one part (bf16) or two (fp16).  So every product is exact and only the sums round.  The rows are
// the instruction's 8 columns: parts side by side where rows x parts <= 8 (one instruction for 16 x 16 weights), else one instruction for
// each part and 8 rows.  The 128-row tiles of the tcgen05 instructions would take operands through shared memory: 2 bytes a weight written and read there
// where this kernel moves half a byte, for rows that fill an eighth of the instruction's smallest tile.
//
// Codes and scales come by cp.async into a ring of each warp's own (no barrier between warps), 32 rows x 128 columns a stage.
#include <algorithm>

#include "weights4.cuh"

namespace bf {
namespace {

constexpr int WARPS = 8, THREADS = 32 * WARPS;
constexpr int CHUNK = 128;                         // columns of a stage
constexpr int TILE_N = 32;                         // rows of a stage
constexpr int ROW_BYTES = 80;                      // 64 and a pad that keeps 8 rows x 4 words on 32 banks
constexpr int STAGE_BYTES = TILE_N * ROW_BYTES + 4 * TILE_N * 4;  // codes; scales of up to 4 groups
constexpr int STAGES = 3;
constexpr int RING_BYTES = WARPS * STAGES * STAGE_BYTES;
constexpr int X_BYTES = 40 * 1024;                 // parts of the rows: with the ring, two blocks share an SM
constexpr int X_MOST = 150 * 1024;                 // and what a block alone on an SM has left of its 227 KB
constexpr int SMS = 148;

__device__ __forceinline__ uint32_t smem_of(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t to, const void* from, bool valid) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(valid ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copies_begin() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

// Codes in bits 0-3 and 16-19 of `w`, minus 8, as two bfloat16: 0x4300 | code is 128 + code.
__device__ __forceinline__ uint32_t weights_of(uint32_t w) {
  uint32_t v = (w & 0x000f000fu) | 0x43004300u;
  const __nv_bfloat162 off = __halves2bfloat162(__ushort_as_bfloat16(0x4308), __ushort_as_bfloat16(0x4308));
  const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), off);
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The bfloat16 parts of v: two and three parts of 8 bits each (the last rounded to the nearest).  Infinities and NaN are one part.
__device__ __forceinline__ void parts_of(float v, int parts, uint32_t (&p)[3]) {
  const uint32_t bits = __float_as_uint(v);
  if ((bits & 0x7fffffffu) >= 0x7f800000u) {
    p[0] = (bits >> 16) | ((bits & 0x007fffffu) ? 0x40u : 0u);
    p[1] = p[2] = 0;
    return;
  }
  if (parts == 3) {
    p[0] = bits >> 16;
    const float r = v - __uint_as_float(bits & 0xffff0000u);
    p[1] = __float_as_uint(r) >> 16;
    p[2] = __float_as_uint(r - __uint_as_float(__float_as_uint(r) & 0xffff0000u)) >> 16;
  } else {
    const __nv_bfloat16 h = __float2bfloat16(v);
    p[0] = __bfloat16_as_ushort(h);
    p[1] = __bfloat16_as_ushort(__float2bfloat16(v - __bfloat162float(h)));
    p[2] = 0;
  }
}

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

// Where the work of a block lies.
struct Split {
  int parts;      // bfloat16 parts of a row
  int kw;         // forward: warps that share rows and split columns (8 / kw row tiles a block)
  int cluster;    // blocks that split the columns (forward) or the outputs (rows)
  int per_phase;  // forward: chunks whose parts fit X_BYTES
  int tile_m;     // rows of a block
};

// Lanes copy a stage: codes [32 rows][64 bytes from column `chunk` * 128], scales of the chunk's groups.
__device__ __forceinline__ void load_stage(const W4& w, long long pitch, int groups, uint32_t to, int n0, int chunk, int lane) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int seg = lane + 32 * j, row = seg >> 2;
    const long long at = (long long)chunk * (CHUNK / 2) + (seg & 3) * 16;
    const bool ok = n0 + row < w.n_out && at < pitch;
    copy16(to + row * ROW_BYTES + (seg & 3) * 16, w.codes + (ok ? (long long)(n0 + row) * pitch + at : 0), ok);
  }
  const int in_chunk = w.group_log2 >= 7 ? 1 : CHUNK >> w.group_log2;
  const int g0 = w.group_log2 >= 7 ? chunk >> (w.group_log2 - 7) : chunk << (7 - w.group_log2);
  for (int i = 0; i < in_chunk; ++i) {
    const bool ok = n0 + lane < w.n_out && g0 + i < groups;
    copy4(to + TILE_N * ROW_BYTES + (i * TILE_N + lane) * 4, w.scales + (ok ? (long long)(g0 + i) * w.n_out + n0 + lane : 0), ok);
  }
}

__device__ __forceinline__ uint32_t lds32(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ float cluster_read(const float* p, uint32_t rank) {
  uint32_t at;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_of(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// ---- y = x W^T --------------------------------------------------------------------
// PARTS instructions for 8 rows (1: one part, or all parts of at most 8 / parts rows side by side), NT tiles of 8 rows, DUAL: W c and |W| r.
// Shared memory: ring | parts of the rows [step of 32 columns][product][part, tile][column][4 lanes][8 columns of the step], where the 8 are stored in the order
// 0 4 1 5 2 6 3 7 that `weights_of` gives the codes of a word in.
template <int PARTS, int NT, bool DUAL>
__global__ void __launch_bounds__(THREADS, PARTS * NT * (DUAL ? 2 : 1) > 6 ? 1 : 2) w4_forward_kernel(const W4LinearArgs p, const Split sp) {
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr int Q = PARTS * NT, SETS = DUAL ? 2 : 1;
  const W4 w = p.w;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int kw = warp % sp.kw, rw = warp / sp.kw, rows_cta = TILE_N * (WARPS / sp.kw);
  const int rank = blockIdx.x % sp.cluster;
  const int nb = (blockIdx.x / sp.cluster) * rows_cta, n0 = nb + rw * TILE_N;
  const int m0 = blockIdx.y * sp.tile_m, M = min(sp.tile_m, p.M - m0);
  const bool packed = PARTS == 1 && NT == 1;
  const int cv = packed ? M * sp.parts : (NT == 1 ? M : 8);  // columns of a tile that are held
  const int chunks = (w.n_in + CHUNK - 1) / CHUNK, share = (chunks + sp.cluster - 1) / sp.cluster;
  const int first = min(rank * share, chunks), end = min(first + share, chunks);
  const int groups = w.groups();
  const long long pitch = w.pitch();
  const uint32_t ring = smem_of(smem) + warp * (STAGES * STAGE_BYTES), xs = smem_of(smem) + RING_BYTES;
  const int step_bytes = SETS * Q * cv * 64, set_bytes = Q * cv * 64;
  const int fold_mask = w.group_log2 >= 7 ? 3 : (1 << (w.group_log2 - 5)) - 1, fold_shift = min(w.group_log2, 7) - 5;

  float tot[SETS][2][NT][4], acc[SETS][2][NT][4];
#pragma unroll
  for (int s = 0; s < SETS; ++s)
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) tot[s][r][j][i] = acc[s][r][j][i] = 0.f;

  int next = first + kw;  // the chunk that is copied next
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) {
    if (next < end) load_stage(w, pitch, groups, ring + s * STAGE_BYTES, n0, next, lane);
    copies_begin();
    next += sp.kw;
  }
  int slot = 0;
  for (int from = first; from < end; from += sp.per_phase) {
    const int to = min(from + sp.per_phase, end);
    if (from != first) __syncthreads();
    // parts of the rows' columns [from, to) * 128: eight columns a thread
    const int blocks = (to - from) * (CHUNK / 8);
    for (int i = threadIdx.x; i < blocks * M; i += THREADS) {
      const int m = i / blocks, blk = i - m * blocks, k = from * CHUNK + blk * 8;
      const long long at = (long long)(m0 + m) * w.n_in + k;
      float v[SETS][8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (DUAL) {
          v[0][j] = v[SETS - 1][j] = 0.f;
          if (k + j < w.n_in) centre_radius(static_cast<const float*>(p.a)[at + j], p.b[at + j], p.mode, p.relu_in, v[0][j], v[SETS - 1][j]);
        } else {
          v[0][j] = k + j < w.n_in ? load_any(p.a, p.type, at + j) : 0.f;
        }
      }
#pragma unroll
      for (int s = 0; s < SETS; ++s) {
        uint32_t e[3][8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          uint32_t q[3];
          parts_of(v[s][j], sp.parts, q);
          e[0][j] = q[0];
          e[1][j] = q[1];
          e[2][j] = q[2];
        }
        for (int part = 0; part < sp.parts; ++part) {
          const int col = packed ? m * sp.parts + part : (m & 7), q = packed ? 0 : part * NT + (m >> 3);
          uint32_t o[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t lo = part == 0 ? e[0][j] : part == 1 ? e[1][j] : e[2][j], hi = part == 0 ? e[0][j + 4] : part == 1 ? e[1][j + 4] : e[2][j + 4];
            o[j] = lo | (hi << 16);
          }
          const uint32_t dst = xs + (blk >> 2) * step_bytes + s * set_bytes + ((q * cv + col) * 4 + (blk & 3)) * 16;
          asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(dst), "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3]) : "memory");
        }
      }
    }
    __syncthreads();
    for (int c = from + kw; c < to; c += sp.kw) {
      copies_wait<STAGES - 2>();
      __syncwarp();
      {  // into the slot that was read last
        const int free_slot = slot == 0 ? STAGES - 1 : slot - 1;
        if (next < end) load_stage(w, pitch, groups, ring + free_slot * STAGE_BYTES, n0, next, lane);
        copies_begin();
        next += sp.kw;
      }
      const uint32_t st = ring + slot * STAGE_BYTES;
      slot = slot == STAGES - 1 ? 0 : slot + 1;
#pragma unroll
      for (int step = 0; step < 4; ++step) {
        uint32_t b[SETS][Q][4];
        const uint32_t xb = xs + ((c - from) * 4 + step) * step_bytes + (g * 4 + t) * 16;
#pragma unroll
        for (int s = 0; s < SETS; ++s)
#pragma unroll
          for (int q = 0; q < Q; ++q) {
            b[s][q][0] = b[s][q][1] = b[s][q][2] = b[s][q][3] = 0;
            if (g < cv)
              asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(b[s][q][0]), "=r"(b[s][q][1]), "=r"(b[s][q][2]), "=r"(b[s][q][3]) : "r"(xb + s * set_bytes + q * cv * 64) : "memory");
          }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint32_t w0 = lds32(st + (r * 16 + g) * ROW_BYTES + (step * 4 + t) * 4), w1 = lds32(st + (r * 16 + g + 8) * ROW_BYTES + (step * 4 + t) * 4);
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
        if (((step + 1) & fold_mask) == 0) {  // the group ends here
          const uint32_t sc = st + TILE_N * ROW_BYTES + ((step >> fold_shift) * TILE_N + g) * 4;
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float s0 = __uint_as_float(lds32(sc + r * 64)), s1 = __uint_as_float(lds32(sc + r * 64 + 32));
#pragma unroll
            for (int s = 0; s < SETS; ++s) {
              const float f0 = s == 0 ? s0 : fabsf(s0), f1 = s == 0 ? s1 : fabsf(s1);
#pragma unroll
              for (int j = 0; j < NT; ++j) {
                tot[s][r][j][0] = fmaf(f0, acc[s][r][j][0], tot[s][r][j][0]);
                tot[s][r][j][1] = fmaf(f0, acc[s][r][j][1], tot[s][r][j][1]);
                tot[s][r][j][2] = fmaf(f1, acc[s][r][j][2], tot[s][r][j][2]);
                tot[s][r][j][3] = fmaf(f1, acc[s][r][j][3], tot[s][r][j][3]);
                acc[s][r][j][0] = acc[s][r][j][1] = acc[s][r][j][2] = acc[s][r][j][3] = 0.f;
              }
            }
          }
        }
      }
    }
  }
  // Sums over the warps that split the columns, then over the blocks that did, each in order.
  constexpr int CC = SETS * NT * 8;
  float* red = reinterpret_cast<float*>(smem);  // [kw][rows of the block][CC]
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
          red[(kw * rows_cta + rw * TILE_N + r * 16 + g + (i >> 1) * 8) * CC + (s * NT + j) * 8 + 2 * t + (i & 1)] = tot[s][r][j][i];
  __syncthreads();
  for (int i = threadIdx.x; i < rows_cta * CC; i += THREADS) {
    float v = red[i];
    for (int k = 1; k < sp.kw; ++k) v += red[k * rows_cta * CC + i];
    red[i] = v;
  }
  if (sp.cluster > 1) cluster_barrier();
  else __syncthreads();
  const int mine = rows_cta / sp.cluster;  // rows of the block that this one finishes
  for (int i = threadIdx.x; i < mine * M; i += THREADS) {
    const int m = i / mine, row = rank * mine + i - m * mine, n = nb + row;
    if (n >= w.n_out) continue;
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int s = 0; s < SETS; ++s) {
      const int count = packed ? sp.parts : 1, col = packed ? m * sp.parts : m;
      for (int part = 0; part < count; ++part) {
        const float* at = red + row * CC + s * NT * 8 + col + part;
        float v = 0.f;
        if (sp.cluster == 1) v = *at;
        else
          for (int k = 0; k < sp.cluster; ++k) v += cluster_read(at, k);
        sum[s] += v;
      }
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
  if (sp.cluster > 1) cluster_barrier();  // the others may still read this block's sums
}

// ---- z = a W ------------------------------------------------------------------------
// A block takes 128 columns and (with its cluster) splits the outputs over its warps, 32 at a time.  The scale belongs to the sum's index here, so it goes
// into the rows: a[m, n] * scale[group, n], rounded to 32 bits and split into parts, by each warp for the outputs it reads.
// Columns are the instruction's rows: lane (g, t) takes half a word (four columns) of each of the outputs 2t, 2t + 1, 2t + 8, 2t + 9.
template <int PARTS, int NT, bool DUAL>
__global__ void __launch_bounds__(THREADS, 2) w4_rows_kernel(const W4RowsArgs p, const Split sp) {
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr int Q = PARTS * NT, SETS = DUAL ? 2 : 1, MT = 8 * NT;
  const W4 w = p.w;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int rank = blockIdx.x % sp.cluster, kb = blockIdx.x / sp.cluster;
  const int m0 = blockIdx.y * sp.tile_m, M = min(sp.tile_m, p.M - m0);
  const bool packed = PARTS == 1;
  const int cv = packed ? M * sp.parts : (NT == 1 ? M : 8);
  const int tiles = (w.n_out + TILE_N - 1) / TILE_N, share = (tiles + sp.cluster - 1) / sp.cluster;
  const int first = min(rank * share, tiles), end = min(first + share, tiles);
  const int groups = w.groups();
  const long long pitch = w.pitch();
  const uint32_t ring = smem_of(smem) + warp * (STAGES * STAGE_BYTES);
  const int set_bytes = Q * cv * 64;
  const uint32_t as = smem_of(smem) + RING_BYTES + warp * (SETS * set_bytes);  // [set][part, tile][column][32 outputs, in the order the lanes read them]
  const int in_chunk = w.group_log2 >= 7 ? 1 : CHUNK >> w.group_log2, steps = 4 / in_chunk;
  const int half = lane >> 4, in16 = lane & 15, place = half * 16 + (in16 & 6) * 2 + ((in16 >> 3) << 1) + (in16 & 1);

  float acc[SETS][4][2][NT][4];
#pragma unroll
  for (int s = 0; s < SETS; ++s)
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[s][r][e][j][i] = 0.f;

  auto rows_at = [&](int tile, float (&v)[SETS][MT]) {
    const int n = tile * TILE_N + lane;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      v[0][m] = 0.f;
      if (DUAL) v[SETS - 1][m] = 0.f;
      if (m < M && tile < end && n < w.n_out) {
        const long long at = (long long)(m0 + m) * w.n_out + n;
        if (DUAL) {
          const float lo = static_cast<const float*>(p.a)[at], up = p.b[at];
          v[0][m] = lo + up;
          v[SETS - 1][m] = up - lo;
        } else {
          v[0][m] = load_any(p.a, p.type, at);
        }
      }
    }
  };

  int next = first + warp;
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) {
    if (next < end) load_stage(w, pitch, groups, ring + s * STAGE_BYTES, next * TILE_N, kb, lane);
    copies_begin();
    next += WARPS;
  }
  float av[SETS][MT];
  rows_at(first + warp, av);
  int slot = 0;
  for (int tile = first + warp; tile < end; tile += WARPS) {
    float now[SETS][MT];
#pragma unroll
    for (int s = 0; s < SETS; ++s)
#pragma unroll
      for (int m = 0; m < MT; ++m) now[s][m] = av[s][m];
    rows_at(tile + WARPS, av);
    copies_wait<STAGES - 2>();
    __syncwarp();
    {
      const int free_slot = slot == 0 ? STAGES - 1 : slot - 1;
      if (next < end) load_stage(w, pitch, groups, ring + free_slot * STAGE_BYTES, next * TILE_N, kb, lane);
      copies_begin();
      next += WARPS;
    }
    const uint32_t st = ring + slot * STAGE_BYTES;
    slot = slot == STAGES - 1 ? 0 : slot + 1;
#pragma unroll
    for (int step = 0; step < 4; ++step) {
      if (step % steps == 0) {  // a group begins: its rows
        const float scale = __uint_as_float(lds32(st + TILE_N * ROW_BYTES + ((step / steps) * TILE_N + lane) * 4));
        __syncwarp();
#pragma unroll
        for (int s = 0; s < SETS; ++s) {
          const float f = s == 0 ? scale : fabsf(scale);
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            if (m < M) {
              uint32_t q[3];
              parts_of(now[s][m] * f, sp.parts, q);
#pragma unroll
              for (int part = 0; part < 3; ++part)
                if (part < sp.parts) {
                  const int col = packed ? m * sp.parts + part : (m & 7), tq = packed ? 0 : part * NT + (m >> 3);
                  const uint32_t dst = as + s * set_bytes + ((tq * cv + col) * 32 + place) * 2;
                  asm volatile("st.shared.b16 [%0], %1;" ::"r"(dst), "h"((unsigned short)q[part]) : "memory");
                }
            }
          }
        }
        __syncwarp();
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t row = st + (h * 16 + 2 * t) * ROW_BYTES + (step * 4 + (g & 3)) * 4;
        const uint32_t w0 = lds32(row), w1 = lds32(row + ROW_BYTES), w8 = lds32(row + 8 * ROW_BYTES), w9 = lds32(row + 9 * ROW_BYTES);
        const uint32_t sel = g >= 4 ? 0x7632u : 0x5410u;
        const uint32_t lo = __byte_perm(w0, w1, sel), hi = __byte_perm(w8, w9, sel);
        uint32_t b[SETS][Q][2];
#pragma unroll
        for (int s = 0; s < SETS; ++s)
#pragma unroll
          for (int q = 0; q < Q; ++q) {
            b[s][q][0] = b[s][q][1] = 0;
            if (g < cv)
              asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(b[s][q][0]), "=r"(b[s][q][1]) : "r"(as + s * set_bytes + ((q * cv + g) * 32 + h * 16 + 4 * t) * 2) : "memory");
          }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          uint32_t a[4] = {weights_of(lo >> (8 * e)), weights_of(lo >> (8 * e + 4)), weights_of(hi >> (8 * e)), weights_of(hi >> (8 * e + 4))};
#pragma unroll
          for (int q = 0; q < Q; ++q) mma(acc[0][step][e][q % NT], a[0], a[1], a[2], a[3], b[0][q][0], b[0][q][1]);
          if (DUAL) {
#pragma unroll
            for (int i = 0; i < 4; ++i) a[i] &= 0x7fff7fffu;
#pragma unroll
            for (int q = 0; q < Q; ++q) mma(acc[SETS - 1][step][e][q % NT], a[0], a[1], a[2], a[3], b[SETS - 1][q][0], b[SETS - 1][q][1]);
          }
        }
      }
    }
  }
  // Sums over the warps, eight columns of rows at a time, then over the blocks of the cluster, each in order.
  float* red = reinterpret_cast<float*>(smem);                    // [warp][128][8]
  float* part = red + WARPS * CHUNK * 8;                          // [set, tile][128][8]
  copies_wait<0>();
#pragma unroll
  for (int s = 0; s < SETS; ++s)
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      __syncthreads();
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            red[(warp * CHUNK + r * 32 + 8 * (g & 3) + 4 * (g >> 2) + 2 * e + (i >> 1)) * 8 + 2 * t + (i & 1)] = acc[s][r][e][j][i];
      __syncthreads();
      for (int i = threadIdx.x; i < CHUNK * 8; i += THREADS) {
        float v = red[i];
#pragma unroll
        for (int k = 1; k < WARPS; ++k) v += red[k * CHUNK * 8 + i];
        part[(s * NT + j) * CHUNK * 8 + i] = v;
      }
    }
  if (sp.cluster > 1) cluster_barrier();
  else __syncthreads();
  const int mine = CHUNK / sp.cluster;
  for (int i = threadIdx.x; i < mine * M; i += THREADS) {
    const int m = i / mine, k = rank * mine + i - m * mine;
    if (kb * CHUNK + k >= w.n_in) continue;
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int s = 0; s < SETS; ++s) {
      const int count = packed ? sp.parts : 1;
      for (int q = 0; q < count; ++q) {
        const int col = packed ? m * sp.parts + q : (m & 7);
        const float* at = part + ((s * NT + (packed ? 0 : m >> 3)) * CHUNK + k) * 8 + col;
        float v = 0.f;
        if (sp.cluster == 1) v = *at;
        else
          for (int c = 0; c < sp.cluster; ++c) v += cluster_read(at, c);
        sum[s] += v;
      }
    }
    const long long at = (long long)(m0 + m) * w.n_in + kb * CHUNK + k;
    if (DUAL) {
      static_cast<float*>(p.z)[at] = 0.5f * (sum[0] - sum[1]);
      p.z2[at] = 0.5f * (sum[0] + sum[1]);
    } else {
      store_any(p.z, p.type, at, sum[0]);
    }
  }
  if (sp.cluster > 1) cluster_barrier();
}

template <typename Args>
int launch_clustered(void (*kernel)(Args, Split), const char* name, SmemOptIn& table, const Args& p, const Split& sp, long long blocks, int tiles_m, int smem,
                     cudaStream_t stream) {
  const int rc = ensure_dynamic_smem(kernel, smem, table, name);
  if (rc != BF_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks, tiles_m);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)sp.cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = sp.cluster > 1 ? 1 : 0;
  (void)cudaLaunchKernelEx(&cfg, kernel, p, sp);
  BF_CHECK_LAUNCH(name);
  return BF_OK;
}

int power_below(int v) {
  int p = 1;
  while (2 * p <= v) p *= 2;
  return p;
}

template <int PARTS, int NT, bool DUAL>
int forward(const W4LinearArgs& p, Split sp, int tiles_m, cudaStream_t stream) {
  static SmemOptIn table;
  const int tiles_n = ceil_div(p.w.n_out, TILE_N), chunks = ceil_div(p.w.n_in, CHUNK);
  // 16 warps an SM: as many splits of the columns as give each a stage's work, within a block first, then over a cluster
  const long long units = (long long)tiles_n * tiles_m;
  const int split = (int)std::max<long long>(1, std::min<long long>(chunks, (16LL * SMS) / units));
  sp.kw = std::min(WARPS, power_below(split));
  const int cv = PARTS == 1 && NT == 1 ? sp.tile_m * sp.parts : (NT == 1 ? sp.tile_m : 8);
  const int chunk_bytes = 4 * (DUAL ? 2 : 1) * PARTS * NT * cv * 64;
  while (sp.kw * chunk_bytes > X_MOST) sp.kw /= 2;  // the warps of a block take a chunk each
  sp.cluster = std::min(8, power_below(std::max(1, split / sp.kw)));
  sp.per_phase = std::max(sp.kw, X_BYTES / chunk_bytes / sp.kw * sp.kw);
  const int share = ceil_div(chunks, sp.cluster);
  const int x_bytes = std::min(sp.per_phase, share) * chunk_bytes;
  const long long blocks = (long long)ceil_div(p.w.n_out, TILE_N * (WARPS / sp.kw)) * sp.cluster;
  return launch_clustered(w4_forward_kernel<PARTS, NT, DUAL>, "w4_forward_kernel", table, p, sp, blocks, tiles_m, RING_BYTES + x_bytes, stream);
}

template <int PARTS, int NT, bool DUAL>
int backward(const W4RowsArgs& p, Split sp, int tiles_m, cudaStream_t stream) {
  static SmemOptIn table;
  const int kblocks = ceil_div(p.w.n_in, CHUNK), tiles = ceil_div(p.w.n_out, TILE_N);
  const long long units = (long long)kblocks * tiles_m;
  const int split = (int)std::max<long long>(1, std::min<long long>(ceil_div(tiles, WARPS), (2LL * SMS) / units));
  sp.cluster = std::min(8, power_below(split));
  const int cv = PARTS == 1 ? sp.tile_m * sp.parts : (NT == 1 ? sp.tile_m : 8);
  const int rows_bytes = WARPS * (DUAL ? 2 : 1) * PARTS * NT * cv * 64;
  const int sums = (WARPS + (DUAL ? 2 : 1) * NT) * CHUNK * 8 * 4;
  return launch_clustered(w4_rows_kernel<PARTS, NT, DUAL>, "w4_rows_kernel", table, p, sp, (long long)kblocks * sp.cluster, tiles_m,
                          std::max(RING_BYTES + rows_bytes, sums), stream);
}

constexpr int MOST_TILES = 65535;  // of a grid's second axis

}  // namespace

int launch_w4_linear(const W4LinearArgs& all, cudaStream_t stream) {
  Split sp = {};
  sp.parts = all.type == BF_TYPE_F32 ? 3 : all.type == BF_TYPE_F16 ? 2 : 1;
  const bool dual = all.b != nullptr, side_by_side = all.M * sp.parts <= 8;
  const int nt = side_by_side || all.M <= 8 ? 1 : 2;
  sp.tile_m = std::min(all.M, 8 * nt);
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
      rc = side_by_side ? forward<1, 1, true>(p, sp, here, stream) : nt == 1 ? forward<3, 1, true>(p, sp, here, stream) : forward<3, 2, true>(p, sp, here, stream);
    else if (side_by_side) rc = forward<1, 1, false>(p, sp, here, stream);
    else if (sp.parts == 1) rc = forward<1, 2, false>(p, sp, here, stream);
    else if (sp.parts == 2) rc = nt == 1 ? forward<2, 1, false>(p, sp, here, stream) : forward<2, 2, false>(p, sp, here, stream);
    else rc = nt == 1 ? forward<3, 1, false>(p, sp, here, stream) : forward<3, 2, false>(p, sp, here, stream);
    if (rc != BF_OK) return rc;
  }
  return BF_OK;
}

int launch_w4_rows(const W4RowsArgs& all, cudaStream_t stream) {
  Split sp = {};
  sp.parts = all.type == BF_TYPE_F32 ? 3 : 2;  // a 16-bit row times a 32-bit scale: two parts hold it to 2^-18
  const bool dual = all.b != nullptr, side_by_side = all.M * sp.parts <= 8;
  const int nt = dual || side_by_side || all.M <= 8 ? 1 : 2;
  sp.tile_m = std::min(all.M, 8 * nt);
  const long long tiles = ceil_div(all.M, sp.tile_m);
  for (long long first = 0; first < tiles; first += MOST_TILES) {
    const int here = (int)std::min<long long>(MOST_TILES, tiles - first);
    W4RowsArgs p = all;
    const long long skip = first * sp.tile_m, size = all.type == BF_TYPE_F32 ? 4 : 2;
    p.M = (int)std::min<long long>(all.M - skip, (long long)here * sp.tile_m);
    p.a = static_cast<const char*>(all.a) + skip * all.w.n_out * size;
    p.b = dual ? all.b + skip * all.w.n_out : nullptr;
    p.z = static_cast<char*>(all.z) + skip * all.w.n_in * size;
    p.z2 = dual ? all.z2 + skip * all.w.n_in : nullptr;
    int rc;
    if (dual) rc = side_by_side ? backward<1, 1, true>(p, sp, here, stream) : backward<3, 1, true>(p, sp, here, stream);
    else if (side_by_side) rc = backward<1, 1, false>(p, sp, here, stream);
    else if (sp.parts == 2) rc = nt == 1 ? backward<2, 1, false>(p, sp, here, stream) : backward<2, 2, false>(p, sp, here, stream);
    else rc = nt == 1 ? backward<3, 1, false>(p, sp, here, stream) : backward<3, 2, false>(p, sp, here, stream);
    if (rc != BF_OK) return rc;
  }
  return BF_OK;
}

}  // namespace bf
