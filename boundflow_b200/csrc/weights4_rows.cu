// z = a W for few rows a and 4-bit weights, and the gradients of interval bounds (W and |W|); weights4_mma.cuh says how.
#include "weights4_mma.cuh"

namespace bf {
namespace {

// A block takes 128 columns and (with its cluster) splits the outputs over its warps, 32 at a time.  The scale belongs to the sum's index here, so it goes
// into the rows: a[m, n] * scale[group, n], rounded to 32 bits and split into parts, by each warp for the outputs it reads.
// Columns are the instruction's rows: lane (g, t) takes half a word (four columns) of each of the outputs 2t, 2t + 1, 2t + 8, 2t + 9.
//
// Measured (B200): nine fp32 rows back through 4096 x 4096 12.0 us, 16 bf16 rows through 8192 x 4096 18.1, one bf16 row through 16384 x 16384 48 us (2.9 TB/s).  With more than a
// row or two the tensor cores are 41% and the issue slots 49% busy with 16 warps an SM; with one row the parts, which each warp makes for every 32 outputs, and four
// loads of shared memory for 1024 codes bound it.
//
// The matrix instruction truncates what it adds to, always in the same direction: sums that stay in it over 192 instructions are off by 7e-6 where all terms are positive.  Three and more fp32 rows
// end them after at most MOST_IN_ONE outputs times 32, by more blocks or (SHORT) by an addition in 32 bits after every 32 outputs; `backward` chooses.  (16-bit rows do not: their results
// are rounded to 2^-9 or 2^-12.)
//
// P parts of a row, side by side (PACKED, one tile) or an instruction each for NT tiles of 8 rows; STEPS of 32 columns share a scale (1, 2, or 4 and more).
constexpr int MOST_IN_ONE = 8;
template <int P, bool PACKED, int NT, bool DUAL, int STEPS, bool SHORT>
__global__ void __launch_bounds__(THREADS, 2) w4_rows_kernel(const W4RowsArgs p, const Split sp) {
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr int Q = PACKED ? 1 : P * NT, SETS = DUAL ? 2 : 1;
  constexpr int MT = PACKED ? 8 / P : 8 * NT;   // most rows of a block
  constexpr int TURNS = (MT + 1) / 2;           // rows of a half warp
  const W4 w = p.w;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int rank = blockIdx.x & (sp.cluster - 1), kb = blockIdx.x >> sp.cluster_log2;  // (cluster is a power of two)
  const int m0 = blockIdx.y * sp.tile_m, M = min(sp.tile_m, p.M - m0);
  const int cv = PACKED ? M * P : (NT == 1 ? M : 8);
  const int tiles = (w.n_out + TILE_N - 1) / TILE_N, share = (tiles + sp.cluster - 1) >> sp.cluster_log2;
  const int first = min(rank * share, tiles), end = min(first + share, tiles);
  const int groups = w.groups();
  const long long pitch = w.pitch();
  const uint32_t inbox = smem_of(smem) + RING_BYTES + WARPS * (SETS * Q * cv * 64), ring = smem_of(smem) + warp * (STAGES * STAGE_BYTES);
  if (sp.cluster > 1) cluster_arrive();  // (before the sums go out all blocks of the cluster have to be there)
  const int set_bytes = Q * cv * 64;
  const uint32_t as = smem_of(smem) + RING_BYTES + warp * (SETS * set_bytes);  // [set][part, tile][column][32 outputs, in the order the lanes read them]
  // a lane makes the parts of two neighbouring outputs of every other row
  const int pair = lane & 15, odd = lane >> 4, in8 = pair & 7;
  const uint32_t place = as + ((pair >> 3) * 16 + (in8 & 3) * 4 + (in8 >> 2) * 2) * 2;
  const int size = p.type == BF_TYPE_F32 ? 4 : 2;
  const bool wide = w.n_out % 2 == 0 && (((uintptr_t)p.a | (uintptr_t)p.b) & (2 * size - 1)) == 0;
  const int bytes = (int)min((long long)CHUNK, pitch - (long long)kb * (CHUNK / 2));
  const uint8_t* codes = w.codes + (long long)kb * (CHUNK / 2) + min((lane & 3) * 16, bytes - 16);

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

  // (as they lie in memory: a conversion here would wait for each load in turn)
  constexpr int WORDS = P == 3 ? 2 : 1;
  auto rows_at = [&](int tile, uint32_t (&v)[SETS][TURNS][WORDS]) {
    const int n = tile * TILE_N + 2 * pair;
    const bool here = tile < end && n < w.n_out, two = n + 1 < w.n_out;
#pragma unroll
    for (int i = 0; i < TURNS; ++i) {
      const int m = 2 * i + odd;
#pragma unroll
      for (int s = 0; s < SETS; ++s) {
        v[s][i][0] = v[s][i][WORDS - 1] = 0;
        if (m < M && here) {
          const long long at = (long long)(m0 + m) * w.n_out + n;
          if (P == 3) {
            const uint32_t* from = reinterpret_cast<const uint32_t*>(s == 0 ? static_cast<const float*>(p.a) : p.b) + at;
            if (wide) {
              const uint2 f = *reinterpret_cast<const uint2*>(from);
              v[s][i][0] = f.x;
              v[s][i][WORDS - 1] = f.y;
            } else {
              v[s][i][0] = from[0];
              if (two) v[s][i][WORDS - 1] = from[1];
            }
          } else {
            const uint16_t* from = static_cast<const uint16_t*>(p.a) + at;
            if (wide) v[0][i][0] = *reinterpret_cast<const uint32_t*>(from);
            else v[0][i][0] = from[0] | (two ? (uint32_t)from[1] << 16 : 0u);
          }
        }
      }
    }
  };
  auto numbers = [&](const uint32_t (&v)[WORDS]) {
    if (P == 3) return make_float2(__uint_as_float(v[0]), __uint_as_float(v[WORDS - 1]));
    if (p.type == BF_TYPE_BF16) return make_float2(__uint_as_float(v[0] << 16), __uint_as_float(v[0] & 0xffff0000u));
    return __half22float2(*reinterpret_cast<const __half2*>(&v[0]));
  };

  uint32_t av[SETS][TURNS][WORDS];
  rows_at(first + warp, av);  // before the codes, which would keep these waiting for the memory's first microsecond
  int next = first + warp;
  auto load_next = [&](uint32_t to) {
    if (next < end) {
      const int n0 = next * TILE_N, rows = min(TILE_N, w.n_out - n0);
      const uint8_t* from = codes + (long long)(n0 + min(lane >> 2, rows - 1)) * pitch;
      load_codes(to, from, from, 8 * pitch, rows, bytes, lane);
      load_scales(to, w, groups, n0, kb, lane);
    }
    copies_begin();
    next += WARPS;
  };
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) load_next(ring + s * STAGE_BYTES);
  int slot = 0;
  for (int tile = first + warp; tile < end; tile += WARPS) {
    float2 now[SETS][TURNS];
#pragma unroll
    for (int i = 0; i < TURNS; ++i) {
      now[0][i] = numbers(av[0][i]);
      if (DUAL) {  // gradients of lower and upper bounds to those of centre and radius
        const float2 lo = now[0][i], up = numbers(av[SETS - 1][i]);
        now[0][i] = make_float2(lo.x + up.x, lo.y + up.y);
        now[SETS - 1][i] = make_float2(up.x - lo.x, up.y - lo.y);
      }
    }
    rows_at(tile + WARPS, av);
    copies_wait<STAGES - 2>();
    __syncwarp();
    load_next(ring + (slot == 0 ? STAGES - 1 : slot - 1) * STAGE_BYTES);
    const uint32_t st = ring + slot * STAGE_BYTES;
    slot = slot == STAGES - 1 ? 0 : slot + 1;
#pragma unroll
    for (int group = 0; group < 4 / STEPS; ++group) {
      {
        const uint32_t at = st + TILE_N * ROW_BYTES + (group * TILE_N + 2 * pair) * 4;
        const float f0 = __uint_as_float(lds32(at)), f1 = __uint_as_float(lds32(at + 4));
        if (group > 0) __syncwarp();
#pragma unroll
        for (int i = 0; i < TURNS; ++i) {
          const int m = 2 * i + odd;
          if (m < M) {
#pragma unroll
            for (int s = 0; s < SETS; ++s) {
              uint32_t q[P];
              two_numbers_checked<P>(now[s][i].x * (s == 0 ? f0 : fabsf(f0)), now[s][i].y * (s == 0 ? f1 : fabsf(f1)), q);
#pragma unroll
              for (int part = 0; part < P; ++part) {
                const int j = PACKED ? m * P + part : part * NT * cv + m;  // column, counted through the tiles
                asm volatile("st.shared.b32 [%0], %1;" ::"r"(place + s * set_bytes + j * 64), "r"(q[part]) : "memory");
              }
            }
          }
        }
        __syncwarp();
      }
      auto load_b = [&](int h, uint32_t (&b)[SETS][Q][2]) {
#pragma unroll
        for (int s = 0; s < SETS; ++s)
#pragma unroll
          for (int q = 0; q < Q; ++q)
            asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];"
                         : "=r"(b[s][q][0]), "=r"(b[s][q][1])
                         : "r"(as + s * set_bytes + ((q * cv + min(g, cv - 1)) * 32 + h * 16 + 4 * t) * 2)
                         : "memory");
      };
      // Codes of 32 columns and 16 outputs: lo, hi as the instruction takes them.
      auto load_codes_of = [&](int h, int step, uint32_t& lo, uint32_t& hi) {
        const uint32_t row = st + (h * 16 + 2 * t) * ROW_BYTES + (step * 4 + (g & 3)) * 4;
        const uint32_t w0 = lds32(row), w1 = lds32(row + ROW_BYTES), w8 = lds32(row + 8 * ROW_BYTES), w9 = lds32(row + 9 * ROW_BYTES);
        const uint32_t sel = g >= 4 ? 0x7632u : 0x5410u;
        lo = __byte_perm(w0, w1, sel);
        hi = __byte_perm(w8, w9, sel);
      };
      auto weights = [&](uint32_t lo, uint32_t hi, int e, uint32_t (&a)[4]) {
        a[0] = weights_of(lo >> (8 * e));
        a[1] = weights_of(lo >> (8 * e + 4));
        a[2] = weights_of(hi >> (8 * e));
        a[3] = weights_of(hi >> (8 * e + 4));
      };
      if constexpr (SHORT) {
        uint32_t b[2][SETS][Q][2];
        load_b(0, b[0]);
        load_b(1, b[1]);
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
          const int step = group * STEPS + i;
          uint32_t lo[2], hi[2];
          load_codes_of(0, step, lo[0], hi[0]);
          load_codes_of(1, step, lo[1], hi[1]);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int s = 0; s < SETS; ++s) {
              float sum[NT][4];
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                uint32_t a[4];
                weights(lo[h], hi[h], e, a);
                if (s == 1) {
#pragma unroll
                  for (int k = 0; k < 4; ++k) a[k] &= 0x7fff7fffu;
                }
#pragma unroll
                for (int q = 0; q < Q; ++q) {
                  if (h == 0 && q < NT) mma_anew(sum[q % NT], a[0], a[1], a[2], a[3], b[h][s][q][0], b[h][s][q][1]);
                  else mma(sum[q % NT], a[0], a[1], a[2], a[3], b[h][s][q][0], b[h][s][q][1]);
                }
              }
#pragma unroll
              for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int k = 0; k < 4; ++k) acc[s][step][e][j][k] += sum[j][k];
            }
          }
        }
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t b[SETS][Q][2];
          load_b(h, b);
#pragma unroll
          for (int i = 0; i < STEPS; ++i) {
            const int step = group * STEPS + i;
            uint32_t lo, hi;
            load_codes_of(h, step, lo, hi);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              uint32_t a[4];
              weights(lo, hi, e, a);
#pragma unroll
              for (int q = 0; q < Q; ++q) mma(acc[0][step][e][q % NT], a[0], a[1], a[2], a[3], b[0][q][0], b[0][q][1]);
              if (DUAL) {
#pragma unroll
                for (int k = 0; k < 4; ++k) a[k] &= 0x7fff7fffu;
#pragma unroll
                for (int q = 0; q < Q; ++q) mma(acc[SETS - 1][step][e][q % NT], a[0], a[1], a[2], a[3], b[SETS - 1][q][0], b[SETS - 1][q][1]);
              }
            }
          }
        }
      }
    }
  }
  // Sums over the warps, eight columns at a time, go to the block of the cluster that finishes the input features, [product, row][block][feature]; the sums over
  // the blocks are taken there, each in a fixed order.
  constexpr int LINE = CHUNK + 4;
  float* red = reinterpret_cast<float*>(smem);  // [warp][8][128 and a pad]
  const int each_log2 = 7 - sp.cluster_log2, mine = 1 << each_log2;
  copies_wait<0>();
  if (sp.cluster > 1) cluster_wait();
  const int feature = threadIdx.x & (CHUNK - 1), owner = feature >> each_log2;
  uint32_t out = inbox + ((rank << each_log2) + feature - (owner << each_log2)) * 4;
  if (sp.cluster > 1) out = cluster_address(out, owner);
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
            red[(warp * 8 + 2 * t + (i & 1)) * LINE + r * 32 + 8 * (g & 3) + 4 * (g >> 2) + 2 * e + (i >> 1)] = acc[s][r][e][j][i];
      __syncthreads();
      const int here = PACKED ? M : min(8, M - j * 8);  // rows of the tile
      for (int m = threadIdx.x >> 7; m < here; m += THREADS / CHUNK) {
        float v = 0.f;
#pragma unroll
        for (int q = 0; q < (PACKED ? P : 1); ++q)
#pragma unroll
          for (int x = 0; x < WARPS; ++x) v += red[(x * 8 + (PACKED ? m * P + q : m)) * LINE + feature];
        cluster_store(out + (s * M + j * 8 + m) * CHUNK * 4, v, sp.cluster > 1);
      }
    }
  if (sp.cluster > 1) cluster_barrier();
  else __syncthreads();
  const float* box = reinterpret_cast<const float*>(smem + (inbox - smem_of(smem)));
  for (int i = threadIdx.x; i < M << each_log2; i += THREADS) {
    const int m = i >> each_log2, k = (rank << each_log2) + (i & (mine - 1));
    if (kb * CHUNK + k >= w.n_in) continue;
    float sum[2];
#pragma unroll
    for (int s = 0; s < SETS; ++s) {
      const float* at = box + (s * M + m) * CHUNK + (i & (mine - 1));
      float v[4] = {0.f, 0.f, 0.f, 0.f};
      if (sp.cluster < 4) {
        for (int c = 0; c < sp.cluster; ++c) v[0] += at[c << each_log2];
      } else {
        for (int c = 0; c < sp.cluster; c += 4) {
#pragma unroll
          for (int x = 0; x < 4; ++x) v[x] += at[(c + x) << each_log2];
        }
      }
      sum[s] = (v[0] + v[1]) + (v[2] + v[3]);
    }
    const long long at = (long long)(m0 + m) * w.n_in + kb * CHUNK + k;
    if (DUAL) {
      static_cast<float*>(p.z)[at] = 0.5f * (sum[0] - sum[1]);
      p.z2[at] = 0.5f * (sum[0] + sum[1]);
    } else {
      store_any(p.z, p.type, at, sum[0]);
    }
  }
}

template <int P, bool PACKED, int NT, bool DUAL, bool SHORT>
int launch_groups(const W4RowsArgs& p, const Split& sp, long long blocks, int tiles_m, int smem, cudaStream_t stream) {
  static SmemOptIn table[3];
  if (p.w.group_log2 == 5) return launch_clustered(w4_rows_kernel<P, PACKED, NT, DUAL, 1, SHORT>, "w4_rows_kernel", table[0], p, sp, blocks, tiles_m, THREADS, smem, stream);
  if (p.w.group_log2 == 6) return launch_clustered(w4_rows_kernel<P, PACKED, NT, DUAL, 2, SHORT>, "w4_rows_kernel", table[1], p, sp, blocks, tiles_m, THREADS, smem, stream);
  return launch_clustered(w4_rows_kernel<P, PACKED, NT, DUAL, 4, SHORT>, "w4_rows_kernel", table[2], p, sp, blocks, tiles_m, THREADS, smem, stream);
}
template <int P, bool PACKED, int NT, bool DUAL>
int backward(const W4RowsArgs& p, Split sp, int tiles_m, cudaStream_t stream) {
  const int kblocks = ceil_div(p.w.n_in, CHUNK), tiles = ceil_div(p.w.n_out, TILE_N);
  const long long units = (long long)kblocks * tiles_m;
  const int split = (int)std::max<long long>(1, std::min<long long>(ceil_div(tiles, WARPS), (2LL * SMS) / units));
  sp.cluster = std::min(8, power_below(split));
  // Long sums of fp32 rows (not of one or two, whose parts have columns of their own: 40000 terms are within 1.3e-7).  Up to eight rows the additions are cheap (16384 x 16384, us: eight
  // 69.9 -> 75.9, with four times the blocks 81.7).  More rows
  // and pairs have no registers left for them, and are split over more blocks where 8 of those suffice (16384 x 16384: 16 rows 117 -> 133, with additions 144; 64 rows 445 -> 494, 549;
  // 8192 x 4096: 64 rows 61.9 -> 67.7, 73.8; pairs of 48 125 -> 105, 146).
  constexpr bool CHEAP = NT == 1 && !DUAL;
  bool additions = false;
  if (P == 3 && !PACKED) {
    while (!CHEAP && sp.cluster < 8 && ceil_div(tiles, WARPS * sp.cluster) > MOST_IN_ONE) sp.cluster *= 2;
    additions = ceil_div(tiles, WARPS * sp.cluster) > MOST_IN_ONE;
  }
  sp.cluster_log2 = log2_of(sp.cluster);
  const int cv = PACKED ? sp.tile_m * P : (NT == 1 ? sp.tile_m : 8);
  const int rows_bytes = WARPS * (DUAL ? 2 : 1) * (PACKED ? 1 : P * NT) * cv * 64;
  const int smem = RING_BYTES + rows_bytes + (DUAL ? 2 : 1) * sp.tile_m * CHUNK * 4;  // ring (the sums over the warps at the end need less), parts, sums of the cluster
  const long long blocks = (long long)kblocks * sp.cluster;
  if constexpr (P == 3 && !PACKED) {
    if (additions) return launch_groups<P, PACKED, NT, DUAL, true>(p, sp, blocks, tiles_m, smem, stream);
  }
  return launch_groups<P, PACKED, NT, DUAL, false>(p, sp, blocks, tiles_m, smem, stream);
}

}  // namespace

int launch_w4_rows(const W4RowsArgs& all, cudaStream_t stream) {
  Split sp = {};
  const int parts = all.type == BF_TYPE_F32 ? 3 : 2;  // a 16-bit row times a 32-bit scale: two parts hold it to 2^-17
  const bool dual = all.b != nullptr;
  sp.packed = all.M * parts <= 8;
  const int nt = dual || sp.packed || all.M <= 8 ? 1 : 2;
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
    if (dual) rc = sp.packed ? backward<3, true, 1, true>(p, sp, here, stream) : backward<3, false, 1, true>(p, sp, here, stream);
    else if (sp.packed) rc = parts == 3 ? backward<3, true, 1, false>(p, sp, here, stream) : backward<2, true, 1, false>(p, sp, here, stream);
    else if (parts == 2) rc = nt == 1 ? backward<2, false, 1, false>(p, sp, here, stream) : backward<2, false, 2, false>(p, sp, here, stream);
    else rc = nt == 1 ? backward<3, false, 1, false>(p, sp, here, stream) : backward<3, false, 2, false>(p, sp, here, stream);
    if (rc != BF_OK) return rc;
  }
  return BF_OK;
}

}  // namespace bf
