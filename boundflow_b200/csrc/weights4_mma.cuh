// The parts that both products of 4-bit weights are made of: how codes, scales and rows come to the warp-level tensor-core
// instruction (m16n8k16, bfloat16 in, fp32 sums).
//
// The codes are what has to be read: half a byte a weight, so that at 6.5 TB/s 13 thousand million weights a millisecond pass and a
// multiplication in FP32 registers (convert, scale, multiply-add for every row) would bound the kernel instead.  A code minus 8 is exact in bfloat16:
// `weights_of` makes two of them from a word with three operations, and the rows go in as sums of bfloat16 parts, which hold a
// 32-bit number exactly (8 + 8 + 8 bits), a 16-bit one in one part (bf16) or two (fp16).  So every product is exact and only the sums round.  The rows are
// the instruction's 8 columns: parts side by side where that takes fewer instructions, else one instruction for each part and 8 rows.  The 128-row
// tiles of the tcgen05 instructions would take operands through shared memory: 2 bytes a weight written and read there
// where these kernels move half a byte, for rows that fill an eighth of the instruction's smallest tile; for many rows that is what weights4_many.cu does.
//
// Codes and scales come by cp.async into a ring of each warp's own (no barrier between warps), 32 rows x 128 columns a stage.
#pragma once
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
constexpr int SMS = 148;
constexpr int MOST_TILES = 65535;                  // of a grid's second axis

__device__ __forceinline__ uint32_t smem_of(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t to, const void* from, bool valid) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(valid ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copies_begin() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same on sums of zero: no registers to clear.
__device__ __forceinline__ void mma_anew(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// Codes in the upper halves of the bytes, minus 8 and times 16, as four 8-bit numbers: the highest bit turned makes two's complement of them.
__device__ __forceinline__ uint32_t digits_of(uint32_t w) {
  uint32_t v;
  asm("lop3.b32 %0, %1, %2, %3, 0x6A;" : "=r"(v) : "r"(w), "r"(0xf0f0f0f0u), "r"(0x80808080u));
  return v;
}
__device__ __forceinline__ void mma_digits(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Bit patterns of two numbers to the words (first, second) of their bfloat16 parts: three parts of 8 bits, or two, the second rounded to the nearest.
// Infinities and NaN are one part.
__device__ __forceinline__ void one_number(float v, int parts, uint32_t (&p)[3]) {
  const uint32_t bits = __float_as_uint(v);
  if ((bits & 0x7fffffffu) >= 0x7f800000u) {
    p[0] = (bits >> 16) | ((bits & 0x007fffffu) ? 0x40u : 0u);
    p[1] = p[2] = 0;
  } else if (parts == 3) {
    p[0] = bits >> 16;
    const float r = v - __uint_as_float(bits & 0xffff0000u);
    p[1] = __float_as_uint(r) >> 16;
    p[2] = __float_as_uint(r - __uint_as_float(__float_as_uint(r) & 0xffff0000u)) >> 16;
  } else {
    p[0] = bits >> 16;  // (numbers that would round to infinity come here)
    p[1] = __bfloat16_as_ushort(__float2bfloat16(v - __uint_as_float(bits & 0xffff0000u)));
    p[2] = 0;
  }
}
template <int PARTS>
__device__ __forceinline__ void two_numbers(float a, float b, uint32_t (&p)[PARTS]) {
  if (PARTS == 3) {
    const float ra = a - __uint_as_float(__float_as_uint(a) & 0xffff0000u), rb = b - __uint_as_float(__float_as_uint(b) & 0xffff0000u);
    const float qa = ra - __uint_as_float(__float_as_uint(ra) & 0xffff0000u), qb = rb - __uint_as_float(__float_as_uint(rb) & 0xffff0000u);
    p[0] = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
    p[PARTS > 1 ? 1 : 0] = __byte_perm(__float_as_uint(ra), __float_as_uint(rb), 0x7632);
    p[PARTS > 2 ? 2 : 0] = __byte_perm(__float_as_uint(qa), __float_as_uint(qb), 0x7632);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    const float2 f = __bfloat1622float2(h);
    const __nv_bfloat162 l = __floats2bfloat162_rn(a - f.x, b - f.y);
    p[0] = *reinterpret_cast<const uint32_t*>(&h);
    p[PARTS > 1 ? 1 : 0] = *reinterpret_cast<const uint32_t*>(&l);
  }
}
template <int PARTS>
__device__ __forceinline__ void two_numbers_checked(float a, float b, uint32_t (&p)[PARTS]) {
  float top;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(top) : "f"(fabsf(a)), "f"(fabsf(b)));
  if (top < (PARTS == 3 ? __int_as_float(0x7f800000) : 3.3e38f)) {
    two_numbers<PARTS>(a, b, p);
  } else {  // one of them is an infinity or a NaN, or rounds to one
    uint32_t x[3], y[3];
    one_number(a, PARTS, x);
    one_number(b, PARTS, y);
#pragma unroll
    for (int i = 0; i < PARTS; ++i) p[i] = x[i] | (y[i] << 16);
  }
}

// How the work is split over blocks.
struct Split {
  int packed;     // parts of a row side by side in the instruction's columns
  int kw;         // forward: warps of a block that share rows and split columns
  int rw;         // forward: row tiles of a block (kw * rw warps)
  int cluster;    // blocks that split the columns (forward) or the outputs (rows)
  int kw_log2, cluster_log2;
  int per_phase;  // forward: chunks whose parts are in shared memory at a time
  int tile_m;     // rows of a block
  int inbox;      // forward: bytes of the sums that come from the warps that split the columns
  unsigned mine_inverse;  // forward: 2^32 over the rows that a block finishes
};

// Lanes copy a stage: codes [32 rows][64 bytes], scales of the chunk's groups.  `codes` is the lane's first 16 bytes (row lane / 4, piece lane % 4),
// `rows` how many of the tile's rows there are, `bytes` how many of the 64 lie within the codes' rows; `safe` stands for what is not there.
__device__ __forceinline__ void load_codes(uint32_t to, const uint8_t* codes, const uint8_t* safe, long long pitch8, int rows, int bytes, int lane) {
  const int row = lane >> 2, piece = (lane & 3) * 16;
  const uint32_t dst = to + row * ROW_BYTES + piece;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const bool ok = row + 8 * j < rows && piece < bytes;
    copy16(dst + j * 8 * ROW_BYTES, ok ? codes + j * pitch8 : safe, ok);
  }
}
__device__ __forceinline__ void load_scales(uint32_t to, const W4& w, int groups, int n0, int chunk, int lane) {
  const int in_chunk = w.group_log2 >= 7 ? 1 : CHUNK >> w.group_log2;
  const int g0 = w.group_log2 >= 7 ? chunk >> (w.group_log2 - 7) : chunk << (7 - w.group_log2);
  const bool ok = n0 + lane < w.n_out;
  const float* from = w.scales + (long long)g0 * w.n_out + (ok ? n0 + lane : 0);
  for (int i = 0; i < in_chunk; ++i) copy4(to + TILE_N * ROW_BYTES + (i * TILE_N + lane) * 4, g0 + i < groups ? from + (long long)i * w.n_out : w.scales, ok && g0 + i < groups);
}

__device__ __forceinline__ uint32_t lds32(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t cluster_address(uint32_t at, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(at), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_store(uint32_t at, float v, bool cluster) {
  if (cluster) asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at), "f"(v) : "memory");
  else asm volatile("st.shared.f32 [%0], %1;" ::"r"(at), "f"(v) : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

template <typename Args>
int launch_clustered(void (*kernel)(Args, Split), const char* name, SmemOptIn& table, const Args& p, const Split& sp, long long blocks, int tiles_m, int threads,
                     int smem, cudaStream_t stream) {
  // (the most that any call asks for: with each call's own size, the limit of a first call could be lowered by that of another thread's before its launch)
  const int rc = ensure_dynamic_smem(kernel, 227 * 1024, table, name);
  if (rc != BF_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks, tiles_m);
  cfg.blockDim = dim3(threads);
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

int log2_of(int v) {
  int l = 0;
  while ((1 << l) < v) ++l;
  return l;
}
int power_below(int v) {
  int p = 1;
  while (2 * p <= v) p *= 2;
  return p;
}

}  // namespace
}  // namespace bf
