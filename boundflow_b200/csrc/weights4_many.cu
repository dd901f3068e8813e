// Products of many rows with 4-bit weights on the 5th-generation tensor cores: y = x W^T + bias and z = a W, and the second product of interval bounds (|W|).
//
// With many rows the arithmetic bounds, and the weights unpacked for 256 of them cost less than the products.  The features (outputs of x W^T, columns of a W) are
// the accumulators' 128 lanes, the rows their columns (64, 128 or 256 of a block).  Eight warps unpack the weights of 64 summed indices into shared memory, one thread
// issues the products, and what the rows contribute lies ready in images of 64 columns by so many rows (swizzled as the tensor cores read them,
// w4_rows_images_kernel) that another fetches by bulk copies.
//
//   x W^T: codes minus 8 are exact in bfloat16, and so are the rows in one part (bf16), two (fp16) or three (fp32), as in weights4_mma.cuh.  The sum over the
//     columns that share a scale (at most 128 of them) is taken on the tensor cores, into one of two accumulators; from there the eight warps add it, times the scale,
//     to sums in their registers while the other is filled.
//   a W: the scale belongs to the summed index, so it goes into the weight: scale * (code - 8) as a sum of two bfloat16 numbers (16-bit rows: off by 2^-17 at most) or
//     three (fp32 rows), rounded to the nearest each.  All products of parts are taken beside 16-bit rows; beside fp32 rows six of nine, what is left out is below 2^-24 of the whole.  Tensor-memory accumulators truncate, by half a unit in the last
//     place of the running sum for every 16 terms of a product and always in the same direction, so a sum ends after `back_stages` and is added to the registers in the same way
//     (fp32 rows of 1024 to 65536 terms against 64 bits, 2-norm: 1.1e-6 to 1.2e-6; 8192 terms in one sum 5.3e-5, the FP32 kernel on the dense weight 5e-7 to 4e-6).  A weight's
//     second part would make NaN of a row's infinity, so where a stage's image holds numbers that are not finite (a bit says so) the image as it is meets the weights' first parts, and a
//     copy that the copying warp clears of them in shared memory meets the others.
//
// Waits are bounded: where one runs out, the block raises the status word, frees its tensor memory and stores NaN.
//
// Bounds and measurements (B200, images included).  4096 bf16 rows through 8192 x 4096: 319 us, 861 TFLOP/s (half of the measured rate of a library's plain product); fp32 rows, three
// products for one, 617 us (1340 TFLOP/s of bfloat16 products); back, bf16 616 us (two products: 892), fp16 794 (four), fp32 1387 to 1470 us (six: 1120 to 1190), 2.7 ms where every number is infinite.  Of a stage of x W^T with 256 bf16 rows (512 clocks of
// products) 950 clocks are taken: eight warps need 730 of them for their sums, unpacking 570, issuing 380; beginning and end of a block are another 5 us that nothing hides.  Back, three pairs unpack a
// stage in 1300 clocks and hold its slot meanwhile.  What was tried: the products issued by a thread that also unpacks (twice the time), by a thread chosen by its number instead of
// elect.sync (41 us for 64 rows, 31 now), sums back of one stage of fp32 rows (7e-7 off instead of 1.1e-6, 5 % slower), eight warps that both unpack and sum (528 us for 4096 rows, 319 now).
#include <math.h>

#include <algorithm>

#include "tc_primitives.cuh"
#include "weights4.cuh"

namespace bf {
namespace {

using namespace tc;

constexpr int LANES = 128;            // features of a block
constexpr int STEP = 64;              // summed indices of a stage: 128 bytes of bfloat16
constexpr int A_BYTES = LANES * STEP * 2;
// Warps: eight that sum, pairs that unpack a stage each in turn, one that copies, one that issues.  Launched with 128 registers a thread; the eight take 168 (they hold up
// to 128 sums), for which the others give up all but 80: 256 * 168 + 256 * 80 is within 512 * 128.
constexpr int SUMMERS = 8, TEAM = 64, COPIER = 14, ISSUER = 15, THREADS = 512;
__host__ __device__ constexpr int back_stages(int weight_parts) { return weight_parts == 3 ? 2 : 8; }  // of a sum of a W: 48 MMA steps (six products of parts), or 64 to 128 beside a result of 16 bits
constexpr int HEADER = 1024;          // of the workspace: the status word, then a bit for each tile of rows and 64 summed indices that hold a number that is not finite
constexpr int RING = 224 * 1024;

enum { TAKE_ROWS = 0, TAKE_CENTRE = 1, TAKE_RADIUS = 2, TAKE_SUM = 3, TAKE_DIFFERENCE = 4 };
__host__ __device__ constexpr int words_of(int steps) { return (steps + 31) / 32; }  // of the bits of a tile of rows

struct ManyArgs {
  W4 w;
  const uint8_t* images;
  const uint32_t* odd;  // a W: bits [row tile][step]
  const void* a;
  const float* b;
  const void* bias;
  void* out;
  float* out2;          // second pass of a pair (|W|): bounds or gradients of both ends from the first pass's result and this one's
  int type, bias_type, M, take, steps;
  int* status;
};

struct Control {
  unsigned long long a_full[4], a_empty[4], b_full[8], b_empty[8], d_full[2], d_empty[2], copied;
  uint32_t tmem;
  int abort_flag;
};

// One thread of a converged warp.  (The compiler knows that it is one: what the tensor cores' instructions take from uniform registers is then moved there without a loop over lanes.)
__device__ __forceinline__ bool elected() {
  uint32_t one;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(one));
  return one != 0;
}
// The products of a stage's four times 16 summed indices; `slice` is the step of A's descriptor.
template <int SLICE>
__device__ __forceinline__ void mma_step(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, one;\n\t.reg .b64 x, y;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.eq.b32 one, %5, %5;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t"
      "add.u64 x, %1, %6;\n\tadd.u64 y, %2, 2;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, {%5, %5, %5, %5}, one;\n\t"
      "add.u64 x, %1, %7;\n\tadd.u64 y, %2, 4;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, {%5, %5, %5, %5}, one;\n\t"
      "add.u64 x, %1, %8;\n\tadd.u64 y, %2, 6;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, {%5, %5, %5, %5}, one;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1u : 0u), "r"(0u),
      "n"(SLICE), "n"(2 * SLICE), "n"(3 * SLICE)
      : "memory");
}
__device__ __forceinline__ void mma_bf16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1u : 0u), "r"(0u)
      : "memory");
}
__device__ __forceinline__ uint32_t bits_of(__nv_bfloat162 v) { return *reinterpret_cast<const uint32_t*>(&v); }

// ---- images of the rows ----------------------------------------------------------------
struct ImageArgs {
  const void* a;
  const float* b;
  uint8_t* images;
  uint32_t* odd;
  int* status;
  int type, take, mode, relu_in, M, n, tile_m, steps;
};
// [row tile][64 columns][part][row of the tile][128 bytes, in eights, the eight e of row r in place e ^ (r % 8)].  FORWARD: the eights in the order 0 4 1 5 2 6 3 7 that
// `weights_of` gives the codes of a word in.  What is outside the rows is zero.  Eight columns of a row a thread.
template <int PARTS, bool FORWARD>
__global__ void __launch_bounds__(256) w4_rows_images_kernel(const ImageArgs p) {
  const long long row_eights = (long long)p.steps * 8, rows = (long long)((p.M + p.tile_m - 1) / p.tile_m) * p.tile_m, total = rows * row_eights;
  if (p.status && blockIdx.x == 0 && threadIdx.x == 0) *p.status = 0;
  const bool wide = p.n % 8 == 0 && ((reinterpret_cast<uintptr_t>(p.a) | reinterpret_cast<uintptr_t>(p.b)) & 15) == 0;
  for (long long i = blockIdx.x * 256LL + threadIdx.x; i < total; i += gridDim.x * 256LL) {
    const long long m = total < (1LL << 32) ? (long long)((unsigned)i / (unsigned)row_eights) : i / row_eights;
    const int eight = (int)(i - m * row_eights), n = eight * 8, r = (int)m & (p.tile_m - 1);  // (tiles of 64, 128 or 256)
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 0.f;
    if (m < p.M && n < p.n) {
      const long long at = m * p.n + n;
      if (p.type == BF_TYPE_F32) {
        const float *a = static_cast<const float*>(p.a) + at, *b = p.b + at;
        float u[8];
        if (wide) {
          *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(a);
          *reinterpret_cast<float4*>(v + 4) = *reinterpret_cast<const float4*>(a + 4);
          if (p.take != TAKE_ROWS) {
            *reinterpret_cast<float4*>(u) = *reinterpret_cast<const float4*>(b);
            *reinterpret_cast<float4*>(u + 4) = *reinterpret_cast<const float4*>(b + 4);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            v[j] = n + j < p.n ? a[j] : 0.f;
            u[j] = p.take != TAKE_ROWS && n + j < p.n ? b[j] : 0.f;
          }
        }
        if (p.take != TAKE_ROWS) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            float x = v[j], y = u[j];
            if (p.take == TAKE_CENTRE || p.take == TAKE_RADIUS) {
              if (p.mode == BF_IN_LOWER_UPPER) {
                if (p.relu_in) { x = x < 0.f ? 0.f : x; y = y < 0.f ? 0.f : y; }  // (a comparison with a NaN is false: it stays)
                v[j] = p.take == TAKE_CENTRE ? 0.5f * (x + y) : 0.5f * (y - x);
              } else {
                v[j] = p.take == TAKE_CENTRE ? x : y;
              }
            } else {
              v[j] = p.take == TAKE_SUM ? x + y : y - x;
            }
          }
        }
      } else if (wide) {
        const uint4 q = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.a) + at);
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f = p.type == BF_TYPE_BF16 ? __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[j])) : __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
          v[2 * j] = f.x;
          v[2 * j + 1] = f.y;
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = n + j < p.n ? load_any(p.a, p.type, at + j) : 0.f;
      }
    }
    uint32_t out[PARTS][4];
    bool strange = false, infinite = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      strange |= !(fabsf(v[j]) < 3.3e38f);  // (above that a number rounds to infinity)
      infinite |= !(fabsf(v[j]) < INFINITY);
    }
    if (!FORWARD && infinite) {
      uint32_t* word = p.odd + (long long)((unsigned)m >> (31 - __clz(p.tile_m))) * words_of(p.steps) + (eight >> 8);
      const uint32_t bit = 1u << ((eight >> 3) & 31);
      if ((*reinterpret_cast<volatile uint32_t*>(word) & bit) == 0) atomicOr(word, bit);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float x = FORWARD ? v[j] : v[2 * j], y = FORWARD ? v[j + 4] : v[2 * j + 1];
      const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
      out[0][j] = bits_of(h);
      if (PARTS > 1) {
        const float2 f = __bfloat1622float2(h);
        const float rx = x - f.x, ry = y - f.y;
        const __nv_bfloat162 l = __floats2bfloat162_rn(rx, ry);
        out[PARTS > 1 ? 1 : 0][j] = bits_of(l);
        if (PARTS > 2) {
          const float2 g = __bfloat1622float2(l);
          out[PARTS > 2 ? 2 : 0][j] = bits_of(__floats2bfloat162_rn(rx - g.x, ry - g.y));
        }
      }
    }
    if (PARTS > 1 && strange) {  // infinities and NaN are one part; the largest numbers are cut to theirs
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (fabsf(v[j]) < 3.3e38f) continue;
        uint16_t part[3] = {0, 0, 0};
        const uint32_t bits = __float_as_uint(v[j]);
        part[0] = (uint16_t)((bits >> 16) | ((bits & 0x7fffffffu) > 0x7f800000u ? 0x40u : 0u));
        if ((bits & 0x7fffffffu) < 0x7f800000u) {
          const float rest = v[j] - __uint_as_float(bits & 0xffff0000u);
          part[1] = (uint16_t)(__float_as_uint(rest) >> 16);
          part[2] = (uint16_t)(__float_as_uint(rest - __uint_as_float(__float_as_uint(rest) & 0xffff0000u)) >> 16);
        }
        const int word = FORWARD ? j & 3 : j >> 1, high = FORWARD ? j >> 2 : j & 1;
#pragma unroll
        for (int k = 0; k < PARTS; ++k) {
          const uint32_t keep = high ? 0x0000ffffu : 0xffff0000u;
#pragma unroll
          for (int x = 0; x < 4; ++x)
            if (x == word) out[k][x] = (out[k][x] & keep) | ((uint32_t)part[k] << (16 * high));
        }
      }
    }
    uint8_t* to = p.images + ((((long long)((unsigned)m >> (31 - __clz(p.tile_m)))) * p.steps + (eight >> 3)) * PARTS * p.tile_m + r) * 128 + (((eight & 7) ^ (r & 7)) << 4);
#pragma unroll
    for (int k = 0; k < PARTS; ++k) *reinterpret_cast<uint4*>(to + (long long)k * p.tile_m * 128) = make_uint4(out[k][0], out[k][1], out[k][2], out[k][3]);
  }
}

// ---- the products -----------------------------------------------------------------------
// XP parts of the rows, WP of the weights (1: x W^T), CW columns of the accumulators a warp (half of the block's rows), UNIT: steps of 32 columns that share a scale in
// x W^T (1, 2, or 4 and more).
template <int XP, int WP, int CW, int UNIT>
__global__ void __launch_bounds__(THREADS, 1) w4_many_kernel(const ManyArgs p) {
  constexpr bool FORWARD = WP == 1;
  constexpr int TM = 2 * CW, B_BYTES = TM * 128;
  constexpr int AS = FORWARD ? 4 : WP == 2 ? 3 : 2;                                                     // stages of weights
  constexpr int BS = (RING - AS * WP * A_BYTES) / B_BYTES > 8 ? 8 : (RING - AS * WP * A_BYTES) / B_BYTES;  // and of images
  // Pairs that unpack.  No more than stages: a pair that comes to stage h has seen stage h - TEAMS's slot free, so stage h - TEAMS - AS done; a phase of h's own slot could
  // pass for the one before it unless stage h - 2 AS is.
  constexpr int TEAMS = AS >= 3 ? 3 : 2;
  static_assert(BS >= XP && TEAMS <= AS, "the parts of a stage have to fit");
  extern __shared__ unsigned char raw_smem[];
  unsigned char* tiles = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw_smem) + 1024 + 1023) & ~(uintptr_t)1023);
  Control* ctl = reinterpret_cast<Control*>(tiles - 1024);
  const uint32_t a_ring = smem_u32(tiles), b_ring = a_ring + AS * WP * A_BYTES;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const W4 w = p.w;
  const int H = p.steps, m0 = blockIdx.y * TM, f0 = blockIdx.x * LANES;
  const int groups = w.groups();
  const long long pitch = w.pitch();
  volatile int* abort_flag = &ctl->abort_flag;
  const bool absolute = p.out2 != nullptr;

  if (tid == 0) {
    for (int s = 0; s < AS; ++s) {
      mbar_init(smem_u32(&ctl->a_full[s]), TEAM / 32);
      mbar_init(smem_u32(&ctl->a_empty[s]), 1);
    }
    for (int s = 0; s < BS; ++s) {
      mbar_init(smem_u32(&ctl->b_full[s]), 1);
      mbar_init(smem_u32(&ctl->b_empty[s]), 1);
    }
    mbar_init(smem_u32(&ctl->copied), 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(smem_u32(&ctl->d_full[s]), 1);
      mbar_init(smem_u32(&ctl->d_empty[s]), SUMMERS);
    }
    ctl->abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  constexpr uint32_t COLUMNS = 2 * TM < 128 ? 128 : 2 * TM;
  if (warp == ISSUER) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctl->tmem)), "r"(COLUMNS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ctl->tmem;
  constexpr int SPAN = !FORWARD ? back_stages(WP) : UNIT >= 4 ? 2 : 1;  // stages of a sum (x W^T with scales for 32 columns: half a stage)
  const int units = FORWARD && UNIT == 1 ? 2 * H : (H + SPAN - 1) / SPAN;

  const uint8_t* images = p.images + (long long)blockIdx.y * H * XP * B_BYTES;
  const uint32_t* odd = p.odd + (long long)blockIdx.y * words_of(H);
  if (warp >= SUMMERS) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    if (warp == COPIER) {
      // The numbers of a stage's image that are not finite, with zeros in their place: what the weights' later parts are multiplied by.
      auto clear = [&](uint32_t at) {
        for (int i = lane * 16; i < B_BYTES; i += 512) {
          uint32_t v[4];
          asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(at + i) : "memory");
          bool some = false;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t keep = ((v[j] & 0x7f80u) == 0x7f80u ? 0u : 0xffffu) | ((v[j] & 0x7f800000u) == 0x7f800000u ? 0u : 0xffff0000u);
            some |= keep != 0xffffffffu;
            v[j] &= keep;
          }
          if (some) put16(at + i, v[0], v[1], v[2], v[3]);
        }
      };
      const bool one = elected();
      bool ok = true;  // (of the one)
      int asked = 0;
      uint32_t copied_phase = 0, bits = 0;
      for (int h = 0; h < H; ++h) {
        if (!FORWARD && (h & 31) == 0) bits = __ldg(odd + (h >> 5));
        const bool infinite = !FORWARD && ((bits >> (h & 31)) & 1u) != 0;
        for (int part = 0; part < XP; ++part) {
          const uint8_t* image = images + ((long long)h * XP + part) * B_BYTES;
          if (one && ok) {
            const int s = asked % BS;
            ok = asked < BS || mbar_wait(smem_u32(&ctl->b_empty[s]), (uint32_t)(asked / BS - 1) & 1u, abort_flag);
            if (ok) {
              mbar_arrive_expect_tx(smem_u32(&ctl->b_full[s]), B_BYTES);
              bulk_copy_g2s(b_ring + s * B_BYTES, image, B_BYTES, smem_u32(&ctl->b_full[s]));
              ++asked;
            }
          }
          if (part == 0 && infinite) {
            int at = -1;
            if (one && ok) {
              const int s = asked % BS;
              ok = asked < BS || mbar_wait(smem_u32(&ctl->b_empty[s]), (uint32_t)(asked / BS - 1) & 1u, abort_flag);
              if (ok) {
                mbar_arrive_expect_tx(smem_u32(&ctl->copied), B_BYTES);
                bulk_copy_g2s(b_ring + s * B_BYTES, image, B_BYTES, smem_u32(&ctl->copied));
                at = s;
              }
            }
            at = __reduce_max_sync(0xffffffffu, at);
            if (at < 0) continue;
            if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&ctl->copied), copied_phase, abort_flag))) {
              if (one) drain_bulk_copies(&ctl->copied, 1, (int)copied_phase + 1);
              ok = false;
              continue;
            }
            copied_phase ^= 1u;
            clear(b_ring + at * B_BYTES);
            fence_proxy_async();
            __syncwarp();
            if (one) mbar_arrive(smem_u32(&ctl->b_full[at]));
            ++asked;
          }
        }
      }
      if (one && !ok) drain_bulk_copies(ctl->b_full, BS, asked);  // copies in flight land before the block ends
      __syncwarp();
    } else if (warp == ISSUER) {
      if (elected()) {
        // Bits: fp32 sums, bfloat16 operands, weights of a W stored with the features side by side (bit 15), rows / 8, lanes / 16.
        constexpr uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | (FORWARD ? 0u : 1u << 15) | ((uint32_t)(TM >> 3) << 17) | ((uint32_t)(LANES >> 4) << 24);
        constexpr int SLICE = FORWARD ? 2 : 128;  // 16 summed indices on, in units of 16 bytes
        // Features side by side: atoms of 64 features x 8 summed indices, 1024 bytes; the next 8 indices 1024 bytes on, the next 64 features 8192.
        const uint64_t a_first = FORWARD ? make_desc(a_ring) : (uint64_t)((a_ring & 0x3FFFFu) >> 4) | (512ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
        const uint64_t b_first = make_desc(b_ring);
        int slot = 0, unit = 0, as = 0;
        uint32_t b_phase = 0, a_phase = 0;
        bool ok = true;
        auto wait = [&](unsigned long long& bar, uint32_t phase) { return ok = ok && mbar_wait(smem_u32(&bar), phase, abort_flag); };
        auto unit_begins = [&]() {
          if (unit >= 2) wait(ctl->d_empty[unit & 1], (uint32_t)(unit / 2 - 1) & 1u);
        };
        uint32_t bits = FORWARD ? 0u : __ldg(odd), next_bits = FORWARD ? 0u : __ldg(odd + min(1, words_of(H) - 1));
        for (int h = 0; ok && h < H; ++h) {
          if (!FORWARD && h > 0 && (h & 31) == 0) {
            bits = next_bits;
            next_bits = __ldg(odd + min((h >> 5) + 1, words_of(H) - 1));
          }
          wait(ctl->a_full[as], a_phase);
          const uint64_t a = a_first + (uint64_t)(as * WP * (A_BYTES >> 4));
          if (FORWARD && UNIT == 1) {  // two units a stage
            const int first = slot;
            const uint32_t first_phase = b_phase;
            for (int half = 0; half < 2; ++half) {
              unit_begins();
              const uint32_t d = tmem + (unit & 1) * TM;
              slot = first;
              b_phase = first_phase;
              for (int part = 0; part < XP; ++part) {
                if (half == 0) wait(ctl->b_full[slot], b_phase);
                tc_fence_after();
                if (!ok) break;
                const uint64_t b = b_first + (uint64_t)(slot * (B_BYTES >> 4));
                mma_bf16(d, a + 4 * half, b + 4 * half, idesc, part > 0);
                mma_bf16(d, a + 4 * half + 2, b + 4 * half + 2, idesc, true);
                if (half == 1) mma_commit(smem_u32(&ctl->b_empty[slot]));
                if (++slot == BS) { slot = 0; b_phase ^= 1u; }
              }
              if (!ok) break;
              if (half == 1) mma_commit(smem_u32(&ctl->a_empty[as]));
              mma_commit(smem_u32(&ctl->d_full[unit & 1]));
              ++unit;
            }
          } else {
            const bool anew = h % SPAN == 0;
            if (anew) unit_begins();
            const uint32_t d = tmem + (unit & 1) * TM;
            for (int part = 0; part < XP; ++part) {
              wait(ctl->b_full[slot], b_phase);
              tc_fence_after();
              if (!ok) break;
              uint64_t b = b_first + (uint64_t)(slot * (B_BYTES >> 4));
#pragma unroll
              for (int q = 0; q < WP; ++q) {
                if (!FORWARD && part == 0 && q == 1 && ((bits >> (h & 31)) & 1u) != 0) {  // from here on without what is not finite
                  mma_commit(smem_u32(&ctl->b_empty[slot]));
                  if (++slot == BS) { slot = 0; b_phase ^= 1u; }
                  wait(ctl->b_full[slot], b_phase);
                  tc_fence_after();
                  if (!ok) break;
                  b = b_first + (uint64_t)(slot * (B_BYTES >> 4));
                }
                if (FORWARD || WP == 2 || q + part < WP) mma_step<SLICE>(d, a + (uint64_t)(q * (A_BYTES >> 4)), b, idesc, !(anew && part == 0 && q == 0));
              }
              if (!ok) break;
              mma_commit(smem_u32(&ctl->b_empty[slot]));
              if (++slot == BS) { slot = 0; b_phase ^= 1u; }
            }
            if (!ok) break;
            mma_commit(smem_u32(&ctl->a_empty[as]));
            if (h == H - 1 || h % SPAN == SPAN - 1) {
              mma_commit(smem_u32(&ctl->d_full[unit & 1]));
              ++unit;
            }
          }
          if (++as == AS) { as = 0; a_phase ^= 1u; }
        }
      }
      __syncwarp();
    } else {
      // Unpacking: a team of 64 threads a stage.  x W^T: 64 columns of two features of the block a thread; a W: the block's 128 columns of one output a thread.  What a team
      // needs is fetched two of its stages ahead.
      const int team = (warp - SUMMERS) >> 1, t = tid & (TEAM - 1);
      const uint8_t* from[2];
      const float* scales[FORWARD ? 1 : 4];
      if (FORWARD) {
        for (int r = 0; r < 2; ++r) from[r] = w.codes + (long long)min(f0 + t + 64 * r, w.n_out - 1) * pitch;
      } else {
        from[0] = w.codes + (long long)f0 / 2;
        for (int r = 0; r < 4; ++r) scales[FORWARD ? 0 : r] = w.scales + (long long)min((f0 + r * 32) >> w.group_log2, groups - 1) * w.n_out;
      }
      uint4 codes[2][4];
      float scale[2][4];
      auto fetch = [&](int h, int b) {
        if (h >= H) return;
        if (FORWARD) {
#pragma unroll
          for (int r = 0; r < 4; ++r) codes[b][r] = __ldg(reinterpret_cast<const uint4*>(from[r >> 1] + min((long long)h * (STEP / 2) + (r & 1) * 16, pitch - 16)));
        } else {
          const int n = min(h * STEP + t, w.n_out - 1);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            codes[b][r] = __ldg(reinterpret_cast<const uint4*>(from[0] + n * pitch + min((long long)r * 16, pitch - 16 - f0 / 2)));
            scale[b][r] = __ldg(scales[FORWARD ? 0 : r] + n);
          }
        }
      };
      if (team < TEAMS) {
        fetch(team, 0);
        fetch(team + TEAMS, 1);
      }
      for (int h2 = team < TEAMS ? team : H; h2 < H; h2 += 2 * TEAMS) {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const int h = h2 + b * TEAMS;
          if (h >= H) break;
          const int as = h % AS;
          if (h >= AS && !mbar_wait_warp(smem_u32(&ctl->a_empty[as]), (uint32_t)(h / AS - 1) & 1u, abort_flag)) { h2 = H; break; }
          // Piece r: x W^T: feature t + 64 (r / 2), eights 4 (r % 2) + e; a W: features 32 r and on: eights 4 (r % 2) + e, the upper 64 features 8192 bytes on.  Swizzled by the row.
          const uint32_t to = a_ring + as * WP * A_BYTES + (t >> 3) * 1024 + (t & 7) * 128;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const uint32_t word[4] = {codes[b][r].x, codes[b][r].y, codes[b][r].z, codes[b][r].w};
            const float f = FORWARD ? 1.f : absolute ? fabsf(scale[b][r]) : scale[b][r];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t at = to + (r >> 1) * 8192 + (((uint32_t)((r & 1) * 4 + e) ^ (uint32_t)(t & 7)) << 4);
              uint32_t q[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                q[i] = weights_of(word[e] >> (4 * i));
                if (absolute) q[i] &= 0x7fff7fffu;
              }
              if (FORWARD) {
                put16(at, q[0], q[1], q[2], q[3]);
              } else {
                uint32_t part[WP][4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  if (WP == 2) {  // the product rounded to the nearest, and what that leaves of it
                    const float c0 = __uint_as_float(q[i] << 16), c1 = __uint_as_float(q[i] & 0xffff0000u);
                    part[0][i] = bits_of(__floats2bfloat162_rn(c0 * f, c1 * f));
                    part[WP - 1][i] = bits_of(__floats2bfloat162_rn(fmaf(c0, f, -__uint_as_float(part[0][i] << 16)), fmaf(c1, f, -__uint_as_float(part[0][i] & 0xffff0000u))));
                    continue;
                  }
                  float x = __uint_as_float(q[i] << 16) * f, y = __uint_as_float(q[i] & 0xffff0000u) * f;
#pragma unroll
                  for (int k = 0; k < WP; ++k) {
                    const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
                    part[k][i] = bits_of(v);
                    x -= __uint_as_float(part[k][i] << 16);
                    y -= __uint_as_float(part[k][i] & 0xffff0000u);
                  }
                }
#pragma unroll
                for (int k = 0; k < WP; ++k) put16(at + k * A_BYTES, part[k][0], part[k][1], part[k][2], part[k][3]);
              }
            }
          }
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&ctl->a_full[as]));
          fetch(h + 2 * TEAMS, b);
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
    float acc[CW];
#pragma unroll
    for (int j = 0; j < CW; ++j) acc[j] = 0.f;
    bool alive = true;
    const int feature = f0 + (warp & 3) * 32 + lane;  // of the accumulators' lane
    const uint32_t sums = tmem + ((uint32_t)((warp & 3) * 32) << 16) + (warp >> 2) * CW;
    auto unit_scale = [&](int u) {
      const long long k = (long long)u * (UNIT >= 4 ? 128 : 32 * UNIT);
      const int g = (int)min(k >> w.group_log2, (long long)groups - 1);
      const float s = __ldg(w.scales + (long long)g * w.n_out + min(feature, w.n_out - 1));
      return absolute ? fabsf(s) : s;
    };
    float next_scale = FORWARD ? unit_scale(0) : 1.f;
    for (int u = 0; u < units; ++u) {
      const int buffer = u & 1;
      const float s = next_scale;
      if (FORWARD && u + 1 < units) next_scale = unit_scale(u + 1);
      if (!FORWARD)  // (they wait for long: asleep, they leave the others the issue slots)
        for (int i = 0; i < 4000000 && !mbar_try_wait(smem_u32(&ctl->d_full[buffer]), (uint32_t)(u / 2) & 1u) && *abort_flag == 0; ++i) __nanosleep(500);
      if (!mbar_wait_warp(smem_u32(&ctl->d_full[buffer]), (uint32_t)(u / 2) & 1u, abort_flag)) { alive = false; break; }
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < CW; c += 32) {
        float v[32];
        tmem_ld32(sums + buffer * TM + c, v);
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
          if (FORWARD) {  // two multiply-adds an instruction
            asm("{\n\t.reg .b64 x, y, z;\n\t"
                "mov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %3};\n\tmov.b64 z, {%4, %4};\n\t"
                "fma.rn.f32x2 x, y, z, x;\n\t"
                "mov.b64 {%0, %1}, x;\n\t}"
                : "+f"(acc[c + j]), "+f"(acc[c + j + 1])
                : "f"(v[j]), "f"(v[j + 1]), "f"(s));
          } else {
            acc[c + j] += v[j];
            acc[c + j + 1] += v[j + 1];
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&ctl->d_empty[buffer]));
    }

    // A lane holds a feature, its registers the rows: neighbouring lanes store neighbouring features.
    const int of = FORWARD ? feature : (feature & ~7) + ((feature & 7) >> 1) + 4 * (feature & 1), width = FORWARD ? w.n_out : w.n_in;
    const float bias = FORWARD && p.bias && !absolute && of < width ? load_any(p.bias, p.bias_type, of) : 0.f;
    if (of < width) {
      const int m1 = m0 + (warp >> 2) * CW;
      const long long first = (long long)m1 * width + of;
      auto rows = [&](auto* out, auto round) {
#pragma unroll
        for (int j = 0; j < CW; ++j)
          if (m1 + j < p.M) out[first + (long long)j * width] = round(acc[j]);
      };
#pragma unroll
      for (int j = 0; j < CW; ++j) acc[j] = alive ? acc[j] + bias : __int_as_float(0x7fffffff);
      if (absolute) {
        constexpr int BATCH = 16;  // of the first pass's results, on their way together
#pragma unroll
        for (int j0 = 0; j0 < CW; j0 += BATCH) {
          float* out = static_cast<float*>(p.out) + first;
          float c[BATCH];
#pragma unroll
          for (int j = 0; j < BATCH; ++j) c[j] = m1 + j0 + j < p.M ? out[(long long)(j0 + j) * width] : 0.f;
#pragma unroll
          for (int j = 0; j < BATCH; ++j) {
            if (m1 + j0 + j >= p.M) continue;
            const float v = acc[j0 + j];
            out[(long long)(j0 + j) * width] = FORWARD ? c[j] - v : 0.5f * (c[j] - v);
            p.out2[first + (long long)(j0 + j) * width] = FORWARD ? c[j] + v : 0.5f * (c[j] + v);
          }
        }
      } else if (p.type == BF_TYPE_F32) {
        rows(static_cast<float*>(p.out), [](float v) { return v; });
      } else if (p.type == BF_TYPE_BF16) {
        rows(static_cast<__nv_bfloat16*>(p.out), [](float v) { return __float2bfloat16(v); });
      } else {
        rows(static_cast<__half*>(p.out), [](float v) { return __float2half(v); });
      }
    }
    if (!alive && lane == 0) *p.status = 1;
  }
  tc_fence_before();
  __syncthreads();
  if (warp == ISSUER) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(COLUMNS) : "memory");
  }
}

// Rows of a block: 256 where those blocks fill the chip, fewer where more blocks are needed or the rows are few.
int rows_of_block(int M, int features) {
  const long long tiles = ceil_div(features, LANES);
  if (M > 128 && tiles * ceil_div(M, 256) >= 148) return 256;
  return M > 64 ? 128 : 64;
}
int steps_of(int n) { return ceil_div(n, STEP); }
size_t odd_bytes(int M, int sum) { return (size_t)ceil_div(M, 64) * words_of(steps_of(sum)) * 4; }  // (the smallest tiles)
size_t header_of(int M, int sum) { return HEADER + (odd_bytes(M, sum) + 1023) / 1024 * 1024; }
int parts_of(int type) { return type == BF_TYPE_F32 ? 3 : type == BF_TYPE_F16 ? 2 : 1; }

template <int XP, int WP, int CW, int UNIT>
int launch(const ManyArgs& p, dim3 grid, cudaStream_t stream) {
  static SmemOptIn table;
  constexpr int smem = RING + 2048;
  const int rc = ensure_dynamic_smem(w4_many_kernel<XP, WP, CW, UNIT>, smem, table, "w4_many_kernel");
  if (rc != BF_OK) return rc;
  w4_many_kernel<XP, WP, CW, UNIT><<<grid, THREADS, smem, stream>>>(p);
  BF_CHECK_LAUNCH("w4_many_kernel");
  g_tc_launches.fetch_add(1, std::memory_order_relaxed);
  return BF_OK;
}
template <int XP, int WP, int CW>
int launch_unit(const ManyArgs& p, dim3 grid, cudaStream_t stream) {
  if (WP > 1 || p.w.group_log2 >= 7) return launch<XP, WP, CW, 4>(p, grid, stream);
  if constexpr (WP == 1) return p.w.group_log2 == 6 ? launch<XP, WP, CW, 2>(p, grid, stream) : launch<XP, WP, CW, 1>(p, grid, stream);
  return BF_OK;
}
template <int XP, int WP>
int launch_rows(const ManyArgs& p, int tile_m, dim3 grid, cudaStream_t stream) {
  if (tile_m == 256) return launch_unit<XP, WP, 128>(p, grid, stream);
  return tile_m == 128 ? launch_unit<XP, WP, 64>(p, grid, stream) : launch_unit<XP, WP, 32>(p, grid, stream);
}

// Rows of one launch: their images are kept to 256 MB, more rows go slab by slab through the same workspace.
int slab_of(int M, int sum, int type) {
  const long long row = (long long)steps_of(sum) * 128 * parts_of(type), most = std::max(1LL, (256LL << 20) / row / 256) * 256;
  return (int)std::min<long long>({M, most, 64LL * 65535});
}
template <bool FORWARD>
int pass(const ManyArgs& all, int mode, int relu_in, void* workspace, bool first_pass, cudaStream_t stream) {
  const int sum = FORWARD ? all.w.n_in : all.w.n_out, features = FORWARD ? all.w.n_out : all.w.n_in, parts = parts_of(all.type), slab = slab_of(all.M, sum, all.type);
  const int size = all.type == BF_TYPE_F32 ? 4 : 2;
  uint8_t* base = static_cast<uint8_t*>(workspace);
  for (long long done = 0; done < all.M; done += slab) {
    ManyArgs p = all;
    p.M = (int)std::min<long long>(slab, all.M - done);
    p.a = static_cast<const char*>(all.a) + done * sum * size;
    p.b = all.b ? all.b + done * sum : nullptr;
    p.out = static_cast<char*>(all.out) + done * features * size;
    p.out2 = all.out2 ? all.out2 + done * features : nullptr;
    p.steps = steps_of(sum);
    p.status = reinterpret_cast<int*>(base);
    uint32_t* odd = reinterpret_cast<uint32_t*>(base + HEADER);
    p.odd = odd;
    p.images = base + header_of(slab, sum);
    const int tile_m = rows_of_block(p.M, features);
    const ImageArgs im = {p.a, p.b, base + header_of(slab, sum), odd, first_pass && done == 0 ? p.status : nullptr, p.type, p.take, mode, relu_in, p.M, sum, tile_m, p.steps};
    if (!FORWARD && cudaMemsetAsync(odd, 0, odd_bytes(p.M, sum), stream) != cudaSuccess) {
      set_error("w4_rows_images_kernel: cannot clear the workspace");
      return BF_E_CUDA;
    }
    const long long eights = (long long)ceil_div(p.M, tile_m) * tile_m * p.steps * 8;
    const int blocks = (int)std::min<long long>((eights + 255) / 256, 148 * 64);
    if (parts == 1) w4_rows_images_kernel<1, FORWARD><<<blocks, 256, 0, stream>>>(im);
    else if (parts == 2) w4_rows_images_kernel<2, FORWARD><<<blocks, 256, 0, stream>>>(im);
    else w4_rows_images_kernel<3, FORWARD><<<blocks, 256, 0, stream>>>(im);
    BF_CHECK_LAUNCH("w4_rows_images_kernel");
    const dim3 grid(ceil_div(features, LANES), ceil_div(p.M, tile_m));
    int rc;
    if constexpr (FORWARD) rc = parts == 1 ? launch_rows<1, 1>(p, tile_m, grid, stream) : parts == 2 ? launch_rows<2, 1>(p, tile_m, grid, stream) : launch_rows<3, 1>(p, tile_m, grid, stream);
    else rc = parts == 1 ? launch_rows<1, 2>(p, tile_m, grid, stream) : parts == 2 ? launch_rows<2, 2>(p, tile_m, grid, stream) : launch_rows<3, 3>(p, tile_m, grid, stream);
    if (rc != BF_OK) return rc;
  }
  return BF_OK;
}

}  // namespace

// Whether these kernels are faster than those for few rows, by a model of both.  Few rows: a launch and so many microseconds for 10^9 products.  Here: launches, ends and
// beginnings, and a time for each 64 summed indices of every wave of blocks, which grows with the parts and hardly with the rows (the latency of unpacking bounds it).
// Measured (us, many / few): 64 bf16 rows through 8192 x 4096 30.5 / 32.8, 48 fp32 ones 40.9 / 56.3, boxes of 48 82 / 122; 256 bf16 rows through 2048 x 2048
// 21.3 / 19.8, 512 22.0 / 33.4; 1024 through 512 x 784 22.1 / 14.1; back through 8192 x 4096 128 bf16 rows 130 / 103, 192 131 / 162, 256 fp32 ones 267 / 228, 512 275 / 396.
bool w4_many_pays(int M, int n_in, int n_out, int group, int type, bool forward, bool pair) {
  const int features = forward ? n_out : n_in, tile = rows_of_block(slab_of(M, forward ? n_in : n_out, type), features), parts = parts_of(type);
  const double few = 4.0 + 1e-9 * M * (double)n_in * n_out * (forward ? (pair ? 55.0 : parts == 1 ? 13.5 : parts == 2 ? 18.0 : 24.0) : (pair ? 60.0 : parts == 3 ? 27.0 : 24.0));
  const double waves = (double)ceil_div((long long)ceil_div(features, LANES) * ceil_div(M, tile), 148);
  const double large = tile == 256 ? 1.0 : tile == 128 ? 0.15 : 0.0;
  double stage = forward ? (parts == 1 ? 0.37 + 0.33 * large : parts == 2 ? 0.45 + 0.45 * large : 0.53 + 0.62 * large) : (parts == 3 ? 1.85 + 0.7 * large : 0.9 + 0.25 * large);
  if (forward && group == 32) stage *= 2.0;  // (two sums a stage)
  const double many = (pair ? 2.0 : 1.0) * (8.0 + waves * steps_of(forward ? n_in : n_out) * stage);
  return many < few;
}

long long w4_many_bytes(int M, int sum, int type) {
  const int slab = slab_of(M, sum, type);
  return (long long)header_of(slab, sum) + (long long)ceil_div(slab, 256) * 256 * steps_of(sum) * 128 * parts_of(type);  // enough for blocks of any size
}
int launch_w4_linear_many(const W4LinearArgs& l, void* workspace, cudaStream_t stream) {
  ManyArgs p = {};
  p.w = l.w;
  p.a = l.a;
  p.b = l.b;
  p.bias = l.bias;
  p.out = l.y;
  p.type = l.type;
  p.bias_type = l.bias_type;
  p.M = l.M;
  p.take = l.b ? TAKE_CENTRE : TAKE_ROWS;
  const int rc = pass<true>(p, l.mode, l.relu_in, workspace, true, stream);
  if (rc != BF_OK || !l.b) return rc;
  p.take = TAKE_RADIUS;
  p.out2 = l.y2;
  return pass<true>(p, l.mode, l.relu_in, workspace, false, stream);
}
int launch_w4_rows_many(const W4RowsArgs& r, void* workspace, cudaStream_t stream) {
  ManyArgs p = {};
  p.w = r.w;
  p.a = r.a;
  p.b = r.b;
  p.out = r.z;
  p.type = r.type;
  p.M = r.M;
  p.take = r.b ? TAKE_SUM : TAKE_ROWS;
  const int rc = pass<false>(p, 0, 0, workspace, true, stream);
  if (rc != BF_OK || !r.b) return rc;
  p.take = TAKE_DIFFERENCE;
  p.out2 = r.z2;
  return pass<false>(p, 0, 0, workspace, false, stream);
}

}  // namespace bf
