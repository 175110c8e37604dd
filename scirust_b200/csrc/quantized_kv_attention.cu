// Attention of single tokens over the paged KV cache in 8 bits (its layout: quantized_kv.cu).
//
//   o = sum_j w_j s_v(j) c_v(j) / sum_j w_j,   w_j = exp(scale * s_k(j) * (q . c_k(j)) - m),
// with codes c and the scales s of the position's block and head.
//
// Bound by the codes' bytes, half of a bf16 cache's, so everything done for a byte has half the time: 64 sequences of up to 2048 positions, 32
// / 8 heads of 128, take 37.8 us (0.82 of the copy rate), one of 131072 46 (0.89). Calls of a few tiles a CTA are bound by latency, from 4.5 us on.
// One CTA per SM holds a ring of 16 KB tiles (keys and values of 64 positions, or 128 of heads of 64: 32.9 us with tiles of 64, 25.5 so, for
// 64 sequences of 16 / 4 such heads) that one warp fills by TMA and another with the tile's scales; the tiles of all jobs (a sequence and up
// to 24 query heads of one kv head) lie end to end and are dealt out evenly, however ragged the lengths. Consumer warps take the tiles in
// groups of four, warp w of a group a quarter of the tile's positions, in sixteens:
//  - mma.sync takes codes as the A operand, 16 positions (S = K q) or 16 dimensions (O = V w), and eight query heads as columns: a warp's
//    16 positions times 16 query rows would be half empty with eight query heads a kv head or fewer. With more, each group takes all tiles for
//    eight of them. ldmatrix moves pairs of bytes, so the even and the odd dimensions of V come apart as rows of two halves of the A operand,
//    and for K the dimensions of a step are in another order, in which q is loaded.
//  - Codes become fp16, which holds every one of either type exactly: int8 by a byte permute (a byte behind 0x64 is 1024 + it) and one
//    subtraction of two halves, e4m3 by its conversion. K in int8 goes into the product as it is: q, scaled by a power of two so that its
//    row's largest magnitude is just below 2^14 and rounded to whole numbers, is two bytes, whose products are summed apart, exactly. That
//    rounding is off by 2^-14 of the row's largest at most, and bf16 values from 2^-6 of it on are kept as they are; 50 conversions a tile and
//    lane of 130 are saved (one sequence of 131072 positions: 52 us with halves, 49 so, as the rest then was). For e4m3 q's largest is just
//    below 2^15, and fp16 holds it without loss.
//  - The reference of the exponentials is a score seen before, not the maximum: it moves when a score exceeds it by 2^6, so that few
//    tiles need a reduction over positions and a pass over O. Weights are 2^9 at the reference: at most 2^15, and what lies 2^-33 below the
//    reference is still a number of fp16. Their sum is taken in 32 bits before they are rounded (half a step of 2^-11) and weighed.
//  - A value's scale goes into its weight, as a ratio to a power of two that weighs the sums at the end: a product of its own for each block of 16
//    positions would need a pass over O for each. That power is a head's own and, where weights allow it, no less than the largest scale that the
//    warp has seen of the piece, so that few tiles move it. But it is at most half of the largest product of a weight and a scale, so that
//    what is rounded to fp16 loses no more than 2^-26 of that product (half of fp16's smallest step, 2^-25, against 2) wherever a
//    scale without weight lies. Scales up to 2^100 times as large as another may lie beside it.
//  - A warp takes its positions' bytes into registers and gives the stage back before it computes, so that nearly the whole ring is always
//    under way from memory.
// At the end of a piece of a job the warps leave their sums in shared memory and go on; two finishing warps join them, or, with more than
// eight heads, all consumers, since two warps take ten turns for twenty heads (32 sequences of one kv head with 20 27.3 us so, 21.5
// by all). A job that is cut has its pieces joined by the CTA that ends last, in the order of the tiles (a counter, no atomics on data).
// Only the warp that brings the codes works out which piece is next; the others find its sequence, heads and tiles beside its queries.
#include <cfloat>
#include <cuda_bf16.h>
#include "api.h"
#include "dependent.cuh"
#include "per_device.h"
#include "quantized_kv.cuh"
#include "sm100_ptx.cuh"

namespace sb {
int num_sms();                                                 // gemm_tcgen05.cu
int make_tmap_3d_u8_rows(CUtensorMap* out, const void* base, uint32_t row_bytes, uint64_t rows, uint64_t groups, uint32_t box_rows,
                         uint32_t box_groups);

namespace kv8 {

constexpr int MAX_B = 1024;                  // sequences of a launch, whose offsets lie in shared memory
constexpr int STAGES_MAX = 24;
constexpr int SET = 8, HEADS_MAX = 3 * SET;  // query heads of a set, which is what a warp takes, and of a job
constexpr int SMEM = 225 * 1024;
constexpr int SHARES = 4;                    // of the pieces of a job that is joined, at most
constexpr float LOWEST = -FLT_MAX;           // reference of no score: no finite one lies below it, and what lies above by 15 moves it

struct AttendParams {
  const __nv_bfloat16* q; long long ldq;
  const float* scales;
  int n_blocks, page, page_bits, block_bits;         // page_bits: 3, 4 or 5, or for multiples of 64 6
  int page_shift;                            // log2 of the page, -1 where it is no power of two
  const int* table; int max_blocks;
  const int* seq_len;
  int B, Hkv, G, subs;                       // a kv head's G query heads in `subs` jobs
  int sets, heads;                           // of so many sets of so many heads
  float scale_log2;
  float* part;                               // [2 * grid] of [HEADS_MAX][DH] values and [HEADS_MAX][2] maxima and sums
  unsigned int* counters;                    // [B * Hkv * subs], zero between calls
  __nv_bfloat16* out; long long ldo;
  int* status;
  int stages;
};

// The tiles [t_beg, t_end) of a job that lie in a CTA's range.
struct __align__(16) Piece {
  int b, h0, live, len;                      // sequence, query heads [h0, h0 + live), positions
  int t_beg, t_end, nt, last;                // nt: tiles of the job; last: of the CTA
  int start, counter, pad[2];                // the job's first unit, its counter
};

template <int DH>
struct Cfg {
  static constexpr int GROUPS = 3, CONSUMERS = 4 * GROUPS;     // of four warps, and warps
  static constexpr int CODES = CONSUMERS, SCALES = CONSUMERS + 1, FINISHERS = CONSUMERS + 2;      // two producers, two finishers
  static constexpr int THREADS = CONSUMERS * 32 + 128;
  static constexpr int TK = 8192 / DH;                         // positions of a tile: 64, or 128 at half the head dimension
  static constexpr int TILE = TK * DH;                         // bytes of a tile's keys, and of its values
  static constexpr int PARTS = TK / 64;                        // a warp's positions of a tile, in sixteens
  static constexpr int SCALES_OF_V = TK / 8;                   // where values' scales begin: one for eight positions of keys, then of values
  static constexpr int PITCH = DH + 4;                         // of a head's sums between warps
  static constexpr int QSLOTS = 4;                             // pieces whose queries lie in shared memory
  static constexpr int fixed_bytes(int sets, int heads, int B) {
    return CONSUMERS * heads * (PITCH + 4) * 4 + QSLOTS * (sets * heads * DH * 2 + static_cast<int>(sizeof(Piece))) + (2 * B + 1) * 4 +
           STAGES_MAX * (2 * SCALES_OF_V * 4 + 16) + (2 * QSLOTS + 2) * 8 + 1024;
  }
  // A stage is always taken by the same groups: a parity wait tells a fill from the one after next only by whoever has seen the one between.
  static constexpr int stages(int sets, int heads, int B) {
    const int n = (SMEM - fixed_bytes(sets, heads, B)) / (2 * TILE), most = n < STAGES_MAX ? n : STAGES_MAX;
    return sets == 1 ? most / GROUPS * GROUPS : most;
  }
  static constexpr int smem_bytes(int sets, int heads, int B) { return stages(sets, heads, B) * 2 * TILE + fixed_bytes(sets, heads, B); }
};
static_assert(Cfg<128>::stages(1, 8, MAX_B) >= 9 && Cfg<128>::stages(3, 8, MAX_B) >= 8, "128 KB in flight");

__device__ __forceinline__ void ldsm(uint32_t addr, uint32_t (&a)[2], uint32_t (&b)[2]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(a[0]), "=r"(a[1]), "=r"(b[0]), "=r"(b[1]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm_t(uint32_t addr, uint32_t (&a)[2], uint32_t (&b)[2]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(a[0]), "=r"(a[1]), "=r"(b[0]), "=r"(b[1]) : "r"(addr) : "memory");
}
// c += a b, or with FIRST c = a b
template <bool FIRST>
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (FIRST)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <bool FIRST>
__device__ __forceinline__ void mma_s8(int (&c)[4], const uint32_t (&a)[2], const uint32_t (&a_next)[2], uint32_t b0, uint32_t b1) {
  if constexpr (FIRST)
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a_next[0]), "r"(a_next[1]), "r"(b0), "r"(b1), "r"(0));
  else
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a_next[0]), "r"(a_next[1]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t half2_bits(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// One over a power of two between 2^-126 and 2^126.
__device__ __forceinline__ float inverse(float x) { return __uint_as_float(0x7f000000u - __float_as_uint(x)); }

// The reference of values' scales, a power of two, after scales of up to `scale`, whose largest product with a weight is `product`, and a weight
// of `a` for what was there: no less than the scales, so that nothing moves it before larger ones, but at most half of the largest product
// so far (of which the old reference was at most half). A product is at most 2^15 of it: weights are, and where it lies below the scales it is
// a quarter of the product or more. Numbers of one sign compare as their bits do.
__device__ __forceinline__ float values_reference(float old, float scale, float product, float a) {
  const uint32_t up = min((__float_as_uint(fmaxf(scale, old)) + 0x7fffffu) & 0x7f800000u, 0x7e800000u);
  const uint32_t most = __float_as_uint(fmaxf(0.5f * product, a * old)) & 0x7f800000u;
  const uint32_t least = __float_as_uint(fmaxf(scale * 0x1p-100f, 0x1p-126f)) & 0x7f800000u;      // the scales' ratio stays a number
  return __uint_as_float(max(min(up, most), least));
}

// Bytes (0, 1) and (2, 3) of w as pairs of halves, or with APART (0, 2) and (1, 3).
template <bool E4M3, bool APART>
__device__ __forceinline__ void widen(uint32_t w, uint32_t& x, uint32_t& y) {
  if constexpr (E4M3) {
    if (APART) w = __byte_perm(w, 0, 0x3120);
    asm("{\n"
        ".reg .b16 lo, hi;\n"
        "mov.b32 {lo, hi}, %2;\n"
        "cvt.rn.f16x2.e4m3x2 %0, lo;\n"
        "cvt.rn.f16x2.e4m3x2 %1, hi;\n"
        "}\n" : "=r"(x), "=r"(y) : "r"(w));
  } else {
    const uint32_t u = w ^ 0x80808080u;
    x = __byte_perm(u, 0x64646464u, APART ? 0x4240 : 0x4140);
    y = __byte_perm(u, 0x64646464u, APART ? 0x4341 : 0x4342);
    asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(x) : "r"(0x64806480u));          // 1152
    asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(y) : "r"(0x64806480u));
  }
}

// Tiles of one sequence: an empty one keeps a tile without positions, whose job writes zeros.
template <int TK>
__device__ __forceinline__ int tiles_of(int len) { return len > 0 ? (len + TK - 1) / TK : 1; }

// How the units (tiles of all jobs, end to end; or whole jobs) are dealt out: the first `more` CTAs have one more than the others.
struct Deal {
  int ctas, each, more, whole;
  __device__ __forceinline__ int first(int c) const { return c * each + min(c, more); }
  __device__ __forceinline__ int cta(int u) const {
    const int at = more * (each + 1);
    return u < at ? u / (each + 1) : more + (u - at) / each;
  }
};

// Four shares (reference and sum of weights, weighted values) as one; those of no piece have a sum of zero.
__device__ __forceinline__ void join_shares(const float2 (&ml)[SHARES], const float4 (&e)[SHARES], float4& v, float& sum) {
  const float top = fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x));
  sum = 0.f;
  v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int k = 0; k < SHARES; ++k) {
    const float a = ex2(ml[k].x - top);
    sum += ml[k].y * a;
    v.x += e[k].x * a; v.y += e[k].y * a; v.z += e[k].z * a; v.w += e[k].w * a;
  }
}

// MANY: jobs of more than one set of heads; SMALL: both producers ask for a tile's boxes
template <int DH, bool E4M3, bool MANY, bool SMALL>
__global__ void __launch_bounds__(Cfg<DH>::THREADS, 1)
attend_kernel(const __grid_constant__ CUtensorMap tmap, const __grid_constant__ AttendParams p) {
  using C = Cfg<DH>;
  constexpr int CHUNKS = DH / 16, GROUPS = C::GROUPS, CONSUMERS = C::CONSUMERS, TK = C::TK, PARTS = C::PARTS, SCALES_OF_V = C::SCALES_OF_V;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int stages = p.stages, sets = MANY ? p.sets : 1, heads = p.heads, jobs_b = p.Hkv * p.subs;
  float* sc = reinterpret_cast<float*>(ring + stages * 2 * C::TILE);                // [stages][keys | values], of 8 positions each
  __nv_bfloat16* sm_q = reinterpret_cast<__nv_bfloat16*>(sc + STAGES_MAX * 2 * SCALES_OF_V);     // [slots][sets * heads][DH]
  Piece* pieces = reinterpret_cast<Piece*>(sm_q + C::QSLOTS * sets * heads * DH);          // [slots]
  float* sm_o = reinterpret_cast<float*>(pieces + C::QSLOTS);                       // [warps][heads][PITCH]
  float4* sm_ml = reinterpret_cast<float4*>(sm_o + CONSUMERS * heads * C::PITCH);   // [warps][heads]: reference, sum, that of values' scales
  uint64_t* full = reinterpret_cast<uint64_t*>(sm_ml + CONSUMERS * heads);
  uint64_t* empty = full + STAGES_MAX;
  uint64_t* q_full = empty + STAGES_MAX;
  uint64_t* q_empty = q_full + C::QSLOTS;
  uint64_t* o_full = q_empty + C::QSLOTS;                                           // the warps' sums of a piece, but for the last one's
  uint64_t* o_empty = o_full + 1;
  int* prefix = reinterpret_cast<int*>(o_empty + 1);                                // [B + 1] tiles before sequence b
  int* lens = prefix + p.B + 1;                                                     // [B]
  // of the finishers and the consumers: whether their job's other pieces are there, its first CTA, its pieces
  __shared__ int s_last[2], s_join[2][2];
  __shared__ int s_end, s_ready, s_ready_now, s_ready_join[2];
  __shared__ Deal s_deal;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (warp == 0) {
    if (lane < stages) { mbar_init(&full[lane], 1 + 2 * SCALES_OF_V); mbar_init(&empty[lane], 4 * sets); }
    if (lane < C::QSLOTS) { mbar_init(&q_full[lane], 1); mbar_init(&q_empty[lane], CONSUMERS + 2); }
    if (lane == 0) { mbar_init(o_full, CONSUMERS); mbar_init(o_empty, 1); s_end = s_ready = 0; }
    fence_barrier_init();
  } else if (threadIdx.x == C::CODES * 32) {
    prefetch_tmap(&tmap);
  }
  __syncthreads();
  pdl_trigger();
  {
    // lengths and tables are the first things read, one after the other: L2 has them when they are
    const size_t line = (static_cast<size_t>(blockIdx.x) * C::THREADS + threadIdx.x) * 128, bytes = static_cast<size_t>(p.B) * 4;
    if (line < bytes * p.max_blocks) asm volatile("prefetch.global.L2 [%0];" ::"l"(reinterpret_cast<const char*>(p.table) + line));
    if (line < bytes) asm volatile("prefetch.global.L2 [%0];" ::"l"(reinterpret_cast<const char*>(p.seq_len) + line));
  }
  pdl_wait();

  if (warp == C::CODES || warp == C::SCALES) {
    // ------------------------------ producers: one warp brings queries and codes, one scales ------------------------------
    const bool brings_codes = warp == C::CODES;
    Deal deal;
    if (brings_codes) {
      const int cap = static_cast<int>(min(static_cast<long long>(p.max_blocks) * p.page, 0x7fffffffll - TK));
      int base = 0, longest = 0;
      int next = lane < p.B ? p.seq_len[lane] : 0;
      for (int b0 = 0; b0 < p.B; b0 += 32) {
        const int len = min(next, cap);
        next = b0 + 32 + lane < p.B ? p.seq_len[b0 + 32 + lane] : 0;
        const int n = b0 + lane < p.B ? tiles_of<TK>(len) : 0;
        int inc = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, inc, o);
          if (lane >= o) inc += v;
        }
        if (b0 + lane < p.B) { prefix[b0 + lane] = base + inc - n; lens[b0 + lane] = len; }
        base += __shfl_sync(0xffffffffu, inc, 31);
        longest = max(longest, n);
      }
      longest = __reduce_max_sync(0xffffffffu, longest);
      const int tiles = base * jobs_b, jobs = p.B * jobs_b, grid = gridDim.x;
      deal.ctas = min(grid, MANY ? tiles : (tiles + GROUPS - 1) / GROUPS);
      deal.each = tiles / deal.ctas;
      deal.whole = 0;
      // What it costs to cut jobs (writing sums, asking for the count, reading them), at the end, where nothing else is under way, is as long
      // as sixteen tiles: up to there jobs are dealt out whole. us cut / whole, 32 / 8 heads of 128: 1 x 600 positions 9.9 / 7.1, 4 x 800 10.6 /
      // 8.4, 4 x 1600 (21 tiles more) 11.1 / 12.0, 16 x 300 10.7 / 6.3, 16 x 1500 14.2 / 11.9, 16 x 2500 18.1 / 16.7, 64 x 1000 26.5 / 27.2, 9
      // of up to 5003 on 4 / 1 heads 12.8 / 28.1; 16 / 4 heads of 64, whose tiles are twice as long: 1 x 600 8.1 / 5.5, 4 x 1600 8.5 / 8.3, 4 x
      // 3000 8.9 / 12.4, 16 x 1500 9.7 / 8.5, 16 x 3000 11.0 / 12.7, 64 x 1000 14.5 / 11.5, 64 x 2000 17.3 / 16.8. A tile of several sets takes
      // twice as long or more, so that with few such jobs sixteen are too many, at worst by a third: 20 / 1 heads of 128 1 x 600 9.9 / 10.9, 4
      // x 800 10.2 / 12.8, 16 x 300 9.0 / 8.2, 16 x 1000 14.1 / 14.8, 32 x 400 11.7 / 9.4, 148 x 1000 23.2 / 17.5; 32 / 2 of 128 16 x 600
      // 13.0 / 10.2, 74 x 1000 20.1 / 14.6; 24 / 2 of 64 8 x 1200 7.4 / 9.7, 16 x 2000 12.1 / 13.5, 74 x 1000 15.0 / 10.6.
      const int each = jobs <= grid ? 1 : jobs / grid, most = each + (each * grid < jobs);
      if (longest <= 4096 && most * longest - deal.each <= 16) {
        deal.ctas = min(grid, jobs);
        deal.each = each;
        deal.whole = 1;
      }
      deal.more = (deal.whole ? jobs : tiles) - deal.each * deal.ctas;
      if (lane == 0) { prefix[p.B] = base; s_deal = deal; }
    }
    asm volatile("bar.sync 3, 64;" ::: "memory");
    deal = s_deal;
    const bool idle = static_cast<int>(blockIdx.x) >= deal.ctas;
    int b = 0, job = 0, t_beg = 0, left = 0;                                                // the first piece; units of the CTA to come
    if (!idle) {
      const int u0 = deal.first(blockIdx.x);
      left = deal.first(blockIdx.x + 1) - u0;
      if (deal.whole) {
        b = u0 / jobs_b;
        job = u0 - b * jobs_b;
      } else {
        // the last sequence whose first unit is not behind the CTA's, by steps of a 32nd of those left
        for (int n = p.B - 1; n > 0;) {
          const int step = (n + 31) / 32, at = b + (lane + 1) * step;
          const int c = __popc(__ballot_sync(0xffffffffu, at <= b + n && prefix[min(at, p.B)] * jobs_b <= u0));
          b += c * step;
          n = min(step - 1, n - c * step);
        }
        t_beg = u0 - prefix[b] * jobs_b;
        job = t_beg / tiles_of<TK>(lens[b]);
        t_beg -= job * tiles_of<TK>(lens[b]);
      }
    }
    int len = lens[b], nt = tiles_of<TK>(len), start = prefix[b] * jobs_b;
    start += job * nt;
    int kvh = p.subs == 1 ? job : job / p.subs, sub = job - kvh * p.subs;

    const int box_bits = min(p.page_bits, 6), box = 1 << box_bits, nbx = TK >> box_bits;    // positions of a TMA box, boxes of a tile
    // of a tile, a lane has one box of codes, of keys and of values, or one scale, of eight positions
    const int first = brings_codes ? lane << box_bits : lane % SCALES_OF_V * 8;                     // its first position in the tile
    const int x = first >> box_bits;
    const int per_page = p.page >> p.block_bits;                                            // scales of a page and head
    const int step = lane / SCALES_OF_V * p.Hkv * per_page + ((first & (box - 1)) >> p.block_bits);
    // with SMALL every other box is the scales' warp's to ask for
    const bool asks = brings_codes ? !(x & 1) : (x & 1) && lane < SCALES_OF_V && !(first & (box - 1));
    int stage = 0, q_slot = 0;
    uint32_t phase = 0, q_phase = 0;
    // of box (fetched + lane) of sequence b: its page, -1 outside the pool, and its first position there
    int fetched = -1, id_of_lane = -1, slot_of_lane = 0;
    do {
      const int t_end = deal.whole ? nt : min(nt, t_beg + left);
      left -= deal.whole ? 1 : t_end - t_beg;
      const int* table = p.table + static_cast<size_t>(b) * p.max_blocks;
      auto fetch = [&] {
        const long long pos = static_cast<long long>(fetched + lane) << box_bits;
        const int at = pos >= len ? 0 : p.page_shift >= 0 ? static_cast<int>(pos) >> p.page_shift : static_cast<int>(pos) / p.page;
        slot_of_lane = static_cast<int>(pos) - at * p.page;
        id_of_lane = -1;
        if (pos < len) id_of_lane = table[at];
      };
      if (!idle && fetched != t_beg * nbx) {             // the kv heads of a sequence have one table
        fetched = t_beg * nbx;
        fetch();                                         // the ids come while the queries are seen to
      }
      if (brings_codes) {
        mbar_wait_converged(&q_empty[q_slot], q_phase ^ 1, p.status, ST_TIMEOUT_EMPTY);
        if (lane == 0) {
          const int h0 = kvh * p.G + sub * sets * heads, live = min(sets * heads, p.G - sub * sets * heads);
          if (!idle)
            asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                         ::"r"(smem_u32(sm_q + q_slot * sets * heads * DH)), "l"(p.q + b * p.ldq + static_cast<long long>(h0) * DH),
                         "r"(live * DH * 2), "r"(smem_u32(&q_full[q_slot])) : "memory");
          Piece* to = pieces + q_slot;
          to->b = b; to->h0 = h0; to->live = live; to->len = len;
          to->t_beg = t_beg; to->t_end = idle ? t_beg : t_end; to->nt = nt; to->last = left <= 0;
          to->start = start; to->counter = b * jobs_b + job;
          mbar_arrive_expect_tx(&q_full[q_slot], idle ? 0 : live * DH * 2);
        }
        if (++q_slot == C::QSLOTS) { q_slot = 0; q_phase ^= 1; }
      }
      if (idle) break;
      for (int t = t_beg; t < t_end; ++t) {
        const int bx0 = t * nbx;
        if (bx0 + nbx > fetched + 32) {                  // nbx divides 32: a tile's boxes are fetched together
          fetched = bx0;
          fetch();
        }
        const int id = __shfl_sync(0xffffffffu, id_of_lane, bx0 + x - fetched);
        const int slot = __shfl_sync(0xffffffffu, slot_of_lane, bx0 + x - fetched);
        const bool known = static_cast<unsigned>(id) < static_cast<unsigned>(p.n_blocks);
        const int rest = len - t * TK;                                                      // positions of the tile that exist, or more
        const int live = rest >= TK ? nbx : max(0, (rest + box - 1) >> box_bits);           // boxes with one of them
        mbar_wait_converged(&empty[stage], phase ^ 1, p.status, ST_TIMEOUT_EMPTY);
        auto ask = [&] {
          tma_load_3d(ring + stage * 2 * C::TILE + first * 2 * DH, &tmap, &full[stage], 0, kvh * p.page + slot, known ? 2 * id : 2 * p.n_blocks);
        };
        if (brings_codes) {
          // A box of keys and, behind it, that of values; ids outside the pool: one behind its last page, all zeros. The stage is not full
          // before lane 0 has arrived, whichever comes first, its bytes or that they are expected.
          if (SMALL ? asks && x < live : x < live) ask();
          if (lane == 0) mbar_arrive_expect_tx(&full[stage], live * 2 * box * DH);
        } else if (lane < 2 * SCALES_OF_V) {
          const bool real = first < rest && known;
          const int at = (id * 2 * p.Hkv + kvh) * per_page + (slot >> p.block_bits) + step;
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;"
                       ::"r"(smem_u32(sc + stage * 2 * SCALES_OF_V + lane)), "l"(p.scales + (real ? at : 0)), "r"(real ? 4 : 0) : "memory");
          asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(smem_u32(&full[stage])) : "memory");
          if (SMALL && asks && x < live) ask();
        }
        if (++stage == stages) { stage = 0; phase ^= 1; }
      }
      start += nt;                                       // the next job's
      t_beg = 0;
      if (++sub == p.subs) { sub = 0; ++kvh; }
      if (++job == jobs_b) {
        job = kvh = 0;
        fetched = -1;
        if (++b < p.B) { len = lens[b]; nt = tiles_of<TK>(len); }
      }
    } while (left > 0);
    asm volatile("cp.async.wait_all;" ::: "memory");
    return;
  }

  // ------------------------------ consumers, and finishers: these join the warps' sums of all pieces but the last -----------------------
  const bool consumes = warp < CONSUMERS;
  const int quad = lane >> 2, tq = lane & 3, mi = lane >> 3;
  const int group = warp >> 2, pw = warp & 3;
  // the groups take turns at the tiles, or, with more than one set of heads, each takes all tiles for a set of its own
  const int my_set = MANY ? group : 0, stride = MANY ? 1 : GROUPS;
  const int wrow = pw * (16 * PARTS) + (mi & 1) * 8 + (lane & 7);                              // the lane's row of a tile, for ldmatrix
  // its first sixteen bytes of that row, swizzled; those of step c are at this address ^ (c << 4), and those of values a box behind
  const int box = 1 << p.page_bits;
  const uint32_t my_row = smem_u32(ring) + ((wrow & ~(box - 1)) * 2 + (wrow & (box - 1))) * DH +
                          (((mi >> 1) ^ (DH == 128 ? wrow & 7 : (wrow >> 1) & 3)) << 4);
  const uint32_t my_scales = smem_u32(sc) + pw * (8 * PARTS);
  const int next_part = (box <= 16 ? 32 : 16) * DH;                                    // sixteen positions further on
  const int team = consumes ? CONSUMERS * 32 : 64, tid = consumes ? threadIdx.x : threadIdx.x - C::FINISHERS * 32;
  auto team_sync = [&] { asm volatile("bar.sync %0, %1;" ::"r"(consumes ? 1 : 2), "r"(team) : "memory"); };
  int turn = group - my_set;                 // tiles of the next piece before the first that this group takes
  int stage = turn, q_slot = 0;
  uint32_t phase = 0, q_phase = 0, o_phase = 0;
  for (bool last = false; !last;) {
    if (!mbar_wait_warp(&q_full[q_slot], q_phase, p.status, ST_TIMEOUT_FULL)) return;
    const Piece* piece = pieces + q_slot;                // the last one stays
    const int t_beg = piece->t_beg, t_end = piece->t_end, len = piece->len, live = piece->live, mine = min(heads, live - my_set * heads);
    last = piece->last;
    Piece to;
    const __nv_bfloat16* my_q = sm_q + (q_slot * sets + my_set) * heads * DH;
    uint64_t* q_done = &q_empty[q_slot];
    if (++q_slot == C::QSLOTS) { q_slot = 0; q_phase ^= 1; }
    if (consumes) {
      // q as B fragments: column `quad` is a query head; of a step of 16 dimensions the lane's four are 4 tq .. 4 tq + 3, as K's bytes come
      uint32_t qb[CHUNKS][2];
      float qf[2];
      {
        const __nv_bfloat16* src = my_q + quad * DH + tq * 4;
        uint32_t top = 0;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
          const uint2 v = quad < mine ? *reinterpret_cast<const uint2*>(src + c * 16) : make_uint2(0, 0);
          qb[c][0] = v.x;
          qb[c][1] = v.y;
          top = largest(top, largest(v.x, v.y));
        }
        top = largest(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = largest(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const uint32_t e = max(max(top & 0x7fffu, top >> 16 & 0x7fffu) >> 7, 15u);     // the exponent of the largest, biased
        float down;
        if constexpr (E4M3) {
          const float up = __uint_as_float((268u - e) << 23);                          // 2^(14 - (e - 127)), and back
          down = __uint_as_float((e - 14u) << 23);
#pragma unroll
          for (int c = 0; c < CHUNKS; ++c) {
            qb[c][0] = half2_bits(bf16_lo(qb[c][0]) * up, bf16_hi(qb[c][0]) * up);
            qb[c][1] = half2_bits(bf16_lo(qb[c][1]) * up, bf16_hi(qb[c][1]) * up);
          }
        } else {
          // Whole numbers of up to 2^14: 1.5 * 2^23 + q is a float whose last bytes are it. The lower byte counts from -128 on, so that the
          // upper one is that of q + 128, and the lower one that of q + 128 less 128, which is its first bit the other way.
          const float up = __uint_as_float((267u - e) << 23);
          down = e == 255 ? __uint_as_float(0x7fffffffu) : __uint_as_float((e - 13u) << 23);      // no whole number is a NaN or an infinity
#pragma unroll
          for (int c = 0; c < CHUNKS; ++c) {
            auto whole_number = [up](float x) { return __float_as_uint(fmaf(x, up, 12582912.f + 128.f)); };
            const uint32_t w0 = whole_number(bf16_lo(qb[c][0])), w1 = whole_number(bf16_hi(qb[c][0]));
            const uint32_t w2 = whole_number(bf16_lo(qb[c][1])), w3 = whole_number(bf16_hi(qb[c][1]));
            const uint32_t w01 = __byte_perm(w0, w1, 0x5140), w23 = __byte_perm(w2, w3, 0x5140);      // lower bytes, upper bytes
            qb[c][0] = __byte_perm(w01, w23, 0x7632);
            qb[c][1] = __byte_perm(w01, w23, 0x5410) ^ 0x80808080u;
          }
        }
        const float f = down * p.scale_log2;
        qf[0] = __shfl_sync(0xffffffffu, f, tq * 8);                                   // of heads 2 tq and 2 tq + 1, the columns of a result
        qf[1] = __shfl_sync(0xffffffffu, f, tq * 8 + 4);
      }
      __syncwarp();
      if (lane == 0 && !MANY) mbar_arrive(q_done);
      float m[2] = {LOWEST, LOWEST}, l[2] = {0.f, 0.f}, o[CHUNKS][4];
      float vinv[2] = {0x1p126f, 0x1p126f};                                            // one over the references of values' scales
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) o[c][0] = o[c][1] = o[c][2] = o[c][3] = 0.f;

      int t = my_set < sets ? t_beg + turn : t_end;                                    // with two sets one group has none
      for (; t < t_end; t += stride) {
        const int st = stage;
        const uint32_t ph = phase;
        stage += stride;
        if (stage >= stages) { stage -= stages; phase ^= 1; }
        mbar_wait_converged(&full[st], ph, p.status, ST_TIMEOUT_FULL);
        const uint32_t row = my_row + st * (2 * C::TILE);
        float2 ks_of[PARTS], vs_of[PARTS];
#pragma unroll
        for (int i = 0; i < PARTS; ++i) {
          const uint32_t at = my_scales + st * (8 * SCALES_OF_V) + i * 8;
          asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(ks_of[i].x), "=f"(ks_of[i].y) : "r"(at) : "memory");
          asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(vs_of[i].x), "=f"(vs_of[i].y) : "r"(at + 4 * SCALES_OF_V) : "memory");
        }
        // the bytes of the warp's positions go to registers, and the stage back to the producers
        uint32_t k_of[PARTS][CHUNKS][2], v_of[PARTS][CHUNKS][2];
#pragma unroll
        for (int i = 0; i < PARTS; ++i) {
#pragma unroll
          for (int c = 0; c < CHUNKS; c += 2) ldsm((row + i * next_part) ^ (c << 4), k_of[i][c], k_of[i][c + 1]);
#pragma unroll
          for (int c = 0; c < CHUNKS; c += 2) ldsm_t((row + i * next_part + box * DH) ^ (c << 4), v_of[i][c], v_of[i][c + 1]);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[st]);
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
          const float2 ks = ks_of[part], vs = vs_of[part];
          uint32_t (&rk)[CHUNKS][2] = k_of[part], (&rv)[CHUNKS][2] = v_of[part];
          const int valid = len - t * TK - (pw * PARTS + part) * 16;                     // positions of these 16 that exist
          float s[4];
          if constexpr (E4M3) {
            float s1[4];                                                                 // two sums of products, so that they need not wait so long
#pragma unroll
            for (int c = 0; c < CHUNKS; c += 2) {
              uint32_t a[4];
              widen<E4M3, false>(rk[c][0], a[0], a[2]);
              widen<E4M3, false>(rk[c][1], a[1], a[3]);
              if (c == 0) mma_f16<true>(s, a[0], a[1], a[2], a[3], qb[c][0], qb[c][1]);
              else mma_f16<false>(s, a[0], a[1], a[2], a[3], qb[c][0], qb[c][1]);
              widen<E4M3, false>(rk[c + 1][0], a[0], a[2]);
              widen<E4M3, false>(rk[c + 1][1], a[1], a[3]);
              if (c == 0) mma_f16<true>(s1, a[0], a[1], a[2], a[3], qb[c + 1][0], qb[c + 1][1]);
              else mma_f16<false>(s1, a[0], a[1], a[2], a[3], qb[c + 1][0], qb[c + 1][1]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] += s1[e];
          } else {
            int hi[4], lo[4];
#pragma unroll
            for (int c = 0; c < CHUNKS; c += 2) {
              if (c == 0) {
                mma_s8<true>(hi, rk[c], rk[c + 1], qb[c][0], qb[c + 1][0]);
                mma_s8<true>(lo, rk[c], rk[c + 1], qb[c][1], qb[c + 1][1]);
              } else {
                mma_s8<false>(hi, rk[c], rk[c + 1], qb[c][0], qb[c + 1][0]);
                mma_s8<false>(lo, rk[c], rk[c + 1], qb[c][1], qb[c + 1][1]);
              }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] = __int2float_rn(hi[e] * 256 + lo[e]);
          }
          float x[4], top = -INFINITY;                                                   // scores less the reference
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            s[e] *= ks.x * qf[e];
            s[2 + e] *= ks.y * qf[e];
          }
          if (valid < 16) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (quad + (e >> 1) * 8 >= valid) s[e] = -INFINITY;
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            x[e] = s[e] - m[e & 1];
            top = fmaxf(top, x[e]);
          }
          const float vs_top = fmaxf(vs.x, vs.y);
          if (__any_sync(0xffffffffu, top > 15.f || vs_top * fmaxf(vinv[0], vinv[1]) > 1.f)) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float most = fmaxf(s[e], s[2 + e]) - 9.f;
#pragma unroll
              for (int d = 4; d < 32; d <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
              const float m_new = fmaxf(m[e], most), a = ex2(m[e] - m_new);
              m[e] = m_new;
              l[e] *= a;
              x[e] = s[e] - m_new;
              x[2 + e] = s[2 + e] - m_new;
              float product = fmaxf(ex2(x[e]) * vs.x, ex2(x[2 + e]) * vs.y);
#pragma unroll
              for (int d = 4; d < 32; d <<= 1) product = fmaxf(product, __shfl_xor_sync(0xffffffffu, product, d));
              const float v_old = inverse(vinv[e]);
              vinv[e] = inverse(values_reference(v_old, vs_top, product, a));
              const float keep = a * v_old * vinv[e];                                  // v_old shrinks no faster than a
#pragma unroll
              for (int c = 0; c < CHUNKS; ++c) {
                o[c][e] *= keep;
                o[c][2 + e] *= keep;
              }
            }
          }
          uint32_t w[2];
          {
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = ex2(x[e]);
            l[0] += x[0] + x[2];
            l[1] += x[1] + x[3];
            w[0] = transpose8x8(half2_bits(x[0] * (vs.x * vinv[0]), x[1] * (vs.x * vinv[1])));
            w[1] = transpose8x8(half2_bits(x[2] * (vs.y * vinv[0]), x[3] * (vs.y * vinv[1])));
          }
          // what lies behind the last position may be NaN, which a weight of zero does not make zero
          uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;
          if (E4M3 && valid < 16) {
            keep0 = (2 * tq < valid ? 0xffffu : 0u) | (2 * tq + 1 < valid ? 0xffff0000u : 0u);
            keep1 = (2 * tq + 8 < valid ? 0xffffu : 0u) | (2 * tq + 9 < valid ? 0xffff0000u : 0u);
          }
#pragma unroll
          for (int c = 0; c < CHUNKS; ++c) {
            uint32_t a[4];
            if (E4M3) { rv[c][0] &= keep0; rv[c][1] &= keep1; }
            widen<E4M3, true>(rv[c][0], a[0], a[1]);
            widen<E4M3, true>(rv[c][1], a[2], a[3]);
            mma_f16<false>(o[c], a[0], a[1], a[2], a[3], w[0], w[1]);
          }
        }
      }
      turn = t - t_end;

#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[e] += __shfl_xor_sync(0xffffffffu, l[e], d);
      if (!MANY) {
        mbar_wait_converged(o_empty, o_phase ^ 1, p.status, ST_TIMEOUT_EMPTY);         // those of the piece before have been read
        o_phase ^= 1;
      }
      // a lane's values of a head lie behind one another: dimensions 16 c + 2 quad and the next, for all c
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int h = 2 * tq + e;
        if (h >= mine) continue;
        float4* dst = reinterpret_cast<float4*>(sm_o + (warp * heads + h) * C::PITCH + quad * (2 * CHUNKS));
#pragma unroll
        for (int c = 0; c < CHUNKS; c += 2) dst[c / 2] = make_float4(o[c][e], o[c][2 + e], o[c + 1][e], o[c + 1][2 + e]);
        if (quad == 0) sm_ml[warp * heads + h] = make_float4(m[e], l[e], inverse(vinv[e]), 0.f);
      }
      if (!last && !MANY) {
        __syncwarp();
        if (lane == 0) mbar_arrive(o_full);
        continue;
      }
    } else {
      to = *piece;
      __syncwarp();
      if (lane == 0) mbar_arrive(q_done);
      if (last) {
        // Mostly the other piece of the job has long been there, at the start of the next CTA's range: then the consumers need neither write
        // theirs nor ask for the count when they are done.
        if (tid == 0 && t_beg != t_end && !(t_beg == 0 && t_end == to.nt)) {
          const Deal deal = s_deal;
          const int c0 = deal.cta(to.start), n = deal.cta(to.start + to.nt - 1) - c0 + 1;
          for (int i = 0; i < (1 << 20) && !*const_cast<volatile int*>(&s_end); ++i) {
            unsigned int there;
            asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(there) : "l"(p.counters + to.counter) : "memory");
            if (there == static_cast<unsigned int>(n) - 1) {
              s_ready_join[0] = c0;
              s_ready_join[1] = n;
              __threadfence_block();
              *const_cast<volatile int*>(&s_ready) = 1;
              break;
            }
            __nanosleep(200);
          }
        }
        return;
      }
      if (MANY) continue;
      if (!mbar_wait_warp(o_full, o_phase, p.status, ST_TIMEOUT_FULL)) return;
      o_phase ^= 1;
    }
    if (t_beg == t_end) return;                          // a CTA without units

    if (consumes) {
      to = *piece;
      __syncwarp();
      if (lane == 0 && MANY) mbar_arrive(q_done);
    }
    const bool whole = t_beg == 0 && t_end == to.nt;
    auto part_of = [&](int c) { return p.part + static_cast<size_t>(c) * (HEADS_MAX * (DH + 2)); };
    // item i: four values of a head, in the order in which the warps left them
    auto write_out = [&](int i, float4 v, float sum) {
      const int h = i / (DH / 4), j = i % (DH / 4), d = 32 * (j % (CHUNKS / 2)) + 2 * (j / (CHUNKS / 2));
      const float inv = len > 0 ? 1.f / sum : 0.f;
      __nv_bfloat16* dst = p.out + to.b * p.ldo + static_cast<long long>(to.h0 + h) * DH + d;
      *reinterpret_cast<uint32_t*>(dst) = pack_bf16x2(v.x * inv, v.y * inv);
      *reinterpret_cast<uint32_t*>(dst + 16) = pack_bf16x2(v.z * inv, v.w * inv);
    };
    const int items = live * (DH / 4);
    // The pieces of a job are joined in shares, piece i in share i % shares, and these in their order; how many there are follows from the
    // heads (as many as the consumers have threads for). So which CTA does it, and which of its warps, does not show in the result.
    const int shares = items <= 96 ? 4 : items <= 192 ? 2 : 1;
    bool ready = false;                                  // all other pieces are there
    if (consumes) {
      if (tid == 0 && last) {
        *const_cast<volatile int*>(&s_end) = 1;
        s_ready_now = *const_cast<volatile int*>(&s_ready);
      }
      team_sync();
      ready = last && s_ready_now;
    }
    const int r_c0 = s_ready_join[0], r_own = static_cast<int>(blockIdx.x) - r_c0, r_pieces = ready ? s_ready_join[1] : 0;
    ready = ready && r_pieces <= (shares == 1 ? SHARES : shares);      // a piece a share, or one share: they can be joined at once
    // ---- the warps' sums are joined in the order of the warps ----
    constexpr int WARPS = MANY ? 4 : CONSUMERS;              // of a set
    for (int base = tid & ~31; base < items; base += team) {
      const int i = min(base + lane, items - 1), h = i / (DH / 4), set = (h >= heads) + (h >= 2 * heads), at = h - set * heads;
      const int from = MANY ? 4 * set : 0, x = lane & 15;
      float4 other[SHARES];
      float2 other_ml[SHARES];
#pragma unroll
      for (int k = 0; k < SHARES; ++k) {
        other_ml[k] = make_float2(LOWEST, 0.f);
        other[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (ready && k < r_pieces && k != r_own) {
          const float* src = part_of(2 * (r_c0 + k) + (k == 0));
          other_ml[k] = __ldcg(reinterpret_cast<const float2*>(src + HEADS_MAX * DH + 2 * h));
          other[k] = __ldcg(reinterpret_cast<const float4*>(src + i * 4));
        }
      }
      // lane x has the weight of warp x; all sums are under way while the weights are worked out
      const float4 ml = x < WARPS ? sm_ml[(from + x) * heads + at] : make_float4(LOWEST, 0.f, 0.f, 0.f);
      const float* src = sm_o + (from * heads + at) * C::PITCH + i % (DH / 4) * 4;
      float4 e[WARPS];
#pragma unroll
      for (int k = 0; k < WARPS; ++k) e[k] = *reinterpret_cast<const float4*>(src + k * (heads * C::PITCH));
      float top = ml.x;
#pragma unroll
      for (int d = 1; d < 16; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
      // both 2^-24 times as large: a value near the largest number would leave the range beside a weight of 2^9 and more
      const float a = ex2(ml.x - top), weight = a * (ml.z * 0x1p-24f);
      float sum = a * (ml.y * 0x1p-24f);
#pragma unroll
      for (int d = 1; d < 16; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < WARPS; ++k) {
        const float w = __shfl_sync(0xffffffffu, weight, (lane & 16) + k);
        v.x += e[k].x * w; v.y += e[k].y * w; v.z += e[k].z * w; v.w += e[k].w * w;
      }
      if (ready) {
#pragma unroll
        for (int k = 0; k < SHARES; ++k)
          if (k == r_own) { other_ml[k] = make_float2(top, sum); other[k] = v; }
        join_shares(other_ml, other, v, sum);
      }
      if (base + lane >= items) continue;
      if (whole || ready) {
        write_out(i, v, sum);
      } else {
        float* dst = part_of(2 * blockIdx.x + (t_beg == 0));
        *reinterpret_cast<float4*>(dst + i * 4) = v;
        if (i % (DH / 4) == 0) *reinterpret_cast<float2*>(dst + HEADS_MAX * DH + 2 * h) = make_float2(top, sum);
      }
    }
    if (ready) {
      if (tid == 0) p.counters[to.counter] = 0;
      return;
    }
    if (whole && last) return;
    team_sync();
    if (!consumes && tid == 0) mbar_arrive(o_empty);
    if (whole) continue;
    // ---- the CTA that ends last joins the pieces, in the order of the tiles ----
    if (tid == 0) {
      unsigned int before;
      asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(before) : "l"(p.counters + to.counter) : "memory");
      const Deal deal = s_deal;                          // while the count is under way
      const int c0 = deal.cta(to.start), n = deal.cta(to.start + to.nt - 1) - c0 + 1;
      s_join[consumes][0] = c0;
      s_join[consumes][1] = n;
      s_last[consumes] = before == static_cast<unsigned int>(n) - 1;
      if (s_last[consumes]) p.counters[to.counter] = 0;
    }
    team_sync();
    if (!s_last[consumes]) continue;
    const int c0 = s_join[consumes][0], n_pieces = s_join[consumes][1];
    // item i of a share of the pieces: the loads of eight pieces are under way together
    auto join_share = [&](int i, int share, float2& ml, float4& v) {
      const int h = i / (DH / 4);
      ml = make_float2(LOWEST, 0.f);
      v = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int c = share; c < n_pieces; c += 8 * shares) {
        float2 next_ml[8];
        float4 next[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int at = c + k * shares;
          next_ml[k] = make_float2(LOWEST, 0.f);
          next[k] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (at < n_pieces) {
            const float* src = part_of(2 * (c0 + at) + (at == 0));
            next_ml[k] = __ldcg(reinterpret_cast<const float2*>(src + HEADS_MAX * DH + 2 * h));
            next[k] = __ldcg(reinterpret_cast<const float4*>(src + i * 4));
          }
        }
        float top = ml.x;
#pragma unroll
        for (int k = 0; k < 8; ++k) top = fmaxf(top, next_ml[k].x);
        const float keep = ex2(ml.x - top);
        ml.x = top;
        ml.y *= keep;
        v.x *= keep; v.y *= keep; v.z *= keep; v.w *= keep;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float a = ex2(next_ml[k].x - top);
          ml.y += next_ml[k].y * a;
          v.x += next[k].x * a; v.y += next[k].y * a; v.z += next[k].z * a; v.w += next[k].w * a;
        }
      }
    };
    float4* sm_v = reinterpret_cast<float4*>(sm_o);          // [shares][items], then [shares][live]
    float2* sm_vml = reinterpret_cast<float2*>(sm_v + shares * items);
    const bool spread = consumes && shares > 1;              // of the last piece: there is room where the sums were, which have been read
    if (spread) {
      if (tid < items * shares) {
        const int share = tid / items, i = tid - share * items;
        float2 ml;
        float4 v;
        join_share(i, share, ml, v);
        sm_v[tid] = v;
        if (i % (DH / 4) == 0) sm_vml[share * live + i / (DH / 4)] = ml;
      }
      team_sync();
    }
    for (int i = tid; i < items; i += team) {
      float2 ml[SHARES];
      float4 e[SHARES], v;
      float sum;
#pragma unroll
      for (int k = 0; k < SHARES; ++k) {
        ml[k] = make_float2(LOWEST, 0.f);
        e[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (spread && k < shares) {
          e[k] = sm_v[k * items + i];
          ml[k] = sm_vml[k * live + i / (DH / 4)];
        }
      }
      if (!spread) {
#pragma unroll 1
        for (int k = 0; k < shares; ++k) {
          float2 next_ml;
          float4 next;
          join_share(i, k, next_ml, next);
#pragma unroll
          for (int x = 0; x < SHARES; ++x)
            if (x == k) { ml[x] = next_ml; e[x] = next; }
        }
      }
      join_shares(ml, e, v, sum);
      write_out(i, v, sum);
    }
    if (consumes && !last) team_sync();                      // the next piece's sums go where the shares were
  }
}

template <int DH, bool E4M3, bool MANY, bool SMALL>
static int launch_kind(const CUtensorMap& tm, AttendParams p, int grid, cudaStream_t s) {
  using C = Cfg<DH>;
  static PerDeviceOnce attr;
  if (allow_smem(attr, attend_kernel<DH, E4M3, MANY, SMALL>, SMEM, SB_ERR_LAUNCH)) return SB_ERR_LAUNCH;
  p.stages = C::stages(p.sets, p.heads, p.B);
  return launch_dep(attend_kernel<DH, E4M3, MANY, SMALL>, dim3(grid), dim3(C::THREADS), C::smem_bytes(p.sets, p.heads, p.B), s, tm, p) == cudaSuccess
             ? 0 : SB_ERR_LAUNCH;
}

template <int DH, bool E4M3>
static int launch_attend(const CUtensorMap& tm, const AttendParams& p, int grid, cudaStream_t s) {
  // A box takes one warp some 90 cycles to ask for, whatever its size: a tile of four or more is shared by the two producers. us for one /
  // two asking, 64 sequences of up to 2304 positions, 8 heads of 128, pages of 8 65.9 / 58.2, 16 52.4 / 50.3, 32 (two boxes) 46.5 / 47.1;
  // 4 heads of 64, pages of 8 36.6 / 29.8, 16 25.9 / 22.9, 32 21.0 / 19.8, 64 (two boxes) 18.6 / 18.4.
  const bool small = (Cfg<DH>::TK >> p.page_bits) >= 4;
  if (p.sets > 1) return small ? launch_kind<DH, E4M3, true, true>(tm, p, grid, s) : launch_kind<DH, E4M3, true, false>(tm, p, grid, s);
  return small ? launch_kind<DH, E4M3, false, true>(tm, p, grid, s) : launch_kind<DH, E4M3, false, false>(tm, p, grid, s);
}

}  // namespace kv8
}  // namespace sb

using namespace sb;

// Floats of `part` for launches on the current device at head dimension dh.
extern "C" int sb_quant_kv_attention_floats(int dh) { return 2 * num_sms() * kv8::HEADS_MAX * (dh + 2); }

// q: [B, ldq] bf16 (H * dh used, rotated), out: [B, ldo] bf16, rows 16-byte aligned. A sequence of no positions gets zeros; ids outside the
// pool count as zeros. page 8, 16, 32 or a multiple of 64; B <= 1024. max_tiles: an upper bound of the 64-position tiles of all
// jobs, which only caps the grid. counters: B * Hkv * ceil(H / Hkv / 24) words, zero before the first call (every call leaves them zero).
extern "C" int sb_quant_kv_attention(const void* q, long long ldq, const void* codes, int e4m3, const float* scales, int n_blocks, int page,
                                     int block, const int* table, int max_blocks, const int* seq_len, int B, int H, int Hkv, int dh,
                                     long long max_tiles, float scale, float* part, unsigned int* counters, void* out, long long ldo,
                                     int* status, void* stream_) {
  if (!q || !codes || !scales || !table || !seq_len || !out || !part || !counters || !status || B <= 0 || B > kv8::MAX_B || H <= 0 ||
      max_blocks <= 0 || max_tiles <= 0 || !kv8::layout_ok(Hkv, dh, n_blocks, page, block) || H % Hkv)
    return SB_ERR_ARG;
  if (page != 8 && page != 16 && page != 32 && page % 64) return SB_ERR_ARG;
  if ((reinterpret_cast<uintptr_t>(q) & 15) || (reinterpret_cast<uintptr_t>(out) & 15) || (ldq & 7) || (ldo & 7)) return SB_ERR_ALIGN;
  if (static_cast<double>(n_blocks) * 2 * Hkv * (page / block) > 2147483647.0 || static_cast<double>(Hkv) * page > 2147483647.0)
    return SB_ERR_TOO_LARGE;
  CUtensorMap tm;
  const int rc = make_tmap_3d_u8_rows(&tm, codes, dh, static_cast<uint64_t>(Hkv) * page, static_cast<uint64_t>(n_blocks) * 2,
                                      page < 64 ? page : 64, 2);
  if (rc) return rc;
  kv8::AttendParams p;
  p.q = static_cast<const __nv_bfloat16*>(q); p.ldq = ldq;
  p.scales = scales;
  p.n_blocks = n_blocks; p.page = page;
  for (p.page_bits = 3; p.page_bits < 6 && (1 << p.page_bits) < page;) ++p.page_bits;
  p.page_shift = -1;
  if (!(page & (page - 1)))
    for (p.page_shift = 3; (1 << p.page_shift) < page;) ++p.page_shift;
  for (p.block_bits = 3; (1 << p.block_bits) < block;) ++p.block_bits;
  p.table = table; p.max_blocks = max_blocks; p.seq_len = seq_len;
  p.B = B; p.Hkv = Hkv; p.G = H / Hkv;
  p.subs = (p.G + kv8::HEADS_MAX - 1) / kv8::HEADS_MAX;
  const int per_job = (p.G + p.subs - 1) / p.subs;
  p.sets = (per_job + kv8::SET - 1) / kv8::SET;
  p.heads = (per_job + p.sets - 1) / p.sets;
  const double most = static_cast<double>(B) * ((static_cast<double>(max_blocks) * page + 63) / 64) * Hkv * p.subs;
  if (most > 2147483647.0) return SB_ERR_TOO_LARGE;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.part = part; p.counters = counters;
  p.out = static_cast<__nv_bfloat16*>(out); p.ldo = ldo;
  p.status = status;
  // the kernel leaves a tile to each group of consumers
  const long long shared = p.sets == 1 ? (max_tiles + 2) / 3 : max_tiles, jobs = static_cast<long long>(B) * Hkv * p.subs;
  const long long want = shared > jobs ? shared : jobs;
  const int grid = want < num_sms() ? static_cast<int>(want) : num_sms();
  cudaStream_t s = static_cast<cudaStream_t>(stream_);
  if (dh == 64) return e4m3 ? kv8::launch_attend<64, true>(tm, p, grid, s) : kv8::launch_attend<64, false>(tm, p, grid, s);
  return e4m3 ? kv8::launch_attend<128, true>(tm, p, grid, s) : kv8::launch_attend<128, false>(tm, p, grid, s);
}

// The capture that `stream` is in, 0 where it is in none: what a graph's launches share is apart from every other graph's.
extern "C" int sb_stream_capture_id(void* stream_, unsigned long long* id) {
  cudaStreamCaptureStatus status;
  unsigned long long capture = 0;
  if (!id || cudaStreamGetCaptureInfo(static_cast<cudaStream_t>(stream_), &status, &capture) != cudaSuccess) return SB_ERR_RUNTIME;
  *id = status == cudaStreamCaptureStatusActive ? capture : 0;
  return 0;
}
