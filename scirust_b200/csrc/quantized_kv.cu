// Paged KV cache in 8 bits: keys and values quantised as they are written, and pages read back in bf16.
//
// A pool is codes [n_blocks, 2 (k|v), Hkv, page, dh], int8 or e4m3, and scales [n_blocks, 2, Hkv, page / block] in fp32; `block` consecutive
// positions of a head share one, and a value is code * scale. The scale is the smallest power of two that holds the block's largest magnitude
// m, with k = floor(log2 m): 2^(k-6) for int8 (127 steps; what lies above 127 of them is less than half a step off), for e4m3 the least
// with 448 * scale >= m. A power of two costs int8 up to one of its eight bits, and makes everything after it exact: x / scale, a block's
// rescaling by a ratio of scales (e4m3 loses nothing by it, but below its smallest normal value), and the value in bf16. Since a block of
// positions fills up over many calls, its scale can grow: what it holds is then rounded to the new steps. The steps at least double each
// time, so that a code is off by less than one of its last steps, however often. A block that is given an infinity or a NaN gets NaN as its
// scale and keeps it until its first position is written again: what the format cannot hold is not lost silently.
#include <cuda_bf16.h>
#include "api.h"
#include "dependent.cuh"
#include "quantized_kv.cuh"
#include "sm100_ptx.cuh"

namespace sb {
int num_sms();                                                                 // gemm_tcgen05.cu

namespace kv8 {

// ---- writing -------------------------------------------------------------------------------------------------------------------
// A warp takes one key or value head of a chunk of rows (or several, where there are more than enough warps) and walks over the blocks of
// positions that begin in it; a block's rows that reach into the next chunk are its own. Which sequence and position a row has follows from cu_q and seq_len, so that no two warps can write one
// block. Sixteen rows at a time stay in registers between the maximum and the codes; of larger blocks the rows are read twice, the second
// time from L2. Query heads are only turned: a warp has one row, or as many as fill it, with their part of the rotation's table in registers
// for a quarter of the heads.
// Bound by memory for prompts and by latency for single tokens.
constexpr int WARPS = 4;

struct AppendParams {
  __nv_bfloat16* qkv; long long ld;
  int n, H, Hkv;
  const float *cos_t, *sin_t; int n_pos;       // null: the rows hold what is to be written
  uint8_t* codes; float* scales;
  int n_blocks, page, block;
  const int* table; int max_blocks;
  const int *seq_len, *cu_q;                   // cu_q null: row b is sequence b's only one
  int B, chunk;
  int head_ctas, kv_ctas;                      // CTAs of a chunk's key and value heads, and of all chunks; queries' CTAs come behind
};

// The sequence that row t belongs to: how many of cu[1 .. B] are at most t, by steps of a 32nd of what is left.
__device__ __forceinline__ int find_sequence(const int* cu, int B, int t) {
  const int lane = threadIdx.x & 31;
  int lo = 0, n = B;
  while (n > 0) {
    const int step = (n + 31) / 32, at = lo + (lane + 1) * step;
    const int c = __popc(__ballot_sync(0xffffffffu, at <= lo + n && cu[at] <= t));
    lo += c * step;
    n = min(step - 1, n - c * step);
  }
  return lo;
}

// Products and their sum are rounded one by one: fused, a value that lies between two of bf16 may go the other way than in the formula's
// plain evaluation, and take a code with it.
__device__ __forceinline__ uint32_t rotate(uint32_t x, float c, float s) {
  const float a = bf16_lo(x), b = bf16_hi(x);
  return pack_bf16x2(__fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s)), __fadd_rn(__fmul_rn(a, s), __fmul_rn(b, c)));
}

template <bool E4M3>
__device__ __forceinline__ uint32_t to_codes(float a, float b, float c, float d) {
  if constexpr (E4M3) {
    return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3) |
           static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3)) << 16;
  } else {
    // 1.5 * 2^23 + x is rounded to a whole number, whose last byte is x's (a conversion takes four times as long)
    auto code = [](float x) { return __float_as_uint(fminf(fmaxf(x, -127.f), 127.f) + 12582912.f); };
    return __byte_perm(__byte_perm(code(a), code(b), 0x0040), __byte_perm(code(c), code(d), 0x0040), 0x5410);
  }
}

// The scale that a largest magnitude needs, from its bits in bf16 (NaN and infinity have the largest ones). From 1.9375 * 2^127 on e4m3
// would round to 2^128, an infinity.
template <bool E4M3>
__device__ __forceinline__ float scale_for(uint32_t bits) {
  if (bits >= (E4M3 ? 0x7f78u : 0x7f80u)) return __uint_as_float(0x7fffffffu);
  int k = static_cast<int>(bits >> 7) - 127, more = (bits & 0x7f) > 0x60;       // above 1.75 * 2^k
  if (k < -90) { k = -90; more = 0; }                                          // no scale, and no ratio of two, leaves the normal numbers
  const int e = E4M3 ? k - 8 + more : k - 6;
  return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

struct Place { int rows, pos; };               // rows of a sequence from some row on, the first one's position; rows 0: that has no place

// Where row t of sequence b is, which its first row is not behind and which has more.
__device__ __forceinline__ Place place_of(const AppendParams& p, int b, int t, int stop, int& skip) {
  const int rows = min(stop, p.n) - t;
  const long long at = static_cast<long long>(p.seq_len[b]) - (stop - t);
  long long limit = min(static_cast<long long>(p.max_blocks) * p.page, 0x7fffffffll);
  if (p.cos_t) limit = min(limit, static_cast<long long>(p.n_pos));
  if (at < 0 || at >= limit) {
    skip = at < 0 ? static_cast<int>(min(-at, static_cast<long long>(rows))) : rows;
    return {0, 0};
  }
  return {min(rows, static_cast<int>(limit - at)), static_cast<int>(at)};
}

__device__ __forceinline__ uint4 rotate8(uint4 v, const float4& c, const float4& s) {
  return make_uint4(rotate(v.x, c.x, s.x), rotate(v.y, c.y, s.y), rotate(v.z, c.z, s.z), rotate(v.w, c.w, s.w));
}

template <int DH>
__device__ __forceinline__ void turn_queries(const AppendParams& p, int cta) {
  constexpr int LANES = DH / 8, ROWS = 32 / LANES, AHEAD = 8;                  // lanes of a row, rows of a warp, heads under way
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane / LANES, ch = lane % LANES;
  const int t0 = cta * ROWS, t = t0 + sub;
  __nv_bfloat16* x = p.qkv + min(t, p.n - 1) * p.ld + ch * 8;
  uint4 v[AHEAD];
  auto load = [&](int h0) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (h0 + i * WARPS < p.H) v[i] = *reinterpret_cast<const uint4*>(x + (h0 + i * WARPS) * DH);
  };
  load(warp);                                  // while the row's place is looked for
  int b = p.cu_q ? find_sequence(p.cu_q, p.B, t0) : t;
  if (t >= p.n) return;
  int stop = t + 1;
  if (p.cu_q) {
    while (b < p.B && p.cu_q[b + 1] <= t) ++b;
    if (b >= p.B || t < p.cu_q[b]) return;
    stop = p.cu_q[b + 1];
  } else if (b >= p.B) {
    return;
  }
  int skip;
  const Place at = place_of(p, b, t, stop, skip);
  if (at.rows == 0) return;
  const size_t a = static_cast<size_t>(at.pos) * (DH / 2) + ch * 4;
  const float4 c = *reinterpret_cast<const float4*>(p.cos_t + a), s = *reinterpret_cast<const float4*>(p.sin_t + a);
  for (int h0 = warp;;) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (h0 + i * WARPS < p.H) *reinterpret_cast<uint4*>(x + (h0 + i * WARPS) * DH) = rotate8(v[i], c, s);
    h0 += WARPS * AHEAD;
    if (h0 >= p.H) break;
    load(h0);
  }
}

// BATCH: rows at a time, 8 for blocks of 8 and else 16
template <int DH, bool E4M3, int BATCH>
__global__ void __launch_bounds__(WARPS * 32, 6) append_kernel(const __grid_constant__ AppendParams p) {
  constexpr int LANES = DH / 8, ROWS = 32 / LANES, WORDS = BATCH / ROWS;       // lanes of a row, rows of a load, loads of a batch
  pdl_trigger();
  pdl_wait();
  if (static_cast<int>(blockIdx.x) >= p.kv_ctas) {
    turn_queries<DH>(p, blockIdx.x - p.kv_ctas);
    return;
  }
  const int lane = threadIdx.x & 31, sub = lane / LANES, ch = lane % LANES;
  const int chunk = blockIdx.x / p.head_ctas, first_head = (blockIdx.x - chunk * p.head_ctas) * WARPS + (threadIdx.x >> 5);
  if (first_head >= 2 * p.Hkv) return;
  int t = chunk * p.chunk;
  const int end = min(p.n - t, p.chunk) + t;
  int b = p.cu_q ? find_sequence(p.cu_q, p.B, t) : t;
  while (t < end) {
    int start = t, stop = t + 1;                                               // rows of the sequence
    if (p.cu_q) {
      while (b < p.B && p.cu_q[b + 1] <= t) ++b;
      if (b >= p.B) return;
      start = p.cu_q[b];
      stop = p.cu_q[b + 1];
      if (t < start) { t = start; continue; }
    } else {
      b = t;
      if (b >= p.B) return;
    }
    int skip;
    const Place place = place_of(p, b, t, stop, skip);
    if (place.rows == 0) { t += skip; continue; }
    const int pos = place.pos, off = pos & (p.block - 1), cnt = min(p.block - off, place.rows), t0 = t;
    t += cnt;
    if (off && t0 != start) continue;                                          // a block that began in an earlier chunk

    const int at = pos / p.page, slot = pos - at * p.page, id = p.table[static_cast<size_t>(b) * p.max_blocks + at];
    const bool known = static_cast<unsigned>(id) < static_cast<unsigned>(p.n_blocks);
    for (int head = first_head; head < 2 * p.Hkv; head += p.head_ctas * WARPS) {
      const int kv = head >= p.Hkv, h = head - kv * p.Hkv;
      const bool turns = p.cos_t && !kv;
      __nv_bfloat16* x = p.qkv + (t0 + sub) * p.ld + (p.H + head) * DH + ch * 8;
      uint4 v[WORDS];
      auto load = [&](int r0) {
#pragma unroll
        for (int i = 0; i < WORDS; ++i) {
          v[i] = make_uint4(0, 0, 0, 0);
          if (r0 + i * ROWS + sub < cnt) v[i] = *reinterpret_cast<const uint4*>(x + (r0 + i * ROWS) * p.ld);
        }
      };
      load(0);
      // while the rows are under way: the scale of what the block holds
      const size_t row = (static_cast<size_t>(known ? id : 0) * 2 + kv) * p.Hkv + h;
      float* scale_at = p.scales + row * (p.page / p.block) + slot / p.block;
      const float old = off && known ? *scale_at : 0.f;
      uint32_t top = 0;
      for (int r0 = 0; r0 < cnt; r0 += BATCH) {
        if (r0) load(r0);
        if (turns) {
          const size_t a = static_cast<size_t>(pos + r0 + sub) * (DH / 2) + ch * 4;
#pragma unroll
          for (int i = 0; i < WORDS; ++i) {
            const bool in = r0 + i * ROWS + sub < cnt;
            float4 c = make_float4(0, 0, 0, 0), s = c;
            if (in) c = *reinterpret_cast<const float4*>(p.cos_t + a + i * ROWS * (DH / 2)), s = *reinterpret_cast<const float4*>(p.sin_t + a + i * ROWS * (DH / 2));
            v[i] = rotate8(v[i], c, s);
            if (in) *reinterpret_cast<uint4*>(x + (r0 + i * ROWS) * p.ld) = v[i];
          }
        }
#pragma unroll
        for (int i = 0; i < WORDS; ++i)
          top = max16x2(top, max16x2(max16x2(v[i].x & 0x7fff7fffu, v[i].y & 0x7fff7fffu), max16x2(v[i].z & 0x7fff7fffu, v[i].w & 0x7fff7fffu)));
      }
      if (!known) continue;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) top = max16x2(top, __shfl_xor_sync(0xffffffffu, top, o));
      top = max(top & 0xffffu, top >> 16);
      const float need = scale_for<E4M3>(top);
      const float scale = off && (old > need || old != old) ? old : need;
      if (lane == 0) *scale_at = scale;                                          // all lanes have read it: they have met since
      const bool holds = scale == scale;
      const float inv = 1.f / scale;
      uint8_t* dst = p.codes + (row * p.page + slot) * DH;
      for (int r0 = 0; r0 < cnt; r0 += BATCH) {
        if (cnt > BATCH) load(r0);
#pragma unroll
        for (int i = 0; i < WORDS; ++i) {
          uint2 c;
          c.x = to_codes<E4M3>(bf16_lo(v[i].x) * inv, bf16_hi(v[i].x) * inv, bf16_lo(v[i].y) * inv, bf16_hi(v[i].y) * inv);
          c.y = to_codes<E4M3>(bf16_lo(v[i].z) * inv, bf16_hi(v[i].z) * inv, bf16_lo(v[i].w) * inv, bf16_hi(v[i].w) * inv);
          if (!holds) c = make_uint2(0, 0);
          if (r0 + i * ROWS + sub < cnt) *reinterpret_cast<uint2*>(dst + (r0 + i * ROWS + sub) * DH + ch * 8) = c;
        }
      }
      if (off && holds && old != scale) {                                        // what the block holds, in the new steps
        const float ratio = old * inv;
        uint4* before = reinterpret_cast<uint4*>(dst - off * DH);
#pragma unroll 4
        for (int i = lane; i < off * (DH / 16); i += 32) {
          uint4 w = before[i];
          uint32_t* e = &w.x;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float4 f = from_codes<E4M3>(e[j]);
            e[j] = to_codes<E4M3>(f.x * ratio, f.y * ratio, f.z * ratio, f.w * ratio);
          }
          before[i] = w;
        }
      }
    }
  }
}

// ---- reading back --------------------------------------------------------------------------------------------------------------
// A page's codes and its values in bf16 lie in the same order, and the scale of an element is the one at its index / (block * dh). A thread
// expands sixteen codes. Bound by memory: one byte read and two written an element.
struct ReadParams {
  const uint8_t* codes; const float* scales;
  const int* pages; int n, n_blocks;
  long long page_words;                        // 16 codes each
  int shift;                                   // log2 of the words that share a scale
  int page_scales;
  __nv_bfloat16* out;
};

template <bool E4M3>
__global__ void __launch_bounds__(256) read_kernel(const __grid_constant__ ReadParams p) {
  pdl_trigger();
  pdl_wait();
  const long long w = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  if (w >= p.page_words) return;
  for (int i = blockIdx.y; i < p.n; i += gridDim.y) {
    const int id = p.pages[i];
    uint4 o[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
    if (static_cast<unsigned>(id) < static_cast<unsigned>(p.n_blocks)) {
      const uint4 c = *(reinterpret_cast<const uint4*>(p.codes) + id * p.page_words + w);
      const float s = p.scales[static_cast<size_t>(id) * p.page_scales + (w >> p.shift)];
      const float4 f0 = from_codes<E4M3>(c.x), f1 = from_codes<E4M3>(c.y), f2 = from_codes<E4M3>(c.z), f3 = from_codes<E4M3>(c.w);
      o[0] = make_uint4(pack_bf16x2(f0.x * s, f0.y * s), pack_bf16x2(f0.z * s, f0.w * s), pack_bf16x2(f1.x * s, f1.y * s),
                        pack_bf16x2(f1.z * s, f1.w * s));
      o[1] = make_uint4(pack_bf16x2(f2.x * s, f2.y * s), pack_bf16x2(f2.z * s, f2.w * s), pack_bf16x2(f3.x * s, f3.y * s),
                        pack_bf16x2(f3.z * s, f3.w * s));
    }
    uint4* dst = reinterpret_cast<uint4*>(p.out) + (i * p.page_words + w) * 2;
    dst[0] = o[0];
    dst[1] = o[1];
  }
}

}  // namespace kv8
}  // namespace sb

using namespace sb;

// qkv: [n, ld] bf16, H + 2 Hkv heads a row, 16-byte aligned rows; with cos_t and sin_t ([n_pos, dh / 2]) its query and key heads are rotated
// in place first. Sequence b has rows cu_q[b] .. cu_q[b + 1] - 1 (without cu_q row b), its last positions of seq_len[b]. Rows without a
// place (in front of position 0, behind the table or the rotation's, of no sequence) stay as they are; ids outside the pool are skipped.
// chunk: rows a warp looks for blocks in.
extern "C" int sb_quant_kv_append(void* qkv, long long ld, int n, int H, int Hkv, int dh, const float* cos_t, const float* sin_t, int n_pos,
                                  void* codes, int e4m3, float* scales, int n_blocks, int page, int block, const int* table, int max_blocks,
                                  const int* seq_len, const int* cu_q, int B, int chunk, void* stream_) {
  if (!qkv || !codes || !scales || !table || !seq_len || n <= 0 || H < 0 || B <= 0 || max_blocks <= 0 || chunk <= 0 || !cos_t != !sin_t ||
      !kv8::layout_ok(Hkv, dh, n_blocks, page, block))
    return SB_ERR_ARG;
  const uintptr_t all = reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(cos_t) |
                        reinterpret_cast<uintptr_t>(sin_t);
  if ((all & 15) || (ld & 7)) return SB_ERR_ALIGN;
  kv8::AppendParams p;
  p.qkv = static_cast<__nv_bfloat16*>(qkv); p.ld = ld; p.n = n; p.H = H; p.Hkv = Hkv;
  p.cos_t = cos_t; p.sin_t = sin_t; p.n_pos = n_pos;
  p.codes = static_cast<uint8_t*>(codes); p.scales = scales;
  p.n_blocks = n_blocks; p.page = page; p.block = block;
  p.table = table; p.max_blocks = max_blocks; p.seq_len = seq_len; p.cu_q = cu_q; p.B = B; p.chunk = chunk;
  const long long chunks = (static_cast<long long>(n) + chunk - 1) / chunk, rows = 256 / dh;                     // rows of a warp of queries
  // A warp finds its place by five loads, each of which waits for the one before: beyond two rounds of CTAs it takes more heads with that.
  const long long most = (2 * Hkv + kv8::WARPS - 1) / kv8::WARPS, rounds = chunks * most / (num_sms() * 12ll);
  p.head_ctas = static_cast<int>(rounds < 2 ? most : rounds < most ? (most + rounds - 1) / rounds : 1);
  const long long kv_ctas = chunks * p.head_ctas, ctas = kv_ctas + (cos_t && H ? (n + rows - 1) / rows : 0);
  if (ctas > 0x7fffffffll) return SB_ERR_TOO_LARGE;
  p.kv_ctas = static_cast<int>(kv_ctas);
  const dim3 grid(static_cast<unsigned>(ctas));
  using Kernel = void (*)(kv8::AppendParams);
  static const Kernel kernels[8] = {kv8::append_kernel<64, false, 16>, kv8::append_kernel<64, false, 8>, kv8::append_kernel<64, true, 16>,
                                    kv8::append_kernel<64, true, 8>, kv8::append_kernel<128, false, 16>, kv8::append_kernel<128, false, 8>,
                                    kv8::append_kernel<128, true, 16>, kv8::append_kernel<128, true, 8>};
  const Kernel kern = kernels[(dh == 128) * 4 + (e4m3 != 0) * 2 + (block == 8)];
  return launch_dep(kern, grid, dim3(kv8::WARPS * 32), 0, static_cast<cudaStream_t>(stream_), p) == cudaSuccess ? 0 : SB_ERR_LAUNCH;
}

// out [n, 2, Hkv, page, dh] bf16: the pages' values; zeros for ids outside the pool.
extern "C" int sb_quant_kv_read(const void* codes, int e4m3, const float* scales, int n_blocks, int Hkv, int page, int block, int dh,
                                const int* pages, int n, void* out, void* stream_) {
  if (!codes || !scales || !pages || !out || n <= 0 || !kv8::layout_ok(Hkv, dh, n_blocks, page, block)) return SB_ERR_ARG;
  if ((reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(out)) & 15) return SB_ERR_ALIGN;
  kv8::ReadParams p;
  p.codes = static_cast<const uint8_t*>(codes); p.scales = scales; p.pages = pages; p.n = n; p.n_blocks = n_blocks;
  p.page_words = 2ll * Hkv * page * dh / 16;
  p.shift = 0;
  while ((16 << p.shift) < block * dh) ++p.shift;
  p.page_scales = 2 * Hkv * (page / block);
  p.out = static_cast<__nv_bfloat16*>(out);
  if (p.page_words > (1ll << 31) * 256 - 256) return SB_ERR_TOO_LARGE;
  const dim3 grid(static_cast<unsigned>((p.page_words + 255) / 256), n < 65535 ? n : 65535);
  auto kern = e4m3 ? kv8::read_kernel<true> : kv8::read_kernel<false>;
  return launch_dep(kern, grid, dim3(256), 0, static_cast<cudaStream_t>(stream_), p) == cudaSuccess ? 0 : SB_ERR_LAUNCH;
}
