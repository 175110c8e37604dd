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
#include <type_traits>
#include "api.h"
#include "dependent.cuh"
#include "quantized_kv.cuh"
#include "sm100_ptx.cuh"

namespace sb {
int num_sms();                                                                 // gemm_tcgen05.cu

namespace kv8 {

// ---- writing -------------------------------------------------------------------------------------------------------------------
// A warp, or two that exchange their maxima, takes one key or value head of a chunk of rows and walks over the blocks of positions that begin
// in it; a block's rows that reach into the next chunk are its own. Which sequence and position a row has follows from cu_q and seq_len and is
// looked for once a sequence and chunk (once a block: 17.2 for 15.4 us, for 16 sequences of 700 rows). No two warps can write one block. Eight
// rows a warp stay in registers between the maximum and the codes; of larger blocks the rows are read twice, the second time from L2. (The
// next block's or head's rows under way meanwhile take registers that more warps use better: 17.8 us.) Query heads are only turned: a warp has
// one row, or as many as fill it, with their part of the rotation's table in registers for a quarter of the heads.
// Bound by latency: 2.3 us for one token, 3.2 for one of each of 64 sequences of an 8B model. Runs of rows take longer than their bytes do, since a
// warp sees to its blocks one after the other, each a chain of loads, a maximum, codes and stores: a prompt of 2048 rows 11.0 us (0.72 of
// the copy rate), four of up to 1000 16.7 (0.80), 16 runs of up to 700 without rotation, 2080 CTAs for 1184 places, in blocks of 8 or 16
// 14.2 and 15.0 (0.55, 0.52), in blocks of 64, whose rows are read twice, 19.0 (0.41).
constexpr int HEADS = 4;                       // key or value heads of a CTA, with `SPLIT` warps each

struct AppendParams {
  __nv_bfloat16* qkv; long long ld;
  int n, H, Hkv;
  const float *cos_t, *sin_t; int n_pos;       // null: the rows hold what is to be written
  uint8_t* codes; float* scales;
  int n_blocks, page, block, block_bits, per_page;      // per_page: blocks of a page
  const int* table; int max_blocks;
  const int *seq_len, *cu_q;                   // cu_q null: row b is sequence b's only one
  int B, chunk;
  int head_ctas, kv_ctas;                      // CTAs of a chunk's key and value heads, and of all chunks; queries' CTAs come behind
};

// The sequence that row t belongs to: how many of cu[1 .. B] are at most t, by steps of a 32nd of what is left.
__device__ __forceinline__ int find_sequence(const int* cu, int B, int t) {
  const int lane = threadIdx.x & 31;
  if (B == 1) return cu[1] <= t;
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

// x * f as codes. int8: 1.5 * 2^23 + x is rounded to a whole number, whose last byte is x's (a conversion takes four times as long); CLAMP: it
// may be 128.
template <bool E4M3, bool CLAMP>
__device__ __forceinline__ uint32_t to_codes(float a, float b, float c, float d, float f) {
  if constexpr (E4M3) {
    return __nv_cvt_float2_to_fp8x2(make_float2(a * f, b * f), __NV_SATFINITE, __NV_E4M3) |
           static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(c * f, d * f), __NV_SATFINITE, __NV_E4M3)) << 16;
  } else {
    auto code = [f](float x) {
      return __float_as_uint(CLAMP ? fminf(fmaxf(x * f, -127.f), 127.f) + 12582912.f : fmaf(x, f, 12582912.f));
    };
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

struct Place { int start, stop, rows, pos; };  // a sequence's rows; from some row on, those that have a place and the first one's position

// Where row t of sequence b is. Where it has no place, `rows` is 0 and `skip` how many rows have none.
__device__ __forceinline__ Place place_of(const AppendParams& p, int b, int t, int& skip) {
  Place at = {t, t + 1, 0, 0};
  const int len = p.seq_len[b];                // three loads that do not wait for one another
  if (p.cu_q) { at.start = p.cu_q[b]; at.stop = p.cu_q[b + 1]; }
  if (t < at.start) { skip = at.start - t; return at; }
  const int rows = min(at.stop, p.n) - t;
  if (rows <= 0) { skip = 1; return at; }      // offsets that do not ascend
  const long long pos = static_cast<long long>(len) - (at.stop - t);
  long long limit = min(static_cast<long long>(p.max_blocks) * p.page, 0x7fffffffll);
  if (p.cos_t) limit = min(limit, static_cast<long long>(p.n_pos));
  if (pos < 0 || pos >= limit) {
    skip = pos < 0 ? static_cast<int>(min(-pos, static_cast<long long>(rows))) : rows;
    return at;
  }
  at.rows = min(rows, static_cast<int>(limit - pos));
  at.pos = static_cast<int>(pos);
  return at;
}

__device__ __forceinline__ uint4 rotate8(uint4 v, const float4& c, const float4& s) {
  return make_uint4(rotate(v.x, c.x, s.x), rotate(v.y, c.y, s.y), rotate(v.z, c.z, s.z), rotate(v.w, c.w, s.w));
}

template <int DH>
__device__ __forceinline__ void turn_queries(const AppendParams& p, int team, int warp) {
  constexpr int WARPS = HEADS;
  constexpr int LANES = DH / 8, ROWS = 32 / LANES, AHEAD = 8;                  // lanes of a row, rows of a warp, heads under way
  const int lane = threadIdx.x & 31, sub = lane / LANES, ch = lane % LANES;
  const int t0 = team * ROWS, t = t0 + sub;
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
  if (p.cu_q && t > t0)
    while (b < p.B && p.cu_q[b + 1] <= t) ++b;
  if (b >= p.B) return;
  int skip;
  const Place at = place_of(p, b, t, skip);
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

template <int DH, bool E4M3, int SPLIT>
__global__ void __launch_bounds__(HEADS * SPLIT * 32, SPLIT == 1 ? 8 : 4) append_kernel(const __grid_constant__ AppendParams p) {
  constexpr int LANES = DH / 8, ROWS = 32 / LANES, WORDS = 8 / ROWS;           // lanes of a row, rows of a load, loads of eight rows
  constexpr int BATCH = 8 * SPLIT;
  pdl_trigger();
  pdl_wait();
  if (static_cast<int>(blockIdx.x) >= p.kv_ctas) {
    const int warp = threadIdx.x >> 5;
    turn_queries<DH>(p, (blockIdx.x - p.kv_ctas) * SPLIT + warp / HEADS, warp % HEADS);
    return;
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, ch = lane % LANES;
  const int sub = lane / LANES + (SPLIT == 1 ? 0 : warp % SPLIT * 8);          // the lane's first row of a batch
  const int chunk = blockIdx.x / p.head_ctas, head = (blockIdx.x - chunk * p.head_ctas) * HEADS + warp / SPLIT;
  __shared__ uint32_t s_top[HEADS * SPLIT];
  if (head >= 2 * p.Hkv) return;
  const int kv = head >= p.Hkv, h = head - kv * p.Hkv;
  const bool turns = p.cos_t && !kv;
  __nv_bfloat16* const rows = p.qkv + sub * p.ld + (p.H + head) * DH + ch * 8;
  int t = chunk * p.chunk;
  const int end = min(p.n - t, p.chunk) + t;
  int b = p.cu_q ? find_sequence(p.cu_q, p.B, t) : t;
  while (t < end) {                                                            // b: the sequence of row t, or the next one
    if (!p.cu_q) b = t;
    if (b >= p.B) return;
    int skip;
    const Place place = place_of(p, b, t, skip);
    const int* table = p.table + static_cast<size_t>(b) * p.max_blocks;
    int pos = place.pos;
    const int stop = t + place.rows;                                           // of the sequence's rows that have a place
    if (place.rows == 0) {
      t += skip;
    } else if ((pos & (p.block - 1)) && t != place.start) {                    // a block that began in an earlier chunk
      const int rest = min(p.block - (pos & (p.block - 1)), place.rows);
      t += rest;
      pos += rest;
    }
    auto load = [&](uint4 (&to)[WORDS], int t0, int cnt) {
#pragma unroll
      for (int i = 0; i < WORDS; ++i) {
        to[i] = make_uint4(0, 0, 0, 0);
        if (i * ROWS + sub < cnt) to[i] = *reinterpret_cast<const uint4*>(rows + (t0 + i * ROWS) * p.ld);
      }
    };
    for (int cnt; t < end && t < stop; t += cnt, pos += cnt) {
      const int off = pos & (p.block - 1), t0 = t;
      cnt = min(p.block - off, stop - t);
      uint4 v[WORDS];
      load(v, t, cnt);
      const int id = table[pos / p.page];
      const bool known = static_cast<unsigned>(id) < static_cast<unsigned>(p.n_blocks);
      const int slot = pos % p.page;
      __nv_bfloat16* x = rows + t0 * p.ld;
      const size_t row = (static_cast<size_t>(known ? id : 0) * 2 + kv) * p.Hkv + h;
      float* scale_at = p.scales + row * p.per_page + (slot >> p.block_bits);
      const float old = off && known ? *scale_at : 0.f;
      uint32_t top = 0;
      for (int r0 = 0; r0 < cnt; r0 += BATCH) {
        if (r0) load(v, t0 + r0, cnt - r0);
        if (turns) {
          const size_t a = static_cast<size_t>(pos + r0 + sub) * (DH / 2) + ch * 4;
#pragma unroll
          for (int i = 0; i < WORDS; ++i) {
            const bool in = r0 + i * ROWS + sub < cnt;
            float4 c = make_float4(0, 0, 0, 0), s = c;
            const size_t at = a + i * ROWS * (DH / 2);
            if (in) {
              c = *reinterpret_cast<const float4*>(p.cos_t + at);
              s = *reinterpret_cast<const float4*>(p.sin_t + at);
            }
            v[i] = rotate8(v[i], c, s);
            if (in) *reinterpret_cast<uint4*>(x + (r0 + i * ROWS) * p.ld) = v[i];
          }
        }
#pragma unroll
        for (int i = 0; i < WORDS; ++i)
          top = largest(top, largest(largest(v[i].x, v[i].y), largest(v[i].z, v[i].w)));
      }
      if (!known) continue;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) top = largest(top, __shfl_xor_sync(0xffffffffu, top, o));
      top = max(top & 0x7fffu, top >> 16 & 0x7fffu);
      if (SPLIT > 1) {                                                         // both warps of the head come here equally often
        if (lane == 0) s_top[warp] = top;
        asm volatile("bar.sync %0, 64;" ::"r"(1 + warp / 2) : "memory");
        top = max(top, s_top[warp ^ 1]);
      }
      const float need = scale_for<E4M3>(top);
      const float scale = off && (old > need || old != old) ? old : need;
      if (lane == 0 && sub == 0) *scale_at = scale;                            // all lanes have read it: they have met since
      const bool holds = scale == scale;
      const float inv = 1.f / scale;
      uint8_t* dst = p.codes + (row * p.page + slot) * DH;
      auto write = [&](auto clamp) {
        constexpr bool CLAMP = decltype(clamp)::value;
        for (int r0 = 0; r0 < cnt; r0 += BATCH) {
          if (cnt > BATCH) load(v, t0 + r0, cnt - r0);
#pragma unroll
          for (int i = 0; i < WORDS; ++i) {
            uint2 c;
            c.x = to_codes<E4M3, CLAMP>(bf16_lo(v[i].x), bf16_hi(v[i].x), bf16_lo(v[i].y), bf16_hi(v[i].y), inv);
            c.y = to_codes<E4M3, CLAMP>(bf16_lo(v[i].z), bf16_hi(v[i].z), bf16_lo(v[i].w), bf16_hi(v[i].w), inv);
            if (!holds) c = make_uint2(0, 0);
            if (r0 + i * ROWS + sub < cnt) *reinterpret_cast<uint2*>(dst + (r0 + i * ROWS + sub) * DH + ch * 8) = c;
          }
        }
      };
      // only a mantissa of all ones is more than 127 steps of its own scale
      if (!E4M3 && (top & 0x7f) == 0x7f) write(std::true_type());
      else write(std::false_type());
      if (off && holds && old != scale) {                                        // what the block holds, in the new steps
        const float ratio = old * inv;
        uint4* before = reinterpret_cast<uint4*>(dst - off * DH);
#pragma unroll 4
        for (int i = lane + warp % SPLIT * 32; i < off * (DH / 16); i += 32 * SPLIT) {
          uint4 w = before[i];
          uint32_t* e = &w.x;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float4 f = from_codes<E4M3>(e[j]);
            e[j] = to_codes<E4M3, true>(f.x, f.y, f.z, f.w, ratio);
          }
          before[i] = w;
        }
      }
      if (SPLIT > 1) asm volatile("bar.sync %0, 64;" ::"r"(1 + warp / 2) : "memory");      // the maxima have been read
    }
    if (p.cu_q && t < end)
      while (b < p.B && p.cu_q[b + 1] <= t) ++b;
  }
}

// ---- reading back --------------------------------------------------------------------------------------------------------------
// A page's codes and its values in bf16 lie in the same order, and the scale of an element is the one at its index / (block * dh). A thread
// expands two words of eight codes, or four where there are many, all of whose loads are under way before the first store; a warp's stores are
// whole lines (sixteen codes a thread, whose stores are halves of lines: 66.5 us for 1000 pages). Bound by memory: one byte read and two written
// an element. us for two / four / eight words a thread, 8 heads of 128: 1000 pages of 64 64.7 / 61.1 / 61.7 (0.98 of the copy rate), 100
// 6.6 / 7.0 / 10.2, 30 3.2 / 3.8 / 5.5.
constexpr int READ_THREADS = 256;

struct ReadParams {
  const uint2* codes; const float* scales;
  const int* pages; int n, n_blocks;
  long long page_words;                        // 8 codes each
  int shift;                                   // log2 of the words that share a scale
  int page_scales;
  uint4* out;
};

template <bool E4M3, int READ_WORDS>
__global__ void __launch_bounds__(READ_THREADS) read_kernel(const __grid_constant__ ReadParams p) {
  pdl_trigger();
  pdl_wait();
  const long long first = static_cast<long long>(blockIdx.x) * (READ_THREADS * READ_WORDS) + threadIdx.x;
  for (int i = blockIdx.y; i < p.n; i += gridDim.y) {
    const int id = p.pages[i];
    const bool known = static_cast<unsigned>(id) < static_cast<unsigned>(p.n_blocks);
    const uint2* src = p.codes + (known ? id : 0) * p.page_words;
    const float* scales = p.scales + static_cast<size_t>(known ? id : 0) * p.page_scales;
    uint4* dst = p.out + i * p.page_words;
    uint2 c[READ_WORDS];
    float s[READ_WORDS];
#pragma unroll
    for (int k = 0; k < READ_WORDS; ++k) {
      const long long w = first + k * READ_THREADS;
      c[k] = make_uint2(0, 0);
      s[k] = 0.f;
      if (known && w < p.page_words) {
        c[k] = src[w];
        s[k] = scales[w >> p.shift];
      }
    }
#pragma unroll
    for (int k = 0; k < READ_WORDS; ++k) {
      const long long w = first + k * READ_THREADS;
      const float4 f0 = from_codes<E4M3>(c[k].x), f1 = from_codes<E4M3>(c[k].y);
      if (w < p.page_words)
        dst[w] = make_uint4(pack_bf16x2(f0.x * s[k], f0.y * s[k]), pack_bf16x2(f0.z * s[k], f0.w * s[k]),
                            pack_bf16x2(f1.x * s[k], f1.y * s[k]), pack_bf16x2(f1.z * s[k], f1.w * s[k]));
    }
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
  p.n_blocks = n_blocks; p.page = page; p.block = block; p.per_page = page / block;
  for (p.block_bits = 3; (1 << p.block_bits) < block;) ++p.block_bits;
  p.table = table; p.max_blocks = max_blocks; p.seq_len = seq_len; p.cu_q = cu_q; p.B = B; p.chunk = chunk;
  const long long chunks = (static_cast<long long>(n) + chunk - 1) / chunk, rows = 256 / dh;                     // rows of a warp of queries
  // Two warps a head: for blocks of more than sixteen, whose rows one warp would read in twice as many turns (16 sequences of 700 rows, blocks
  // of 64: 19.1 against 25.3 us), and for blocks of sixteen where there are too few warps to hide how long a block takes. us for two / one: 8
  // heads of 128, 500 rows 5.9 / 7.8, 2048 rows 11.0 / 12.4, three sequences of 1000 14.3 / 14.0, four 18.4 / 16.8; 4 heads of 64, whose
  // rows a warp loads in half the turns, 2048 rows 5.1 / 6.5, eight sequences of up to 1000 11.9 / 9.9.
  const bool few = chunks * 2 * Hkv < num_sms() * (dh == 128 ? 20ll : 10ll);
  const int split = chunk > 8 && (block > 16 || (block > 8 && few)) ? 2 : 1;
  const int warps = kv8::HEADS * split;
  p.head_ctas = (2 * Hkv + kv8::HEADS - 1) / kv8::HEADS;
  const long long kv_ctas = chunks * p.head_ctas, ctas = kv_ctas + (cos_t && H ? (n + rows * split - 1) / (rows * split) : 0);
  if (ctas > 0x7fffffffll) return SB_ERR_TOO_LARGE;
  p.kv_ctas = static_cast<int>(kv_ctas);
  const dim3 grid(static_cast<unsigned>(ctas));
  using Kernel = void (*)(kv8::AppendParams);
  static const Kernel kernels[8] = {kv8::append_kernel<64, false, 1>, kv8::append_kernel<64, false, 2>, kv8::append_kernel<64, true, 1>,
                                    kv8::append_kernel<64, true, 2>, kv8::append_kernel<128, false, 1>, kv8::append_kernel<128, false, 2>,
                                    kv8::append_kernel<128, true, 1>, kv8::append_kernel<128, true, 2>};
  const Kernel kern = kernels[(dh == 128) * 4 + (e4m3 != 0) * 2 + split - 1];
  return launch_dep(kern, grid, dim3(warps * 32), 0, static_cast<cudaStream_t>(stream_), p) == cudaSuccess ? 0 : SB_ERR_LAUNCH;
}

// out [n, 2, Hkv, page, dh] bf16: the pages' values; zeros for ids outside the pool.
extern "C" int sb_quant_kv_read(const void* codes, int e4m3, const float* scales, int n_blocks, int Hkv, int page, int block, int dh,
                                const int* pages, int n, void* out, void* stream_) {
  if (!codes || !scales || !pages || !out || n <= 0 || !kv8::layout_ok(Hkv, dh, n_blocks, page, block)) return SB_ERR_ARG;
  if ((reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(out)) & 15) return SB_ERR_ALIGN;
  kv8::ReadParams p;
  p.codes = static_cast<const uint2*>(codes); p.scales = scales; p.pages = pages; p.n = n; p.n_blocks = n_blocks;
  p.page_words = 2ll * Hkv * page * dh / 8;
  p.shift = 0;
  while ((8 << p.shift) < block * dh) ++p.shift;
  p.page_scales = 2 * Hkv * (page / block);
  p.out = static_cast<uint4*>(out);
  const int words = n * static_cast<double>(p.page_words) < 4e6 ? 2 : 4;
  const long long ctas = (p.page_words + kv8::READ_THREADS * words - 1) / (kv8::READ_THREADS * words);
  if (ctas > 0x7fffffffll) return SB_ERR_TOO_LARGE;
  const dim3 grid(static_cast<unsigned>(ctas), n < 65535 ? n : 65535);
  using Kernel = void (*)(kv8::ReadParams);
  static const Kernel kernels[4] = {kv8::read_kernel<false, 2>, kv8::read_kernel<false, 4>, kv8::read_kernel<true, 2>,
                                    kv8::read_kernel<true, 4>};
  const Kernel kern = kernels[(e4m3 != 0) * 2 + (words == 4)];
  return launch_dep(kern, grid, dim3(kv8::READ_THREADS), 0, static_cast<cudaStream_t>(stream_), p) == cudaSuccess ? 0 : SB_ERR_LAUNCH;
}
