// Attention of single tokens over the paged KV cache in 8 bits (its layout: quantized_kv.cu).
//
// o = sum_j w_j s_v(j) c_v(j) / sum_j w_j with w_j = exp(scale * s_k(j) * (q . c_k(j)) - m): codes c, scales s of the position's block. One CTA
// for a query head of a sequence; each of its warps takes every fourth position, lanes hold dimensions, and the warps' running maxima,
// sums and values are joined at the end.
#include <cuda_bf16.h>
#include "api.h"
#include "dependent.cuh"
#include "quantized_kv.cuh"
#include "sm100_ptx.cuh"

namespace sb {
namespace kv8 {

struct AttendParams {
  const __nv_bfloat16* q; long long ldq;
  const uint8_t* codes; const float* scales;
  int n_blocks, page, block;
  const int* table; int max_blocks;
  const int* seq_len;
  int H, Hkv;
  float scale;
  __nv_bfloat16* out; long long ldo;
};

template <int DH, bool E4M3>
__global__ void __launch_bounds__(128) attend_kernel(const __grid_constant__ AttendParams p) {
  constexpr int LANES = DH / 4;                                // lanes that hold a position: all, or half of them
  pdl_trigger();
  pdl_wait();
  const int head = blockIdx.x, b = blockIdx.y, kvh = head / (p.H / p.Hkv);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d = lane % LANES * 4, part = lane / LANES;
  const long long cap = static_cast<long long>(p.max_blocks) * p.page;
  const int len = static_cast<int>(min(static_cast<long long>(p.seq_len[b]), cap));
  const __nv_bfloat16* q = p.q + b * p.ldq + head * DH + d;
  float4 qv;
  qv.x = __bfloat162float(q[0]); qv.y = __bfloat162float(q[1]); qv.z = __bfloat162float(q[2]); qv.w = __bfloat162float(q[3]);
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0, 0, 0, 0);
  constexpr int STEP = 4 * (32 / LANES);
  for (int j0 = warp * (32 / LANES); j0 < len; j0 += STEP) {
    const int j = j0 + part;
    const bool live = j < len;
    const int id = live ? p.table[static_cast<size_t>(b) * p.max_blocks + j / p.page] : 0;
    const bool known = live && static_cast<unsigned>(id) < static_cast<unsigned>(p.n_blocks);
    const size_t row = known ? (static_cast<size_t>(id) * 2 * p.Hkv + kvh) : 0;
    const int slot = j % p.page, blocks = p.page / p.block;
    float4 k = make_float4(0, 0, 0, 0), v = k;
    float ks = 0.f, vs = 0.f;
    if (known) {
      const size_t vrow = row + p.Hkv;
      k = from_codes<E4M3>(*reinterpret_cast<const uint32_t*>(p.codes + (row * p.page + slot) * DH + d));
      v = from_codes<E4M3>(*reinterpret_cast<const uint32_t*>(p.codes + (vrow * p.page + slot) * DH + d));
      ks = p.scales[row * blocks + slot / p.block];
      vs = p.scales[vrow * blocks + slot / p.block];
    }
    float s = qv.x * k.x + qv.y * k.y + qv.z * k.z + qv.w * k.w;
#pragma unroll
    for (int x = 1; x < LANES; x <<= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    s = live ? s * ks * p.scale : -INFINITY;
    if (!live) continue;                                       // the upper half of a warp, at the last position only
    const float top = fmaxf(m, s), w = s == top && top == m ? 1.f : expf(s - top), a = top == m ? 1.f : expf(m - top);
    m = top;
    l = l * a + w;
    o.x = o.x * a + w * vs * v.x; o.y = o.y * a + w * vs * v.y; o.z = o.z * a + w * vs * v.z; o.w = o.w * a + w * vs * v.w;
  }
  __shared__ float sm_m[8], sm_l[8], sm_o[8][DH];
  const int who = warp * (32 / LANES) + part;
  sm_o[who][d] = o.x; sm_o[who][d + 1] = o.y; sm_o[who][d + 2] = o.z; sm_o[who][d + 3] = o.w;
  if (d == 0) { sm_m[who] = m; sm_l[who] = l; }
  __syncthreads();
  if (threadIdx.x < DH) {
    float top = -INFINITY, lt = 0.f, ot = 0.f;
    for (int w = 0; w < STEP; ++w) top = fmaxf(top, sm_m[w]);
    for (int w = 0; w < STEP; ++w) {
      if (w >= len) break;                                     // it has seen no position
      const float a = sm_m[w] == top ? 1.f : expf(sm_m[w] - top);
      lt += sm_l[w] * a;
      ot += sm_o[w][threadIdx.x] * a;
    }
    p.out[b * p.ldo + head * DH + threadIdx.x] = __float2bfloat16_rn(len > 0 ? ot / lt : 0.f);
  }
}

}  // namespace kv8
}  // namespace sb

using namespace sb;

// q: [B, ldq] bf16 (H * dh used, rotated); out: [B, ldo] bf16. A sequence of no positions gets zeros; ids outside the pool count as zeros.
extern "C" int sb_quant_kv_attention(const void* q, long long ldq, const void* codes, int e4m3, const float* scales, int n_blocks, int page,
                                     int block, const int* table, int max_blocks, const int* seq_len, int B, int H, int Hkv, int dh,
                                     float scale, void* out, long long ldo, void* stream_) {
  if (!q || !codes || !scales || !table || !seq_len || !out || B <= 0 || H <= 0 || max_blocks <= 0 || !kv8::layout_ok(Hkv, dh, n_blocks, page, block) ||
      H % Hkv)
    return SB_ERR_ARG;
  if (B > 65535) return SB_ERR_TOO_LARGE;
  kv8::AttendParams p;
  p.q = static_cast<const __nv_bfloat16*>(q); p.ldq = ldq;
  p.codes = static_cast<const uint8_t*>(codes); p.scales = scales;
  p.n_blocks = n_blocks; p.page = page; p.block = block;
  p.table = table; p.max_blocks = max_blocks; p.seq_len = seq_len;
  p.H = H; p.Hkv = Hkv; p.scale = scale;
  p.out = static_cast<__nv_bfloat16*>(out); p.ldo = ldo;
  auto kern = dh == 64 ? (e4m3 ? kv8::attend_kernel<64, true> : kv8::attend_kernel<64, false>)
                       : (e4m3 ? kv8::attend_kernel<128, true> : kv8::attend_kernel<128, false>);
  return launch_dep(kern, dim3(H, B), dim3(128), 0, static_cast<cudaStream_t>(stream_), p) == cudaSuccess ? 0 : SB_ERR_LAUNCH;
}
