// Pages of a paged KV cache to other pages, in the pools of all layers at once.
//
// A page is `page_bytes` contiguous bytes; what is copied of it are `segs` segments of `seg_bytes`, `seg_pitch` apart: the page as a whole
// (one segment), or the first positions of each head of K and of V. Copy i goes from page src[i] of the source pools to page dst[i] of the
// destination pools; no destination is a source or another copy's destination, so the order of copies does not matter. Ids outside their
// pools are skipped.
//
// Bound by memory: each byte is read and written once. A CTA copies up to 16 KB of one page of one layer, four 16-byte words a thread, all
// of whose loads are under way before the first store; layers are the slowest grid index, so a page that goes to many (a fork) is read
// from L2 by all but the first. What is written is marked as the first to leave L2: a fork of all layers is more than fits beside what the
// next steps read. 128 pages of 256 KB in eight layers 83 us, 0.99 of the copy rate; 301 pages of 8 KB in 32 layers 26.3, 0.92; 40 of 64
// positions to 16 pages in 32 layers 15.0, of which 84 MB are writes, 0.91 (stores without the mark 17.1; two words a thread 18.2, eight
// 21.3; copies as the fastest index 19.2; four copies a CTA, which hold a source that stays the same in registers, gain nothing).
#include "api.h"
#include "dependent.cuh"

namespace sb {
namespace pages {

constexpr int MAX_LAYERS = 64, THREADS = 256, WORDS = 4;      // pools of a launch; words of a thread

struct Params {
  const void* src[MAX_LAYERS];
  void* dst[MAX_LAYERS];
  const int *from, *to;
  int n, src_blocks, dst_blocks, segs;
  long long page_words, seg_words, seg_pitch_words;
  int step_segs, step_words;                       // THREADS words further on: segments, and words into the one behind them
};

// One segment: no division.
template <typename W, bool ONE>
__global__ void __launch_bounds__(THREADS) copy_pages_kernel(const __grid_constant__ Params p) {
  pdl_trigger();
  pdl_wait();
  const long long words = p.seg_words * p.segs, first = static_cast<long long>(blockIdx.x) * (THREADS * WORDS) + threadIdx.x;
  const W* src = static_cast<const W*>(p.src[blockIdx.z]);
  W* dst = static_cast<W*>(p.dst[blockIdx.z]);
  long long at[WORDS];
  {
    int seg = ONE ? 0 : static_cast<int>(static_cast<unsigned>(first) / static_cast<unsigned>(p.seg_words));      // words < 2^31 (host)
    long long in = first - seg * p.seg_words;
#pragma unroll
    for (int k = 0; k < WORDS; ++k) {
      at[k] = ONE ? first + k * THREADS : seg * p.seg_pitch_words + in;
      seg += p.step_segs;
      in += p.step_words;
      if (in >= p.seg_words) { in -= p.seg_words; ++seg; }
    }
  }
  for (int i = blockIdx.y; i < p.n; i += gridDim.y) {
    const int a = p.from[i], b = p.to[i];
    if (static_cast<unsigned>(a) >= static_cast<unsigned>(p.src_blocks) || static_cast<unsigned>(b) >= static_cast<unsigned>(p.dst_blocks))
      continue;
    const W* s = src + a * p.page_words;
    W* d = dst + b * p.page_words;
    W v[WORDS];
#pragma unroll
    for (int k = 0; k < WORDS; ++k)
      if (first + k * THREADS < words) v[k] = s[at[k]];
#pragma unroll
    for (int k = 0; k < WORDS; ++k)
      if (first + k * THREADS < words) __stcs(d + at[k], v[k]);
  }
}

template <typename W>
static int launch(Params p, int layers, const void* const* src, void* const* dst, long long page_bytes, long long seg_bytes,
                  long long seg_pitch, cudaStream_t s) {
  p.page_words = page_bytes / sizeof(W);
  p.seg_words = seg_bytes / sizeof(W);
  p.seg_pitch_words = seg_pitch / sizeof(W);
  const long long words = p.seg_words * p.segs, chunks = (words + THREADS * WORDS - 1) / (THREADS * WORDS);
  p.step_segs = static_cast<int>(THREADS / p.seg_words);
  p.step_words = static_cast<int>(THREADS % p.seg_words);
  for (int l0 = 0; l0 < layers; l0 += MAX_LAYERS) {
    const int n = layers - l0 < MAX_LAYERS ? layers - l0 : MAX_LAYERS;
    for (int l = 0; l < n; ++l) {
      p.src[l] = src[l0 + l];
      p.dst[l] = dst[l0 + l];
    }
    const dim3 grid(static_cast<unsigned>(chunks), p.n < 65535 ? p.n : 65535, n);
    const cudaError_t rc = p.segs == 1 ? launch_dep(copy_pages_kernel<W, true>, grid, dim3(THREADS), 0, s, p)
                                       : launch_dep(copy_pages_kernel<W, false>, grid, dim3(THREADS), 0, s, p);
    if (rc != cudaSuccess) return SB_ERR_LAUNCH;
  }
  return 0;
}

}  // namespace pages
}  // namespace sb

using namespace sb;

// src, dst: host arrays of `layers` pool addresses. from, to: [n] page ids on the device. Segments may not reach into one another or past
// the page.
extern "C" int sb_copy_pages(const void* const* src, void* const* dst, int layers, const int* from, const int* to, int n, int src_blocks,
                             int dst_blocks, long long page_bytes, int segs, long long seg_bytes, long long seg_pitch, void* stream_) {
  if (!src || !dst || !from || !to || layers <= 0 || n <= 0 || src_blocks <= 0 || dst_blocks <= 0 || segs <= 0 || seg_bytes <= 0 ||
      seg_pitch < seg_bytes || page_bytes < (segs - 1) * seg_pitch + seg_bytes)
    return SB_ERR_ARG;
  if (page_bytes >= (1ll << 31)) return SB_ERR_TOO_LARGE;
  uintptr_t all = static_cast<uintptr_t>(page_bytes) | static_cast<uintptr_t>(seg_bytes) | static_cast<uintptr_t>(segs > 1 ? seg_pitch : 0);
  for (int l = 0; l < layers; ++l) {
    if (!src[l] || !dst[l]) return SB_ERR_ARG;
    all |= reinterpret_cast<uintptr_t>(src[l]) | reinterpret_cast<uintptr_t>(dst[l]);
  }
  pages::Params p;
  p.from = from; p.to = to; p.n = n; p.src_blocks = src_blocks; p.dst_blocks = dst_blocks; p.segs = segs;
  cudaStream_t s = static_cast<cudaStream_t>(stream_);
  if ((all & 15) == 0) return pages::launch<uint4>(p, layers, src, dst, page_bytes, seg_bytes, seg_pitch, s);
  if ((all & 3) == 0) return pages::launch<uint32_t>(p, layers, src, dst, page_bytes, seg_bytes, seg_pitch, s);
  return pages::launch<uint8_t>(p, layers, src, dst, page_bytes, seg_bytes, seg_pitch, s);
}
