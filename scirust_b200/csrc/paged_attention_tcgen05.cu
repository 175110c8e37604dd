// Attention of a batch whose sequences share a prefix in the paged cache, on the tensor cores of sm_100a.
//
// Row (t, h) of the batch, token t of sequence b, sees the first `limit` positions of b:
//   s_j = scale q.k_j,  m = max s_j,  l = sum exp(s_j - m),  o = sum exp(s_j - m) v_j / l,   j < limit;   limit <= 0: o = 0.
// Positions below P (the whole pages of the prefix) are the same for all sequences, so the sum is taken in two parts: the rows of all
// sequences against one copy of K and V, and each sequence's rows against what it has for itself. Parts (m_i, l_i, o_i) of a row,
// o_i not divided by l_i, join as m = max m_i, w_i = exp(scale (m_i - m)), o = sum w_i o_i / sum w_i l_i (here m_i is a maximum of q.k).
//
// Both parts are the same work for a CTA: a tile of 128 rows (tokens times the query heads of one kv head), a table of pages and a
// range of 64-position blocks of keys. An item is all of that for one tile of rows:
//   shared: (kv head, tile of consecutive tokens, whatever their sequences), blocks [0, P / 64)
//   own:    (sequence, tile of its tokens, kv head), blocks of [P, limit of its last row)
// Where the sequences bring a whole tile of rows each there is nothing to share, and their own items start at position 0.
// The blocks of all items form one line, which is dealt out evenly over the CTAs; what lies in a CTA's share of an item is a piece.
// An item that is not cut and has no other part is written out at once, pieces of the others go to a workspace and a second,
// dependent launch joins them in a fixed order.
#include "sm100_ptx.cuh"
#include "api.h"
#include "dependent.cuh"
#include "per_device.h"

namespace sb {

int num_sms();
int make_tmap_2d_bf16(CUtensorMap* out, const void* base, uint64_t inner, uint64_t outer, uint64_t ld,
                      uint32_t box_inner, uint32_t box_outer);

namespace spa {

constexpr int BM = 128;        // rows of a tile
constexpr int BN = 64;         // positions of a block
constexpr int THREADS = 192;   // producer, issuer, four softmax warps
constexpr int TMEM_COLS = 256;
constexpr int MAX_DIRECT = 1024;   // sequences of one token each whose plan every CTA makes for itself, in shared memory
constexpr float LOWEST = -3.402823466e38f;   // reference of a row that has seen nothing: 2^(-inf - LOWEST) is 0

template <int DH>
struct Cfg {
  static constexpr int NCH = DH / 64;                // 64-column chunks of a head
  static constexpr int SLOTS = DH == 128 ? 4 : 8;    // ring of K and V blocks
  static constexpr int Q_BYTES = BM * DH * 2;
  static constexpr int KV_BYTES = BN * DH * 2;
  static constexpr int PLAN_BYTES = (2 * MAX_DIRECT + 2) * 4;
  static constexpr int SMEM_BYTES = Q_BYTES + SLOTS * KV_BYTES + 256 /* barriers */ + PLAN_BYTES + 1024 /* alignment */;
  static_assert(2 * (SMEM_BYTES + 1024) <= 228 * 1024, "two CTAs per SM");
  // tensor memory: scores, two buffers of P as bf16 pairs, O
  static constexpr int COL_S = 0, COL_P = BN, COL_O = COL_P + 2 * (BN / 2);
  static_assert(COL_O + DH <= TMEM_COLS, "tensor memory");
};

// What the plan says of an item of its own: tokens [t0, t0 + n), sequence, position behind the last one that a row sees.
struct Pair {
  int t0, n, b, kend;
};

struct Header {        // at the start of the workspace
  int units, units_shared, q_lo, q_hi, pairs;
  int pad[3];
};

struct Params {
  const __nv_bfloat16* q;
  long long ldq;
  const int* block_table;
  int max_blocks;
  const int* seq_len;
  const int* prefix_table;
  const int* cu_q;
  int prefix;          // shared positions: whole pages; 0 where every sequence's own items start at 0
  int page, n_blocks, box;
  int B, NT, H, Hkv, G, TT;
  float scale_log2;
  __nv_bfloat16* out;
  long long ldo;
  int fill;            // rows of no sequence become zero instead of staying as they are
  Header* hdr;
  int* cum;            // [pairs + 1] blocks of own items before a pair, of one kv head
  Pair* pair;
  int* row_limit;      // [NT]
  int* row_pair;       // [NT], -1: of no sequence
  float* whole;        // [2][NT][H][dh], and [2][NT][H][2] behind it: items that were not cut
  float* cut;          // [2 * CTAs][128][dh], and [2 * CTAs][128][2] behind it: first and last pieces of the CTAs
  int max_pairs;
  int* status;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ int clampi(int v, int lo, int hi) { return min(max(v, lo), hi); }

// The even deal of `units` over `ctas`: the first `rem` of them get one more.
struct Deal {
  int per, rem;
  __device__ Deal(int units, int ctas) : per(units / ctas), rem(units - units / ctas * ctas) {}
  __device__ int begin(int c) const { return c * per + min(c, rem); }
  __device__ int owner(int u) const {
    const int edge = rem * (per + 1);
    return u < edge ? u / (per + 1) : rem + (u - edge) / per;      // per == 0: all units lie below the edge
  }
};

__device__ __forceinline__ int blocks_of(int positions) { return positions > 0 ? (positions + BN - 1) / BN : 0; }

// Inclusive sum over a warp.
__device__ __forceinline__ int warp_scan(int v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += x;
  }
  return v;
}

// A piece of an item, as all roles of a CTA see it.
struct Piece {
  int h, t0, n_tok, kbase, kend, j0, j1;   // blocks [j0, j1) of kbase + 64 j, positions below kend
  const int* table;
  bool shared, cut, first;                 // cut: only a part of its item; first: the first piece of this CTA
};

struct Walk {
  const Params& p;
  const int* cum;
  const int* len;        // lengths of sequences of one token each, or null: pairs come from the plan
  int units_shared, q_lo, q_hi, tiles_q, blocks_shared, pairs;
  int u, u1, u_first;
  int pair_at;

  __device__ Walk(const Params& p_, const int* cum_, const int* len_, const Header& h, int u0, int u1_)
      : p(p_), cum(cum_), len(len_), units_shared(h.units_shared), q_lo(h.q_lo), q_hi(h.q_hi),
        tiles_q((h.q_hi - h.q_lo + p_.TT - 1) / p_.TT), blocks_shared(blocks_of(p_.prefix)), pairs(h.pairs), u(u0), u1(u1_),
        u_first(u0), pair_at(-1) {}

  __device__ bool next(Piece& x) {
    if (u >= u1) return false;
    int off, size;
    if (u < units_shared) {
      size = blocks_shared;
      const int item = u / size;
      off = u - item * size;
      x.h = item / tiles_q;
      x.t0 = q_lo + (item - x.h * tiles_q) * p.TT;
      x.n_tok = min(p.TT, q_hi - x.t0);
      x.kbase = 0;
      x.kend = p.prefix;
      x.table = p.prefix_table;
      x.shared = true;
    } else {
      const int v = u - units_shared;
      if (pair_at < 0) {                        // last pair that starts at v or before
        int lo = 0, hi = pairs - 1;
        while (lo < hi) {
          const int mid = (lo + hi + 1) >> 1;
          if (cum[mid] * p.Hkv <= v) lo = mid; else hi = mid - 1;
        }
        pair_at = lo;
      }
      while (cum[pair_at + 1] * p.Hkv <= v) ++pair_at;      // v lies below the last pair's end
      size = cum[pair_at + 1] - cum[pair_at];
      const int rest = v - cum[pair_at] * p.Hkv;
      x.h = rest / size;
      off = rest - x.h * size;
      int b;
      if (len) {
        b = pair_at;
        x.t0 = b; x.n_tok = 1; x.kend = len[b];
      } else {
        const int4 i = *reinterpret_cast<const int4*>(p.pair + pair_at);
        x.t0 = i.x; x.n_tok = i.y; x.kend = i.w;
        b = i.z;
      }
      x.kbase = p.prefix;
      x.table = p.block_table + static_cast<size_t>(b) * p.max_blocks;
      x.shared = false;
    }
    x.j0 = off;
    x.j1 = min(size, off + (u1 - u));
    x.cut = x.j1 - x.j0 != size;
    x.first = u == u_first;
    u += x.j1 - x.j0;
    return true;
  }
};

// Plan of a ragged batch, or of more sequences than the CTAs plan for themselves: one CTA.
__global__ void __launch_bounds__(1024) plan_kernel(const Params p) {
  __shared__ int s_warp[32];
  __shared__ int s_hi, s_pairs, s_sum;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_trigger();
  pdl_wait();
  if (tid == 0) { s_hi = p.cu_q ? clampi(p.cu_q[0], 0, p.NT) : 0; s_pairs = 0; s_sum = 0; }
  for (int t = tid; t < p.NT; t += 1024) { p.row_limit[t] = 0; p.row_pair[t] = -1; }
  __syncthreads();
  const int q_lo = s_hi;
  const int cap = p.max_blocks * p.page;
  for (int b0 = 0; b0 < p.B; b0 += 1024) {
    const int b = b0 + tid;
    int start = 0, end = 0;
    if (b < p.B) {
      start = p.cu_q ? clampi(p.cu_q[b], 0, p.NT) : b;
      end = p.cu_q ? clampi(p.cu_q[b + 1], 0, p.NT) : b + 1;
    }
    // offsets that fall back would give rows to two sequences: the largest end so far is where a sequence starts at least
    int top = b < p.B ? max(start, end) : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, top, o);
      if (lane >= o) top = max(top, x);
    }
    if (lane == 31) s_warp[warp] = top;
    __syncthreads();
    int before = s_hi;
    for (int w = 0; w < warp; ++w) before = max(before, s_warp[w]);
    int prev = __shfl_up_sync(0xffffffffu, top, 1);
    before = lane > 0 ? max(before, prev) : before;
    __syncthreads();
    if (tid == 1023) s_hi = max(before, top);
    start = max(start, before);
    const int n = b < p.B ? max(0, end - start) : 0;
    int tiles = (n + p.TT - 1) / p.TT;
    const int scan = warp_scan(tiles, lane);
    if (lane == 31) s_warp[warp] = scan;
    __syncthreads();
    int at = s_pairs;
    for (int w = 0; w < warp; ++w) at += s_warp[w];
    at += scan - tiles;
    __syncthreads();
    if (tid == 1023) s_pairs = min(at + tiles, p.max_pairs);
    if (b < p.B) {
      const int len = clampi(p.seq_len[b], 0, cap);
      for (int i = 0; i < tiles && at + i < p.max_pairs; ++i) {
        Pair x;
        x.t0 = start + i * p.TT;
        x.n = min(p.TT, n - i * p.TT);
        x.b = b;
        x.kend = len - n + i * p.TT + x.n;
        *reinterpret_cast<int4*>(p.pair + at + i) = make_int4(x.t0, x.n, x.b, x.kend);
      }
    }
    __syncthreads();
  }
  const int pairs = s_pairs, q_hi = max(q_lo, s_hi);
  for (int i = warp; i < pairs; i += 32) {
    const int4 x = *reinterpret_cast<const int4*>(p.pair + i);
    for (int r = lane; r < x.y; r += 32) {
      p.row_limit[x.x + r] = x.w - x.y + r + 1;
      p.row_pair[x.x + r] = i;
    }
  }
  for (int i0 = 0; i0 < pairs; i0 += 1024) {
    const int i = i0 + tid;
    const int n = i < pairs ? blocks_of(p.pair[i].kend - p.prefix) : 0;
    const int scan = warp_scan(n, lane);
    if (lane == 31) s_warp[warp] = scan;
    __syncthreads();
    int at = s_sum;
    for (int w = 0; w < warp; ++w) at += s_warp[w];
    if (i < pairs) p.cum[i] = at + scan - n;
    __syncthreads();
    if (tid == 1023) s_sum = at + scan;
    __syncthreads();
  }
  if (tid == 0) {
    p.cum[pairs] = s_sum;
    const int shared = p.Hkv * ((q_hi - q_lo + p.TT - 1) / p.TT) * blocks_of(p.prefix);
    p.hdr->units = shared + p.Hkv * s_sum;
    p.hdr->units_shared = shared;
    p.hdr->q_lo = q_lo; p.hdr->q_hi = q_hi; p.hdr->pairs = pairs;
  }
}

template <int DH>
__global__ void __launch_bounds__(THREADS, 2)
attend_kernel(const __grid_constant__ CUtensorMap tmap, const __grid_constant__ Params p) {
  using C = Cfg<DH>;
  constexpr int SLOTS = C::SLOTS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sQ = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ring = sQ + C::Q_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + SLOTS * C::KV_BYTES);   // [SLOTS]
  uint64_t* empty = full + SLOTS;        // [SLOTS]
  uint64_t* q_full = empty + SLOTS;      // rows of a piece are in shared memory (4 warp arrivals)
  uint64_t* s_full = q_full + 1;         // scores of a block are in tensor memory
  uint64_t* s_free = s_full + 1;         // and in registers (4 warp arrivals)
  uint64_t* p_full = s_free + 1;         // [2] P of a block is in tensor memory and O rescaled (4 warp arrivals)
  uint64_t* pv_done = p_full + 2;        // P V of a block has completed
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(pv_done + 1);
  int* s_cum = reinterpret_cast<int*>(ring + SLOTS * C::KV_BYTES + 256);     // [B + 1]
  int* s_len = s_cum + MAX_DIRECT + 1;                                       // [B]
  static_assert((2 * SLOTS + 7) * 8 + 4 <= 256, "barriers");

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < SLOTS; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    mbar_init(q_full, 4);
    mbar_init(s_full, 1);
    mbar_init(s_free, 4);
    mbar_init(&p_full[0], 4);
    mbar_init(&p_full[1], 4);
    mbar_init(pv_done, 1);
    fence_barrier_init();
    fence_proxy_async_smem();
    prefetch_tmap(&tmap);
  }
  if (warp == 1) {
    tmem_alloc(tmem_holder, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *reinterpret_cast<volatile uint32_t*>(tmem_holder), 0);
  pdl_trigger();
  pdl_wait();

  // ---- plan: one token per sequence is summed up here, anything else has been by plan_kernel
  const bool direct = p.pair == nullptr;
  Header hdr;
  if (direct) {
    if (warp == 0) {
      const int cap = p.max_blocks * p.page;
      int base = 0;
      for (int b0 = 0; b0 < p.B; b0 += 32) {
        const int b = b0 + lane;
        const int len = b < p.B ? clampi(p.seq_len[b], 0, cap) : 0;
        const int n = blocks_of(len - p.prefix);
        const int scan = warp_scan(n, lane);
        if (b < p.B) {
          s_cum[b] = base + scan - n;
          s_len[b] = len;
          if (blockIdx.x == 0) { p.cum[b] = base + scan - n; }
        }
        base += __shfl_sync(0xffffffffu, scan, 31);
      }
      if (lane == 0) {
        s_cum[p.B] = base;
        if (blockIdx.x == 0) p.cum[p.B] = base;
      }
    }
    __syncthreads();
    hdr.q_lo = 0; hdr.q_hi = p.B; hdr.pairs = p.B;
    hdr.units_shared = p.Hkv * ((p.B + p.TT - 1) / p.TT) * blocks_of(p.prefix);
    hdr.units = hdr.units_shared + p.Hkv * s_cum[p.B];
    if (blockIdx.x == 0 && threadIdx.x == 0) {
      p.hdr->units = hdr.units; p.hdr->units_shared = hdr.units_shared;
      p.hdr->q_lo = 0; p.hdr->q_hi = p.B; p.hdr->pairs = p.B;
    }
  } else {
    hdr.units = p.hdr->units; hdr.units_shared = p.hdr->units_shared;
    hdr.q_lo = p.hdr->q_lo; hdr.q_hi = p.hdr->q_hi; hdr.pairs = p.hdr->pairs;
  }
  const Deal deal(hdr.units, gridDim.x);
  Walk walk(p, direct ? s_cum : p.cum, direct ? s_len : nullptr, hdr, deal.begin(blockIdx.x), deal.begin(blockIdx.x + 1));
  Piece x;

  if (warp == 0) {
    // ------------------------------------ TMA producer ------------------------------------
    // Blocks arrive in the order in which the issuer takes them: K0 K1 V0 K2 V1 ... K(n-1) V(n-2) V(n-1) of a piece.
    int slot = 0;
    uint32_t phase = 0;
    bool ok = true;
    const int nbx = BN / p.box;               // boxes of a block, at most 8
    while (ok && walk.next(x)) {
      int fetched = -(1 << 30), page_of_lane = 0;      // lane i: page of box (fetched + i)
      int fetched_v = -(1 << 30), page_of_lane_v = 0;
      auto load = [&](int j, bool v, int& at, int& pages) -> bool {
        if (!mbar_wait_warp(&empty[slot], phase ^ 1, p.status, ST_TIMEOUT_EMPTY)) return false;
        const int bx0 = j * nbx;
        if (bx0 < at || bx0 + nbx > at + 32) {         // nbx divides 32: a block's boxes are fetched together
          at = bx0;
          const int pos = x.kbase + (at + lane) * p.box;
          pages = pos < x.kend ? x.table[pos / p.page] : 0;
          if (static_cast<unsigned>(pages) >= static_cast<unsigned>(p.n_blocks)) pages = p.n_blocks;   // reads as zeros
        }
        const int live = min(nbx, (x.kend - x.kbase - j * BN + p.box - 1) / p.box);     // boxes with a position below kend
        uint8_t* to = ring + slot * C::KV_BYTES;
        if (lane == 0) mbar_arrive_expect_tx(&full[slot], live * p.box * DH * 2);
        for (int i = 0; i < live; ++i) {
          const int blk = __shfl_sync(0xffffffffu, pages, bx0 + i - at);
          if (lane == 0) {
            const int row = (blk * 2 * p.Hkv + (v ? p.Hkv : 0) + x.h) * p.page + (x.kbase + (bx0 + i) * p.box) % p.page;
#pragma unroll
            for (int c = 0; c < C::NCH; ++c)
              tma_load_2d(to + c * (BN * 128) + i * p.box * 128, &tmap, &full[slot], c * 64, row);
          }
        }
        __syncwarp();
        if (++slot == SLOTS) { slot = 0; phase ^= 1; }
        return true;
      };
      ok = load(x.j0, false, fetched, page_of_lane);
      for (int j = x.j0; j < x.j1 && ok; ++j) {
        if (j + 1 < x.j1) ok = load(j + 1, false, fetched, page_of_lane);
        ok = ok && load(j, true, fetched_v, page_of_lane_v);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------- MMA issuer -------------------------------------
    const bool leader = elect_one();
    constexpr uint32_t idesc_s = make_idesc_bf16(BM, BN, false, false);
    constexpr uint32_t idesc_o = make_idesc_bf16(BM, DH, false, true);
    int slot = 0, n_blocks = 0, n_pieces = 0;      // blocks whose scores were issued, pieces begun
    uint32_t phase = 0;
    bool ok = true;
    const uint64_t dq = make_smem_desc(smem_u32(sQ), 16, 1024);
    auto advance = [&] { if (++slot == SLOTS) { slot = 0; phase ^= 1; } };
    auto scores = [&]() -> bool {                  // S = Q K^T
      if (!mbar_wait_warp(&full[slot], phase, p.status, ST_TIMEOUT_FULL)) return false;
      if (n_blocks > 0 && !mbar_wait_warp(s_free, (n_blocks - 1) & 1, p.status, ST_TIMEOUT_TMEM_EMPTY)) return false;
      tc_fence_after();
      const uint64_t dk = make_smem_desc(smem_u32(ring + slot * C::KV_BYTES), 16, 1024);
      if (leader) {
#pragma unroll
        for (int k = 0; k < DH / 16; ++k)
          umma_bf16_ss(tmem + C::COL_S, smem_desc_at(dq, (k >> 2) * (BM * 128) + (k & 3) * 32),
                       smem_desc_at(dk, (k >> 2) * (BN * 128) + (k & 3) * 32), idesc_s, k > 0 ? 1u : 0u);
        umma_commit(s_full);
        umma_commit(&empty[slot]);
      }
      ++n_blocks;
      advance();
      return true;
    };
    auto values = [&](int i, int live, bool begins) -> bool {     // O (+)= P V of block i, of which `live` positions count
      if (!mbar_wait_warp(&full[slot], phase, p.status, ST_TIMEOUT_FULL)) return false;
      uint8_t* v = ring + slot * C::KV_BYTES;
      if (live < BN) {
        // The weights of positions behind the end are zero, but what lies there may be no number: zero times it would be none either.
        for (int c = lane; c < (BN - live) * (DH / 8); c += 32) {
          const int row = live + c / (DH / 8), w = c % (DH / 8);       // rows are whole, so their swizzle does not matter
          *reinterpret_cast<uint4*>(v + (w >> 3) * (BN * 128) + row * 128 + (w & 7) * 16) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
        __syncwarp();
      }
      if (!mbar_wait_warp(&p_full[i & 1], (i >> 1) & 1, p.status, ST_TIMEOUT_MISC)) return false;
      tc_fence_after();
      const uint64_t dv = make_smem_desc(smem_u32(v), BN * 128, 1024);
      if (leader) {
#pragma unroll
        for (int k = 0; k < BN / 16; ++k)
          umma_bf16_ts(tmem + C::COL_O, tmem + C::COL_P + (i & 1) * (BN / 2) + k * 8, smem_desc_at(dv, k * (16 * 128)), idesc_o,
                       (!begins || k > 0) ? 1u : 0u);
        umma_commit(pv_done);
        umma_commit(&empty[slot]);
      }
      advance();
      return true;
    };
    while (ok && walk.next(x)) {
      ok = mbar_wait_warp(q_full, n_pieces & 1, p.status, ST_TIMEOUT_MISC);
      ++n_pieces;
      const int i0 = n_blocks;
      ok = ok && scores();
      for (int j = x.j0; j < x.j1 && ok; ++j) {
        if (j + 1 < x.j1) ok = scores();
        ok = ok && values(i0 + j - x.j0, min(BN, x.kend - x.kbase - j * BN), j == x.j0);
      }
    }
  } else {
    // ------------------------------------ softmax warps ------------------------------------
    const int quarter = warp & 3;          // lanes of tensor memory that this warp may read
    const int r = quarter * 32 + lane;     // row of the tile
    const int tok = r / p.G, g = r - tok * p.G;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t tm_S = tmem + C::COL_S + lane_off, tm_O = tmem + C::COL_O + lane_off;
    const float sl2 = p.scale_log2;
    int n_blocks = 0;
    auto load_q = [&](const Piece& y) {
      if (tok < y.n_tok) {
        const uint4* from = reinterpret_cast<const uint4*>(p.q + (y.t0 + tok) * p.ldq + (y.h * p.G + g) * DH);
        uint8_t* to = sQ + r * 128;
#pragma unroll
        for (int c = 0; c < DH / 8; ++c)
          *reinterpret_cast<uint4*>(to + (c >> 3) * (BM * 128) + (((c & 7) ^ (r & 7)) << 4)) = from[c];
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
    };
    bool more = walk.next(x);
    if (more) load_q(x);
    while (more) {
      const bool active = quarter * 32 < x.n_tok * p.G;      // whether any row of this warp counts
      const bool valid = tok < x.n_tok;
      const int t = x.t0 + tok;
      // positions that the row sees of this piece's
      const int limit = valid ? min(x.kend, direct ? s_len[t] : p.row_limit[t]) : x.kend;
      float m_ref = LOWEST, l = 0.f;
      for (int j = x.j0; j < x.j1; ++j, ++n_blocks) {
        mbar_wait_converged(s_full, n_blocks & 1, p.status, ST_TIMEOUT_TMEM_FULL);
        if (!active) {
          __syncwarp();
          if (lane == 0) { mbar_arrive(s_free); mbar_arrive(&p_full[n_blocks & 1]); }
          continue;
        }
        tc_fence_after();
        uint32_t v[BN];
        __syncwarp();
        tmem_ld_32x32_converged(tm_S, v);
        tmem_ld_32x32_converged(tm_S + 32, v + 32);
        tmem_ld_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(s_free);
        const int lim = limit - (x.kbase + j * BN);          // columns from here on are masked
        if (lim < BN) {
#pragma unroll
          for (int i = 0; i < BN; ++i)
            if (i >= lim) v[i] = 0xff800000u;
        }
        float m4[4] = {LOWEST, LOWEST, LOWEST, LOWEST};
#pragma unroll
        for (int i = 0; i < BN; i += 2)
          m4[(i >> 1) & 3] = max3(m4[(i >> 1) & 3], __uint_as_float(v[i]), __uint_as_float(v[i + 1]));
        const float m_blk = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
        const bool grow = m_blk > m_ref;
        const float alpha = grow ? ex2((m_ref - m_blk) * sl2) : 1.f;
        if (grow) m_ref = m_blk;
        const float neg_m = -m_ref;
        if (j > x.j0) {
          mbar_wait_converged(pv_done, (n_blocks - 1) & 1, p.status, ST_TIMEOUT_TMEM_FULL);
          tc_fence_after();
          if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
            for (int c = 0; c < DH / 32; ++c) {
              uint32_t o[32];
              tmem_ld_32x32_converged(tm_O + c * 32, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; i += 2) mul2(o[i], o[i + 1], alpha, alpha);
              tmem_st_32x32_converged(tm_O + c * 32, o);
            }
          }
        }
        float sum4[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        uint32_t pk[BN / 2];
#pragma unroll
        for (int i = 0; i < BN; i += 2) {
          // Subtracted before it is scaled: one fused step leaves the rounding of scale * m between a row's largest score and zero,
          // which is everything once scores are beyond 2^24.
          fma2(v[i], v[i + 1], 1.f, neg_m);
          mul2(v[i], v[i + 1], sl2, sl2);
          const float e0 = ex2(__uint_as_float(v[i])), e1 = ex2(__uint_as_float(v[i + 1]));
          add2(sum4[i & 6], sum4[(i & 6) + 1], __float_as_uint(e0), __float_as_uint(e1));
          pk[i >> 1] = pack_bf16x2(e0, e1);
        }
        tmem_st_32x32(tmem + C::COL_P + (n_blocks & 1) * (BN / 2) + lane_off, pk);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[n_blocks & 1]);
        const float sum = ((sum4[0] + sum4[1]) + (sum4[2] + sum4[3])) + ((sum4[4] + sum4[5]) + (sum4[6] + sum4[7]));
        l = __fadd_rn(__fmul_rn(l, alpha), sum);
      }
      // all products of this piece with its rows are done: the next piece's may take their place
      const Piece y = x;
      more = walk.next(x);
      if (more) load_q(x);
      if (!active) continue;
      mbar_wait_warp(pv_done, (n_blocks - 1) & 1, p.status, ST_TIMEOUT_TMEM_FULL);
      tc_fence_after();
      const int head = y.h * p.G + g;
      const bool out_now = !y.cut && p.prefix == 0;
      float* to = nullptr;
      if (valid && !out_now) {
        size_t row;
        float* base;
        size_t rows;
        if (y.cut) {
          row = static_cast<size_t>(2 * blockIdx.x + (y.first ? 0 : 1)) * BM + r;
          rows = static_cast<size_t>(2) * gridDim.x * BM;
          base = p.cut;
        } else {
          row = (static_cast<size_t>(y.shared ? 0 : p.NT) + t) * p.H + head;
          rows = static_cast<size_t>(2) * p.NT * p.H;
          base = p.whole;
        }
        to = base + row * DH;
        *reinterpret_cast<float2*>(base + rows * DH + row * 2) = make_float2(m_ref, l);
      }
      const float inv_l = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
      for (int c = 0; c < DH / 32; ++c) {
        uint32_t o[32];
        tmem_ld_32x32(tm_O + c * 32, o);
        tmem_ld_wait();
        if (valid && out_now) {
          __nv_bfloat16* orow = p.out + t * p.ldo + head * DH + c * 32;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint4 w;
            w.x = pack_bf16x2(__uint_as_float(o[i * 8 + 0]) * inv_l, __uint_as_float(o[i * 8 + 1]) * inv_l);
            w.y = pack_bf16x2(__uint_as_float(o[i * 8 + 2]) * inv_l, __uint_as_float(o[i * 8 + 3]) * inv_l);
            w.z = pack_bf16x2(__uint_as_float(o[i * 8 + 4]) * inv_l, __uint_as_float(o[i * 8 + 5]) * inv_l);
            w.w = pack_bf16x2(__uint_as_float(o[i * 8 + 6]) * inv_l, __uint_as_float(o[i * 8 + 7]) * inv_l);
            *reinterpret_cast<uint4*>(orow + i * 8) = w;
          }
        } else if (valid) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            *reinterpret_cast<uint4*>(to + c * 32 + i * 4) = make_uint4(o[i * 4], o[i * 4 + 1], o[i * 4 + 2], o[i * 4 + 3]);
        }
        __syncwarp();
      }
      tc_fence_before();      // O is in registers before the next piece's first P is handed over
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, TMEM_COLS);
}

// Joins the parts of a row: one CTA of four warps for each (token, head), the warps take every fourth part and add theirs in order.
template <int DH>
__global__ void __launch_bounds__(128) join_kernel(const __grid_constant__ Params p, int ctas) {
  constexpr int F = DH / 32;               // columns of a lane
  __shared__ float s_o[4][DH];
  __shared__ float s_m[4], s_l[4];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t = blockIdx.x, head = blockIdx.y, h = head / p.G;
  pdl_trigger();
  pdl_wait();
  const Header hdr = *p.hdr;
  const int pair = p.pair ? p.row_pair[t] : t;
  __nv_bfloat16* to = p.out + t * p.ldo + head * DH;
  if (pair < 0) {                          // a row of no sequence
    if (p.fill && threadIdx.x < DH) to[threadIdx.x] = __float2bfloat16_rn(0.f);
    return;
  }
  const Deal deal(hdr.units, ctas);
  // the row's two items: [begin, end) in the line of blocks, row inside the tile
  int beg[2], end[2], row[2];
  {
    const int blocks = blocks_of(p.prefix), tiles_q = (hdr.q_hi - hdr.q_lo + p.TT - 1) / p.TT;
    const int tile = (t - hdr.q_lo) / p.TT;
    beg[0] = (h * tiles_q + tile) * blocks;
    end[0] = beg[0] + blocks;
    row[0] = (t - hdr.q_lo - tile * p.TT) * p.G + head - h * p.G;
    const int before = p.cum[pair], size = p.cum[pair + 1] - before;
    beg[1] = hdr.units_shared + before * p.Hkv + h * size;
    end[1] = beg[1] + size;
    row[1] = (t - (p.pair ? p.pair[pair].t0 : t)) * p.G + head - h * p.G;
  }
  int c0[2], n[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const bool some = end[i] > beg[i];
    c0[i] = some ? deal.owner(beg[i]) : 0;
    n[i] = some ? deal.owner(end[i] - 1) - c0[i] + 1 : 0;
  }
  if (p.prefix == 0 && n[1] == 1) return;  // written out by its CTA
  const int parts = n[0] + n[1];
  const size_t rows_cut = static_cast<size_t>(2) * ctas * BM, rows_whole = static_cast<size_t>(2) * p.NT * p.H;
  auto part = [&](int k, const float*& o, const float*& ml) {
    const int i = k < n[0] ? 0 : 1;
    if (n[i] == 1) {
      const size_t at = (static_cast<size_t>(i ? p.NT : 0) + t) * p.H + head;
      o = p.whole + at * DH;
      ml = p.whole + rows_whole * DH + at * 2;
    } else {
      const int c = c0[i] + k - (i ? n[0] : 0);
      const size_t at = static_cast<size_t>(2 * c + (deal.begin(c) >= beg[i] ? 0 : 1)) * BM + row[i];
      o = p.cut + at * DH;
      ml = p.cut + rows_cut * DH + at * 2;
    }
  };
  float m = LOWEST, l = 0.f, acc[F];
#pragma unroll
  for (int f = 0; f < F; ++f) acc[f] = 0.f;
  // this warp's parts: a lane looks up one of up to 32, then all lanes read them one after the other
  for (int k0 = warp; k0 < parts; k0 += 4 * 32) {
    const int k = k0 + 4 * lane;
    const float* o = nullptr;
    float2 x = make_float2(LOWEST, 0.f);
    if (k < parts) {
      const float* ml;
      part(k, o, ml);
      x = *reinterpret_cast<const float2*>(ml);
    }
    float top = x.x;
#pragma unroll
    for (int s = 16; s; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
    if (top > m) {
      const float a = ex2((m - top) * p.scale_log2);
      l *= a;
#pragma unroll
      for (int f = 0; f < F; ++f) acc[f] *= a;
      m = top;
    }
    const float w = ex2((x.x - m) * p.scale_log2);
    float sum = w * x.y;
#pragma unroll
    for (int s = 16; s; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
    l += sum;
    const int count = min(32, (parts - k0 + 3) / 4);
#pragma unroll 4
    for (int i = 0; i < count; ++i) {
      const float* from = reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(o), i));
      const float wi = __shfl_sync(0xffffffffu, w, i);
#pragma unroll
      for (int f = 0; f < F; f += 2) {
        const float2 y = *reinterpret_cast<const float2*>(from + lane * F + f);
        acc[f] = fmaf(wi, y.x, acc[f]);
        acc[f + 1] = fmaf(wi, y.y, acc[f + 1]);
      }
    }
  }
#pragma unroll
  for (int f = 0; f < F; ++f) s_o[warp][lane * F + f] = acc[f];
  if (lane == 0) { s_m[warp] = m; s_l[warp] = l; }
  __syncthreads();
  if (threadIdx.x < DH) {
    const float top = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
    float sum = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float a = ex2((s_m[w] - top) * p.scale_log2);
      sum = fmaf(a, s_l[w], sum);
      o = fmaf(a, s_o[w][threadIdx.x], o);
    }
    to[threadIdx.x] = __float2bfloat16_rn(sum > 0.f ? o / sum : 0.f);
  }
}

// Bytes of the parts of the workspace, in the order in which they lie.
struct Layout {
  size_t cum, pair, limit, row_pair, whole, cut, total;
  Layout(long long NT, int H, int dh, int ctas, int max_pairs, bool planned, bool shared) {
    auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    cum = up(sizeof(Header));
    pair = cum + up((static_cast<size_t>(max_pairs) + 1) * 4);
    limit = pair + (planned ? up(static_cast<size_t>(max_pairs) * sizeof(Pair)) : 0);
    row_pair = limit + (planned ? up(static_cast<size_t>(NT) * 4) : 0);
    whole = row_pair + (planned ? up(static_cast<size_t>(NT) * 4) : 0);
    cut = whole + (shared ? up(static_cast<size_t>(2) * NT * H * (dh + 2) * 4) : 0);
    total = cut + up(static_cast<size_t>(2) * ctas * BM * (dh + 2) * 4);
  }
};

template <int DH>
static int launch(const CUtensorMap& tm, const Params& p, int ctas, cudaStream_t s) {
  static PerDeviceOnce attr;
  if (allow_smem(attr, attend_kernel<DH>, Cfg<DH>::SMEM_BYTES, SB_ERR_LAUNCH)) return SB_ERR_LAUNCH;
  if (p.pair && launch_dep(plan_kernel, dim3(1), dim3(1024), 0, s, p) != cudaSuccess) return SB_ERR_LAUNCH;
  if (launch_dep(attend_kernel<DH>, dim3(ctas), dim3(THREADS), Cfg<DH>::SMEM_BYTES, s, tm, p) != cudaSuccess) return SB_ERR_LAUNCH;
  return launch_dep(join_kernel<DH>, dim3(p.NT, p.H), dim3(128), 0, s, p, ctas) == cudaSuccess ? 0 : SB_ERR_LAUNCH;
}

static int ctas_for(long long units) {
  const long long most = 2ll * num_sms();
  return static_cast<int>(units < 1 ? 1 : units < most ? units : most);
}

}  // namespace spa
}  // namespace sb

using namespace sb;

// Bytes of workspace that sb_shared_prefix_attention needs (16-byte aligned); 0 where it would refuse the sizes.
extern "C" size_t sb_shared_prefix_attention_bytes(int NT, int B, int H, int Hkv, int dh, int ragged, int shared) {
  if (NT <= 0 || B <= 0 || H <= 0 || Hkv <= 0 || H % Hkv || H / Hkv > spa::BM) return 0;
  const bool planned = ragged || B > spa::MAX_DIRECT;
  const int max_pairs = ragged ? B + NT / (spa::BM / (H / Hkv)) : B;
  return spa::Layout(NT, H, dh, 2 * num_sms(), max_pairs, planned, shared != 0).total;
}

// q: bf16 [NT, ldq], query heads first, positions already rotated in. pool: n_blocks pages [2, Hkv, page, dh], page a multiple of 8.
// cu_q: [B + 1] rows of the sequences, or null: one row each (NT == B). seq_len: positions of each sequence, its rows' among them.
// prefix_table: pages of the first `prefix` positions, which all sequences share (prefix a multiple of page; 0: none). max_units bounds
// the blocks of 64 positions of all (sequence, kv head, tile of rows), which caps the grid.
extern "C" int sb_shared_prefix_attention(const void* q, long long ldq, const void* pool, int n_blocks, const int* block_table,
                                          int max_blocks, int page, const int* seq_len, const int* prefix_table, int prefix,
                                          const int* cu_q, int B, int NT, int H, int Hkv, int dh, long long max_units, float scale,
                                          void* workspace, size_t workspace_bytes, void* out, long long ldo, int fill, int* status,
                                          void* stream) {
  if (B <= 0 || NT <= 0 || H <= 0 || Hkv <= 0 || H % Hkv || H / Hkv > spa::BM || (dh != 64 && dh != 128) || n_blocks < 1 ||
      max_blocks < 1 || page < 8 || page % 8 || prefix < 0 || prefix % page || (prefix && !prefix_table) || (!cu_q && NT != B) ||
      !(scale > 0.f) || !status || !workspace)
    return SB_ERR_ARG;
  if ((reinterpret_cast<uintptr_t>(q) & 15) || (ldq & 7) || (reinterpret_cast<uintptr_t>(out) & 15) || (ldo & 7) ||
      (reinterpret_cast<uintptr_t>(workspace) & 15))
    return SB_ERR_ALIGN;
  const uint64_t rows = static_cast<uint64_t>(n_blocks) * 2 * Hkv * page;
  // coordinates of the pool's rows, and of the page behind the last that stands for a bad one; positions; the line of blocks
  if (rows + 2ull * Hkv * page >= (1ull << 31) || static_cast<uint64_t>(max_blocks) * page >= (1ull << 30) ||
      H > 65535)
    return SB_ERR_TOO_LARGE;
  const int G = H / Hkv, TT = spa::BM / G;
  const bool planned = cu_q || B > spa::MAX_DIRECT;
  const int max_pairs = cu_q ? B + NT / TT : B;
  const uint64_t cap = static_cast<uint64_t>(max_blocks) * page;
  if (static_cast<uint64_t>(Hkv) * max_pairs * (cap / spa::BN + 1) + static_cast<uint64_t>(Hkv) * (NT / TT + 1) * (prefix / spa::BN + 1) >=
      (1ull << 31))
    return SB_ERR_TOO_LARGE;
  const int ctas = spa::ctas_for(max_units);
  const spa::Layout at(NT, H, dh, ctas, max_pairs, planned, prefix > 0);
  if (at.total > workspace_bytes) return SB_ERR_ARG;
  int box = 64;
  while (page % box) box >>= 1;
  CUtensorMap tm;
  const int rc = make_tmap_2d_bf16(&tm, pool, dh, rows, dh, 64, box);
  if (rc) return rc;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  spa::Params p;
  p.q = static_cast<const __nv_bfloat16*>(q); p.ldq = ldq;
  p.block_table = block_table; p.max_blocks = max_blocks; p.seq_len = seq_len; p.prefix_table = prefix_table; p.cu_q = cu_q;
  p.prefix = prefix; p.page = page; p.n_blocks = n_blocks; p.box = box;
  p.B = B; p.NT = NT; p.H = H; p.Hkv = Hkv; p.G = G; p.TT = TT;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.out = static_cast<__nv_bfloat16*>(out); p.ldo = ldo; p.fill = fill;
  p.hdr = reinterpret_cast<spa::Header*>(ws);
  p.cum = reinterpret_cast<int*>(ws + at.cum);
  p.pair = planned ? reinterpret_cast<spa::Pair*>(ws + at.pair) : nullptr;
  p.row_limit = planned ? reinterpret_cast<int*>(ws + at.limit) : nullptr;
  p.row_pair = planned ? reinterpret_cast<int*>(ws + at.row_pair) : nullptr;
  p.whole = reinterpret_cast<float*>(ws + at.whole);
  p.cut = reinterpret_cast<float*>(ws + at.cut);
  p.max_pairs = max_pairs;
  p.status = status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dh == 64 ? spa::launch<64>(tm, p, ctas, s) : spa::launch<128>(tm, p, ctas, s);
}
