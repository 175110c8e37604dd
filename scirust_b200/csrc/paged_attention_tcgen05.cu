// Attention of a batch whose sequences share a prefix in the paged cache, on the tensor cores of sm_100a.
//
// Row (t, h) of the batch, token t of sequence b, sees the first `limit` positions of b:
//   s_j = scale q.k_j,  m = max s_j,  l = sum exp(s_j - m),  o = sum exp(s_j - m) v_j / l,   j < limit;   limit <= 0: o = 0.
// Positions below P (the whole pages of the prefix) are the same for all sequences, so the sum is taken in two parts: the rows of all
// sequences against one copy of K and V, and each sequence's rows against what it has for itself. Parts (m_i, l_i, o_i) of a row,
// o_i not divided by l_i, join as m = max m_i, w_i = 2^(m_i - m), o = sum w_i o_i / sum w_i l_i (scores in units of log 2).
//
// Both parts are the same work for a CTA: up to two tiles of 128 rows (tokens times the query heads of one kv head), a table of pages and
// a range of 128-position blocks of keys. An item is all of that for one set of rows:
//   shared: (kv head, consecutive tokens, whatever their sequences), blocks [0, P / 128)
//   own:    (sequence, tokens of it, kv head), blocks of [P, limit of its last row)
// Where the sequences bring a whole tile of rows each there is nothing to share, and their own items start at position 0.
// The blocks of all items form one line, which is dealt out over the CTAs, one a SM; what lies in a CTA's share of an item is a piece.
// An item that is not cut and has no other part is written out at once, pieces of the others go to a workspace and a second,
// dependent launch joins them in a fixed order, so that answers do not depend on what ran when.
//
// In a CTA a warp brings rows and K by TMA, one V, one issues S = Q K^T, one O += P V, and two lanes of four warps each turn scores into
// weights: lane by lane a tile each, or every second block of one tile, so that one lane's exponentials (128 x 128 of them take 1024
// cycles) run beside the products of the other. Scores, weights and both sums are in tensor memory, K and V in rings of blocks.
//
// What bounds it, B200, 32 / 8 heads of 128, a call in a graph:
//   many rows and a long prefix: the exponentials and what lies between them. A block of two tiles takes some 3700 cycles, 2048 of them
//     exponentials on each SM sub-partition, and 2048 products beside them: 520 tokens of 16 sequences behind 8192 positions 83 us, 0.54 of the matrix
//     rate.
//   one token a sequence: 64 sequences behind 16384 positions, up to 512 of their own, 60.5 us where memory would take 21: the sequences'
//     own items, 512 of two or three blocks, are as many starts and ends, and what they fetch of their own code; shared blocks are read
//     once, but a CTA's ten of them bring a new maximum, thus a pass over O, almost every time.
//   few sequences: latency. 4 samples behind 512 positions 10.8 us: 7 until the last CTA is done (3 of them until the first block has
//     come), 1 to the joining launch, 2 for that to find and to add up its parts.
// Code counts: pieces of one block go through most of the kernel once each. From 148 KB to 107 (and 76 where the batch is ragged, by a
// kernel of its own) the times above fell by 5 to 15 %.
#include "sm100_ptx.cuh"
#include "api.h"
#include "dependent.cuh"
#include "per_device.h"
#include <limits.h>
#include <type_traits>

namespace sb {

int num_sms();
int make_tmap_3d_bf16_box(CUtensorMap* out, const void* base, uint64_t d0, uint64_t d1, uint64_t d2, uint64_t pitch1, uint64_t pitch2,
                          uint32_t box0, uint32_t box1, uint32_t box2);
int make_tmap_2d_bf16(CUtensorMap* out, const void* base, uint64_t inner, uint64_t outer, uint64_t ld,
                      uint32_t box_inner, uint32_t box_outer);

namespace spa {

constexpr int BM = 128;        // rows of a tile
constexpr int BN = 128;        // positions of a block
constexpr int BN_LOG = 7;
constexpr int HALF = BN / 2;   // columns of P that are handed over at once
constexpr int THREADS = 384;   // loaders of rows and K, and of V, issuers of both products, two lanes of four softmax warps
// Registers a thread: 168 at launch for all three warpgroups, shared out as 72 + 2 x 216.
constexpr int REGS_ISSUE = 72, REGS_SOFTMAX = 216;
static_assert(REGS_ISSUE + 2 * REGS_SOFTMAX <= 3 * 168, "the shares draw on the registers of the launch");
constexpr int TMEM_COLS = 512;
constexpr int FEW = 8;         // rows of an item whose products are taken the other way round (few_rows)
constexpr int QUEUE = 4;       // pieces that the producer may be ahead
// Units (below) of a block of few rows, of one tile and of two, and of what an item costs besides its blocks, about half a microsecond each.
// 16 sequences behind 4000 positions 17.6 us, 33 behind 5003 32.1, 64 behind 16384 60.5, 256 of a block each behind 1024 76; with blocks of
// 2, 2, 4 and items of 4, 6, 10 they take 18.2, 32.9, 59.0 and 82, with 3, 2, 4 and 3, 5, 10 18.9, 32.9, 63.1 and 82.
constexpr int BLOCK_FEW = 3, BLOCK_ONE = 2, BLOCK_TWO = 4, ITEM_FEW = 1, ITEM_ONE = 4, ITEM_TWO = 10;
// A row's reference is its running maximum, so its largest weight is 1 and loses nothing when weights become bf16, and the sum is one of
// weights before that. A reference that may lag behind by 2^8 saves rescales of O (520 tokens behind 8192 positions 77 us for 83, 64
// sequences behind 16384 positions 58 for 60), for an error of 2.2e-3 in place of 2.0e-3 on unit scores and 1.3e-3 in place of 0.5e-3 on
// scores of four times the spread; with a sum of the rounded weights that is 1.0e-3, but the sum costs more than the rescales.
constexpr float LOWEST = -3.402823466e38f;   // reference of a row that has seen nothing: 2^(-inf - LOWEST) is 0

template <int DH>
struct Cfg {
  static constexpr int NCH = DH / 64;                // 64-column chunks of a head
  static constexpr int KV_BYTES = BN * DH * 2;
  static constexpr int SB = DH == 64 ? 2 : 1;        // score accumulators: one that the lanes take turns with at 128, one each at 64
  // Shared memory holds two tiles of the rows that the largest tile of the batch has, and as many blocks of K and V as go in beside them.
  static constexpr int MAX_SLOTS = DH == 128 ? 7 : 14;
  static constexpr int BAR_BYTES = (8 * (2 * MAX_SLOTS + 2 * QUEUE + 2 + 2 + 2 + 2 + 4 + 2 + 4 + 4 + 2) + 8 + 15) / 16 * 16;
  static constexpr int FIXED_BYTES = BAR_BYTES + QUEUE * 32 + BM * 8 + 2 * 2 * 4 * FEW * 4 + 1024 /* alignment */;
  static int slots(int q_rows) {
    const int n = (227 * 1024 - FIXED_BYTES - 2 * q_rows * DH * 2) / KV_BYTES;
    return n < MAX_SLOTS ? n : MAX_SLOTS;
  }
  static int smem_bytes(int q_rows) { return 2 * q_rows * DH * 2 + slots(q_rows) * KV_BYTES + FIXED_BYTES; }
  static_assert((227 * 1024 - FIXED_BYTES - 2 * BM * DH * 2) / KV_BYTES >= 5, "three blocks of K and two of V beside two full tiles");
  // tensor memory: scores, P of each lane as bf16 pairs, O of each lane
  static constexpr int COL_P = SB * BN, COL_O = COL_P + 2 * (BN / 2);
  static_assert(COL_O + 2 * DH <= TMEM_COLS, "tensor memory");
};

// What the plan says of an item of its own: tokens [t0, t0 + n), sequence, position behind the last one that a row sees.
struct Pair {
  int t0, n, b, kend;
};

struct Header {        // at the start of the workspace, of a batch that has been planned
  int units_shared, units_own, q_lo, q_hi, pairs;
  int least;           // no row sees fewer positions
  int pad[2];
};

// a / d for 0 <= a < 2^31 by a multiplication, where the host knows d: m = 2^k / d rounded up with k = 31 + log2 d rounded up, so that
// m d - 2^k < 2^(k - 31).
struct Divisor {
  unsigned m;
  int shift;
  __host__ void set(int d) {
    int log = 0;
    while ((1ll << log) < d) ++log;
    shift = 31 + log;
    m = static_cast<unsigned>(((1ull << shift) + d - 1) / d);
  }
  __device__ __forceinline__ int of(int a) const { return static_cast<int>((static_cast<unsigned long long>(a) * m) >> shift); }
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
  int page, n_blocks, box_log;
  Divisor by_page, by_heads, by_span;     // page, Hkv, 2 TT
  int B, NT, H, Hkv, G, TT;
  int few;             // items whose products are taken the other way round: 1 a sequence's own, 2 shared ones (few_rows)
  int q_tokens;        // of the box that brings a tile of rows
  int q_rows;          // of a tile in shared memory, a multiple of 8; the tensor core reads 128, those behind are rows of no one
  int ks, vs;          // blocks of K and V in shared memory
  float scale_log2;
  __nv_bfloat16* out;
  long long ldo;
  int fill;            // rows of no sequence become zero instead of staying as they are
  Header* hdr;
  int* cum;            // [pairs + 1] blocks of own items before a pair, of one kv head
  Pair* pair;
  int* row_limit;      // [NT]
  int* row_pair;       // [NT], -1: of no sequence
  int2* part;          // [Hkv][shared tiles] and then [pairs][Hkv]: CTAs that have a piece of the item; twice the first of these, 1 more for
                       // its second piece
  int* row_t0;         // [NT] first token of its pair
  float* whole;        // [slots][NT][H][dh], and [slots][NT][H][2] behind it: items that were not cut, shared and then own
  float* cut;          // [2 * CTAs][256][dh], and [2 * CTAs][256][2] behind it: first and last pieces of the CTAs
  int shared_items;    // entries of `part` that shared items have
  int max_pairs;
  int* status;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 32 bytes, a whole sector.
__device__ __forceinline__ void st_global_v8(float* to, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]),
               "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
constexpr int kTries = 1 << 21;
// Wait of a whole warp, all lanes with one result; bounded like mbar_wait, in a third of the instructions, since there are some
// forty in the kernel.
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, int* status, int code) {
  int tries = 0;
#pragma unroll 1
  while (!__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) {
    // a try takes 20 cycles at least, some thousand as a rule
    if (++tries > kTries || ((tries & 15) == 0 && __any_sync(0xffffffffu, *reinterpret_cast<volatile int*>(status) != 0))) {
      atomicCAS(status, 0, code);
      return false;
    }
  }
  return true;
}
// Lane 0's value: the same for the whole warp, as the compiler then knows.
__device__ __forceinline__ uint32_t same(uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); }
__device__ __forceinline__ int clampi(int v, int lo, int hi) { return min(max(v, lo), hi); }

// a / d for 0 <= a < 2^31, d > 0 and results below 2^20, where the estimate is off by one at most: the compiler's own division takes four
// times the instructions.
__device__ __forceinline__ int quotient(int a, int d) {
  const int q = static_cast<int>(__fdividef(static_cast<float>(a), static_cast<float>(d))), r = a - q * d;
  return q - (r < 0) + (r >= d);
}

__device__ __forceinline__ int blocks_of(int positions) { return positions > 0 ? (positions + BN - 1) / BN : 0; }
// An item lies in the line with the units of its blocks, in front of which are those for what it costs besides.
__device__ __forceinline__ int block_units(int n_tok, int TT, bool few) { return few ? BLOCK_FEW : n_tok > TT ? BLOCK_TWO : BLOCK_ONE; }
__device__ __forceinline__ int head_units(int n_tok, int TT, bool few) { return few ? ITEM_FEW : n_tok > TT ? ITEM_TWO : ITEM_ONE; }
__device__ __forceinline__ int units_of(int positions, int n_tok, int TT, bool few) {
  return positions > 0 ? blocks_of(positions) * block_units(n_tok, TT, few) + head_units(n_tok, TT, few) : 0;
}
// a / block_units
__device__ __forceinline__ int blocks_in(int units, int each) {
  return each == BLOCK_FEW ? static_cast<int>(__umulhi(units, 0xaaaaaaabu) >> 1) : units >> (each >> 1);
}

// The deal of the line over the CTAs: shared items to the first of them, own ones to the others, the units of either evenly. A CTA also
// has to begin a piece that its neighbour's share has cut, which is dearer for shared items (of two tiles) than for own ones (of a few
// rows). With U and V units, `more` units dearer: U / n + more = V / (ctas - n) for n CTAs. Shares that do not mind the border leave some
// CTAs with many ends of shared items, others with none: 12.5 us in place of 10.9 (4 samples behind 512), 20.0 / 18.6 (16 behind 4000).
// At least the units of a block a CTA, so that one between the ends of an item has a block of it, whose units may lie with two CTAs (the
// first unit's CTA has the block).
struct Deal {                              // the part of it that CTA c has a share of
  int from, units, first, per, rem;        // where it begins in the line, its units, its first CTA
  __device__ Deal(int units_shared, int units_own, int grid, int c, int more) {
    int n = units_shared > 0 ? grid : 0;   // CTAs of the shared part
    if (units_shared > 0 && units_own > 0) {
      const float U = units_shared, V = units_own, N = grid, b = more * N - U - V;
      n = clampi(__float2int_ru(2.f * U * N / (sqrtf(b * b + 4.f * more * U * N) - b)), 1, grid - 1);
    }
    const bool own = c >= n;
    from = own ? units_shared : 0;
    units = own ? units_own : units_shared;
    first = own ? n : 0;
    const int share = max(1, min(own ? grid - n : n, units / BLOCK_TWO));
    per = units / share;                   // may be large
    rem = units - per * share;
  }
  __device__ int begin(int c) const { return from + min(units, (c - first) * per + min(c - first, rem)); }
  __device__ int owner(int u) const {
    const int v = u - from, edge = rem * (per + 1);
    const bool low = v < edge;
    return first + quotient(low ? v : v - edge, low ? per + 1 : max(per, 1)) + (low ? 0 : rem);
  }
};

// The shared items of one kv head: tiles of two times TT tokens, the last of which may have one tile of rows.
struct Shared {
  int tiles, size, last, head;        // items of a head, units of an item and of the last one, of a head
  __device__ Shared(const Params& p, int tokens) {
    const int prefix = p.prefix, TT = p.TT;
    const bool few = p.few & 2;
    tiles = prefix > 0 ? p.by_span.of(tokens + 2 * TT - 1) : 0;
    size = units_of(prefix, 2 * TT, TT, false);
    last = units_of(prefix, tokens - (tiles - 1) * 2 * TT, TT, few);
    head = tiles > 0 ? (tiles - 1) * size + last : 0;
  }
};

__device__ __forceinline__ float warp_max(float x) {
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}
// Inclusive sum over a warp.
__device__ __forceinline__ int warp_scan(int v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += x;
  }
  return v;
}

// A piece of an item. The producer finds a CTA's pieces, one after the other, and hands them to the other warps.
struct Piece {
  int h, t0, n_tok, kbase, kend, j0, j1;   // blocks [j0, j1) of kbase + 128 j, positions below kend
  int flags;                               // and the sequence, whose table it is, from SEQUENCE on
};
// CUT: not all of its item; FIRST: begins where the CTA's share does; SHORT: some row may end inside
constexpr int PIECE_SHARED = 1, PIECE_CUT = 2, PIECE_FIRST = 4, PIECE_SHORT = 8, SEQUENCE = 4;

// Slots of the rows of items that were not cut: of shared items (of few rows by kv head, token and query head, of others as the batch has
// them), then of own ones.
__host__ __device__ __forceinline__ int own_slot(const Params& p) { return p.prefix == 0 ? 0 : 1; }
__host__ __device__ __forceinline__ int whole_slots(const Params& p) { return own_slot(p) + 1; }

// Whether the products are taken the other way round, S^T = K Q^T and O^T = V^T P^T, of up to eight rows (a sequence of one token has as
// many as query heads share a kv head). In a tile of 128 rows they would be lanes 0 to 7 of one warp, which would go through 128 columns
// of scores and dh of O one by one; here a thread has a position, or a column of O, of all rows, an eighth of the instructions. 64
// sequences behind 16384 positions, 500 of their own: 57 us, as tiles of 128 rows 65 to 71; 64 of their own, a block each, where the code
// of both weighs more than what it saves, 55 and 50; 16 sequences with 1 of their own 27.5 and 25.
template <bool PLANNED>
__device__ __forceinline__ bool few_rows(const Params& p, const Piece& x) {
  return !PLANNED && (x.flags & PIECE_SHARED ? p.few & 2 : p.few & 1) != 0;
}

// A CTA's pieces, found by a whole warp. The plan of a batch of one token a sequence is summed up on the way, 32 sequences at a time; a
// ragged one has been planned (plan_kernel). From one item to the next there is no division and no search, which took 4000 cycles a piece,
// as long as the others take for one of one block.
template <bool PLANNED>
struct Walk {
  const Params& p;
  const Shared shared;
  int units_shared, q_lo, q_hi, pairs;
  int u, u1, u_first;
  int h, tile, size;             // the item: kv head; tile of shared items, or lane that has the pair; units
  int last, index;               // the first unit of its last block, its entry of p.part
  int window, c_lo, c_hi;        // pairs window + lane: units of one kv head before and behind
  int4 info;

  __device__ Walk(const Params& p_, const Header& hd, int u0, int u1_)
      : p(p_), shared(p_, hd.q_hi - hd.q_lo), units_shared(hd.units_shared), q_lo(hd.q_lo), q_hi(hd.q_hi),
        pairs(hd.pairs), u(u0), u1(u1_), u_first(u0), h(0), tile(0), size(0), last(0), index(0), window(-32), c_lo(0), c_hi(0),
        info(make_int4(0, 0, 0, 0)) {}

  // The pairs behind those of the window.
  __device__ void advance(int lane) {
    const int before = window < 0 || PLANNED ? 0 : __shfl_sync(0xffffffffu, c_hi, 31), i = (window += 32) + lane;
    if (PLANNED) {
      c_lo = c_hi = -1;
      if (i < pairs) {
        c_lo = p.cum[i];
        c_hi = p.cum[i + 1];
        info = *reinterpret_cast<const int4*>(p.pair + i);
      }
    } else {
      const int len = i < pairs ? clampi(p.seq_len[i], 0, p.max_blocks * p.page) : 0;
      const int n = units_of(len - p.prefix, 1, p.TT, p.few & 1);
      c_hi = before + warp_scan(n, lane);
      c_lo = c_hi - n;
      info = make_int4(i, 1, i, len);
    }
  }

  // False: no more pieces.
  __device__ bool next(Piece& x) {
    const int lane = threadIdx.x & 31;
    for (;;) {
      if (u >= u1) return false;
      int off = 0;
      x.flags = 0;
      if (u < units_shared) {
        if (u == u_first) {
          h = quotient(u, shared.head);
          const int rest = u - h * shared.head;
          tile = min(quotient(rest, shared.size), shared.tiles - 1);
          off = rest - tile * shared.size;
        } else if (++tile == shared.tiles) {
          tile = 0;
          ++h;
        }
        size = tile == shared.tiles - 1 ? shared.last : shared.size;
        x.t0 = q_lo + tile * 2 * p.TT;
        x.n_tok = min(2 * p.TT, q_hi - x.t0);
        index = h * shared.tiles + tile;
        x.kbase = 0;
        x.kend = p.prefix;
        x.flags = PIECE_SHARED;
      } else {
        // the first lane whose pair has units beyond v
        int v = -1;
        unsigned mask = 0;                        // nothing in the window yet
        if (u == u_first) {
          v = u - units_shared;
          if (PLANNED) {                           // last pair that starts at v or before
            int lo = 0, hi = pairs - 1;
            while (lo < hi) {
              const int mid = (lo + hi + 1) >> 1;
              if (p.cum[mid] * p.Hkv <= v) lo = mid; else hi = mid - 1;
            }
            window = lo - 32;
          }
        } else if (++h == p.Hkv) {
          mask = tile == 31 ? 0u : 0xffffffffu << (tile + 1);
        }
        if (u == u_first || h == p.Hkv) {
          unsigned open;
          while (!(open = __ballot_sync(0xffffffffu, c_hi * p.Hkv > v && c_hi > c_lo) & mask)) {
            if (window + 32 >= pairs) return false;
            advance(lane);
            mask = 0xffffffffu;
          }
          tile = __ffs(open) - 1;
          const int before = __shfl_sync(0xffffffffu, c_lo, tile);
          size = __shfl_sync(0xffffffffu, c_hi, tile) - before;
          h = 0;
          if (u == u_first) {
            const int rest = v - before * p.Hkv;
            h = quotient(rest, size);
            off = rest - h * size;
          }
        }
        x.t0 = __shfl_sync(0xffffffffu, info.x, tile);
        x.n_tok = __shfl_sync(0xffffffffu, info.y, tile);
        x.kend = __shfl_sync(0xffffffffu, info.w, tile);
        x.kbase = p.prefix;
        index = p.shared_items + (window + tile) * p.Hkv + h;
        x.flags = __shfl_sync(0xffffffffu, info.z, tile) << SEQUENCE;
      }
      x.h = h;
      if (u == u_first) x.flags |= PIECE_FIRST;
      const int stop = min(size, off + (u1 - u)), begin = u - off;
      u += stop - off;
      // a block belongs to the CTA that has its first unit
      const bool few = few_rows<PLANNED>(p, x);
      const int head = head_units(x.n_tok, p.TT, few), each = block_units(x.n_tok, p.TT, few), blocks = blocks_in(size - head, each);
      x.j0 = blocks_in(max(0, off - head) + each - 1, each);
      x.j1 = blocks_in(max(0, stop - head) + each - 1, each);
      if (x.j1 == x.j0) continue;
      if (x.j1 - x.j0 != blocks) x.flags |= PIECE_CUT;
      last = begin + head + (blocks - 1) * each;
      return true;
    }
  }
};

// Plan of a ragged batch: one CTA.
__global__ void __launch_bounds__(1024) plan_kernel(const Params p) {
  __shared__ int s_warp[32];
  __shared__ int s_hi, s_pairs, s_sum, s_least;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_trigger();
  pdl_wait();
  if (tid == 0) { s_hi = clampi(p.cu_q[0], 0, p.NT); s_pairs = 0; s_sum = 0; s_least = INT_MAX; }
  for (int t = tid; t < p.NT; t += 1024) { p.row_limit[t] = 0; p.row_pair[t] = -1; }
  __syncthreads();
  const int q_lo = s_hi;
  const int cap = p.max_blocks * p.page;
  for (int b0 = 0; b0 < p.B; b0 += 1024) {
    const int b = b0 + tid;
    int start = 0, end = 0;
    if (b < p.B) {
      start = clampi(p.cu_q[b], 0, p.NT);
      end = clampi(p.cu_q[b + 1], 0, p.NT);
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
    const int span = 2 * p.TT;             // tokens of an item
    int tiles = (n + span - 1) / span;
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
      if (n > 0) atomicMin(&s_least, len - n + 1);
      for (int i = 0; i < tiles && at + i < p.max_pairs; ++i) {
        Pair x;
        x.t0 = start + i * span;
        x.n = min(span, n - i * span);
        x.b = b;
        x.kend = len - n + i * span + x.n;
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
      p.row_t0[x.x + r] = x.x;
    }
  }
  for (int i0 = 0; i0 < pairs; i0 += 1024) {
    const int i = i0 + tid;
    const int n = i < pairs ? units_of(p.pair[i].kend - p.prefix, p.pair[i].n, p.TT, false) : 0;
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
    p.hdr->units_shared = p.Hkv * Shared(p, q_hi - q_lo).head;
    p.hdr->units_own = p.Hkv * s_sum;
    p.hdr->q_lo = q_lo; p.hdr->q_hi = q_hi; p.hdr->pairs = pairs;
    p.hdr->least = s_least;
  }
}

// What brings the blocks of K, or of V, whole warp. The table is read ahead: 32 boxes of the piece while the 32 in front of them are
// brought, and the first of the next piece while this one is.
struct Boxes {
  int from, page, in;            // lane i: page of box (from + i) of a piece, and where in it the box begins
};
struct Ring {
  uint8_t* at;
  uint64_t *full, *empty;
  const int* table;
  int slots, slot, head, row;    // lane i: first row in the pool of its box
  uint32_t phase;
  Boxes now, then;

  __device__ Ring(uint8_t* at_, uint64_t* full_, uint64_t* empty_, int slots_)
      : at(at_), full(full_), empty(empty_), table(nullptr), slots(slots_), slot(0), head(0), row(0), phase(0) {}

  __device__ static const int* table_of(const Params& p, const Piece& x) {
    return x.flags & PIECE_SHARED ? p.prefix_table : p.block_table + static_cast<size_t>(x.flags >> SEQUENCE) * p.max_blocks;
  }
  __device__ static Boxes boxes(const Params& p, const Piece& x, const int* table, int from) {
    const int pos = x.kbase + ((from + static_cast<int>(threadIdx.x & 31)) << p.box_log), at_page = p.by_page.of(pos);
    Boxes b;
    b.from = from;
    b.in = pos - at_page * p.page;
    b.page = pos < x.kend ? table[at_page] : 0;
    return b;
  }
  __device__ static Boxes first(const Params& p, const Piece& x) { return boxes(p, x, table_of(p, x), x.j0 << (BN_LOG - p.box_log)); }

  __device__ void rows(const Params& p) {
    const int page = static_cast<unsigned>(now.page) >= static_cast<unsigned>(p.n_blocks) ? p.n_blocks : now.page;   // reads as zeros
    row = (page * 2 * p.Hkv + head) * p.page + now.in;
  }
  __device__ void piece(const Params& p, const Piece& x, int head_, const Boxes& first_) {
    table = table_of(p, x);
    head = head_;
    now = first_;
    then.from = -1;
    rows(p);
  }

  template <int DH>
  __device__ bool load(const Params& p, const CUtensorMap& tmap, const Piece& x, int j) {
    const int lane = threadIdx.x & 31, nbx = BN >> p.box_log, bx0 = j << (BN_LOG - p.box_log);       // boxes of a block, at most 16
    if (bx0 >= now.from + 32) {               // nbx divides 32: a block's boxes are read together
      now = then;
      rows(p);
      then.from = -1;
    }
    if (then.from < 0 && (now.from + 32) << p.box_log < x.kend - x.kbase) then = boxes(p, x, table, now.from + 32);
    if (!wait(&empty[slot], phase ^ 1, p.status, ST_TIMEOUT_EMPTY)) return false;
    const int live = min(nbx, (x.kend - x.kbase - j * BN + (1 << p.box_log) - 1) >> p.box_log);     // boxes with a position below kend
    if (lane == 0) mbar_arrive_expect_tx(&full[slot], (live * DH * 2) << p.box_log);
    __syncwarp();
    const int i = lane - (bx0 - now.from);
    if (i >= 0 && i < live) {
      uint8_t* to = at + slot * (BN * DH * 2) + (i << p.box_log) * 128;
#pragma unroll
      for (int c = 0; c < DH / 64; ++c) tma_load_2d(to + c * (BN * 128), &tmap, &full[slot], c * 64, row);
    }
    __syncwarp();
    if (++slot == slots) { slot = 0; phase ^= 1; }
    return true;
  }
};

template <int DH, bool PLANNED>
__global__ void __launch_bounds__(THREADS, 1)
attend_kernel(const __grid_constant__ CUtensorMap tmap, const __grid_constant__ CUtensorMap q_tile,
              const __grid_constant__ Params p) {
  using C = Cfg<DH>;
  const int KS = p.ks, VS = p.vs;
  const int q_chunk = p.q_rows * 128, q_bytes = q_chunk * C::NCH;      // a 64-column chunk of a tile of rows, the tile
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sQ = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sK = sQ + 2 * q_bytes;
  uint8_t* sV = sK + KS * C::KV_BYTES;
  uint64_t* k_full = reinterpret_cast<uint64_t*>(sV + VS * C::KV_BYTES);      // [KS]
  uint64_t* k_empty = k_full + KS;
  uint64_t* v_full = k_empty + KS;       // [VS]
  uint64_t* v_empty = v_full + VS;
  uint64_t* x_full = v_empty + VS;       // [QUEUE] a piece is in the queue
  uint64_t* x_empty = x_full + QUEUE;    // [QUEUE] and has been read (loader of V, issuers, eight softmax warps)
  uint64_t* q_full = x_empty + QUEUE;    // [2] rows of every second piece are in shared memory
  uint64_t* q_empty = q_full + 2;        // [2] and have been multiplied
  uint64_t* s_full = q_empty + 2;        // [2] scores of a lane's block are in tensor memory
  uint64_t* s_free = s_full + 2;         // [SB] the scores that lay in this accumulator are in registers (4 warp arrivals)
  uint64_t* p_full = s_free + 2;         // [2][2] a half of a lane's P is in tensor memory, O rescaled (4 warp arrivals)
  uint64_t* pv_done = p_full + 4;        // [2] P V of a lane's block has completed
  uint64_t* o_full = pv_done + 2;        // [4] a quarter of the rows: lane 1 has its sum ready for lane 0
  uint64_t* o_free = o_full + 4;         // [4] and lane 0 has read it
  uint64_t* r_full = o_free + 4;         // [2] few rows: what the warps of a lane tell each other is in shared memory (4 warp arrivals)
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(r_full + 2);
  Piece* queue = reinterpret_cast<Piece*>(sV + VS * C::KV_BYTES + C::BAR_BYTES);
  // maximum and sum: [BM] of lane 1; of few rows [lane][warp][row]
  float2* s_ml = reinterpret_cast<float2*>(queue + QUEUE);
  float* s_max = reinterpret_cast<float*>(s_ml + BM);                         // [lane][block, even or odd][warp][row]

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
#pragma unroll 1
    for (int s = 0; s < KS; ++s) { mbar_init(&k_full[s], 1); mbar_init(&k_empty[s], 1); }
#pragma unroll 1
    for (int s = 0; s < VS; ++s) { mbar_init(&v_full[s], 1); mbar_init(&v_empty[s], 1); }
#pragma unroll 1
    for (int s = 0; s < QUEUE; ++s) { mbar_init(&x_full[s], 1); mbar_init(&x_empty[s], 11); }
#pragma unroll 1
    for (int s = 0; s < 2; ++s) {
      mbar_init(&q_full[s], 1);
      mbar_init(&q_empty[s], 1);
      mbar_init(&s_full[s], 1);
      mbar_init(&s_free[s], 4);
      mbar_init(&pv_done[s], 1);
      mbar_init(&r_full[s], 4);
    }
#pragma unroll 1
    for (int s = 0; s < 4; ++s) {
      mbar_init(&p_full[s], 4);
      mbar_init(&o_full[s], 1);
      mbar_init(&o_free[s], 1);
    }
    fence_barrier_init();
    fence_proxy_async_smem();
    prefetch_tmap(&tmap);
    prefetch_tmap(&q_tile);
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

  // Pieces as the other warps get them from warp 0; j1 == 0 is the end. A piece of more rows than a tile has gives each lane a
  // tile, and both take every block; of one tile both take the rows, and every second block. The lanes take turns throughout: `steps`
  // counts what both have taken (a block of a lane is a step).
  int at = 0;
  uint32_t at_phase = 0;
  auto take = [&](Piece& x) -> bool {
    if (!wait(&x_full[at], at_phase, p.status, ST_TIMEOUT_MISC)) return false;
    const int4* from = reinterpret_cast<const int4*>(queue + at);
    const int4 a = from[0], b = from[1];
    x.h = a.x; x.t0 = a.y; x.n_tok = a.z; x.kbase = a.w;
    x.kend = b.x; x.j0 = b.y; x.j1 = b.z; x.flags = b.w;
    __syncwarp();
    if (lane == 0) mbar_arrive(&x_empty[at]);
    if (++at == QUEUE) { at = 0; at_phase ^= 1; }
    return x.j1 != 0;
  };
  Piece x = {};

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_ISSUE));
  if (warp == 0) {
    // -------------------------------- pieces, their rows, and K --------------------------------
    Header hdr;
    if (PLANNED) {
      hdr.units_shared = p.hdr->units_shared; hdr.units_own = p.hdr->units_own;
      hdr.q_lo = p.hdr->q_lo; hdr.q_hi = p.hdr->q_hi; hdr.pairs = p.hdr->pairs; hdr.least = p.hdr->least;
    } else {
      const int cap = p.max_blocks * p.page;
      int sum = 0, least = INT_MAX;
#pragma unroll 1
      for (int b0 = 0; b0 < p.B; b0 += 32) {
        const int b = b0 + lane;
        const int len = b < p.B ? clampi(p.seq_len[b], 0, cap) : INT_MAX;
        const int n = b < p.B ? units_of(len - p.prefix, 1, p.TT, p.few & 1) : 0;
        least = min(least, len);
        sum += __reduce_add_sync(0xffffffffu, n);
      }
      hdr.q_lo = 0; hdr.q_hi = p.B; hdr.pairs = p.B; hdr.least = __reduce_min_sync(0xffffffffu, least);
      hdr.units_shared = p.Hkv * Shared(p, p.B).head;
      hdr.units_own = p.Hkv * sum;
    }
    const Deal deal(hdr.units_shared, hdr.units_own, gridDim.x, blockIdx.x,
                    head_units(hdr.q_hi - hdr.q_lo, p.TT, (p.few & 2) != 0) - head_units(1, p.TT, p.few & 1));
    Walk<PLANNED> walk(p, hdr, deal.begin(blockIdx.x), deal.begin(blockIdx.x + 1));
    Ring k(sK, k_full, k_empty, KS);
    int n_pieces = 0;
    bool ok = true, both = false, begun = false;
    Piece y = {};                          // the piece behind x
    Boxes first = {};
    while (ok) {
      if (begun) {
        x = y;
        if (hdr.least < x.kend) x.flags |= PIECE_SHORT;
        ok = wait(&x_empty[at], at_phase ^ 1, p.status, ST_TIMEOUT_EMPTY);
        if (!ok) break;
        if (lane == 0) {
          int4* to = reinterpret_cast<int4*>(queue + at);
          to[0] = make_int4(x.h, x.t0, x.n_tok, x.kbase);
          to[1] = make_int4(x.kend, x.j0, x.j1, x.flags);
          mbar_arrive(&x_full[at]);
        }
        __syncwarp();
        if (++at == QUEUE) { at = 0; at_phase ^= 1; }
        if (x.j1 == 0) break;
        if (x.j0 == 0 && lane == 0)        // for the joining launch
          p.part[walk.index] = make_int2(x.flags & PIECE_CUT ? deal.owner(walk.last) - static_cast<int>(blockIdx.x) + 1 : 1,
                                         2 * blockIdx.x + (x.flags & PIECE_FIRST ? 0 : 1));
        k.piece(p, x, x.h, first);
      }
      if (walk.next(y)) first = Ring::first(p, y);
      else y.j0 = y.j1 = 0;
      if (!begun) {
        begun = true;
        continue;
      }
      const bool two = x.n_tok > p.TT;
#pragma unroll 1
      for (int j = x.j0; j < x.j1 && ok; ++j) {
        ok = k.template load<DH>(p, tmap, x, j);
        if (j > x.j0) continue;
        // Rows of a piece of one tile go to either half of the space, while those of the piece before are multiplied; two tiles take both.
        // So the piece before the last has been multiplied, and where both halves are needed the last too.
#pragma unroll 1
        for (int before = 2; before >= (two || both ? 1 : 2); --before) {
          const int piece = n_pieces - before;
          ok = ok && (piece < 0 || wait(&q_empty[piece & 1], (piece >> 1) & 1, p.status, ST_TIMEOUT_EMPTY));
        }
        both = two;
        if (ok && lane == 0) {
          // The box of a tile brings its tokens and, behind the last of them, rows of others that no one reads. For one token a box of its
          // own gains nothing (256 sequences behind 1024 positions 78.8 us with it, 75.5 without).
          const int tiles = two ? 2 : 1, bytes = p.q_tokens * p.G * 128;
          uint64_t* bar = &q_full[n_pieces & 1];
          mbar_arrive_expect_tx(bar, tiles * C::NCH * bytes);
#pragma unroll 1
          for (int i = 0; i < tiles * C::NCH; ++i) {
            const int tile = i / C::NCH, c = i % C::NCH;
            tma_load_3d(sQ + (two ? tile : n_pieces & 1) * q_bytes + c * q_chunk, &q_tile, bar, c * 64, x.h * p.G, x.t0 + tile * p.TT);
          }
        }
        __syncwarp();
      }
      ++n_pieces;
    }
  } else if (warp == 3) {
    // -------------------------------- V --------------------------------
    Ring v(sV, v_full, v_empty, VS);
    bool ok = true;
    while (ok && take(x)) {
      v.piece(p, x, p.Hkv + x.h, Ring::first(p, x));
#pragma unroll 1
      for (int j = x.j0; j < x.j1 && ok; ++j) ok = v.template load<DH>(p, tmap, x, j);
    }
  } else if (warp == 1) {
    // ------------------------------------- S = Q K^T -------------------------------------
    // The two products have a warp each: what one of them waits for, asks and counts (half of the time of a single warp for both) the
    // tensor core spends on the other's. The warp walks its loop as a whole and one lane issues; what an instruction is given comes from
    // lane 0 by a shuffle, so that it is known to be the same for the warp and stays in uniform registers.
    const bool leader = elect_one();
    constexpr uint64_t desc = (static_cast<uint64_t>(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61) | (1ull << 16);
    constexpr uint64_t desc_same = desc & ~(0x3fffull << 32);        // every eight rows are the same eight
    const uint32_t at_q = smem_u32(sQ), at_k = smem_u32(sK), q_step = same(q_chunk >> 4);
    constexpr uint32_t k_step = BN * 8;
    int ks = 0, n_pieces = 0, steps = 0;
    uint32_t kph = 0;
    bool ok = true;
    while (ok && take(x)) {
      const int half = n_pieces & 1;
      const bool two = same(x.n_tok > p.TT ? 1 : 0);
      const int n = same((x.j1 - x.j0) << (two ? 1 : 0));
      // few rows: a product of 16 columns at least, of which eight are the others again
      ok = wait(&q_full[half], (n_pieces >> 1) & 1, p.status, ST_TIMEOUT_MISC);
      auto steps_of = [&](auto kind) {
        constexpr bool few = decltype(kind)::value;
#pragma unroll 1
        for (int i = 0; i < n && ok; ++i, ++steps) {
          const int L = steps & 1;
          const bool uses = !two || (i & 1) == 0, frees = !two || (i & 1) == 1;      // the block's first step, its last
          const int before = C::SB == 1 ? steps : steps >> 1;                        // scores that were in this accumulator
          const uint32_t q_lo = same((at_q + (two ? L : half) * q_bytes) >> 4), k_lo = same((at_k + ks * C::KV_BYTES) >> 4);
          const uint32_t to = same(tmem + (C::SB == 1 ? 0 : L * BN));
          if (uses) ok = wait(&k_full[ks], kph, p.status, ST_TIMEOUT_FULL);
          if (before > 0) ok = ok && wait(&s_free[C::SB == 1 ? 0 : L], (before - 1) & 1, p.status, ST_TIMEOUT_TMEM_EMPTY);
          if (!ok) break;
          tc_fence_after();
          if (leader) {
            if (few) {
#pragma unroll
              for (int k = 0; k < DH / 16; ++k)
                umma_bf16_ss(to, desc | (k_lo + (k >> 2) * k_step + (k & 3) * 2), desc_same | (q_lo + (k >> 2) * q_step + (k & 3) * 2),
                             make_idesc_bf16(BM, 2 * FEW, false, false), k > 0 ? 1u : 0u);
            } else {
#pragma unroll
              for (int k = 0; k < DH / 16; ++k)
                umma_bf16_ss(to, desc | (q_lo + (k >> 2) * q_step + (k & 3) * 2), desc | (k_lo + (k >> 2) * k_step + (k & 3) * 2),
                             make_idesc_bf16(BM, BN, false, false), k > 0 ? 1u : 0u);
            }
            umma_commit(&s_full[L]);
            if (frees && !few) umma_commit(&k_empty[ks]);
            if (i == n - 1) umma_commit(&q_empty[half]);
          }
          if (frees) {
            if (++ks == KS) { ks = 0; kph ^= 1; }
          }
        }
      };
      if (!PLANNED && same(few_rows<PLANNED>(p, x) ? 1 : 0)) steps_of(std::bool_constant<!PLANNED>{});
      else steps_of(std::false_type{});
      ++n_pieces;
    }
  } else {
    // ------------------------------------- O (+)= P V -------------------------------------
    const bool leader = elect_one();
    constexpr uint32_t idesc = make_idesc_bf16(BM, DH, false, true);
    constexpr uint64_t desc = (static_cast<uint64_t>(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61) | (static_cast<uint64_t>(BN * 8) << 16);
    // few rows: V^T has 128 rows (at dh 64 each of them twice), P^T lies in the block of K, eight rows of a position behind one another
    constexpr uint32_t idesc_few = make_idesc_bf16(BM, 2 * FEW, true, true);
    constexpr uint64_t desc_few = DH == 128 ? desc : desc & ~(0x3fffull << 16);
    constexpr uint64_t desc_p = (1ull << 46) | (static_cast<uint64_t>(8 * FEW * 2 >> 4) << 16);
    const uint32_t a_v = smem_u32(sV), a_k = smem_u32(sK);
    int vs = 0, ks = 0, steps = 0;
    uint32_t vph = 0;
    bool ok = true;
    while (ok && take(x)) {
      const bool two = same(x.n_tok > p.TT ? 1 : 0);
      const int n = same((x.j1 - x.j0) << (two ? 1 : 0)), first_live = same(x.kend - x.kbase - x.j0 * BN);
      auto steps_of = [&](auto kind) {
        constexpr bool few = decltype(kind)::value;
#pragma unroll 1
        for (int i = 0; i < n && ok; ++i, ++steps) {
          const int L = steps & 1, turn = steps >> 1;            // every second step is this lane's
          const bool uses = !two || (i & 1) == 0, frees = !two || (i & 1) == 1;
          const int live = min(BN, first_live - (two ? i >> 1 : i) * BN);            // positions that count
          const uint32_t v_lo = same((a_v + vs * C::KV_BYTES) >> 4), p_lo = same((a_k + ks * C::KV_BYTES) >> 4), o = same(tmem + C::COL_O + L * DH),
                         w = same(tmem + C::COL_P + L * (BN / 2)), begins = same(i < 2 ? 1 : 0);
          if (uses) {
            ok = wait(&v_full[vs], vph, p.status, ST_TIMEOUT_FULL);
            if (ok && (live & 15)) {
              // A product takes 16 positions. The weights of those behind the end are zero, but what lies there may be no number, and zero
              // times it would be none either.
              uint8_t* v = sV + vs * C::KV_BYTES;
#pragma unroll 1
              for (int c = lane; c < (16 - (live & 15)) * (DH / 8); c += 32) {
                const int row = live + c / (DH / 8), e = c % (DH / 8);       // rows are whole, so their swizzle does not matter
                *reinterpret_cast<uint4*>(v + (e >> 3) * (BN * 128) + row * 128 + (e & 7) * 16) = make_uint4(0, 0, 0, 0);
              }
              fence_proxy_async_smem();
              __syncwarp();
            }
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            ok = ok && wait(&p_full[2 * L + h], turn & 1, p.status, ST_TIMEOUT_MISC);
            if (!ok) break;
            tc_fence_after();
            if (leader) {
#pragma unroll
              for (int k2 = 0; k2 < HALF / 16; ++k2) {
                const int k = h * (HALF / 16) + k2;
                if (k * 16 < live) {
                  if (few) umma_bf16_ss(o, desc_few | (v_lo + k * 128), desc_p | (p_lo + k * FEW * 2), idesc_few, (!begins || k > 0) ? 1u : 0u);
                  else umma_bf16_ts(o, w + k * 8, desc | (v_lo + k * 128), idesc, (!begins || k > 0) ? 1u : 0u);
                }
              }
            }
          }
          if (!ok) break;
          if (leader) {
            umma_commit(&pv_done[L]);
            if (frees) umma_commit(&v_empty[vs]);
            if (few) umma_commit(&k_empty[ks]);
          }
          if (frees) {
            if (++ks == KS) ks = 0;
            if (++vs == VS) { vs = 0; vph ^= 1; }
          }
        }
      };
      if (!PLANNED && same(few_rows<PLANNED>(p, x) ? 1 : 0)) steps_of(std::bool_constant<!PLANNED>{});
      else steps_of(std::false_type{});
    }
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_SOFTMAX));
    // ------------------------------------ softmax warps ------------------------------------
    const int L = (warp >> 2) - 1;         // lane
    const int quarter = warp & 3;          // lanes of tensor memory that this warp may read
    const int r = quarter * 32 + lane;     // row of the tile
    const int tile_tok = quotient(r, p.G), tile_g = r - tile_tok * p.G;
    const int few_tok = quotient(lane & (FEW - 1), p.G);       // of row lane & 7
    const uint32_t tm = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t tm_S = tm + (C::SB == 1 ? 0 : L * BN), tm_P = tm + C::COL_P + L * (BN / 2), tm_O = tm + C::COL_O + L * DH;
    const float sl2 = p.scale_log2;
    int n = 0, steps = 0, n_join = 0;      // this lane's blocks; both lanes'; pieces whose lanes were joined
    int slot0 = 0, told = 0;               // few rows: where the piece's first block of K lies; phases of r_full
    bool pending = false;                  // lane 1: its O waits to be read by lane 0
    while (take(x)) {
      const bool two = x.n_tok > p.TT;
      const int nb = x.j1 - x.j0;
      const int first = two ? 0 : (L ^ steps) & 1, step = two ? 1 : 2;           // this lane's blocks
      steps += two ? 2 * nb : nb;
      int slot = 0;
      if (!PLANNED && p.few) {
        slot = slot0 + first;
        if (slot >= KS) slot -= KS;
        slot0 += nb;
        slot0 -= quotient(slot0, KS) * KS;
      }
      if (first >= nb) continue;
      if (few_rows<PLANNED>(p, x)) {
        // A thread has position r of a block, and then column r of O, of all rows.
        const int rows = x.n_tok * p.G;
        int limit = x.kend;                // of row lane & 7
        if ((x.flags & (PIECE_SHARED | PIECE_SHORT)) == (PIECE_SHARED | PIECE_SHORT) && few_tok < x.n_tok)
          limit = min(limit, p.seq_len[x.t0 + few_tok]);
        float m_ref[FEW], l[FEW];
#pragma unroll
        for (int e = 0; e < FEW; ++e) { m_ref[e] = LOWEST; l[e] = 0.f; }
        // What the lane's warps wrote is there for all of them.
        auto meet = [&]() {
          __syncwarp();
          if (lane == 0) mbar_arrive(&r_full[L]);
          wait(&r_full[L], told & 1, p.status, ST_TIMEOUT_MISC);
          ++told;
        };
#pragma unroll 1
        for (int i = first; i < nb; i += step, ++n) {
          // the same waits as below, which do not end the loop either
          wait(&s_full[L], n & 1, p.status, ST_TIMEOUT_TMEM_FULL);
          tc_fence_after();
          uint32_t v[FEW], o[FEW];
          tmem_ld_32x8(tm_S, v);
          tmem_ld_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s_free[C::SB == 1 ? 0 : L]);
          const int pos = x.kbase + (x.j0 + i) * BN + r;
          if (__any_sync(0xffffffffu, limit <= pos - lane + 31)) {
#pragma unroll
            for (int e = 0; e < FEW; ++e)
              if (pos >= __shfl_sync(0xffffffffu, limit, e)) v[e] = 0xff800000u;
          }
          float4* top = reinterpret_cast<float4*>(s_max + (L * 2 + (n & 1)) * 4 * FEW);
          float m[FEW];
#pragma unroll
          for (int e = 0; e < FEW; ++e) m[e] = warp_max(__uint_as_float(v[e]));
          if (lane == 0) {
            top[quarter * 2] = make_float4(m[0], m[1], m[2], m[3]);
            top[quarter * 2 + 1] = make_float4(m[4], m[5], m[6], m[7]);
          }
          meet();
          bool grow = false, huge = false;
          float alpha[FEW];
#pragma unroll
          for (int e = 0; e < FEW; ++e) m[e] = LOWEST;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const float4 a = top[w * 2], b = top[w * 2 + 1];
            m[0] = fmaxf(m[0], a.x); m[1] = fmaxf(m[1], a.y); m[2] = fmaxf(m[2], a.z); m[3] = fmaxf(m[3], a.w);
            m[4] = fmaxf(m[4], b.x); m[5] = fmaxf(m[5], b.y); m[6] = fmaxf(m[6], b.z); m[7] = fmaxf(m[7], b.w);
          }
#pragma unroll
          for (int e = 0; e < FEW; ++e) {
            const float now = fmaxf(m[e] * sl2, m_ref[e]);
            grow |= e < rows && now > m_ref[e];        // what lies in columns behind the last row decides nothing
            alpha[e] = ex2(m_ref[e] - now);
            m_ref[e] = now;
            huge |= e < rows && fabsf(now) > 16777216.f && now != LOWEST;
          }
          if (n > 0) {
            wait(&pv_done[L], (n - 1) & 1, p.status, ST_TIMEOUT_TMEM_FULL);
            tc_fence_after();
            if (i > first && grow) {       // all threads of the lane have the same maxima
              tmem_ld_32x8(tm_O, o);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < FEW; e += 2) mul2(o[e], o[e + 1], alpha[e], alpha[e + 1]);
              tmem_st_32x8(tm_O, o);
              tmem_st_wait();
            }
          }
          if (pending) {
            wait(&o_free[quarter], (n_join - 1) & 1, p.status, ST_TIMEOUT_TMEM_EMPTY);
            pending = false;
          }
          float factor = sl2;
          if (huge) {                      // scaled beforehand, as below
#pragma unroll
            for (int e = 0; e < FEW; e += 2) mul2(v[e], v[e + 1], sl2, sl2);
            factor = 1.f;
          }
          float w[FEW];
#pragma unroll
          for (int e = 0; e < FEW; ++e) {
            w[e] = ex2(__fmaf_rn(__uint_as_float(v[e]), factor, -m_ref[e]));
            l[e] = __fmaf_rn(l[e], alpha[e], w[e]);
          }
          *reinterpret_cast<uint4*>(sK + slot * C::KV_BYTES + r * 16) =
              make_uint4(pack_bf16x2(w[0], w[1]), pack_bf16x2(w[2], w[3]), pack_bf16x2(w[4], w[5]), pack_bf16x2(w[6], w[7]));
          slot += step;
          if (slot >= KS) slot -= KS;
          fence_proxy_async_smem();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) { mbar_arrive(&p_full[2 * L]); mbar_arrive(&p_full[2 * L + 1]); }
        }
        // Sums over the warp: a lane passes on what it has of the rows that the other keeps. Row `own` ends in every fourth lane.
        const int own = lane >> 2;
        const bool up16 = lane & 16, up8 = lane & 8, up4 = lane & 4;
        float a4[4], b4[4], a2[2], b2[2];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          a4[e] = (up16 ? l[e + 4] : l[e]) + __shfl_xor_sync(0xffffffffu, up16 ? l[e] : l[e + 4], 16);
          b4[e] = up16 ? m_ref[e + 4] : m_ref[e];
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          a2[e] = (up8 ? a4[e + 2] : a4[e]) + __shfl_xor_sync(0xffffffffu, up8 ? a4[e] : a4[e + 2], 8);
          b2[e] = up8 ? b4[e + 2] : b4[e];
        }
        float sum = (up4 ? a2[1] : a2[0]) + __shfl_xor_sync(0xffffffffu, up4 ? a2[0] : a2[1], 4), m_own = up4 ? b2[1] : b2[0];
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        const bool joins = nb > 1;
        wait(&pv_done[L], (n - 1) & 1, p.status, ST_TIMEOUT_TMEM_FULL);
        tc_fence_after();
        float2* ml = s_ml + (L * 4 + quarter) * FEW;
        uint32_t o[FEW];
        if (joins && L == 1) {
          if ((lane & 3) == 0) ml[own] = make_float2(m_own, sum);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&o_full[quarter]);
          ++n_join;
          pending = true;
          continue;
        }
        tmem_ld_32x8(tm_O, o);
        if (joins) {
          const float2* other = s_ml + (4 + quarter) * FEW;
          uint32_t o1[FEW];
          wait(&o_full[quarter], n_join & 1, p.status, ST_TIMEOUT_TMEM_FULL);
          tc_fence_after();
          tmem_ld_32x8(tm_O + DH, o1);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < FEW; ++e) {
            const float y = other[e].x, m = fmaxf(m_ref[e], y);
            o[e] = __float_as_uint(__fmaf_rn(ex2(m_ref[e] - m), __uint_as_float(o[e]), __fmul_rn(ex2(y - m), __uint_as_float(o1[e]))));
          }
          const float2 y = other[own];
          const float m = fmaxf(m_own, y.x);
          sum = __fmaf_rn(ex2(m_own - m), sum, __fmul_rn(ex2(y.x - m), y.y));
          m_own = m;
          __syncwarp();
          tc_fence_before();
          if (lane == 0) mbar_arrive(&o_free[quarter]);
          ++n_join;
        }
        if ((lane & 3) == 0) ml[own] = make_float2(m_own, sum);
        meet();
        // Rows of a piece lie behind one another. A CTA has two slots, for its first and its last piece, the only ones that can be cut. What
        // lies between has a place of its own, since a CTA may have any number of these: a shared item, of all tokens, among those of the kv
        // heads, an own one, of one token, where its rows are in the batch.
        const bool cut = x.flags & PIECE_CUT;
        const unsigned row = cut                      ? (2 * blockIdx.x + (x.flags & PIECE_FIRST ? 0 : 1)) * (2 * BM)
                             : x.flags & PIECE_SHARED ? x.h * p.NT * p.G
                                                      : (own_slot(p) * p.NT + x.t0) * p.H + x.h * p.G;
        const size_t n_rows = cut ? static_cast<size_t>(2) * gridDim.x * (2 * BM) : static_cast<size_t>(whole_slots(p)) * p.NT * p.H;
        float* base = cut ? p.cut : p.whole;
        if (quarter == 0 && lane < rows) {
          float2 y = s_ml[L * 4 * FEW + lane];
#pragma unroll
          for (int w = 1; w < 4; ++w) y.y += s_ml[(L * 4 + w) * FEW + lane].y;
          reinterpret_cast<float2*>(base + n_rows * DH)[row + lane] = y;
        }
        __syncwarp();                      // an aligned instruction behind stores of some lanes
        tmem_ld_wait();
        float* to = base + static_cast<size_t>(row) * DH + r;
        if (r < DH) {
#pragma unroll
          for (int e = 0; e < FEW; ++e)
            if (e < rows) to[e * DH] = __uint_as_float(o[e]);
        }
        __syncwarp();
        tc_fence_before();
        continue;
      }
      const int g = tile_g;
      const int toks = two ? min(p.TT, x.n_tok - L * p.TT) : x.n_tok, tok = tile_tok + (two ? L * p.TT : 0);
      const bool active = quarter * 32 < toks * p.G;      // whether any row of this warp counts
      const bool valid = tile_tok < toks;
      const int t = x.t0 + tok;
      // positions that the row sees of this piece's
      int limit = x.kend;
      if (valid) {
        if (!(x.flags & PIECE_SHARED)) limit -= x.n_tok - 1 - tok;
        else if (x.flags & PIECE_SHORT) limit = min(limit, PLANNED ? p.row_limit[t] : p.seq_len[t]);
      }
      float m_ref = LOWEST, l = 0.f;
#pragma unroll 1
      for (int i = first; i < nb; i += step, ++n) {
        // Waits in this loop may give up (the status word says so) but do not end it: lanes that left it one by one would be
        // missing at the warp barriers below.
        wait(&s_full[L], n & 1, p.status, ST_TIMEOUT_TMEM_FULL);
        if (!active) {
          __syncwarp();
          if (lane == 0) mbar_arrive(&s_free[C::SB == 1 ? 0 : L]);
          // P V of the block before: its P was complete then, so these arrivals are this block's
          if (n > 0) wait(&pv_done[L], (n - 1) & 1, p.status, ST_TIMEOUT_TMEM_FULL);
          if (pending) {                   // as below
            wait(&o_free[quarter], (n_join - 1) & 1, p.status, ST_TIMEOUT_TMEM_EMPTY);
            pending = false;
          }
          __syncwarp();
          if (lane == 0) { mbar_arrive(&p_full[2 * L]); mbar_arrive(&p_full[2 * L + 1]); }
          continue;
        }
        tc_fence_after();
        const int lim = limit - (x.kbase + (x.j0 + i) * BN);          // columns from here on are masked
        float m_blk, sum4[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        // The row's reference for this block, P V of the lane's block before, which frees P, and O, if the reference has moved; the factor
        // of what the row has so far.
        auto turn = [&]() -> float {
          const float m_new = m_blk * sl2;
          const bool grow = m_new > m_ref;
          const float alpha = grow ? ex2(m_ref - m_new) : 1.f;
          if (grow) m_ref = m_new;
          if (n > 0) {
            wait(&pv_done[L], (n - 1) & 1, p.status, ST_TIMEOUT_TMEM_FULL);
            tc_fence_after();
            if (i > first && __any_sync(0xffffffffu, grow)) {
#pragma unroll 1
              for (int c = 0; c < DH / 32; ++c) {
                uint32_t o[32];
                tmem_ld_32x32_converged(tm_O + c * 32, o);
                tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 32; e += 2) mul2(o[e], o[e + 1], alpha, alpha);
                tmem_st_32x32_converged(tm_O + c * 32, o);
              }
            }
          }
          if (pending) {                   // O of the piece before is about to be overwritten
            wait(&o_free[quarter], (n_join - 1) & 1, p.status, ST_TIMEOUT_TMEM_EMPTY);
            pending = false;
          }
          return alpha;
        };
        // Weights of two columns, as bf16. Scale and difference are one fused step, whose exponent is off from the rounded reference by up
        // to half a step of it: nothing, unless scores are beyond 2^24. Those are scaled beforehand, rounded as the reference was.
        float factor = sl2;
        auto scaled_first = [&](uint32_t* u) {
          if (__any_sync(0xffffffffu, valid && fabsf(m_ref) > 16777216.f && m_ref != LOWEST)) {
#pragma unroll
            for (int c = 0; c < BN; c += 2) mul2(u[c], u[c + 1], sl2, sl2);
            factor = 1.f;
          }
        };
        auto weigh = [&](uint32_t& a, uint32_t& b, int c) -> uint32_t {
          fma2(a, b, factor, -m_ref);
          const float e0 = ex2(__uint_as_float(a)), e1 = ex2(__uint_as_float(b));
          add2(sum4[c & 6], sum4[(c & 6) + 1], __float_as_uint(e0), __float_as_uint(e1));
          return pack_bf16x2(e0, e1);
        };
        uint32_t v[BN];
        __syncwarp();
#pragma unroll
        for (int c = 0; c < BN / 32; ++c) tmem_ld_32x32_converged(tm_S + c * 32, v + c * 32);
        tmem_ld_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_free[C::SB == 1 ? 0 : L]);
        if (__any_sync(0xffffffffu, lim < BN)) {
#pragma unroll
          for (int w = 0; w < BN / 32; ++w) {
            const int in = clampi(lim - w * 32, 0, 32);
            const uint32_t seen = in == 32 ? 0xffffffffu : (1u << in) - 1;
#pragma unroll
            for (int c = 0; c < 32; ++c)
              if (!(seen >> c & 1)) v[w * 32 + c] = 0xff800000u;
          }
        }
        float m4[4] = {LOWEST, LOWEST, LOWEST, LOWEST};
#pragma unroll
        for (int c = 0; c < BN; c += 2)
          m4[(c >> 1) & 3] = max3(m4[(c >> 1) & 3], __uint_as_float(v[c]), __uint_as_float(v[c + 1]));
        m_blk = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
        const float alpha = turn();
        scaled_first(v);
        const int live = x.kend - (x.kbase + (x.j0 + i) * BN);      // positions that any row sees
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (h == 1 && live <= HALF) {    // nothing of it is multiplied
            if (lane == 0) mbar_arrive(&p_full[2 * L + 1]);
            break;
          }
          uint32_t pk[HALF / 2];
#pragma unroll
          for (int c2 = 0; c2 < HALF; c2 += 2) pk[c2 >> 1] = weigh(v[h * HALF + c2], v[h * HALF + c2 + 1], h * HALF + c2);
          tmem_st_32x32(tm_P + h * (HALF / 2), pk);
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[2 * L + h]);
        }
        const float sum = ((sum4[0] + sum4[1]) + (sum4[2] + sum4[3])) + ((sum4[4] + sum4[5]) + (sum4[6] + sum4[7]));
        l = __fadd_rn(__fmul_rn(l, alpha), sum);
      }
      if (!active) continue;
      const bool joins = !two && nb > 1;        // both lanes have a sum of these rows
      wait(&pv_done[L], (n - 1) & 1, p.status, ST_TIMEOUT_TMEM_FULL);
      tc_fence_after();
      if (joins && L == 1) {
        s_ml[r] = make_float2(m_ref, l);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&o_full[quarter]);
        ++n_join;
        pending = true;
        continue;
      }
      float w0 = 1.f, w1 = 0.f;
      if (joins) {
        wait(&o_full[quarter], n_join & 1, p.status, ST_TIMEOUT_TMEM_FULL);
        tc_fence_after();
        const float2 y = s_ml[r];
        const float m = fmaxf(m_ref, y.x);
        w0 = ex2(m_ref - m);
        w1 = ex2(y.x - m);
        m_ref = m;
        l = __fmaf_rn(w0, l, __fmul_rn(w1, y.y));
      }
      const int head = x.h * p.G + g;
      const bool cut = x.flags & PIECE_CUT;
      const bool out_now = !cut && p.prefix == 0;
      float* to = nullptr;
      if (valid && !out_now) {
        size_t row, rows;
        float* base;
        if (cut) {
          row = static_cast<size_t>(2 * blockIdx.x + (x.flags & PIECE_FIRST ? 0 : 1)) * (2 * BM) + (two ? L * BM : 0) + r;
          rows = static_cast<size_t>(2) * gridDim.x * (2 * BM);
          base = p.cut;
        } else {
          row = (static_cast<size_t>(x.flags & PIECE_SHARED ? 0 : own_slot(p)) * p.NT + t) * p.H + head;
          rows = static_cast<size_t>(whole_slots(p)) * p.NT * p.H;
          base = p.whole;
        }
        to = base + row * DH;
        *reinterpret_cast<float2*>(base + rows * DH + row * 2) = make_float2(m_ref, l);
      }
      const float inv_l = l > 0.f ? 1.f / l : 0.f;
#pragma unroll 1
      for (int c0 = 0; c0 < DH; c0 += 32) {
        uint32_t o[32];
        __syncwarp();
        tmem_ld_32x32_converged(tm_O + c0, o);
        if (joins) {
          uint32_t o1[32];
          tmem_ld_32x32_converged(tm_O + DH + c0, o1);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 32; ++e)
            o[e] = __float_as_uint(__fmaf_rn(w0, __uint_as_float(o[e]), __fmul_rn(w1, __uint_as_float(o1[e]))));
        }
        tmem_ld_wait();
        if (valid && out_now) {
          __nv_bfloat16* orow = p.out + t * p.ldo + head * DH + c0;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint4 w;
            w.x = pack_bf16x2(__uint_as_float(o[e * 8 + 0]) * inv_l, __uint_as_float(o[e * 8 + 1]) * inv_l);
            w.y = pack_bf16x2(__uint_as_float(o[e * 8 + 2]) * inv_l, __uint_as_float(o[e * 8 + 3]) * inv_l);
            w.z = pack_bf16x2(__uint_as_float(o[e * 8 + 4]) * inv_l, __uint_as_float(o[e * 8 + 5]) * inv_l);
            w.w = pack_bf16x2(__uint_as_float(o[e * 8 + 6]) * inv_l, __uint_as_float(o[e * 8 + 7]) * inv_l);
            *reinterpret_cast<uint4*>(orow + e * 8) = w;
          }
        } else if (valid) {
#pragma unroll
          for (int e = 0; e < 32; e += 8) st_global_v8(to + c0 + e, o + e);
        }
      }
      __syncwarp();
      tc_fence_before();      // O is in registers before the next piece's first P is handed over
      if (joins) {
        if (lane == 0) mbar_arrive(&o_free[quarter]);
        ++n_join;
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, TMEM_COLS);
}

// Joins the parts of rows. The heads of a (token, kv head) have the same parts, so they are looked up once. PACKED, for many rows of few
// parts: a warp has the rows of a (token, kv head), two at a time, and a CTA four of these. Otherwise a CTA has them, four at a time, a
// row to WAYS warps, which share its parts; their sums meet in shared memory. What an item's parts are has been left by the CTA that has its
// first block (Params::part): worked out here it takes 1.5 us longer.
template <int DH, int WAYS, bool PACKED>
__global__ void __launch_bounds__(128 * WAYS) join_kernel(const __grid_constant__ Params p, int ctas) {
  constexpr int F = DH / 32;               // columns of a lane
  static_assert(WAYS == 1 || !PACKED, "");
  constexpr int ROWS = PACKED ? 1 : 4, AT_ONCE = PACKED ? 2 : 1, BATCH = PACKED || WAYS > 1 ? 4 : 8;       // rows a CTA, a warp; parts at a time
  using Vec = typename std::conditional<F == 4, float4, float2>::type;
  __shared__ float s_o[WAYS > 1 ? ROWS : 1][WAYS][DH];
  __shared__ float2 s_ml[ROWS][WAYS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, way = warp % WAYS, slot = PACKED ? 0 : warp / WAYS;
  const int job = PACKED ? blockIdx.x * 4 + warp : blockIdx.x;
  const int t = p.by_heads.of(job), h = job - t * p.Hkv;
  pdl_trigger();
  pdl_wait();
  if (t >= p.NT) return;
  const int pair = p.pair ? p.row_pair[t] : t;
  if (pair < 0) {                          // a row of no sequence
    if (p.fill)
      for (int i = PACKED ? lane : threadIdx.x; i < p.G * DH; i += PACKED ? 32 : 32 * ROWS * WAYS)
        p.out[t * p.ldo + h * p.G * DH + i] = __float2bfloat16_rn(0.f);
    return;
  }
  // The row's two items: parts, where the first lies and those of the CTAs behind it, which begin with theirs.
  int q_lo = 0, q_hi = p.NT, t0 = t, kend;
  if (p.pair) {
    q_lo = p.hdr->q_lo;
    q_hi = p.hdr->q_hi;
    t0 = p.row_t0[t];
    kend = p.pair[pair].kend;
  } else {
    kend = clampi(p.seq_len[t], 0, p.max_blocks * p.page);
  }
  const int2 own = p.part[p.shared_items + pair * p.Hkv + h];
  int2 common = make_int2(0, 0);
  int first = 0;                           // token of the shared item
  if (p.prefix > 0) {
    const int tile = p.by_span.of(t - q_lo);
    common = p.part[h * p.by_span.of(q_hi - q_lo + 2 * p.TT - 1) + tile];
    first = q_lo + tile * 2 * p.TT;
  }
  int n[2];
  const float* from[2];
  const float2* ml[2];
  int jump[2];                             // rows from the first part to the second, which is 4 * BM in front of the third
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    // in bounds even where a wait of the other launch has given up and the entry is none
    int2 x = i ? own : common;
    x.y = clampi(x.y, 0, 2 * ctas - 1);
    const int count = i && kend <= p.prefix ? 0 : clampi(x.x, 0, ctas - (x.y >> 1)), tok = t - (i ? t0 : first);
    const bool cut = count > 1;
    const size_t at = cut               ? static_cast<size_t>(x.y) * (2 * BM) + (tok < p.TT ? tok * p.G : BM + (tok - p.TT) * p.G)
                      : !i && p.few & 2 ? (static_cast<size_t>(h) * p.NT + t) * p.G
                                        : (static_cast<size_t>(i ? own_slot(p) : 0) * p.NT + t) * p.H + h * p.G;
    const size_t rows = cut ? static_cast<size_t>(4) * ctas * BM : static_cast<size_t>(whole_slots(p)) * p.NT * p.H;
    const float* base = cut ? p.cut : p.whole;
    n[i] = count;
    from[i] = base + at * DH + lane * F;
    ml[i] = reinterpret_cast<const float2*>(base + rows * DH) + at;
    jump[i] = x.y & 1 ? 2 * BM : 4 * BM;
  }
  if (p.prefix == 0 && !p.few && n[1] == 1) return;  // written out by its CTA
  const int parts = n[0] + n[1];
#pragma unroll 1
  for (int g0 = 0; g0 < p.G; g0 += ROWS * AT_ONCE) {
    const int g = g0 + slot;               // this warp's rows: g, and g + 1
    float m[AT_ONCE], l[AT_ONCE], acc[AT_ONCE][F];
#pragma unroll
    for (int r = 0; r < AT_ONCE; ++r) {
      m[r] = LOWEST;
      l[r] = 0.f;
#pragma unroll
      for (int f = 0; f < F; ++f) acc[r][f] = 0.f;
    }
#pragma unroll 1
    for (int k0 = way; k0 < parts; k0 += WAYS * BATCH) {
      Vec o[AT_ONCE][BATCH];
      float2 x[AT_ONCE][BATCH];
#pragma unroll
      for (int b = 0; b < BATCH; ++b) {
        const int k = k0 + b * WAYS;
        const bool own = k >= n[0];
        const int c = own ? k - n[0] : k;
        const int row = g + (c > 0 ? (own ? jump[1] : jump[0]) + (c - 1) * (4 * BM) : 0);
        const float* at_o = (own ? from[1] : from[0]) + static_cast<long long>(row) * DH;
        const float2* at_ml = (own ? ml[1] : ml[0]) + row;
#pragma unroll
        for (int r = 0; r < AT_ONCE; ++r) {
          x[r][b] = make_float2(LOWEST, 0.f);
          o[r][b] = Vec{};
          if (k < parts && g + r < p.G) {
            o[r][b] = *reinterpret_cast<const Vec*>(at_o + r * DH);
            x[r][b] = at_ml[r];
          }
        }
      }
#pragma unroll
      for (int r = 0; r < AT_ONCE; ++r) {
        float top = m[r];
#pragma unroll
        for (int b = 0; b < BATCH; ++b) top = fmaxf(top, x[r][b].x);
        const float a = ex2(m[r] - top);
        l[r] *= a;
#pragma unroll
        for (int f = 0; f < F; ++f) acc[r][f] *= a;
        m[r] = top;
#pragma unroll
        for (int b = 0; b < BATCH; ++b) {            // a part that is none has no weight: l is 0 and so is o
          const float w = ex2(x[r][b].x - top);
          l[r] = fmaf(w, x[r][b].y, l[r]);
          acc[r][0] = fmaf(w, o[r][b].x, acc[r][0]);
          acc[r][1] = fmaf(w, o[r][b].y, acc[r][1]);
          if constexpr (F == 4) {
            acc[r][2] = fmaf(w, o[r][b].z, acc[r][2]);
            acc[r][3] = fmaf(w, o[r][b].w, acc[r][3]);
          }
        }
      }
    }
    if constexpr (WAYS > 1) {
#pragma unroll
      for (int f = 0; f < F; ++f) s_o[slot][way][lane * F + f] = acc[0][f];
      if (lane == 0) s_ml[slot][way] = make_float2(m[0], l[0]);
      __syncthreads();
      if (way == 0) {
        float top = m[0];
#pragma unroll
        for (int w = 1; w < WAYS; ++w) top = fmaxf(top, s_ml[slot][w].x);
        const float a = ex2(m[0] - top);
        l[0] *= a;
#pragma unroll
        for (int f = 0; f < F; ++f) acc[0][f] *= a;
#pragma unroll 1
        for (int w = 1; w < WAYS; ++w) {
          const float2 y = s_ml[slot][w];
          const float b = ex2(y.x - top);
          l[0] = fmaf(b, y.y, l[0]);
#pragma unroll
          for (int f = 0; f < F; ++f) acc[0][f] = fmaf(b, s_o[slot][w][lane * F + f], acc[0][f]);
        }
      }
      __syncthreads();
    }
#pragma unroll
    for (int r = 0; r < AT_ONCE; ++r) {
      if (g + r < p.G && way == 0) {
        const float inv = l[r] > 0.f ? 1.f / l[r] : 0.f;
        __nv_bfloat16* to = p.out + t * p.ldo + (h * p.G + g + r) * DH + lane * F;
        if constexpr (F == 4)
          *reinterpret_cast<uint2*>(to) =
              make_uint2(pack_bf16x2(acc[r][0] * inv, acc[r][1] * inv), pack_bf16x2(acc[r][2] * inv, acc[r][3] * inv));
        else
          *reinterpret_cast<uint32_t*>(to) = pack_bf16x2(acc[r][0] * inv, acc[r][1] * inv);
      }
    }
  }
}

// Bytes of the parts of the workspace, in the order in which they lie.
struct Layout {
  size_t cum, pair, limit, row_pair, row_t0, part, whole, cut, total;
  Layout(long long NT, int H, int Hkv, int dh, int ctas, int max_pairs, int shared_items, bool planned, int slots) {
    auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    const size_t rows = planned ? up(static_cast<size_t>(NT) * 4) : 0;
    cum = planned ? up(sizeof(Header)) : 0;
    pair = cum + (planned ? up((static_cast<size_t>(max_pairs) + 1) * 4) : 0);
    limit = pair + (planned ? up(static_cast<size_t>(max_pairs) * sizeof(Pair)) : 0);
    row_pair = limit + rows;
    row_t0 = row_pair + rows;
    part = row_t0 + rows;
    whole = part + up((static_cast<size_t>(max_pairs) * Hkv + shared_items) * sizeof(int2));
    cut = whole + up(static_cast<size_t>(slots) * NT * H * (dh + 2) * 4);
    total = cut + up(static_cast<size_t>(4) * ctas * BM * (dh + 2) * 4);
  }
};

template <int DH>
static int launch(const CUtensorMap& tm, Params p, int ctas, cudaStream_t s) {
  CUtensorMap q_tile;
  // (64 columns, the query heads of a kv head, tokens): the rows of a tile in the order in which it has them
  const int rc = make_tmap_3d_bf16_box(&q_tile, p.q, DH, p.H, p.NT, DH, p.ldq, 64, p.G, p.q_tokens);
  if (rc) return rc;
  static PerDeviceOnce attr[2];
  if (allow_smem(attr[0], attend_kernel<DH, false>, 227 * 1024, SB_ERR_LAUNCH) ||
      allow_smem(attr[1], attend_kernel<DH, true>, 227 * 1024, SB_ERR_LAUNCH))
    return SB_ERR_LAUNCH;
  const int slots = Cfg<DH>::slots(p.q_rows);
  p.vs = slots / 2;
  p.ks = slots - p.vs;
  if (p.pair && launch_dep(plan_kernel, dim3(1), dim3(1024), 0, s, p) != cudaSuccess) return SB_ERR_LAUNCH;
  if (launch_dep(p.pair ? attend_kernel<DH, true> : attend_kernel<DH, false>, dim3(ctas), dim3(THREADS), Cfg<DH>::smem_bytes(p.q_rows), s,
                 tm, q_tile, p) != cudaSuccess)
    return SB_ERR_LAUNCH;
  const long long jobs = static_cast<long long>(p.NT) * p.Hkv;
  // Few rows of many parts have a warp for every fourth part, many rows half a warp each, us of a call: 16 sequences behind 4000 positions
  // 17.4 with four ways, 18.4 with one, 4 behind 2048 12.9 / 13.8, 4 behind 1024 (four parts) 12.2 / 10.9, 32 behind 4000 23.9 / 23.4; 2
  // sequences of 4 tokens packed 20.5, else 16.5, 32 of 4 30.3 / 28.0, 64 of 6 50.6 / 54.2. The parts of a shared item: as many as CTAs
  // for each of them, of two blocks at least.
  const long long items = p.Hkv * ((p.NT + 2LL * p.TT - 1) / (2 * p.TT)), blocks = p.prefix / BN;
  const long long parts = blocks / 2 < ctas / items ? blocks / 2 : ctas / items;
  return (jobs > 1024 && p.pair        ? launch_dep(join_kernel<DH, 1, true>, dim3((jobs + 3) / 4), dim3(128), 0, s, p, ctas)
          : jobs <= 192 && parts >= 7 ? launch_dep(join_kernel<DH, 4, false>, dim3(jobs), dim3(512), 0, s, p, ctas)
                                      : launch_dep(join_kernel<DH, 1, false>, dim3(jobs), dim3(128), 0, s, p, ctas)) == cudaSuccess ? 0 : SB_ERR_LAUNCH;
}

static int ctas_for(long long units) {
  const long long most = num_sms();
  return static_cast<int>(units < 2 ? 2 : units < most ? units : most);      // one for either part of the line
}

}  // namespace spa
}  // namespace sb

using namespace sb;

// What the sizes of a call decide.
static void sizes(spa::Params& p, int NT, int B, int H, int Hkv, int prefix, bool ragged) {
  p.B = B; p.NT = NT; p.H = H; p.Hkv = Hkv; p.prefix = prefix;
  p.G = H / Hkv; p.TT = spa::BM / p.G;
  p.q_tokens = NT < p.TT ? NT : p.TT;
  p.q_rows = (p.G * p.q_tokens + 7) / 8 * 8;
  p.max_pairs = ragged ? B + NT / (2 * p.TT) : B;
  p.shared_items = prefix > 0 ? Hkv * (NT / (2 * p.TT) + 1) : 0;
  p.few = ragged || p.G > spa::FEW ? 0 : NT * p.G > spa::FEW ? 1 : 3;
}
static int slots_of(const spa::Params& p) { return p.prefix > 0 || p.few ? spa::whole_slots(p) : 0; }

// Bytes of workspace that sb_shared_prefix_attention needs (32-byte aligned); 0 where it would refuse the sizes.
extern "C" size_t sb_shared_prefix_attention_bytes(int NT, int B, int H, int Hkv, int dh, int ragged, int prefix) {
  if (NT <= 0 || B <= 0 || H <= 0 || Hkv <= 0 || H % Hkv || H / Hkv > spa::BM) return 0;
  spa::Params p;
  sizes(p, NT, B, H, Hkv, prefix, ragged != 0);
  return spa::Layout(NT, H, Hkv, dh, num_sms(), p.max_pairs, p.shared_items, ragged != 0, slots_of(p)).total;
}

// q: bf16 [NT, ldq], query heads first, positions already rotated in. pool: n_blocks pages [2, Hkv, page, dh], page a multiple of 8.
// cu_q: [B + 1] rows of the sequences, or null: one row each (NT == B). seq_len: positions of each sequence, its rows' among them.
// prefix_table: pages of the first `prefix` positions, which all sequences share (prefix a multiple of page; 0: none). max_units, about
// the blocks of 128 positions of all items, caps the grid; lengths beyond what it was counted for are answered all the same.
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
      (reinterpret_cast<uintptr_t>(workspace) & 31))
    return SB_ERR_ALIGN;
  const uint64_t rows = static_cast<uint64_t>(n_blocks) * 2 * Hkv * page;
  // coordinates of the pool's rows, and of the page behind the last that stands for a bad one; positions; the line of blocks
  if (rows + 2ull * Hkv * page >= (1ull << 31) || static_cast<uint64_t>(max_blocks) * page >= (1ull << 30) ||
      static_cast<uint64_t>(NT) * Hkv >= (1ull << 31))
    return SB_ERR_TOO_LARGE;
  const bool planned = cu_q != nullptr;
  spa::Params p;
  sizes(p, NT, B, H, Hkv, prefix, planned);
  const int TT = p.TT, max_pairs = p.max_pairs;
  const uint64_t cap = static_cast<uint64_t>(max_blocks) * page;
  const uint64_t own = spa::BLOCK_TWO * (cap / spa::BN + 1) + spa::ITEM_TWO;           // units of an item
  const uint64_t common = spa::BLOCK_TWO * (prefix / spa::BN + 1) + spa::ITEM_TWO;
  if (Hkv * (max_pairs * own + (NT / (2 * TT) + 1) * common) >= (1ull << 31))
    return SB_ERR_TOO_LARGE;
  const int ctas = spa::ctas_for(max_units);
  const spa::Layout at(NT, H, Hkv, dh, ctas, max_pairs, p.shared_items, planned, slots_of(p));
  if (at.total > workspace_bytes) return SB_ERR_ARG;
  int box_log = 6;
  while (page % (1 << box_log)) --box_log;
  CUtensorMap tm;
  const int rc = make_tmap_2d_bf16(&tm, pool, dh, rows, dh, 64, 1 << box_log);
  if (rc) return rc;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.q = static_cast<const __nv_bfloat16*>(q); p.ldq = ldq;
  p.block_table = block_table; p.max_blocks = max_blocks; p.seq_len = seq_len; p.prefix_table = prefix_table; p.cu_q = cu_q;
  p.page = page; p.n_blocks = n_blocks; p.box_log = box_log;
  p.by_page.set(page); p.by_heads.set(Hkv); p.by_span.set(2 * p.TT);
  p.scale_log2 = scale * 1.4426950408889634f;
  p.out = static_cast<__nv_bfloat16*>(out); p.ldo = ldo; p.fill = fill;
  p.hdr = planned ? reinterpret_cast<spa::Header*>(ws) : nullptr;
  p.cum = planned ? reinterpret_cast<int*>(ws + at.cum) : nullptr;
  p.pair = planned ? reinterpret_cast<spa::Pair*>(ws + at.pair) : nullptr;
  p.row_limit = planned ? reinterpret_cast<int*>(ws + at.limit) : nullptr;
  p.row_t0 = planned ? reinterpret_cast<int*>(ws + at.row_t0) : nullptr;
  p.part = reinterpret_cast<int2*>(ws + at.part);
  p.row_pair = planned ? reinterpret_cast<int*>(ws + at.row_pair) : nullptr;
  p.whole = reinterpret_cast<float*>(ws + at.whole);
  p.cut = reinterpret_cast<float*>(ws + at.cut);
  p.status = status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dh == 64 ? spa::launch<64>(tm, p, ctas, s) : spa::launch<128>(tm, p, ctas, s);
}
