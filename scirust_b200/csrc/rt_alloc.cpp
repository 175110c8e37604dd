// CPU runtime, part 2: host-side allocators that hand out *indices/offsets* into device pools.
//
//  * BlockAllocator: fixed-size KV-cache pages with a LIFO free list and per-sequence block lists
//    (the reference's paged cache keeps a block table per sequence and grows it page by page:
//    scirust-core/src/nn/paged_attention.rs:21-147). Freed pages are reused most-recent-first so
//    a workload's physical layout is reproducible. A page may have several owners (sequences with a
//    common prefix); it returns to the list with the last of them.
//  * Arena: a bump allocator over one preallocated device buffer with mark/release, used for the
//    step-scoped workspace instead of one allocation per op (the reference's op-chain allocates an
//    output for every op: scirust-cuda/src/chain.rs:1049-1052; its CPU arenas:
//    scirust-arena/src/*).
#include <stdint.h>
#include <stdlib.h>

#include <vector>

struct SbBlockAlloc {
  std::vector<int32_t> free_list;
  std::vector<int32_t> more;      // owners of a page beyond the first
  std::vector<uint8_t> used;
  int32_t n_blocks;
};
struct SbArena {
  uint64_t capacity, offset, high_water;
};

extern "C" {

SbBlockAlloc* sbrt_balloc_new(int32_t n_blocks) {
  if (n_blocks <= 0) return nullptr;
  SbBlockAlloc* a = nullptr;
  try {                                   // memory that runs out is an error of the caller's call, not one of C++
    a = new SbBlockAlloc();
    a->free_list.reserve(n_blocks);
    a->more.assign(n_blocks, 0);
    a->used.assign(n_blocks, 0);
  } catch (...) {
    delete a;
    return nullptr;
  }
  a->n_blocks = n_blocks;
  for (int32_t i = n_blocks - 1; i >= 0; --i) a->free_list.push_back(i);  // block 0 is handed out first
  return a;
}
void sbrt_balloc_delete(SbBlockAlloc* a) { delete a; }
int32_t sbrt_balloc_num_free(const SbBlockAlloc* a) { return static_cast<int32_t>(a->free_list.size()); }
// Allocates n blocks into out[]; returns 0, or -1 (and allocates nothing) if fewer than n are free.
int32_t sbrt_balloc_alloc(SbBlockAlloc* a, int32_t n, int32_t* out) {
  if (n < 0 || static_cast<size_t>(n) > a->free_list.size()) return -1;
  for (int32_t i = 0; i < n; ++i) {
    out[i] = a->free_list.back();
    a->free_list.pop_back();
    a->used[out[i]] = 1;
    a->more[out[i]] = 0;
  }
  return 0;
}
// Gives up one owner of each block (an id may occur several times); the last owner's returns to the pool. Ids outside the pool, and more
// owners of a block than it has, are rejected (-1) and nothing is freed.
int32_t sbrt_balloc_free(SbBlockAlloc* a, const int32_t* ids, int32_t n) {
  for (int32_t i = 0; i < n; ++i)
    if (ids[i] < 0 || ids[i] >= a->n_blocks) return -1;
  for (int32_t i = 0; i < n; ++i) {
    const int32_t id = ids[i];
    if (!a->used[id]) {                   // one owner more than it has: as they were, from the last on
      while (i-- > 0) {
        if (a->used[ids[i]]) ++a->more[ids[i]];
        else a->used[ids[i]] = 1;
      }
      return -1;
    }
    if (a->more[id] > 0) --a->more[id];
    else a->used[id] = 0;
  }
  // Freed ids go back in the order in which their last owners are given up: `more` marks the ones that are not in the list yet.
  for (int32_t i = 0; i < n; ++i)
    if (!a->used[ids[i]]) ++a->more[ids[i]];
  for (int32_t i = 0; i < n; ++i)
    if (!a->used[ids[i]] && --a->more[ids[i]] == 0) a->free_list.push_back(ids[i]);        // within what is reserved
  return 0;
}
// One more owner for each block (an id may occur several times); -1, and none, if one of them is not in use.
int32_t sbrt_balloc_share(SbBlockAlloc* a, const int32_t* ids, int32_t n) {
  for (int32_t i = 0; i < n; ++i)
    if (ids[i] < 0 || ids[i] >= a->n_blocks || !a->used[ids[i]]) return -1;
  for (int32_t i = 0; i < n; ++i) ++a->more[ids[i]];
  return 0;
}
// Owners of a block, 0 if it is free, -1 if there is none of this id.
int32_t sbrt_balloc_owners(const SbBlockAlloc* a, int32_t id) {
  if (id < 0 || id >= a->n_blocks) return -1;
  return a->used[id] ? a->more[id] + 1 : 0;
}
// Numbers the blocks in use anew, ascending from 0, in a pool of n_blocks: to[id] gets the new id of block id, or -1 if it is free, and the
// return value is how many are in use. A block below that number keeps its id, the others take the lowest free ones in ascending order.
// -1, and nothing changes, if they are more than n_blocks. Blocks are then handed out from the lowest on.
int32_t sbrt_balloc_compact(SbBlockAlloc* a, int32_t n_blocks, int32_t* to) {
  int32_t live = 0;
  for (int32_t i = 0; i < a->n_blocks; ++i) live += a->used[i];
  if (n_blocks <= 0 || live > n_blocks) return -1;
  std::vector<int32_t> more, list;
  std::vector<uint8_t> used;
  try {
    more.assign(n_blocks, 0);
    used.assign(n_blocks, 0);
    list.reserve(n_blocks);
  } catch (...) {
    return -1;
  }
  int32_t hole = 0;
  for (int32_t i = 0; i < a->n_blocks; ++i) {
    to[i] = -1;
    if (!a->used[i]) continue;
    if (i < live) {
      to[i] = i;
    } else {
      while (a->used[hole]) ++hole;
      to[i] = hole++;
    }
    more[to[i]] = a->more[i];
  }
  for (int32_t i = 0; i < live; ++i) used[i] = 1;
  for (int32_t i = n_blocks - 1; i >= live; --i) list.push_back(i);
  a->n_blocks = n_blocks;
  a->more.swap(more);
  a->used.swap(used);
  a->free_list.swap(list);
  return live;
}

SbArena* sbrt_arena_new(uint64_t capacity) {
  SbArena* a = new SbArena();
  a->capacity = capacity;
  a->offset = 0;
  a->high_water = 0;
  return a;
}
void sbrt_arena_delete(SbArena* a) { delete a; }
// Returns the byte offset of an `align`-aligned block of `bytes`, or UINT64_MAX when exhausted.
uint64_t sbrt_arena_alloc(SbArena* a, uint64_t bytes, uint64_t align) {
  if (align == 0) align = 256;
  const uint64_t start = (a->offset + align - 1) / align * align;
  if (start + bytes > a->capacity) return UINT64_MAX;
  a->offset = start + bytes;
  if (a->offset > a->high_water) a->high_water = a->offset;
  return start;
}
uint64_t sbrt_arena_mark(const SbArena* a) { return a->offset; }
void sbrt_arena_release(SbArena* a, uint64_t mark) {
  if (mark <= a->offset) a->offset = mark;
}
uint64_t sbrt_arena_high_water(const SbArena* a) { return a->high_water; }

}  // extern "C"
