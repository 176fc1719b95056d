// Forks and moves of whole sequences in the paged K/V cache: "slot d becomes the first L tokens of what slot s held".
//
// Pages that end up full are shared by reference count, so a fork copies only what will be written again or lies outside
// the pages: the partly filled last page and the compressed rows (1/16 of the tokens, contiguous per slot).  The host half
// (paged_plan) keeps the page table, the counts and the free list, all or nothing, and turns the call into moves in an
// order in which no slot is overwritten before its readers are done; the device half carries them out, 80 in a launch.
//
// Device half: a thread owns the same 16 bytes of every slot (or one column of the page table) and walks over the moves,
// so even the moves of a permutation need no second buffer: what it has not read yet, nobody has written.  A cycle keeps
// its first slot's 16 bytes in a register.  Loads of up to 8 moves travel together, and moves that read the same slot
// share one load.  Bound by HBM: every source is read once per group of moves, every copy written once (32749 tokens, 4
// heads of 128 / 128 bf16, into 63 slots: 53 us, 5.2 TB/s; half of 64 slots of 16411 tokens onto the other half: 26 us,
// 5.5 TB/s), and by the latency of the walk where the slots hold little (a cycle of 16 slots of 4096 tokens: 8.8 us).
#include <algorithm>
#include <vector>

#include "common.h"
#include "kernels.h"

namespace nsa {

typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));

// Calls store(move, value) for the moves m[0..n) in order, with the value that load(slot) had before the moves.  A round of
// up to kPagedRound moves (as the host marked them) reads all its moves and issues all its loads before its first store.
template <class V, class Load, class Store>
__device__ __forceinline__ void walk_moves(const PagedMove* __restrict__ m, int n, Load load, Store store) {
  V kept = V();
  for (int i = 0; i < n;) {
    const int cnt = m[i].round;
    int src[kPagedRound];
    V val[kPagedRound];
#pragma unroll
    for (int k = 0; k < kPagedRound; ++k) src[k] = m[i + k].src;     // the list is padded by a round
#pragma unroll
    for (int k = 0; k < kPagedRound; ++k) {
      val[k] = V();
      if (k < cnt) {
        if (k > 0 && src[k] == src[k > 0 ? k - 1 : 0]) val[k] = val[k > 0 ? k - 1 : 0];
        else if (src[k] >= 0) val[k] = load(src[k]);
      }
    }
#pragma unroll
    for (int k = 0; k < kPagedRound; ++k) {
      if (k < cnt) {
        const PagedMove& x = m[i + k];
        if (x.dst < 0) kept = val[k];
        else store(x, x.src < 0 ? kept : val[k]);
      }
    }
    i += cnt;
  }
}

constexpr int kPageChunk = 4 * 256;    // 16-byte vectors of a page that one workgroup copies

__device__ __forceinline__ void copy_page(const PagedPools& p, int src, int dst, long chunk) {
  const u32x4_t* k = reinterpret_cast<const u32x4_t*>(p.k_pool);
  const u32x4_t* v = reinterpret_cast<const u32x4_t*>(p.v_pool);
  u32x4_t val[4];
  const long at = chunk * kPageChunk + threadIdx.x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const long j = at + 256 * i;
    if (j < p.k_page) val[i] = k[src * p.k_page + j];
    else if (j < p.k_page + p.v_page) val[i] = v[src * p.v_page + j - p.k_page];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const long j = at + 256 * i;
    if (j < p.k_page) reinterpret_cast<u32x4_t*>(p.k_pool)[dst * p.k_page + j] = val[i];
    else if (j < p.k_page + p.v_page) reinterpret_cast<u32x4_t*>(p.v_pool)[dst * p.v_page + j - p.k_page] = val[i];
  }
}

// The first n (fewer than all) elements of a 16-byte vector: in halves, quarters and eighths, whichever n takes.
template <typename E>
__device__ __forceinline__ void store_head(E* p, u32x4_t val, int n) {
  unsigned x = val[0], y = val[1];
  int bytes = n * (int)sizeof(E);
  char* at = reinterpret_cast<char*>(p);
  if (bytes & 8) {
    *reinterpret_cast<uint2*>(at) = make_uint2(x, y);
    x = val[2]; y = val[3];
    at += 8;
  }
  if (bytes & 4) {
    *reinterpret_cast<unsigned*>(at) = x;
    x = y;
    at += 4;
  }
  if (bytes & 2) *reinterpret_cast<uint16_t*>(at) = (uint16_t)x;
}

// grid: (workgroups for the compressed keys, the compressed values, the page table, the last pages; groups of moves)
template <typename E>
__global__ void __launch_bounds__(256)
paged_move_kernel(const PagedMoveArgs a) {
  constexpr int kVec = 16 / (int)sizeof(E);
  const int group = blockIdx.y, m0 = a.group[group], n = a.group[group + 1] - m0;
  const PagedMove* moves = a.moves + m0;
  long blk = blockIdx.x;
  if (blk < a.ck_blocks) {
    const long j = blk * 256 + threadIdx.x, row = (long)a.hkv * a.dk / kVec;    // vectors per compressed row
    const long slot = (long)a.nc_cap * row;
    if (j >= a.rows_most * row) return;
    u32x4_t* ck = reinterpret_cast<u32x4_t*>(a.ck) + j;
    walk_moves<u32x4_t>(moves, n, [&](int s) { return ck[s * slot]; },
                        [&](const PagedMove& x, u32x4_t val) { if (x.src != x.dst && j < x.rows * row) ck[x.dst * slot] = val; });
    return;
  }
  blk -= a.ck_blocks;
  if (blk < a.cv_blocks) {
    const long j = blk * 256 + threadIdx.x;
    const int wide = (a.rows_most + kVec - 1) / kVec;                            // vectors per value channel
    if (j >= (long)a.hkv * a.dv * wide) return;
    const int chan = (int)(j / wide), col = (int)(j - (long)chan * wide) * kVec;
    const long slot = (long)a.hkv * a.dv * a.nc_cap;
    E* cv = reinterpret_cast<E*>(a.cv) + (long)chan * a.nc_cap + col;
    walk_moves<u32x4_t>(moves, n, [&](int s) { return *reinterpret_cast<const u32x4_t*>(cv + s * slot); },
                        [&](const PagedMove& x, u32x4_t val) {
                          if (x.src == x.dst || col >= x.rows) return;
                          if (col + kVec <= x.rows) {
                            *reinterpret_cast<u32x4_t*>(cv + x.dst * slot) = val;
                          } else {                       // columns behind the last compressed row stay as they are
                            store_head<E>(cv + x.dst * slot, val, x.rows - col);
                          }
                        });
    return;
  }
  blk -= a.cv_blocks;
  if (blk < a.table_blocks) {
    const int col = (int)blk * 256 + threadIdx.x;
    if (col >= a.max_pages) return;
    int32_t* table = a.block_table + col;
    walk_moves<int>(moves, n, [&](int s) { return table[(long)s * a.max_pages]; },
                    [&](const PagedMove& x, int val) {
                      const int full = x.len >> 6;
                      const int id = col < full ? val : (col == full && (x.len & 63)) ? x.tail : 0;
                      table[(long)x.dst * a.max_pages] = id;
                      if (col == 0) a.ctx_lens[x.dst] = x.len;
                    });
    return;
  }
  blk -= a.table_blocks;
  if (group != 0) return;
  const long per = (a.pools.k_page + a.pools.v_page + kPageChunk - 1) / kPageChunk;
  const int pair = (int)(blk / per);
  copy_page(a.pools, a.pairs[pair].src, a.pairs[pair].dst, blk - pair * per);
}

// grid: workgroups for the pages, then for the table entries
__global__ void __launch_bounds__(256)
paged_compact_kernel(const PagedCompactArgs a) {
  const long per = (a.pools.k_page + a.pools.v_page + kPageChunk - 1) / kPageChunk;
  long blk = blockIdx.x;
  if (blk < per * a.n_pairs) {
    const int pair = (int)(blk / per);
    copy_page(a.pools, a.pairs[pair].src, a.pairs[pair].dst, blk - pair * per);
    return;
  }
  blk -= per * a.n_pairs;
  const long i = blk * 256 + threadIdx.x;
  if (i >= a.entries) return;
  const int id = a.block_table[i];
  int now = id;
  for (int k = 0; k < a.n_pairs; ++k) now = a.pairs[k].src == id ? a.pairs[k].dst : now;
  if (now != id) a.block_table[i] = now;
}

// ------------------------------------------------------------------------------------------------ host half

// Whether slot b's pages are pages of the pool, and enough for its tokens.
static bool slot_ok(const PagedBooks& bk, int b) {
  if (bk.held[b] < 0 || bk.held[b] > bk.max_pages || bk.lens[b] < 0 || bk.lens[b] > bk.held[b] * 64L) return false;
  const int32_t* t = bk.table + (long)b * bk.max_pages;
  bool bad = false;
  for (int k = 0; k < bk.held[b]; ++k) bad |= (unsigned)(t[k] - 1) >= (unsigned)(bk.num_pages - 1);
  return !bad;
}

// Slot `slot` comes to hold `pages` pages if it holds fewer; the new ones are the top of the free list.
int paged_grow(const PagedBooks& bk, int slot, int pages) {
  if (slot < 0 || slot >= bk.batch || pages < 0 || pages > bk.max_pages || !slot_ok(bk, slot)) return -1;
  const int more = pages - bk.held[slot];
  if (more <= 0) return 0;
  if (more > *bk.n_free) return -3;
  if (*bk.n_free > bk.num_pages) return -1;
  for (int k = 0; k < more; ++k)
    if ((unsigned)(bk.free_pages[*bk.n_free - 1 - k] - 1) >= (unsigned)(bk.num_pages - 1)) return -1;
  int32_t* t = bk.table + (long)slot * bk.max_pages + bk.held[slot];
  for (int k = 0; k < more; ++k) {
    t[k] = bk.free_pages[--*bk.n_free];
    bk.refs[t[k]] = 1;
  }
  bk.held[slot] = pages;
  return 0;
}

// Moves 0..n-1 (5 ints each: src, dst, len, last page read, last page written) in an order that is right one after the
// other; src -1 / dst -1 is the register that holds a cycle's first slot.  A length of -1 (no lengths: each) is all the parent has.  Returns 0,
// -1 (bad argument) or -3 (pool exhausted); nothing changes unless it returns 0.
int paged_plan(const PagedBooks& bk, const int32_t* slots, const int32_t* parents, const int32_t* asked, int n,
               int32_t* moves, int32_t* n_moves) {
  const int B = bk.batch, W = bk.max_pages;
  std::vector<int> node(B, -1), tail(n, -1), from(n, -1), readers(B, 0), row_of(B, -1), lengths(n), common(n);
  std::vector<char> open(n, 0);
  std::vector<int> ready;
  std::vector<int32_t> old;
  ready.reserve(n);                                      // nothing below the first change allocates
  if (*bk.n_free < 0 || *bk.n_free > bk.num_pages) return -1;
  for (int i = 0; i < n; ++i) {
    const int s = slots[i], p = parents[i];
    if (s < 0 || s >= B || p < 0 || p >= B || node[s] >= 0 || !slot_ok(bk, s)) return -1;
    if (row_of[p] < 0 && !slot_ok(bk, p)) return -1;
    lengths[i] = asked == nullptr || asked[i] == -1 ? bk.lens[p] : asked[i];
    if (lengths[i] < 0 || lengths[i] > bk.lens[p]) return -1;
    node[s] = i;
    if (row_of[p] < 0) {
      row_of[p] = (int)(old.size() / W);
      old.insert(old.end(), bk.table + (long)p * W, bk.table + (long)(p + 1) * W);
    }
  }
  auto row = [&](int i) { return old.data() + (long)row_of[parents[i]] * W; };
  auto own = [&](int i) { return bk.table + (long)slots[i] * W; };
  // full pages that the slot holds already, in the same places, stay with it: beams and samples share most of theirs
  for (int i = 0; i < n; ++i) {
    const int most = std::min(bk.held[slots[i]], lengths[i] / 64);
    const int32_t *x = own(i), *y = row(i);
    int k = 0;
    while (k < most && x[k] == y[k]) ++k;
    common[i] = k;
  }
  auto drop = [&](int by) {
    for (int i = 0; i < n; ++i)
      for (int k = common[i]; k < bk.held[slots[i]]; ++k) bk.refs[own(i)[k]] -= by;
  };
  auto share = [&](int by) {
    for (int i = 0; i < n; ++i)
      for (int k = common[i]; k < lengths[i] / 64; ++k) bk.refs[row(i)[k]] += by;
  };
  drop(1);
  share(1);
  // The partly filled last page is written again by its sequence, so it has one owner.  A page nobody else holds any more
  // goes to the slot that stays, or else to the first of its new owners; the others get copies.
  for (int stay = 1; stay >= 0; --stay)
    for (int i = 0; i < n; ++i) {
      if (lengths[i] % 64 == 0 || (slots[i] == parents[i]) != (stay == 1)) continue;
      from[i] = row(i)[lengths[i] / 64];
      if (bk.refs[from[i]] == 0) {
        bk.refs[from[i]] = 1;
        tail[i] = from[i];
      }
    }
  // a copy goes to the slot's own last page if that has become free, else to a page of the free list
  int missing = 0;
  for (int i = 0; i < n; ++i) {
    if (from[i] < 0 || tail[i] >= 0) continue;
    const int h = bk.held[slots[i]];
    const int last = h > 0 ? own(i)[h - 1] : 0;
    if (last > 0 && bk.refs[last] == 0) {
      bk.refs[last] = 1;
      tail[i] = last;
    } else {
      ++missing;
    }
  }
  const int free0 = *bk.n_free;
  int nf = free0;
  for (int i = n - 1; i >= 0; --i)                       // the first page of the first slot ends on top
    for (int k = bk.held[slots[i]] - 1; k >= common[i]; --k) {
      const int pg = own(i)[k];
      if (bk.refs[pg] == 0) {
        if (nf >= bk.num_pages) continue;                // cannot be while the books are in order
        bk.refs[pg] = -1;
        bk.free_pages[nf++] = pg;
      }
    }
  for (int k = free0; k < nf; ++k) bk.refs[bk.free_pages[k]] = 0;
  bool bad = false;                                      // a free list that names pages outside the pool
  for (int k = 0; k < std::min(missing, nf); ++k) bad |= (unsigned)(bk.free_pages[nf - 1 - k] - 1) >= (unsigned)(bk.num_pages - 1);
  if (missing > nf || bad) {
    for (int i = 0; i < n; ++i)
      if (tail[i] >= 0) bk.refs[tail[i]] = 0;
    share(-1);
    drop(-1);
    return bad ? -1 : -3;
  }
  for (int i = 0; i < n; ++i)
    if (from[i] >= 0 && tail[i] < 0) {
      tail[i] = bk.free_pages[--nf];
      bk.refs[tail[i]] = 1;
    }
  *bk.n_free = nf;
  int count = 0;
  auto emit = [&](int src, int dst, int len, int tail_src, int tail_dst) {
    int32_t* m = moves + 5L * count++;
    m[0] = src; m[1] = dst; m[2] = len; m[3] = tail_src; m[4] = tail_dst;
  };
  auto emit_node = [&](int i, int src) { emit(src, slots[i], lengths[i], from[i] < 0 ? 0 : from[i], tail[i] < 0 ? 0 : tail[i]); };
  // what changes; a slot that stays as it is needs no move
  for (int i = 0; i < n; ++i) {
    const int s = slots[i];
    open[i] = s != parents[i] || lengths[i] != bk.lens[s] || tail[i] != from[i];
    if (s != parents[i]) ++readers[parents[i]];
  }
  for (int i = n - 1; i >= 0; --i)
    if (open[i] && readers[slots[i]] == 0) ready.push_back(i);
  while (!ready.empty()) {
    const int i = ready.back();
    ready.pop_back();
    open[i] = 0;
    emit_node(i, parents[i]);
    const int p = parents[i];
    if (p != slots[i] && --readers[p] == 0 && node[p] >= 0 && open[node[p]]) ready.push_back(node[p]);
  }
  // what is left are cycles; a long one is cut into pieces that fit a launch: the slot at the cut holds the first slot's
  // content until the next piece picks it up
  for (int i = 0; i < n; ++i) {
    if (!open[i]) continue;
    int end = i;                                         // the move that reads slot[i]
    while (parents[end] != slots[i]) end = node[parents[end]];
    int in_piece = 0;
    emit(slots[i], -1, lengths[end], 0, 0);
    for (int j = i;; j = node[parents[j]]) {
      open[j] = 0;
      if (j == end) {
        emit_node(j, -1);
        break;
      }
      if (++in_piece == kPagedCyclePiece) {
        emit(-1, slots[j], lengths[end], 0, 0);
        emit(slots[j], -1, lengths[end], 0, 0);
        in_piece = 1;
      }
      emit_node(j, parents[j]);
    }
  }
  *n_moves = count;
  for (int i = 0; i < n; ++i) {
    int32_t* t = own(i);
    const int full = lengths[i] / 64, h = full + (tail[i] >= 0 ? 1 : 0);
    for (int k = common[i]; k < full; ++k) t[k] = row(i)[k];
    if (tail[i] >= 0) t[full] = tail[i];
    for (int k = h; k < bk.held[slots[i]]; ++k) t[k] = 0;
    bk.held[slots[i]] = h;
    bk.lens[slots[i]] = lengths[i];
  }
  return 0;
}

// Pairs (page, new page) after which the pages in use are 1..used.
int paged_compact_plan(const PagedBooks& bk, int32_t* pairs, int32_t* n_pairs, int32_t* used) {
  for (int b = 0; b < bk.batch; ++b)
    if (!slot_ok(bk, b)) return -1;
  int live = 0;
  for (int p = 1; p < bk.num_pages; ++p) live += bk.refs[p] > 0;
  std::vector<int32_t> to(bk.num_pages, 0);
  int hole = 1, n = 0;
  for (int p = live + 1; p < bk.num_pages; ++p) {
    if (bk.refs[p] <= 0) continue;
    while (bk.refs[hole] > 0) ++hole;
    to[p] = hole;
    pairs[2 * n] = p;
    pairs[2 * n + 1] = hole++;
    ++n;
  }
  for (int k = 0; k < n; ++k) {
    bk.refs[pairs[2 * k + 1]] = bk.refs[pairs[2 * k]];
    bk.refs[pairs[2 * k]] = 0;
  }
  for (int b = 0; b < bk.batch; ++b)
    for (int k = 0; k < bk.held[b]; ++k) {
      int32_t& t = bk.table[(long)b * bk.max_pages + k];
      if (to[t]) t = to[t];
    }
  int nf = 0;
  for (int p = bk.num_pages - 1; p > live; --p) bk.free_pages[nf++] = p;
  *bk.n_free = nf;
  *n_pairs = n;
  *used = live;
  return 0;
}

// ------------------------------------------------------------------------------------------------ launches

static long ceil_div(long a, long b) { return (a + b - 1) / b; }

// Puts the moves of a launch into groups of about kPagedGroup, in which what depends on one another stays together and in
// order; groups run side by side.  4: one walk over all moves is slow where the slots hold little (300 tokens forked into 63
// slots: 31 us, in groups of 32, 8, 4 and 1 13.4, 6.9, 7.0 and 11.4), and a source is read once per group (32749 tokens
// into 63 slots: groups of 32, 8, 4 and 1 58, 54, 53 and 85 us).
constexpr int kPagedGroup = 4;

static void paged_groups(PagedMoveArgs& a, const PagedMove* in, int n) {
  int root[kPagedMoves], order[kPagedMoves];
  for (int i = 0; i < n; ++i) root[i] = i;
  auto find = [&](int i) { while (root[i] != i) i = root[i]; return i; };
  auto join = [&](int i, int j) { i = find(i); j = find(j); root[std::max(i, j)] = std::min(i, j); };
  if (n <= kPagedGroup) {
    for (int i = 1; i < n; ++i) root[i] = 0;
  } else {
    int slot[256], writer[256];                          // a hash from a slot to the first move that writes it
    for (int i = 0; i < 256; ++i) slot[i] = -1;
    auto place = [&](int s) {
      int h = s & 255;
      while (slot[h] >= 0 && slot[h] != s) h = (h + 1) & 255;
      return h;
    };
    int piece = -1;
    for (int i = 0; i < n; ++i) {
      if (in[i].dst < 0) piece = i;                      // a cycle's piece shares the register
      if (piece >= 0) join(piece, i);
      if (in[i].src < 0) piece = -1;
      if (in[i].dst < 0) continue;
      const int h = place(in[i].dst);
      if (slot[h] >= 0) join(writer[h], i);
      else { slot[h] = in[i].dst; writer[h] = i; }
    }
    for (int i = 0; i < n; ++i) {
      if (in[i].src < 0) continue;
      const int h = place(in[i].src);
      if (slot[h] >= 0) join(writer[h], i);
    }
  }
  int at = 0, groups = 0;
  a.group[0] = 0;
  for (int r = 0; r < n; ++r) {
    if (find(r) != r) continue;
    for (int i = r; i < n; ++i)
      if (find(i) == r) order[at++] = i;
    if (at - a.group[groups] >= kPagedGroup) a.group[++groups] = at;
  }
  if (a.group[groups] != at) a.group[++groups] = at;
  for (int i = 0; i < n; ++i) a.moves[i] = in[order[i]];
  a.groups = groups;
  for (int g = 0; g < groups; ++g)
    for (int i = a.group[g]; i < a.group[g + 1];) {
      int cnt = 1;                                       // a move into the register starts a round
      while (cnt < kPagedRound && i + cnt < a.group[g + 1] && a.moves[i + cnt].dst >= 0) ++cnt;
      a.moves[i].round = cnt;
      i += cnt;
    }
}

int launch_paged_move(PagedMoveArgs a, const int32_t* moves, int n, int block, int stride, int elem, hipStream_t st) {
  const long per = ceil_div(a.pools.k_page + a.pools.v_page, kPageChunk);
  for (int i = 0; i < n;) {
    // as many moves as fit, without parting a cycle's piece
    int end = i + 1, whole = i;                          // whole: the moves before it leave the register empty
    for (bool kept = moves[5L * i + 1] < 0;; ++end) {
      if (!kept) whole = end;
      if (end == n || end == i + kPagedMoves) break;
      const int32_t* m = moves + 5L * end;
      kept = m[1] < 0 || (kept && m[0] >= 0);
    }
    end = whole;
    PagedMove list[kPagedMoves];
    a.rows_most = 0;
    int pairs = 0;
    for (int k = i; k < end; ++k) {
      const int32_t* m = moves + 5L * k;
      PagedMove& x = list[k - i];
      x.src = m[0]; x.dst = m[1]; x.len = m[2]; x.tail = m[4]; x.round = 1;
      x.rows = m[2] >= block ? std::min((m[2] - block) / stride + 1, a.nc_cap) : 0;
      if (x.src != x.dst) a.rows_most = std::max(a.rows_most, x.rows);
      if ((m[2] & 63) && m[1] >= 0 && m[3] != m[4]) { a.pairs[pairs].src = m[3]; a.pairs[pairs++].dst = m[4]; }
    }
    const long vec = 16 / elem;
    a.ck_blocks = ceil_div(a.rows_most * ((long)a.hkv * a.dk / vec), 256);
    a.cv_blocks = ceil_div((long)a.hkv * a.dv * ceil_div(a.rows_most, vec), 256);
    a.table_blocks = ceil_div(a.max_pages, 256);
    const long slot_blocks = a.ck_blocks + a.cv_blocks + a.table_blocks;
    paged_groups(a, list, end - i);
    const long blocks = slot_blocks + pairs * per;
    if (blocks > 0x7fffffffL) return -2;
    const dim3 grid((unsigned)blocks, (unsigned)a.groups);
    if (elem == 2) hipLaunchKernelGGL(paged_move_kernel<uint16_t>, grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(paged_move_kernel<uint32_t>, grid, dim3(256), 0, st, a);
    i = end;
  }
  return 0;
}

int launch_paged_compact(PagedCompactArgs a, const int32_t* pairs, int n, hipStream_t st) {
  const long per = ceil_div(a.pools.k_page + a.pools.v_page, kPageChunk);
  for (int i = 0; i < n; i += kPagedPairs) {
    a.n_pairs = std::min(kPagedPairs, n - i);
    for (int k = 0; k < a.n_pairs; ++k) { a.pairs[k].src = pairs[2 * (i + k)]; a.pairs[k].dst = pairs[2 * (i + k) + 1]; }
    const long blocks = a.n_pairs * per + ceil_div(a.entries, 256);
    if (blocks > 0x7fffffffL) return -2;
    hipLaunchKernelGGL(paged_compact_kernel, dim3((unsigned)blocks), dim3(256), 0, st, a);
  }
  return 0;
}

}  // namespace nsa
