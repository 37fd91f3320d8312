// Attention of packed sequences of different lengths with shared key/value
// heads (gfx950), bf16 or fp16 in and out, fp32 softmax: whole prompts whose
// keys lie side by side in one tensor, and new tokens over a paged cache.  The
// kernel templates shared by seq_attn.hip (bf16 instances and the C-ABI entry
// points) and seq_attn_f16.hip (fp16 instances).
//
// For sequence r with n query rows and m keys, query head h and key/value head
// h / G (G = heads / kv_heads):
//   O[t,h,:] = sum_j p_j V[j,h/G,:],  p = softmax_j(scale <Q[t,h,:], K[j,h/G,:]>),
// over j < m or, causal, over j <= t + (m - n): the last query row sees every
// key.  A row that sees none gives O = 0 and LSE = -inf.
//
// Layout of the work.  The G query heads of a key head and the sequence's query
// tokens form one list of n G rows (row = token G + head in group), cut into
// tiles: every key staged for a tile serves all heads of the group.  A tile's
// keys may be cut into parts, whose fp32 partials seq_merge_kernel joins.
// Lengths live on the device, so seq_schedule_kernel lists the (tile, part)
// items there: 128-row tiles longest first, 16-row tiles as one chain of items for
// each workgroup.  The grids are the host's upper bounds, and workgroups past the
// list end at once.  In a call of few tiles every workgroup works its item out by
// itself (own_item) and that kernel is left out.
//
//  * seq_wide_kernel: 128 rows, four waves of 32, the 64-key staged walk of
//    bsa_fwd_kernel (S^T = K Q^T, O^T = V^T P^T on 32x32x16 products).
//  * seq_narrow_kernel: 16 rows, for calls of few rows per sequence (decoding
//    steps): four waves walk different keys of the tile, each through its own
//    LDS stages without workgroup barriers, and join at the end.
#pragma once

#include <type_traits>

#include "bsa_tiles.h"

namespace seq {

using dsa::lds_load16;
using dsa::make_rsrc;

// One (tile, key part) of one sequence, for every key/value head.
struct Item {
  int32_t request, q0, n, k0, m;  // sequence: first query row and count, first key and count
  int32_t tile;                   // rows tile * tile_rows ..
  int32_t s0, s1;                 // key steps
  int32_t slot;                   // partial slot, -1: the whole tile, written to O
  int32_t parts;                  // of the tile
  int32_t chain;                  // 16-row tiles: the workgroup, of its key head's
  int32_t pad[5];
};
static_assert(sizeof(Item) == 64, "items are read as one 64-byte line");

struct Params {
  const void* q;
  const void* k;
  const void* v;
  void* o;
  float* lse;                  // [heads, q_rows] or null
  int64_t q_st, q_sh, o_st, o_sh;
  int64_t k_sp, k_st, k_sh;    // page (paged calls), token and head strides, in elements
  int64_t v_sp, v_st, v_sh;
  const int32_t* q_start;      // [requests + 1]
  const int32_t* k_start;      // [requests + 1] (packed calls)
  const int32_t* kv_lens;      // [requests] (paged calls)
  const int32_t* table;        // [requests, table_width] pages (paged calls)
  int64_t table_stride;
  int32_t table_width, pages, page_shift;
  int32_t requests, q_rows, k_rows;
  int32_t heads, kv_heads, group, head_dim;
  int32_t causal;
  int32_t fill;                // rows of o outside every sequence become 0
  float scale_log2;            // scale * log2(e)
  // Schedule.
  int32_t unlisted;            // no schedule kernel: workgroups work their items out (own_item)
  int32_t tile_shift, step_shift, min_chunk;  // log2 of a tile's rows, of a step's keys
  int32_t slots;               // workgroups that run at a time
  int32_t shared_lines;        // 16-row tiles: key heads lie in the same 128-byte lines
  int32_t max_tiles, max_items, max_splits, max_slots;  // room in the lists, per key head
  float item_cost, part_cost, merge_cost;    // of an item and a partial, in key steps
  int32_t* counts;             // items, split tiles, items that run by head groups
  int32_t* chain_start;        // [kMaxChains] first item of each chain (16-row tiles)
  int32_t* tile_base;          // [requests + 1] tiles before each sequence
  Item* items;
  Item* splits;                // split tiles: slot = the first of `parts` slots
  float* part;                 // partial slots, kv_heads each
};

// One partial: O [tile_rows][kD] relative to the row's reference max (in the order
// of part_at), then m (log2 units of the scaled scores) and l per row, in fp32.
__host__ __device__ constexpr int part_floats(int tile_rows, int dim) {
  return tile_rows * (dim + 2);
}

// Where dim d of row r lies in a partial: 16-row tiles row by row, 128-row tiles as
// the waves hold them, quads of dims of 32 rows side by side.
template <int kD, int kRows>
__device__ __forceinline__ int part_at(int r, int d) {
  return kRows == 16 ? r * kD + d
                     : (r >> 5) * (32 * kD) + ((d >> 2) * 32 + (r & 31)) * 4 + (d & 3);
}

constexpr float kRescaleLog2 = 8.0f;  // move the reference max once a p could exceed 2^8
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kHeadGroup = 8;  // key heads that run together: one per XCD
constexpr int kWideRows = 128, kWideKeys = 64;
// Workgroups of the chip that run at a time: two of 128-row tiles on a compute unit;
// one of 16-row tiles, whose four waves keep the memory busy (two: 2 to 5% slower).
constexpr int kWideSlots = 512, kNarrowSlots = 256;
constexpr int kMaxChains = kNarrowSlots;
constexpr int kNarrowWaves = 4;
constexpr int kNarrowRows = 16, kNarrowKeys = 32 * kNarrowWaves;  // 32 keys for each wave

// ds_read_b64_tr_b16: in each 16-lane group lane j receives element j % 4 of
// the 8 bytes that lane 4 r + j / 4 addresses, r = 0..3.
template <typename T>
__device__ __forceinline__ typename dsa::Elem<T>::x4 read_tr(const unsigned char* lds) {
  const dsa_i16x4 raw = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (__attribute__((address_space(3))) dsa_i16x4*)(lds));
  return __builtin_bit_cast(typename dsa::Elem<T>::x4, raw);
}

// lds_load16 of data that is read once: kOnce marks the load non-temporal, which
// streams past the caches (a plain 3 GB read on this card: 6.3 TB/s, 7.1 with it).
template <bool kOnce>
__device__ __forceinline__ void lds_stream16(__amdgpu_buffer_rsrc_t rsrc, unsigned char* lds,
                                             uint32_t voffset) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (DSA_LDS void*)lds, 16, voffset, 0, 0,
                                           kOnce ? 2 : 0);
}

// s_waitcnt with only vmcnt(n) set.
constexpr int vmcnt(int n) { return 0x0F70 | (n & 15) | ((n >> 4) << 14); }

// Position of 16-byte chunk c in row r of a K stage, distinct banks for the 16
// rows that one chunk of a fragment read touches: rows of 256 bytes (kD 128) by
// their low four bits, rows of 128 bytes, two to a bank round, by bits 1..3.
template <int kD>
__device__ __forceinline__ int k_swz(int r, int c) {
  return kD == 128 ? c ^ (r & 15) : c ^ ((r >> 1) & 7);
}

// The page of a request's key in its block table row, as it stands there: an
// entry outside [0, pages) is a bad page, whose keys are not read and take no part.
__device__ __forceinline__ int page_at(const Params& p, int request, int key) {
  return p.table[(int64_t)request * p.table_stride + (key >> p.page_shift)];
}

// K or V of one key head: a row's bytes start at base + 16 (page page16 + row
// row16), rows counted within the page (paged) or the sequence (packed).
struct Source {
  const unsigned char* base;
  uint32_t page16, row16;
};
template <bool kPaged>
__device__ __forceinline__ Source source_of(const void* tensor, int64_t sp, int64_t st, int64_t sh,
                                            int h, int k0) {
  return {static_cast<const unsigned char*>(tensor) + (h * sh + (kPaged ? 0 : k0 * st)) * 2,
          (uint32_t)(sp >> 3), (uint32_t)(st >> 3)};
}

// Resource of the `rows` (at most 16) staged rows from row `row` of `page`: no
// records, and so zeros, when there are none (the base is then never used).
template <bool kPaged>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_rsrc(const Source& s, uint32_t page, int row,
                                                            int rows, int head_dim) {
  uint64_t at = (uint64_t)(uint32_t)row * s.row16;
  if (kPaged) at += (uint64_t)page * s.page16;
  const uint32_t bytes = rows > 0 ? (uint32_t)(rows - 1) * s.row16 * 16 + head_dim * 2 : 0u;
  return make_rsrc(s.base + (at << 4), bytes);
}

// The kernel's arguments read again from memory: what only the end of a kernel
// uses does not hold registers through its loop.
typedef const __attribute__((address_space(4))) Params* LateParams;
__device__ __forceinline__ LateParams late_params() {
  auto at = (LateParams)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(at));
  return at;
}

__device__ __forceinline__ Item load_item(const Item* at) {
  Item it;
  const dsa::const_i32 s = (dsa::const_i32)(const int32_t*)at;
  it.request = s[0]; it.q0 = s[1]; it.n = s[2]; it.k0 = s[3]; it.m = s[4];
  it.tile = s[5]; it.s0 = s[6]; it.s1 = s[7]; it.slot = s[8]; it.parts = s[9];
  it.chain = s[10];
  return it;
}

// Inclusive sum over the 64 lanes (row shifts by 1, 2, 4, 8, then the row sums
// broadcast into the rows behind).  Every lane of the wave must be active.
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
  v += __builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xA, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xC, 0xF, false);
  return v;
}

struct Sequence {
  int32_t q0, n, k0, m;
};

// Keys of a sequence at most, so that no key index of a step or a page window past
// the last one leaves 32 bits.
constexpr int kMaxKeys = 1 << 30;

// Sequence r, whatever the arrays hold: rows and keys within the tensors.
__device__ __forceinline__ Sequence sequence(const Params& p, int r) {
  Sequence s;
  s.q0 = min(max(p.q_start[r], 0), p.q_rows);
  s.n = min(max(p.q_start[r + 1], s.q0), p.q_rows) - s.q0;
  if (p.kv_lens) {
    s.k0 = 0;
    const int64_t room = (int64_t)p.table_width << p.page_shift;
    s.m = (int32_t)min((int64_t)min(max(p.kv_lens[r], 0), kMaxKeys), room);
  } else {
    s.k0 = min(max(p.k_start[r], 0), p.k_rows);
    s.m = min(min(max(p.k_start[r + 1], s.k0), p.k_rows) - s.k0, kMaxKeys);
  }
  return s;
}

__device__ __forceinline__ int tiles_of(const Params& p, const Sequence& s) {
  return (int)(((int64_t)s.n * p.group + (1 << p.tile_shift) - 1) >> p.tile_shift);
}

// Key steps of a tile: up to the last key its last row sees.
__device__ __forceinline__ int steps_of(const Params& p, const Sequence& s, int tile) {
  int end = s.m;
  if (p.causal) {
    const uint32_t last =
        min((uint32_t)(tile + 1) << p.tile_shift, (uint32_t)s.n * (uint32_t)p.group) - 1;
    end = max(0, min(s.m, s.m - s.n + (int)(last / (uint32_t)p.group) + 1));
  }
  return (int)(((int64_t)end + (1 << p.step_shift) - 1) >> p.step_shift);
}

// Near-equal parts of a tile's steps: part j is [from(j), from(j + 1)).
struct Cut {
  int each, more;  // the first `more` parts hold one step more
  __device__ __forceinline__ Cut(int steps, int parts)
      : each((int)((uint32_t)steps / (uint32_t)parts)), more(steps - each * parts) {}
  __device__ __forceinline__ int from(int j) const { return j * each + min(j, more); }
};

// Parts of at most `chunk` steps, at least one; `per` = 1 / chunk.  (For up to 512
// parts the product is off by one at most.)
__device__ __forceinline__ int parts_in(int steps, int chunk, float per) {
  const int x = steps + chunk - 1;
  int parts = (int)((float)x * per);
  parts += (x >= (parts + 1) * chunk) - (x < parts * chunk);
  return max(1, parts);
}

// Rows that belong to no sequence, the `share`-th of `shares` workgroups' part of
// them: O 0 with p.fill, LSE -inf.
__device__ __forceinline__ void clear_outside(const Params& p, int share, int shares) {
  if (!p.fill && !p.lse) return;
  const int first = min(max(p.q_start[0], 0), p.q_rows);
  const int last = min(max(p.q_start[p.requests], first), p.q_rows);
  const int chunks = p.head_dim / 8 * p.heads;  // 16-byte chunks of a row
  const int empty = first + p.q_rows - last;
  const dsa_u32x4 zero = {0u, 0u, 0u, 0u};
  for (int i = share; i < empty; i += shares) {
    const int row = i < first ? i : last + i - first;
    for (int c = threadIdx.x; p.fill && c < chunks; c += blockDim.x) {
      const int head = c / (p.head_dim / 8), d = c % (p.head_dim / 8) * 8;
      *reinterpret_cast<dsa_u32x4*>(static_cast<uint16_t*>(p.o) + (int64_t)row * p.o_st +
                                    head * p.o_sh + d) = zero;
    }
    if (p.lse)
      for (int head = threadIdx.x; head < p.heads; head += blockDim.x)
        p.lse[(int64_t)head * p.q_rows + row] = -INFINITY;
  }
}

// Unit of workgroup `wg` of `used`, where an XCD takes a range of units instead of every
// eighth: the key heads of an item are neighbours, and where they lie in the same
// 128-byte lines (head dims that are no multiple of 64) the XCD's L2 then reads a line
// once.  (64 requests of 12,000 tokens, 8 key heads: 80 dims 470 -> 350 us, 96 dims 471
// -> 416; 5 key heads of 40 dims 225 -> 155.  Where no line is shared, every eighth
// spreads the reads better: 582 against 628 us at 128 dims.)
__device__ __forceinline__ int unit_of(int wg, int used) {
  const int each = used >> 3, more = used & 7, xcd = wg & 7;
  return xcd * each + min(xcd, more) + (wg >> 3);
}

// The item and key head of workgroup `wg` in a call without a schedule kernel:
// at most 64 sequences and 64 tiles, all of them (times the key heads) at once on
// the chip.  Every wave works it out for itself, a lane per sequence, then per
// tile, then per candidate: the longest tile in 1, 2, 3, .. parts, priced by its
// part and the join, as long as the parts of all tiles still run at once.  The
// first workgroup leaves the split tiles for the merge.  False: no item is left,
// and the workgroup clears its part of the rows outside the sequences.
__device__ __forceinline__ bool own_item(const Params& p, int wg, Item* out, int* head) {
  const int lane = threadIdx.x & 63;
  Sequence s = {0, 0, 0, 0};
  if (lane < p.requests) s = sequence(p, lane);
  const int tiles = tiles_of(p, s);
  const int base = (int)wave_scan((uint32_t)tiles) - tiles;
  // (starts that overlap list more tiles than fit)
  const int count = min(__builtin_amdgcn_readlane(base + tiles, 63), p.max_tiles);
  // Lane i: tile i of sequence r, the last that starts at or before it.
  // (at most 64 sequences: six bisection steps)
  int r = 0;
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) {
    const int at = __shfl(base, r + d);
    if (r + d < p.requests && at <= lane) r += d;
  }
  Sequence t;
  t.q0 = __shfl(s.q0, r); t.n = __shfl(s.n, r); t.k0 = __shfl(s.k0, r); t.m = __shfl(s.m, r);
  const int tile = lane - __shfl(base, r);
  const int steps = lane < count ? steps_of(p, t, tile) : 0;
  int longest = steps;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) longest = max(longest, __shfl_xor(longest, d));
  int chunk = max(longest, 1);
  if (p.max_slots > 0 && longest >= 2 * p.min_chunk) {
    const int parts = lane < 32 ? lane + 1 : 32 + (lane - 31) * 8;
    const int mine = max(p.min_chunk, (longest + parts - 1) / parts);
    const float per = 1.f / (float)mine;
    int items = 0;
    for (int i = 0; i < count; ++i)
      items += parts_in(__builtin_amdgcn_readlane(steps, i), mine, per);
    float price = (float)mine + (lane > 0 ? p.part_cost + p.merge_cost * (float)(items * p.kv_heads)
                                          : 0.f);
    if (lane > 0 && (items * p.kv_heads > p.slots || items > p.max_slots)) price = INFINITY;
    int best = lane;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const float other = __shfl_xor(price, d);
      const int its = __shfl_xor(best, d);
      if (other < price || (other == price && its < best)) {
        price = other;
        best = its;
      }
    }
    chunk = __shfl(mine, best);
  }
  int parts = lane < count ? max(1, (steps + chunk - 1) / chunk) : 0;
  uint32_t split = parts > 1 ? (uint32_t)parts << 16 | 1u : 0u;
  uint32_t splits = wave_scan(split);
  if ((__builtin_amdgcn_readlane((int)splits, 63) >> 16) > p.max_slots) {  // (never by the price)
    parts = min(parts, 1);
    split = splits = 0;
  }
  const int first = (int)wave_scan((uint32_t)parts) - parts;
  const int items = __builtin_amdgcn_readlane(first + parts, 63);
  Item it = {};
  it.request = r;
  it.q0 = t.q0; it.n = t.n; it.k0 = t.k0; it.m = t.m;
  it.tile = tile;
  it.parts = parts;
  it.slot = parts > 1 ? (int)((splits - split) >> 16) : -1;
  if (wg == 0 && threadIdx.x < 64) {
    if (parts > 1) p.splits[(splits - split) & 0xffff] = it;
    if (lane == 63) p.counts[1] = (int)(splits & 0xffff);
  }
  const int used = items * p.kv_heads;
  if (wg >= used) {
    clear_outside(p, wg - used, (int)gridDim.x - used);
    return false;
  }
  if (p.shared_lines) wg = unit_of(wg, used);
  const int item = wg / p.kv_heads;
  const int i = (int)__popcll(__ballot(lane < count && first <= item)) - 1;
  const int part = item - __builtin_amdgcn_readlane(first, i);
  const int len = __builtin_amdgcn_readlane(steps, i);
  out->request = __builtin_amdgcn_readlane(it.request, i);
  out->q0 = __builtin_amdgcn_readlane(it.q0, i);
  out->n = __builtin_amdgcn_readlane(it.n, i);
  out->k0 = __builtin_amdgcn_readlane(it.k0, i);
  out->m = __builtin_amdgcn_readlane(it.m, i);
  out->tile = __builtin_amdgcn_readlane(it.tile, i);
  out->parts = __builtin_amdgcn_readlane(it.parts, i);
  const Cut cut(len, out->parts);
  out->s0 = cut.from(part);
  out->s1 = cut.from(part + 1);
  const int slot = __builtin_amdgcn_readlane(it.slot, i);
  out->slot = slot >= 0 ? slot + part : -1;
  *head = wg - item * p.kv_heads;
  return true;
}

// The item and key head of this workgroup; false: none.  The list's first
// counts[2] items run eight key heads at a time, so that each XCD streams the
// keys of one head through its L2; the others, which even out the end of the call,
// run all heads of one item before the next.  (40 heads of one query head, 16,384
// x 16,384: 5.45 ms all heads at a time, 4.82 ms eight.)
__device__ __forceinline__ bool take_item(const Params& p, Item* it, int* h) {
  const int wg = (int)blockIdx.x;
  if (p.unlisted) return own_item(p, wg, it, h);
  const int count = ((dsa::const_i32)p.counts)[0], grouped = ((dsa::const_i32)p.counts)[2];
  if (wg >= count * p.kv_heads) return false;
  int item = wg / p.kv_heads;
  *h = wg - item * p.kv_heads;
  if (wg < grouped * p.kv_heads) {
    const int first = wg / max(1, grouped * kHeadGroup) * kHeadGroup;
    const int rest = wg - first * grouped, heads = min(kHeadGroup, p.kv_heads - first);
    item = rest / heads;
    *h = first + rest - item * heads;
  }
  *it = load_item(p.items + item);
  return true;
}

// 1 where a value is infinity times `sign`, or NaN, else 0.
template <typename T>
__device__ __forceinline__ T infinite_as(T v, float sign) {
  const float x = sign * (float)v;
  return x < INFINITY ? (T)0.0f : (T)1.0f;  // (NaN compares false)
}

// In the matrix products a hidden key's p is 0, and 0 times a value that is not finite
// is NaN.  True where that may have reached a wave's O: a value of the keys [lo, hi),
// which some of its rows see and others do not, or none, is not finite.
template <typename T, bool kPaged>
__device__ __forceinline__ bool hides_infinity(LateParams p, const Item& it, int h, int lo,
                                               int hi) {
  typedef typename dsa::Elem<T>::x8 x8;
  const int chunks = p->head_dim / 8;
  float sum = 0.f;  // NaN once an element is not finite
  for (int i = threadIdx.x & 63; i < (hi - lo) * chunks; i += 64) {
    const int key = lo + i / chunks, chunk = i % chunks;
    int64_t at = (int64_t)(it.k0 + key) * p->v_st;
    if (kPaged) {
      const int page =
          p->table[(int64_t)it.request * p->table_stride + (key >> p->page_shift)];
      if ((unsigned)page >= (unsigned)p->pages) continue;
      at = page * p->v_sp + (int64_t)(key & ((1 << p->page_shift) - 1)) * p->v_st;
    }
    const x8 v = *reinterpret_cast<const x8*>(static_cast<const T*>(p->v) + at + h * p->v_sh +
                                              chunk * 8);
#pragma unroll
    for (int e = 0; e < 8; ++e) sum = fmaf((float)v[e], 0.f, sum);
  }
  return __any(sum != 0.f);
}

// Rows that overlap (one key of stride 0, a V expanded along its tokens): a granule
// that ends inside holds copies of them behind the last key, hidden from every row.
__device__ __forceinline__ bool holds_copies(LateParams p, int kend) {
  return p->v_st < p->head_dim && (kend & 15) != 0;
}

// A wave's O over again, for a wave that hides_infinity: the same products (kRows = 32:
// 32x32x16, 16: 16x16x32), 32 keys at a time from key0, key0 + stride, .. below `hi`,
// with the final reference `m_use`, operands straight from memory.  Where keys from
// lim_first on (hidden from some row) have values that are not finite, these count as
// 0 in the product, and two products of "visible" with "+inf or NaN" and "-inf or NaN"
// tell which elements they reach.  (4,096 causal tokens x 4 heads: 50 us, with such
// values all over 150; element by element, a key to a lane, 14,000.  One infinity that
// nearly every row sees is hidden from rows of its own wave alone: 55 us.)
template <typename T, int kUse, bool kPaged, int kRows, typename Acc>
__device__ __forceinline__ void walk_again(LateParams p, const Item& it, int h, int64_t q_at,
                                           int lim, int lim_first, int key0, int stride, int hi,
                                           float m_use, Acc* oacc) {
  typedef dsa::Elem<T> E;
  typedef typename E::x8 x8;
  constexpr int kDims = 512 / kRows;          // of one product of scores
  constexpr int kElems = kRows * kRows / 64;  // of one accumulator, per lane
  constexpr int kSteps = kRows / 16;          // products of 32 keys with one tile of dims
  const int lane = threadIdx.x & 63;
  const int grp = lane / kRows, col = lane % kRows;
  auto mfma = [](x8 a, x8 b, Acc c) -> Acc {
    if constexpr (kRows == 32) return E::mfma32(a, b, c);
    else return E::mfma16(a, b, c);
  };
  const Source ks = source_of<kPaged>(p->k, p->k_sp, p->k_st, p->k_sh, h, it.k0);
  const Source vs = source_of<kPaged>(p->v, p->v_sp, p->v_st, p->v_sh, h, it.k0);
  const T* q = static_cast<const T*>(p->q) + q_at;
#pragma unroll
  for (int dt = 0; dt < kUse / kRows; ++dt)
#pragma unroll
    for (int r = 0; r < kElems; ++r) oacc[dt][r] = 0.f;
#pragma unroll 1
  for (; key0 < hi; key0 += stride) {
    // The block's two 16-key granules; a row sees their keys below `bound`.
    __amdgpu_buffer_rsrc_t kr[2], vr[2];
    int bound[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int key = key0 + 16 * i;
      int left = min(16, hi - key), row = key, page = 0;
      if (kPaged) {
        if (left > 0)
          page = __builtin_amdgcn_readfirstlane(
              p->table[(int64_t)it.request * p->table_stride + (key >> p->page_shift)]);
        if ((unsigned)page >= (unsigned)p->pages) left = 0;
        row &= (1 << p->page_shift) - 1;
      }
      kr[i] = rows_rsrc<kPaged>(ks, (uint32_t)page, row, left, p->head_dim);
      vr[i] = rows_rsrc<kPaged>(vs, (uint32_t)page, row, left, p->head_dim);
      bound[i] = left > 0 ? min(lim, hi) - key0 : 0;
    }
    // The block's key of slot t of product j, the same for scores and values, and
    // whether the lane's row sees it.
    auto granule_of = [&](int j, int t) { return kRows == 32 ? j : t >> 2; };
    auto row_of = [&](int t) { return (kRows == 32 ? 8 * (t >> 2) : 0) + 4 * grp + (t & 3); };
    auto visible = [&](int j, int t) {
      const int i = granule_of(j, t);
      return 16 * i + row_of(t) < bound[i];
    };
    x8 prob[kSteps];
    {
      asm volatile("" : "+v"(q));  // (Q is not held through the walk)
      const uint32_t at = (uint32_t)((col & 15) * (int)p->k_st + grp * 8) * 2;
      Acc s[32 / kRows];
#pragma unroll
      for (int i = 0; i < 32 / kRows; ++i)
#pragma unroll
        for (int r = 0; r < kElems; ++r) s[i][r] = 0.f;
#pragma unroll
      for (int dc = 0; dc < kUse / kDims; ++dc) {
        const int d = dc * kDims + grp * 8;
        x8 b;
#pragma unroll
        for (int e = 0; e < 8; ++e) b[e] = (T)0.0f;
        if (d < p->head_dim) b = *reinterpret_cast<const x8*>(q + d);
#pragma unroll
        for (int i = 0; i < 32 / kRows; ++i) {
          // (of 32 rows the upper 16 are the second granule's)
          dsa_u32x4 a = __builtin_amdgcn_raw_buffer_load_b128(kr[i], at + dc * kDims * 2, 0, 0);
          if (kRows == 32) {
            const dsa_u32x4 upper =
                __builtin_amdgcn_raw_buffer_load_b128(kr[1], at + dc * kDims * 2, 0, 0);
            if (col >= 16) a = upper;
          }
          if (d >= p->head_dim) a = dsa_u32x4{0u, 0u, 0u, 0u};
          s[i] = mfma(__builtin_bit_cast(x8, a), b, s[i]);
        }
      }
#pragma unroll
      for (int j = 0; j < kSteps; ++j)
#pragma unroll
        for (int t = 0; t < 8; ++t) {
          const int f = j * 8 + t;
          const float score = fmaf(s[f / kElems][f % kElems], p->scale_log2, -m_use);
          prob[j][t] = (T)(visible(j, t) ? __builtin_amdgcn_exp2f(score) : 0.f);
        }
    }
#pragma unroll
    for (int dt = 0; dt < kUse / kRows; ++dt) {
#pragma unroll
      for (int j = 0; j < kSteps; ++j) {
        x8 a;
        float sum = 0.f;
#pragma unroll
        for (int t = 0; t < 8; ++t) {
          // (dims past head_dim are between the rows' ends or 0, and go nowhere)
          a[t] = __builtin_bit_cast(
              T, __builtin_amdgcn_raw_buffer_load_b16(
                     vr[granule_of(j, t)],
                     (uint32_t)(row_of(t) * (int)p->v_st + col) * 2 + dt * kRows * 2, 0, 0));
          sum = fmaf((float)a[t], 0.f, sum);
        }
        if (key0 + 32 > lim_first && __any(sum != 0.f)) {
          x8 up, down, seen;
          Acc ups, downs;
#pragma unroll
          for (int t = 0; t < 8; ++t) {
            up[t] = infinite_as(a[t], 1.f);
            down[t] = infinite_as(a[t], -1.f);
            seen[t] = (T)(visible(j, t) ? 1.f : 0.f);
            if ((float)a[t] * 0.f != 0.f) a[t] = (T)0.0f;
          }
#pragma unroll
          for (int r = 0; r < kElems; ++r) ups[r] = downs[r] = 0.f;
          ups = mfma(up, seen, ups);
          downs = mfma(down, seen, downs);
#pragma unroll
          for (int r = 0; r < kElems; ++r) {
            if (ups[r] > 0.f) oacc[dt][r] += INFINITY;
            if (downs[r] > 0.f) oacc[dt][r] -= INFINITY;
          }
        }
        oacc[dt] = mfma(a, prob[j], oacc[dt]);
      }
    }
  }
}

// 128 rows x the item's keys.  Each wave owns 32 rows; keys stream as 64-key
// half-tiles of K and V, double-buffered in LDS by direct loads issued one
// half-tile ahead; lane (g, qi) = (lane / 32, lane % 32) holds row qi's scores
// of the keys 32 kt + 8 (r / 4) + 4 g + r % 4 and, of O, the dims 32 dt +
// 8 (r / 4) + 4 g + r % 4.
//
// Staged rows hold kD dims, of which the products take the first kUse: head dims of
// 72 to 96 leave the last quarter of a 128-dim row out (8,192 x 8,192 x 32 heads: 96
// dims 897 -> 804 us, 80 dims 985 -> 896).  64-dim rows take 32 KB of LDS and leave
// room for four workgroups a compute unit, if their registers do (128 a lane).
template <typename T, int kD, int kUse, bool kPaged>
__global__ void __launch_bounds__(256, kD == 64 ? 4 : 2) seq_wide_kernel(Params p) {
  typedef dsa::Elem<T> E;
  typedef typename E::x8 x8;
  constexpr int kRow = kD * 2;               // bytes of a staged row
  constexpr int kStage = kWideKeys * kRow;
  constexpr int kChunks = kD / 8;            // 16-byte chunks per row
  constexpr int kSlices = kD / 32;           // 1 KB loads per wave, K or V
  constexpr int kRowsPer = 64 / kChunks;     // rows of one load
  constexpr int kDt = kUse / 32;             // 32-dim output tiles
  __shared__ __attribute__((aligned(1024))) unsigned char lds_k0[kStage];
  __shared__ __attribute__((aligned(1024))) unsigned char lds_k1[kStage];
  __shared__ __attribute__((aligned(1024))) unsigned char lds_v0[kStage];
  __shared__ __attribute__((aligned(1024))) unsigned char lds_v1[kStage];

  Item it;
  int h;
  if (!take_item(p, &it, &h)) return;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 5, qi = lane & 31;
  const int rows = it.n * p.group;
  const int local = wave * 32 + qi;
  const int row = it.tile * kWideRows + local;
  const bool row_ok = row < rows;
  const int row_c = min(row, rows - 1);
  const int token = row_c / p.group;
  const int head = h * p.group + row_c - token * p.group;
  // Keys [0, lim) are visible to the lane's row.
  const int lim = p.causal ? max(0, min(it.m, it.m - it.n + token + 1)) : it.m;
  const bool wave_active = it.tile * kWideRows + wave * 32 < rows;
  const int lim_first = __builtin_amdgcn_readlane(lim, 0);
  const int lim_last = __builtin_amdgcn_readlane(lim, 31);
  // Keys the tile's last row sees: rows past it stage as zeros.
  const int last_row = min(it.tile * kWideRows + kWideRows, rows) - 1;
  const int kend =
      p.causal ? max(0, min(it.m, it.m - it.n + last_row / p.group + 1)) : it.m;

  x8 qf[kUse / 16];
  {
    const T* qrow = static_cast<const T*>(p.q) + (int64_t)(it.q0 + token) * p.q_st +
                    head * p.q_sh;
#pragma unroll
    for (int dc = 0; dc < kUse / 16; ++dc) {
#pragma unroll
      for (int e = 0; e < 8; ++e) qf[dc][e] = (T)0.0f;
      if (dc * 16 + g * 8 < p.head_dim)
        qf[dc] = *reinterpret_cast<const x8*>(qrow + dc * 16 + g * 8);
    }
  }

  // Wave w stages rows 16 w .. 16 w + 15: one page, one resource.  Lane offsets
  // from the first of them (a chunk past head_dim loads zeros).
  uint32_t koff[kSlices], voff[kSlices];
#pragma unroll
  for (int j = 0; j < kSlices; ++j) {
    const int r = j * kRowsPer + lane / kChunks;  // row in the wave's 16
    const int c = lane % kChunks;
    const int kc = k_swz<kD>(wave * 16 + r, c);
    const int vc = kD == 128 ? c ^ ((0xCA60 >> (4 * (r & 3))) & 15) : c ^ (4 * ((r >> 1) & 1));
    koff[j] = (uint32_t)((r * (int)p.k_st + kc * 8) * 2) | dsa::dead_bits(kc, p.head_dim);
    voff[j] = (uint32_t)((r * (int)p.v_st + vc * 8) * 2) | dsa::dead_bits(vc, p.head_dim);
  }
  int vfrag[kDt];
  {
    const int lam = lane & 15, r = lam >> 2, c = lam & 3;
    const int vrow = 4 * g + r;
    const int sub = 2 * ((lane >> 4) & 1) + (c >> 1);
#pragma unroll
    for (int dt = 0; dt < kDt; ++dt) {
      const int chunk = 4 * dt + sub;
      const int pos = kD == 128 ? chunk ^ ((0xCA60 >> (4 * (vrow & 3))) & 15)
                                : chunk ^ (4 * ((vrow >> 1) & 1));
      vfrag[dt] = vrow * kRow + pos * 16 + (c & 1) * 8;
    }
  }

  // Pages of a 1,024-key window, one 16-key granule per lane; the next window's
  // are loaded a window ahead.
  auto window_ids = [&](int window) -> int {
    const int key = window * 1024 + lane * 16;
    return key < kend ? page_at(p, it.request, key) : -1;
  };
  int ids = -1, ids_next = -1;
  uint64_t bad_ids = 0;  // the window's granules in bad pages
  if constexpr (kPaged) {
    ids = window_ids(it.s0 >> 4);
    ids_next = window_ids((it.s0 >> 4) + 1);
    bad_ids = __ballot((unsigned)ids >= (unsigned)p.pages);
  }
  const Source ks = source_of<kPaged>(p.k, p.k_sp, p.k_st, p.k_sh, h, it.k0);
  const Source vs = source_of<kPaged>(p.v, p.v_sp, p.v_st, p.v_sh, h, it.k0);
  // Where step s of this wave's rows lies, worked out a step before its loads go
  // out; bad: the granules (bits 0..3) of the step whose page is outside the cache.
  __amdgpu_buffer_rsrc_t kr, vr;
  int bad_next = 0;
  auto locate = [&](int s) __attribute__((always_inline)) {
    int row = s * kWideKeys + wave * 16;
    int left = min(16, kend - row);
    uint32_t page = 0;
    if constexpr (kPaged) {
      if ((s & 15) == 0) {  // the next window (step s0's is there already)
        ids = ids_next;
        bad_ids = __ballot((unsigned)ids >= (unsigned)p.pages);
        ids_next = window_ids((s >> 4) + 1);
      }
      page = (uint32_t)__builtin_amdgcn_readlane(ids, (s & 15) * 4 + wave);
      bad_next = (int)(bad_ids >> ((s & 15) * 4)) & 15;
      if (page >= (uint32_t)p.pages) left = 0;
      row &= (1 << p.page_shift) - 1;
    }
    kr = rows_rsrc<kPaged>(ks, page, row, left, p.head_dim);
    vr = rows_rsrc<kPaged>(vs, page, row, left, p.head_dim);
  };
  // (the empty asm keeps the stage addresses from being held for every load)
  auto issue = [&](unsigned char* kdst, unsigned char* vdst) __attribute__((always_inline)) {
    int at = wave * kSlices * 1024;
    asm volatile("" : "+s"(at));
#pragma unroll
    for (int j = 0; j < kSlices; ++j) lds_load16(kr, kdst + at + j * 1024, koff[j], 0);
#pragma unroll
    for (int j = 0; j < kSlices; ++j) lds_load16(vr, vdst + at + j * 1024, voff[j], 0);
  };

  float m_run = -INFINITY, l_run = 0.f;
  dsa_f32x16 oacc[kDt];
#pragma unroll
  for (int dt = 0; dt < kDt; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) oacc[dt][r] = 0.f;

  auto compute = [&](const unsigned char* k_lds, const unsigned char* v_lds, int key0, int bad)
      __attribute__((always_inline)) {
    __builtin_amdgcn_s_setprio(0);
    dsa_f32x16 sacc[2];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int r = 0; r < 16; ++r) sacc[kt][r] = 0.f;
#pragma unroll
    for (int dc = 0; dc < kUse / 16; ++dc)
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        const int krow = kt * 32 + qi;
        const x8 a = *reinterpret_cast<const x8*>(k_lds + krow * kRow +
                                                  k_swz<kD>(krow, dc * 2 + g) * 16);
        sacc[kt] = E::mfma32(a, qf[dc], sacc[kt]);
      }
    // Four K reads in flight ahead of the products.
    __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
    for (int i = 0; i < kUse / 8 - 4; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, 4, 0);
    if (key0 + kWideKeys > lim_first) {
      const int bound = lim - key0 - 4 * g;
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (kt * 32 + 8 * (r >> 2) + (r & 3) >= bound) sacc[kt][r] = -INFINITY;
    }
    if (kPaged && bad != 0) {
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (bad & (1 << (2 * kt + (r >> 3)))) sacc[kt][r] = -INFINITY;
    }
    float mx = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, sacc[kt][r]);
    const float mx2 = dsa::pair32_max(mx) * p.scale_log2;
    const bool up = mx2 > m_run + kRescaleLog2;
    if (__any(up)) {
      const float m_new = up ? mx2 : m_run;
      const float alpha = up ? __builtin_amdgcn_exp2f(m_run - m_new) : 1.0f;
      m_run = m_new;
      l_run *= alpha;
#pragma unroll
      for (int dt = 0; dt < kDt; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) oacc[dt][r] *= alpha;
    }
    const float m_use = m_run == -INFINITY ? 0.f : m_run;
    x8 pf[4];
    float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int t = 0; t < 8; t += 2) {
        const float p0 = __builtin_amdgcn_exp2f(
            fmaf(sacc[j >> 1][(j & 1) * 8 + t], p.scale_log2, -m_use));
        const float p1 = __builtin_amdgcn_exp2f(
            fmaf(sacc[j >> 1][(j & 1) * 8 + t + 1], p.scale_log2, -m_use));
        const dsa_f32x2 two = {p0, p1};
        const typename E::x2 pb = __builtin_convertvector(two, typename E::x2);
        sum0 += p0;
        sum1 += p1;
        pf[j][t] = pb[0];
        pf[j][t + 1] = pb[1];
      }
    l_run += sum0 + sum1;
    // The two waves of a SIMD fall into opposite phases (2 to 4% on every long case).
    // The priority lasts until the next step's first product, so that the barrier
    // and the loads behind it are passed quickly (eight chunks over 30,000 cached
    // tokens 1,262 -> 1,231 us, 3,600 tokens x 40 heads over 57,600 3,870 -> 3,800).
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int dt = 0; dt < kDt; ++dt) {
        // Key rows 16 j + 4 g + r (slots 0..3) and 16 j + 8 + 4 g + r (4..7).
        const unsigned char* at = v_lds + vfrag[dt] + j * 16 * kRow;
        const typename E::x4 lo = read_tr<T>(at);
        const typename E::x4 hi = read_tr<T>(at + 8 * kRow);
        const x8 a = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        oacc[dt] = E::mfma32(a, pf[j], oacc[dt]);
      }
    // Four products' V reads (two each) ahead: 32,760 causal tokens 9,300 -> 9,170 us.
    __builtin_amdgcn_sched_group_barrier(0x100, 8, 1);
#pragma unroll
    for (int i = 0; i < 4 * kDt - 4; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 1);
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 1);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, 4, 1);
  };
  int bad_cur = 0, bad_ahead = 0;  // of the staged step and of the one on its way
  auto step = [&](int s, const unsigned char* kc, const unsigned char* vc, unsigned char* kn,
                  unsigned char* vn) __attribute__((always_inline)) {
    __builtin_amdgcn_s_waitcnt(vmcnt(0));
    __syncthreads();
    if (s + 1 < it.s1) {
      issue(kn, vn);
      bad_ahead = bad_next;
      locate(s + 2);  // (past the last key: no rows)
    }
    // (a wave whose rows see none of the step's keys only stages)
    if (wave_active && s * kWideKeys < lim_last) compute(kc, vc, s * kWideKeys, bad_cur);
    bad_cur = bad_ahead;
  };
  if (it.s0 < it.s1) {
    if constexpr (kPaged) {
      if ((it.s0 & 15) == 0) ids_next = ids;  // locate() takes it up
    }
    locate(it.s0);
    issue(lds_k0, lds_v0);
    bad_cur = bad_next;
    locate(it.s0 + 1);
    for (int s = it.s0; s < it.s1; s += 2) {
      step(s, lds_k0, lds_v0, lds_k1, lds_v1);
      if (s + 1 >= it.s1) break;
      step(s + 1, lds_k1, lds_v1, lds_k0, lds_v0);
    }
  }

  const LateParams late = late_params();
  const float l_tot = dsa::pair32_sum(l_run);
  float unfinite = 0.f;  // NaN once an element of O is not finite
#pragma unroll
  for (int dt = 0; dt < kDt; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) unfinite = fmaf(oacc[dt][r], 0.f, unfinite);
  // (a row whose scores are not finite stays as it is)
  const bool copies = holds_copies(late, kend);
  if (__builtin_expect(
          (lim_first < kend || copies) && __any(unfinite != 0.f && l_tot * 0.f == 0.f), 0)) {
    // Staged with the wave's last steps, but not seen by all of its rows.
    const int last = min((lim_last + kWideKeys - 1) & -kWideKeys, it.s1 * kWideKeys);
    if (copies || hides_infinity<T, kPaged>(late, it, h, max(lim_first, it.s0 * kWideKeys),
                                            min(last, kend)))
      walk_again<T, kUse, kPaged, 32>(
          late, it, h, (int64_t)(it.q0 + token) * late->q_st + head * late->q_sh, lim, lim_first,
          it.s0 * kWideKeys, 32, min(lim_last, it.s1 * kWideKeys),
          m_run == -INFINITY ? 0.f : m_run, oacc);
  }
  if (it.slot >= 0) {
    // A partial keeps the accumulators' own order (part_at): whole lines per store.
    float* const po =
        late->part + ((int64_t)it.slot * late->kv_heads + h) * part_floats(kWideRows, kD);
#pragma unroll
    for (int dt = 0; dt < kDt; ++dt)
#pragma unroll
      for (int rr = 0; rr < 4; ++rr) {
        const dsa_f32x4 v4 = {oacc[dt][rr * 4 + 0], oacc[dt][rr * 4 + 1],
                              oacc[dt][rr * 4 + 2], oacc[dt][rr * 4 + 3]};
        *reinterpret_cast<dsa_f32x4*>(po +
                                      part_at<kD, kWideRows>(local, dt * 32 + rr * 8 + g * 4)) = v4;
      }
    if (g == 0) {
      po[kWideRows * kD + local] = m_run;
      po[kWideRows * (kD + 1) + local] = l_tot;
    }
    return;
  }
  if (late->lse && g == 0 && row_ok)
    late->lse[(int64_t)head * late->q_rows + it.q0 + token] =
        l_tot == 0.f ? -INFINITY : m_run * kLn2 + logf(l_tot);
  // O goes out through the wave's quarter of the stages that the last step left
  // alone (every wave is past its reads of them, and no load is on its way there):
  // written row by row as 16-byte chunks, whole rows to a store.
  const float inv = l_tot > 0.f ? 1.f / l_tot : (l_tot == 0.f ? 0.f : l_tot);
  const bool odd = (it.s1 - it.s0) & 1;
  unsigned char* const mine = (wave < 2 ? (odd ? lds_k1 : lds_k0) : (odd ? lds_v1 : lds_v0)) +
                              (wave & 1) * (kStage / 2);
#pragma unroll
  for (int dt = 0; dt < kDt; ++dt)
#pragma unroll
    for (int rr = 0; rr < 4; ++rr) {
      typename E::x4 v4;
#pragma unroll
      for (int e = 0; e < 4; ++e) v4[e] = (T)(oacc[dt][rr * 4 + e] * inv);
      *reinterpret_cast<typename E::x4*>(mine + qi * kRow + k_swz<kD>(qi, dt * 4 + rr) * 16 +
                                         g * 8) = v4;
    }
  __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
  __builtin_amdgcn_wave_barrier();
  const int64_t o_at = row_ok ? (int64_t)(it.q0 + token) * late->o_st + head * late->o_sh : -1;
#pragma unroll
  for (int i = 0; i < kD / 16; ++i) {
    const int r = i * kRowsPer + lane / kChunks, c = lane % kChunks;
    const x8 y = *reinterpret_cast<const x8*>(mine + r * kRow + k_swz<kD>(r, c) * 16);
    const int64_t at = __shfl(o_at, r);
    if (at >= 0 && c * 8 < late->head_dim)
      *reinterpret_cast<x8*>(static_cast<T*>(late->o) + at + c * 8) = y;
  }
}

// 16 rows x the item's keys, on 16x16x32 products.  Wave w takes keys 128 s +
// 32 w .. + 31 of every step s through its own two LDS stage pairs; lane (q4,
// c16) = (lane / 16, lane % 16) holds row c16's scores of the keys 16 kg + 4 q4
// + r and, of O, the dims 16 dt + 4 q4 + r.
template <typename T, int kD, bool kPaged>
__global__ void __launch_bounds__(kNarrowWaves * 64, 1) seq_narrow_kernel(Params p) {
  typedef dsa::Elem<T> E;
  typedef typename E::x8 x8;
  constexpr int kRow = kD * 2;
  constexpr int kStage = 32 * kRow;         // K or V of one wave's 32 keys
  constexpr int kChunks = kD / 8;
  constexpr int kRowsPer = 64 / kChunks;    // rows of one 1 KB load
  constexpr int kLoads = 16 / kRowsPer;     // loads per 16-key granule
  constexpr int kDt = kD / 16;
  __shared__ __attribute__((aligned(1024))) unsigned char lds_k0[kNarrowWaves * kStage];
  __shared__ __attribute__((aligned(1024))) unsigned char lds_k1[kNarrowWaves * kStage];
  __shared__ __attribute__((aligned(1024))) unsigned char lds_v0[kNarrowWaves * kStage];
  __shared__ __attribute__((aligned(1024))) unsigned char lds_v1[kNarrowWaves * kStage];

  __shared__ float join_ml[2][kNarrowWaves][16];
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int q4 = lane >> 4, c16 = lane & 15;
  auto run = [&](const Item& it, const int h) __attribute__((always_inline)) {
  const int rows = it.n * p.group;
  const int row_c = min(it.tile * kNarrowRows + c16, rows - 1);
  const int token = row_c / p.group;
  const int head = h * p.group + row_c - token * p.group;
  const int lim = p.causal ? max(0, min(it.m, it.m - it.n + token + 1)) : it.m;
  const int lim_first = __builtin_amdgcn_readlane(lim, 0);
  const int kend = __builtin_amdgcn_readlane(lim, 15);

  x8 qf[kD / 32];
  {
    const T* qrow = static_cast<const T*>(p.q) + (int64_t)(it.q0 + token) * p.q_st +
                    head * p.q_sh;
#pragma unroll
    for (int dc = 0; dc < kD / 32; ++dc) {
#pragma unroll
      for (int e = 0; e < 8; ++e) qf[dc][e] = (T)0.0f;
      if (dc * 32 + q4 * 8 < p.head_dim)
        qf[dc] = *reinterpret_cast<const x8*>(qrow + dc * 32 + q4 * 8);
    }
  }
  // V chunk c of row r sits at c ^ 2 (r & 7) (256-byte rows) or c ^ 2 ((r / 2) & 3).
  auto v_swz = [](int r, int c) { return kD == 128 ? c ^ (2 * (r & 7)) : c ^ (2 * ((r >> 1) & 3)); };
  uint32_t koff[kLoads], voff[kLoads];
#pragma unroll
  for (int j = 0; j < kLoads; ++j) {
    const int r = j * kRowsPer + lane / kChunks;  // row in its 16-key granule
    const int c = lane % kChunks;
    const int kc = k_swz<kD>(r, c), vc = v_swz(r, c);
    koff[j] = (uint32_t)((r * (int)p.k_st + kc * 8) * 2) | dsa::dead_bits(kc, p.head_dim);
    voff[j] = (uint32_t)((r * (int)p.v_st + vc * 8) * 2) | dsa::dead_bits(vc, p.head_dim);
  }

  // Keys that no other tile of the request reads stream past the caches (64
  // requests of 1,000 to 16,000 tokens, 8 key heads: 661 -> 601 us).  Keys that
  // still lie in the 256 MB cache from an earlier call take some 12% longer so,
  // but a model's layers each have their own.  (The same in seq_wide_kernel gained
  // 14% on cold single tiles and cost the long calls 2 to 3%.)  Lines that several
  // heads share do not (unit_of).
  const bool only_tile = rows <= kNarrowRows && !p.shared_lines;

  // Pages of a window of 32 steps: lane l holds granule l & 1 of step l / 2.
  auto window_ids = [&](int window) -> int {
    const int key = (window * 32 + (lane >> 1)) * kNarrowKeys + wave * 32 + (lane & 1) * 16;
    return key < kend ? page_at(p, it.request, key) : -1;
  };
  int ids = -1, ids_next = -1, bad_next = 0;
  uint64_t bad_ids = 0;  // the window's granules in bad pages
  if constexpr (kPaged) {
    ids = window_ids(it.s0 >> 5);
    ids_next = (it.s0 & 31) == 0 ? ids : window_ids((it.s0 >> 5) + 1);
    bad_ids = __ballot((unsigned)ids >= (unsigned)p.pages);
  }
  const Source ks = source_of<kPaged>(p.k, p.k_sp, p.k_st, p.k_sh, h, it.k0);
  const Source vs = source_of<kPaged>(p.v, p.v_sp, p.v_st, p.v_sh, h, it.k0);
  auto issue = [&](int s, unsigned char* kdst, unsigned char* vdst)
      __attribute__((always_inline)) {
    const int key = s * kNarrowKeys + wave * 32;
    int at = wave * kStage;
    asm volatile("" : "+s"(at));
    if constexpr (kPaged) {
      if ((s & 31) == 0) {  // the next window (the first step's is there already)
        ids = ids_next;
        bad_ids = __ballot((unsigned)ids >= (unsigned)p.pages);
        ids_next = window_ids((s >> 5) + 1);
      }
      bad_next = (int)(bad_ids >> ((s & 31) * 2)) & 3;
    }
#pragma unroll
    for (int kg = 0; kg < 2; ++kg) {
      int row = key + 16 * kg;
      int left = min(16, kend - row);
      uint32_t page = 0;
      if constexpr (kPaged) {
        page = (uint32_t)__builtin_amdgcn_readlane(ids, (s & 31) * 2 + kg);
        if (page >= (uint32_t)p.pages) left = 0;
        row &= (1 << p.page_shift) - 1;
      }
      const __amdgpu_buffer_rsrc_t kr = rows_rsrc<kPaged>(ks, page, row, left, p.head_dim);
      const __amdgpu_buffer_rsrc_t vr = rows_rsrc<kPaged>(vs, page, row, left, p.head_dim);
      auto load = [&](auto once) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < kLoads; ++j)
          lds_stream16<decltype(once)::value>(kr, kdst + at + (kg * kLoads + j) * 1024, koff[j]);
#pragma unroll
        for (int j = 0; j < kLoads; ++j)
          lds_stream16<decltype(once)::value>(vr, vdst + at + (kg * kLoads + j) * 1024, voff[j]);
      };
      if (only_tile) load(std::true_type{});
      else load(std::false_type{});
    }
  };

  float m_run = -INFINITY, l_run = 0.f;
  dsa_f32x4 oacc[kDt];
#pragma unroll
  for (int dt = 0; dt < kDt; ++dt) oacc[dt] = dsa_f32x4{0.f, 0.f, 0.f, 0.f};
  const int vr_row = 4 * q4 + (c16 >> 2);

  auto compute = [&](const unsigned char* k_lds, const unsigned char* v_lds, int key0, int bad)
      __attribute__((always_inline)) {
    dsa_f32x4 s[2];
#pragma unroll
    for (int kg = 0; kg < 2; ++kg) s[kg] = dsa_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int dc = 0; dc < kD / 32; ++dc)
#pragma unroll
      for (int kg = 0; kg < 2; ++kg) {
        const x8 a = *reinterpret_cast<const x8*>(
            k_lds + wave * kStage + (16 * kg + c16) * kRow + k_swz<kD>(c16, dc * 4 + q4) * 16);
        s[kg] = E::mfma16(a, qf[dc], s[kg]);
      }
    if (key0 + 32 > lim_first) {
      const int bound = lim - key0 - 4 * q4;
#pragma unroll
      for (int kg = 0; kg < 2; ++kg)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (16 * kg + r >= bound) s[kg][r] = -INFINITY;
    }
    if (kPaged && bad != 0) {
#pragma unroll
      for (int kg = 0; kg < 2; ++kg)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (bad & (1 << kg)) s[kg][r] = -INFINITY;
    }
    float mx = -INFINITY;
#pragma unroll
    for (int kg = 0; kg < 2; ++kg)
#pragma unroll
      for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[kg][r]);
    mx = fmaxf(mx, __shfl_xor(mx, 16));
    const float mx2 = dsa::pair32_max(mx) * p.scale_log2;
    const bool up = mx2 > m_run + kRescaleLog2;
    if (__any(up)) {
      const float m_new = up ? mx2 : m_run;
      const float alpha = up ? __builtin_amdgcn_exp2f(m_run - m_new) : 1.0f;
      m_run = m_new;
      l_run *= alpha;
#pragma unroll
      for (int dt = 0; dt < kDt; ++dt) oacc[dt] *= alpha;
    }
    const float m_use = m_run == -INFINITY ? 0.f : m_run;
    x8 pf;
    float sum = 0.f;
#pragma unroll
    for (int kg = 0; kg < 2; ++kg)
#pragma unroll
      for (int r = 0; r < 4; r += 2) {
        const float p0 = __builtin_amdgcn_exp2f(fmaf(s[kg][r], p.scale_log2, -m_use));
        const float p1 = __builtin_amdgcn_exp2f(fmaf(s[kg][r + 1], p.scale_log2, -m_use));
        const dsa_f32x2 two = {p0, p1};
        const typename E::x2 pb = __builtin_convertvector(two, typename E::x2);
        sum += p0 + p1;
        pf[4 * kg + r] = pb[0];
        pf[4 * kg + r + 1] = pb[1];
      }
    l_run += sum;
#pragma unroll
    for (int dt = 0; dt < kDt; ++dt) {
      const int pos = v_swz(vr_row, 2 * dt + ((c16 & 3) >> 1));
      const unsigned char* at =
          v_lds + wave * kStage + vr_row * kRow + pos * 16 + (c16 & 1) * 8;
      const typename E::x4 lo = read_tr<T>(at);
      const typename E::x4 hi = read_tr<T>(at + 16 * kRow);
      const x8 a = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      oacc[dt] = E::mfma16(a, pf, oacc[dt]);
    }
  };
  // A wave's stages are its own: it waits for its loads alone.
  int bad_cur = 0;
  auto step = [&](int s, const unsigned char* kc, const unsigned char* vc, unsigned char* kn,
                  unsigned char* vn) __attribute__((always_inline)) {
    if (s + 1 < it.s1) {
      issue(s + 1, kn, vn);
      __builtin_amdgcn_s_waitcnt(vmcnt(4 * kLoads));
    } else {
      __builtin_amdgcn_s_waitcnt(vmcnt(0));
    }
    const int key0 = s * kNarrowKeys + wave * 32;
    if (key0 < kend) compute(kc, vc, key0, bad_cur);
    bad_cur = bad_next;
  };
  if (it.s0 < it.s1) {
    issue(it.s0, lds_k0, lds_v0);
    bad_cur = bad_next;
    for (int s = it.s0; s < it.s1; s += 2) {
      step(s, lds_k0, lds_v0, lds_k1, lds_v1);
      if (s + 1 >= it.s1) break;
      step(s + 1, lds_k1, lds_v1, lds_k0, lds_v0);
    }
  }

  const LateParams late = late_params();
  // Join the waves: their O, m and l through the K stages (row-major fp32).
  l_run += __shfl_xor(l_run, 16);
  const float l_wave = dsa::pair32_sum(l_run);
  static_assert(kNarrowRows * kD * 4 <= kStage, "a wave joins through its own K stage");
  float unfinite = 0.f;  // NaN once an element of O is not finite
#pragma unroll
  for (int dt = 0; dt < kDt; ++dt)
#pragma unroll
    for (int r = 0; r < 4; ++r) unfinite = fmaf(oacc[dt][r], 0.f, unfinite);
  // (a row whose scores are not finite stays as it is)
  const bool copies = holds_copies(late, kend);
  if (__builtin_expect(
          (lim_first < kend || copies) && __any(unfinite != 0.f && l_wave * 0.f == 0.f), 0) &&
      (copies || hides_infinity<T, kPaged>(late, it, h, max(lim_first, it.s0 * kNarrowKeys),
                                           min(kend, it.s1 * kNarrowKeys))))
    walk_again<T, kD, kPaged, 16>(
        late, it, h, (int64_t)(it.q0 + token) * late->q_st + head * late->q_sh, lim, lim_first,
        it.s0 * kNarrowKeys + wave * 32, kNarrowKeys, min(kend, it.s1 * kNarrowKeys),
        m_run == -INFINITY ? 0.f : m_run, oacc);
  dsa::lds_barrier<true>();
  float* const mine = reinterpret_cast<float*>(lds_k0) + wave * kNarrowRows * kD;
#pragma unroll
  for (int dt = 0; dt < kDt; ++dt)
    *reinterpret_cast<dsa_f32x4*>(mine + c16 * kD + 16 * dt + 4 * q4) = oacc[dt];
  if (q4 == 0) {
    join_ml[0][wave][c16] = m_run;
    join_ml[1][wave][c16] = l_wave;
  }
  dsa::lds_barrier();
  // Thread (r, c): row r, dims 8 c .. 8 c + 7.
  for (int r = tid / kChunks; r < kNarrowRows; r += kNarrowWaves * kRowsPer) {
  const int d0 = (tid % kChunks) * 8;
  const int out_row = it.tile * kNarrowRows + r;
  if (out_row >= rows) break;
  float m_all = -INFINITY, l_all = 0.f, w[kNarrowWaves];
#pragma unroll
  for (int i = 0; i < kNarrowWaves; ++i) m_all = fmaxf(m_all, join_ml[0][i][r]);
#pragma unroll
  for (int i = 0; i < kNarrowWaves; ++i) {
    const float mi = join_ml[0][i][r];
    // (no finite score: l is 0, or NaN from NaN scores)
    w[i] = mi == -INFINITY ? join_ml[1][i][r] : __builtin_amdgcn_exp2f(mi - m_all);
    l_all = fmaf(w[i], join_ml[1][i][r], l_all);
  }
  float acc[8];
#pragma unroll
  for (int x = 0; x < 8; ++x) acc[x] = 0.f;
#pragma unroll
  for (int i = 0; i < kNarrowWaves; ++i) {
    if (w[i] == 0.f) continue;
    const float* src = reinterpret_cast<const float*>(lds_k0) + (i * kNarrowRows + r) * kD + d0;
#pragma unroll
    for (int x = 0; x < 8; ++x) acc[x] = fmaf(w[i], src[x], acc[x]);
  }
  if (it.slot >= 0) {
    float* po = late->part + ((int64_t)it.slot * late->kv_heads + h) * part_floats(kNarrowRows, kD);
#pragma unroll
    for (int c = 0; c < 2; ++c)
      *reinterpret_cast<dsa_f32x4*>(po + r * kD + d0 + 4 * c) =
          dsa_f32x4{acc[4 * c], acc[4 * c + 1], acc[4 * c + 2], acc[4 * c + 3]};
    if (d0 == 0) {
      po[kNarrowRows * kD + r] = m_all;
      po[kNarrowRows * (kD + 1) + r] = l_all;
    }
    continue;
  }
  const int out_token = it.q0 + out_row / late->group;
  const int out_head = h * late->group + out_row % late->group;
  const float inv = l_all > 0.f ? 1.f / l_all : (l_all == 0.f ? 0.f : l_all);
  if (d0 < late->head_dim) {
    x8 y;
#pragma unroll
    for (int x = 0; x < 8; ++x) y[x] = (T)(acc[x] * inv);
    *reinterpret_cast<x8*>(static_cast<T*>(late->o) + (int64_t)out_token * late->o_st +
                           out_head * late->o_sh + d0) = y;
  }
  if (late->lse && d0 == 0)
    late->lse[(int64_t)out_head * late->q_rows + out_token] =
        l_all == 0.f ? -INFINITY : m_all * kLn2 + logf(l_all);
  }  };

  // An unlisted call gives the workgroup one item, a listed one its chain.
  Item it;
  int h;
  if (p.unlisted) {
    if (own_item(p, (int)blockIdx.x, &it, &h)) run(it, h);
    return;
  }
  const int wg = (int)blockIdx.x;
  const int unit = p.shared_lines ? unit_of(wg, (int)gridDim.x) : wg;
  const int chain = unit / p.kv_heads;
  h = unit - chain * p.kv_heads;
  const int count = ((dsa::const_i32)p.counts)[0];
  int i = ((dsa::const_i32)p.chain_start)[chain];
  if (i >= count) return;
  it = load_item(p.items + i);
#pragma unroll 1
  for (;;) {
    run(it, h);
    if (++i >= count) break;
    it = load_item(p.items + i);
    if (it.chain != chain) break;
    dsa::lds_barrier();  // the join's reads are done
  }
}

// Joins the parts of split tiles: with M the largest reference, O = sum_i O_i
// 2^(m_i - M) / sum_i l_i 2^(m_i - M).  Latency-bound, so every thread has four
// parts' loads on their way.  A workgroup takes 16 rows of a tile of few parts, 16
// threads to a row with 8 dims each; of a tile of many parts (few rows over many
// keys) one row, 16 groups of 16 threads taking every 16th part, joined through
// LDS.
constexpr int kFewParts = 16;
template <typename T, int kD, int kRows>
__global__ void __launch_bounds__(256) seq_merge_kernel(Params p) {
  __shared__ float acc_lds[16][kD];
  __shared__ float ml[2][16];
  const int splits = ((dsa::const_i32)p.counts)[1];
  const int h = blockIdx.y;
  const int tid = threadIdx.x;
  // Units of 16 rows along x; z counts the rows of one where each takes a
  // workgroup.
  constexpr int kUnits = kRows / 16;
  for (int work = blockIdx.x; work < splits * kUnits; work += gridDim.x)
  for (int z = blockIdx.z; z < 16; z += gridDim.z) {
    const Item it = load_item(p.splits + work / kUnits);
    const bool few = it.parts <= kFewParts;
    if (few && z > 0) break;
    // (rows side by side where a partial has them so)
    const bool across = kRows != 16 && few;
    const int grp = across ? tid & 15 : tid >> 4, d0 = (across ? tid >> 4 : tid & 15) * 8;
    const int r0 = work % kUnits * 16 + z;
    const int r = few ? r0 + grp : r0;
    const int row = it.tile * kRows + r;
    const int rows = it.n * p.group;
    if (it.tile * kRows + r0 >= rows) break;  // uniform
    const int64_t stride = (int64_t)p.kv_heads * part_floats(kRows, kD);
    const float* base = p.part + ((int64_t)it.slot * p.kv_heads + h) * part_floats(kRows, kD);
    float m = -INFINITY, l = 0.f, acc[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = 0.f;
    const int step = few ? 1 : 16;
    for (int i0 = few ? 0 : grp; i0 < it.parts; i0 += 4 * step) {
      // Parts past the last repeat it, with no weight.
      float mi[4], li[4];
      dsa_f32x4 x[4][2];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float* part = base + min(i0 + u * step, it.parts - 1) * stride;
        mi[u] = part[kRows * kD + r];
        li[u] = part[kRows * (kD + 1) + r];
        if (d0 < kD) {
          x[u][0] = *reinterpret_cast<const dsa_f32x4*>(part + part_at<kD, kRows>(r, d0));
          x[u][1] = *reinterpret_cast<const dsa_f32x4*>(part + part_at<kD, kRows>(r, d0 + 4));
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        // (a part no key of which is visible has l 0)
        if (i0 + u * step >= it.parts || li[u] == 0.f) continue;
        const float m_new = fmaxf(m, mi[u]);
        const float a = m == m_new ? 1.f : __builtin_amdgcn_exp2f(m - m_new);
        // (no finite score: l is NaN)
        const float b = mi[u] == -INFINITY ? li[u] : __builtin_amdgcn_exp2f(mi[u] - m_new);
        l = fmaf(l, a, b * li[u]);
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] = fmaf(acc[e], a, b * x[u][e >> 2][e & 3]);
        m = m_new;
      }
    }
    if (few) {
      if (row < rows) {
        const int token = it.q0 + row / p.group, head = h * p.group + row % p.group;
        const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
        if (d0 < p.head_dim) {
          typename dsa::Elem<T>::x8 y;
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = (T)(acc[e] * inv);
          *reinterpret_cast<typename dsa::Elem<T>::x8*>(
              static_cast<T*>(p.o) + (int64_t)token * p.o_st + head * p.o_sh + d0) = y;
        }
        if (p.lse && d0 == 0)
          p.lse[(int64_t)head * p.q_rows + token] = l == 0.f ? -INFINITY : m * kLn2 + logf(l);
      }
      continue;
    }
    if (d0 < kD) {
#pragma unroll
      for (int e = 0; e < 8; ++e) acc_lds[grp][d0 + e] = acc[e];
    }
    if (d0 == 0) {
      ml[0][grp] = m;
      ml[1][grp] = l;
    }
    dsa::lds_barrier();
    if (tid < kD) {
      float m_all = -INFINITY, l_all = 0.f, o = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) m_all = fmaxf(m_all, ml[0][i]);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float w =
            ml[0][i] == -INFINITY ? ml[1][i] : __builtin_amdgcn_exp2f(ml[0][i] - m_all);
        if (w == 0.f) continue;
        l_all = fmaf(w, ml[1][i], l_all);
        o = fmaf(w, acc_lds[i][tid], o);
      }
      const int token = it.q0 + row / p.group, head = h * p.group + row % p.group;
      const float inv = l_all > 0.f ? 1.f / l_all : (l_all == 0.f ? 0.f : l_all);
      if (tid < p.head_dim)
        static_cast<T*>(p.o)[(int64_t)token * p.o_st + head * p.o_sh + tid] = (T)(o * inv);
      if (p.lse && tid == 0)
        p.lse[(int64_t)head * p.q_rows + token] =
            l_all == 0.f ? -INFINITY : m_all * kLn2 + logf(l_all);
    }
    dsa::lds_barrier();
  }
}

}  // namespace seq

// fp16 instances (seq_attn_f16.hip).
int seq_launch_f16(const seq::Params& p, bool paged, bool narrow, int max_groups, bool merge,
                   hipStream_t stream, const char* who);
