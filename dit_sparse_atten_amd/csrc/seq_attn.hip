// Attention of packed sequences and of new tokens over a paged cache: the
// schedule kernel, the bf16 instances and the C-ABI entry points (seq_attn.h
// has the kernels).
#include "seq_launch.h"

namespace seq {

constexpr int kLdsRequests = 1024;  // sequences the schedule keeps in LDS
constexpr int kLdsTiles = 2048;     // tiles whose lengths it keeps there
constexpr int kBuckets = 256;       // item lengths are ordered to 1/256 of the longest
constexpr int kManyParts = 8;       // tiles of more parts are listed by the whole workgroup
// Parts that the longest tile may be cut into, tried on calls of few tiles.
__constant__ const short kTryParts[32] = {1,  2,  3,  4,  5,  6,  7,  8,   9,   10,  11,  12,  14, 16,
                                          18, 20, 24, 28, 32, 40, 48, 56,  64,  80,  96,  112, 128,
                                          160, 192, 256, 384, 512};

// Inclusive sum over the workgroup, `total` for every thread.
template <int kThreads>
__device__ __forceinline__ uint32_t group_scan(uint32_t v, uint32_t* lds, uint32_t* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  v = wave_scan(v);
  dsa::lds_barrier();  // the last scan's reads are done
  if (lane == 63) lds[wave] = v;
  dsa::lds_barrier();
  uint32_t before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < kThreads / 64; ++i) {
    const uint32_t x = lds[i];
    if (i < wave) before += x;
    all += x;
  }
  *total = all;
  return before + v;
}

// Workgroup 0 lists the call's items and split tiles; the others give the rows
// that belong to no sequence their values (O 0 with p.fill, LSE -inf).
//
// kChains (16-row tiles, bound by the reads of their keys): the tiles of a key
// head in a row, each counted as its key steps and a set-up of p.item_cost steps,
// are cut into as many equal ranges as the head has workgroups, and a workgroup
// walks the tiles and parts of one range, its chain.  (A decoding step of 64
// requests of 1,000 to 16,000 tokens: 582 us with parts listed longest first,
// 554 us with chains.)
//
// Else (128-row tiles, bound by their products) the workgroups of the chip (kWideSlots
// at a time) take items in list order, longest first.  Which tiles are cut, in
// key steps, with `work` the steps of all tiles and heads:
//  * up to one round of tiles: every tile longer than `chunk` in near-equal parts
//    of at most that.  Each candidate (the longest tile in 1, 2, 3, .. 512 parts)
//    costs rounds x (mean length + p.item_cost), or its share of the work plus
//    half the longest part if that is more; the cheapest is taken.
//  * more: whole tiles, longest first, even out by themselves but for the last
//    round.  Tiles longer than a slot's share of the work are cut to it; if there
//    are none, the shortest tiles, as many as the last round is short of full,
//    are cut into as many parts as pay.
// Parts cost their partials (p.part_cost).  No choice depends on the order of
// the atomics that place items of nearly equal length.
template <int kThreads, bool kChains>
__global__ void __launch_bounds__(kThreads) seq_schedule_kernel(Params p) {
  const int tid = threadIdx.x;
  if (blockIdx.x > 0) {
    clear_outside(p, blockIdx.x - 1, gridDim.x - 1);
    return;
  }
  __shared__ uint32_t scan_lds[kThreads / 64];
  __shared__ Sequence seq_lds[kLdsRequests];
  __shared__ int base_lds[kLdsRequests + 1];
  __shared__ int tile_steps[kLdsTiles];
  __shared__ int hist[kBuckets];
  __shared__ uint32_t tried[32];
  __shared__ int many[3][kLdsTiles / kManyParts];  // tile, place, slot of the tiles of many parts
  __shared__ int starts[kMaxChains];
  __shared__ unsigned long long work_lds;
  __shared__ int longest_lds, many_count, grouped_lds, ranked, chunk_lds, tail_parts, cut_bucket, cut_left;
  const bool in_lds = p.requests <= kLdsRequests;
  int* const base = in_lds ? base_lds : p.tile_base;
  auto seq_of = [&](int r) -> Sequence { return in_lds ? seq_lds[r] : sequence(p, r); };
  if (tid == 0) {
    work_lds = 0;
    longest_lds = 0;
    many_count = 0;
    grouped_lds = 0;
    ranked = 0;
    tail_parts = 1;
    cut_bucket = kBuckets;
    cut_left = 0;
  }
  if (tid < 32) tried[tid] = 0;
  // Tiles before each sequence.
  uint32_t total = 0;
  uint64_t before = 0;
  for (int r0 = 0; r0 < p.requests; r0 += kThreads) {
    const int r = r0 + tid;
    int count = 0;
    if (r < p.requests) {
      const Sequence s = sequence(p, r);
      if (in_lds) seq_lds[r] = s;
      count = tiles_of(p, s);
    }
    const uint32_t upto = group_scan<kThreads>((uint32_t)count, scan_lds, &total);
    if (r < p.requests) base[r] = (int)min(before + upto - count, (uint64_t)p.max_tiles);
    before += total;
  }
  // (starts that overlap list more tiles than the lists have room for)
  const int tiles = (int)min(before, (uint64_t)p.max_tiles);
  if (tid == 0) base[p.requests] = tiles;
  __syncthreads();
  auto find = [&](int i) -> int {  // the last sequence with base <= i
    int lo = 0, hi = p.requests;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (base[mid] <= i) lo = mid;
      else hi = mid;
    }
    return lo;
  };
  auto length = [&](int i) -> int {
    const int r = find(i);
    return steps_of(p, seq_of(r), i - base[r]);
  };
  auto steps_at = [&](int i) -> int { return i < kLdsTiles ? tile_steps[i] : length(i); };
  // The work, in key steps of one key head, and the longest tile.
  {
    unsigned long long mine = 0;
    int longest = 0;
    for (int i = tid; i < tiles; i += kThreads) {
      const int steps = length(i);
      if (i < kLdsTiles) tile_steps[i] = steps;
      mine += steps;
      longest = max(longest, steps);
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      mine += __shfl_xor(mine, d);
      longest = max(longest, __shfl_xor(longest, d));
    }
    if ((tid & 63) == 0) {
      atomicAdd(&work_lds, mine);
      atomicMax(&longest_lds, longest);
    }
  }
  __syncthreads();
  if constexpr (kChains) {
    // Units of a tile: its set-up, then its steps; chain c holds the units from c
    // quota on.  A tile starts in the chain of its first step.
    const int setup = (int)p.item_cost;
    const uint32_t chains = max(1, kNarrowSlots / p.kv_heads);
    const uint64_t all_units = work_lds + (uint64_t)tiles * setup;
    // From 2^31 units on (2.7e11 keys of one head, set-ups among them): whole tiles, as
    // many to each chain.  (Not 2^32: an item's range is an int, and the last chain's
    // end, up to a quota past the units, still counts in 32 bits.)
    const bool vast = all_units >> 31 != 0;
    const uint32_t units = vast ? (uint32_t)tiles : (uint32_t)all_units;
    const uint32_t quota =
        max((units + chains - 1) / chains, (uint32_t)(vast ? 1 : setup + p.min_chunk));
    const int last_chain = (int)((units + quota - 1) / quota) - 1;
    for (int c = tid; c < kMaxChains; c += kThreads) starts[c] = 0x7fffffff;
    uint32_t items = 0, split_sums = 0, unit_sum = 0;
    for (int i0 = 0; i0 < tiles; i0 += kThreads) {
      const int i = i0 + tid;
      const int steps = i < tiles ? steps_at(i) : 0;
      const uint32_t own = i < tiles ? (vast ? 1u : (uint32_t)(steps + setup)) : 0u;
      const uint32_t from =
          unit_sum + group_scan<kThreads>(own, scan_lds, &total) - own + (vast ? 0 : setup);
      unit_sum += total;
      const int first = min((int)(from / quota), last_chain);
      int parts = i < tiles ? 1 : 0;
      if (steps > 0 && p.max_slots > 0 && !vast)
        parts += min((int)((from + steps - 1) / quota), last_chain) - first;
      const int place = (int)(items + group_scan<kThreads>((uint32_t)parts, scan_lds, &total)) - parts;
      items += total;
      const uint32_t cuts = parts > 1 ? (uint32_t)parts << 16 | 1u : 0u;
      const uint32_t at = split_sums + group_scan<kThreads>(cuts, scan_lds, &total) - cuts;
      split_sums += total;
      if (parts == 0) continue;
      Item it = {};
      it.request = find(i);
      const Sequence s = seq_of(it.request);
      it.q0 = s.q0; it.n = s.n; it.k0 = s.k0; it.m = s.m;
      it.tile = i - base[it.request];
      it.parts = parts;
      const int slot0 = (int)(at >> 16), split0 = (int)(at & 0xffff);
      if (parts > 1 && split0 < p.max_splits) {
        it.slot = slot0;
        p.splits[split0] = it;
      }
      for (int j = 0; j < parts; ++j) {
        it.chain = first + j;
        it.s0 = j == 0 ? 0 : (int)(it.chain * quota - from);
        it.s1 = j + 1 == parts ? steps : (int)((it.chain + 1) * quota - from);
        it.slot = parts > 1 ? slot0 + j : -1;
        if (place + j < p.max_items) {
          p.items[place + j] = it;
          atomicMin(&starts[it.chain], place + j);
        }
      }
    }
    __syncthreads();
    for (int c = tid; c < kMaxChains; c += kThreads) p.chain_start[c] = starts[c];
    if (tid == 0) {
      p.counts[0] = (int)min(items, (uint32_t)p.max_items);
      p.counts[1] = (int)min(split_sums & 0xffff, (uint32_t)p.max_splits);
    }
    return;
  }
  const int longest = longest_lds;
  const int64_t work = (int64_t)work_lds * p.kv_heads, count = (int64_t)tiles * p.kv_heads;
  constexpr int slots = kWideSlots;
  const int whole = max(longest, 1);  // a chunk that cuts nothing
  // Bucket of a length, the longest first (by a multiplication: any monotone map
  // serves).
  auto bucket_of = [](int steps, float per) {
    return (kBuckets - 1) - min(kBuckets - 1, (int)((float)steps * per));
  };
  const float per_whole = (float)(kBuckets - 1) / (float)whole;
  auto bucket = [&](int steps) { return bucket_of(steps, per_whole); };  // of whole tiles
  const int share =
      (int)min(max((work + slots - 1) / slots, (int64_t)p.min_chunk), (int64_t)0x7fffffff);
  if (p.max_slots == 0 || longest < 2 * p.min_chunk || tiles == 0) {
    if (tid == 0) chunk_lds = whole;
  } else if (count <= slots) {
    // Up to a round of tiles: at most `slots` <= kLdsTiles of them.
    const int which = tid & 31;
    const int chunk = max(p.min_chunk, (longest + kTryParts[which] - 1) / kTryParts[which]);
    const float per_chunk = 1.f / (float)chunk;
    uint32_t items = 0;
#pragma unroll 4
    for (int i = tid >> 5; i < tiles; i += kThreads / 32)
      items += parts_in(tile_steps[i], chunk, per_chunk);
    atomicAdd(&tried[which], items);
    __syncthreads();
    if (tid < 64) {
      const uint32_t n = tried[which] * (uint32_t)p.kv_heads;  // (up to 512 parts of 512 tiles)
      const bool cuts = chunk < whole;
      const float cost = p.item_cost + (cuts ? p.part_cost : 0.f);
      const float mean = (float)work / (float)n + cost;
      const float rounds = (float)((n + slots - 1) / slots);  // (slots: a power of two)
      const float even = ((float)work + cost * (float)n) / (float)slots;
      float price = n <= slots ? (float)chunk + cost
                               : fmaxf(rounds * mean, even + 0.5f * ((float)chunk + cost));
      if (cuts) price += p.merge_cost * (float)n;
      if (cuts && tried[which] > (uint32_t)p.max_slots) price = INFINITY;
      int best = which;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const float other = __shfl_xor(price, d);
        const int its = __shfl_xor(best, d);
        if (other < price || (other == price && its < best)) {
          price = other;
          best = its;
        }
      }
      const int taken = __shfl(chunk, best);
      if (tid == 0) chunk_lds = taken;
    }
  } else {
    if (longest > share) {
      if (tid == 0) chunk_lds = share;
    } else {
      // The K shortest tiles fill the last round: found by their bucket, and in
      // the bucket that K ends in by their order.
      const int k = (int)((count % slots + p.kv_heads - 1) / p.kv_heads);
      if (tid < kBuckets) hist[tid] = 0;
      __syncthreads();
      for (int i = tid; i < tiles; i += kThreads) atomicAdd(&hist[bucket(steps_at(i))], 1);
      __syncthreads();
      const uint32_t own = tid < kBuckets ? hist[tid] : 0;
      const uint32_t upto = group_scan<kThreads>(own, scan_lds, &total);
      // (bucket tid holds the ranks upto - own .. upto - 1, longest first: where
      // nothing is cut, the places of its items)
      if (tid < kBuckets) hist[tid] = (int)(upto - own);
      if (tid == kBuckets / 2) grouped_lds = (int)upto;
      if (tid == 0) ranked = 1;
      const int from = tiles - k;  // first rank of the tail
      if (k > 0 && tid < kBuckets && (int)upto > from && (int)(upto - own) <= from) {
        const float steps = (float)(kBuckets - tid) * (float)whole / (float)(kBuckets - 1);
        float best = steps + p.item_cost;
        int parts = 1;
        for (int q = 2; q <= 8; ++q) {
          const uint32_t n = (uint32_t)(k * q * p.kv_heads);  // (k heads: a round and less than one more)
          if (k * q > p.max_slots || steps < (float)(q * p.min_chunk)) break;
          const float price =
              (float)((n + slots - 1) / slots) * (steps / (float)q + p.item_cost + p.part_cost) +
              p.merge_cost * (float)n;
          if (price < best) {
            best = price;
            parts = q;
          }
        }
        tail_parts = parts;
        cut_bucket = tid;
        cut_left = (int)upto - from;  // of this bucket, its first tiles in order
      }
      if (tid == 0) chunk_lds = whole;
    }
  }
  __syncthreads();
  const int chunk = chunk_lds, tail = tail_parts, cut_at = cut_bucket;
  // Parts of tile i; `seen`: tiles of the cut bucket before it.
  auto parts_of = [&](int steps, uint32_t seen) -> int {
    if (tail > 1) {
      const int at = bucket(steps);
      return at > cut_at || (at == cut_at && (int)seen < cut_left) ? tail : 1;
    }
    return max(1, (int)((uint32_t)(steps + chunk - 1) / (uint32_t)chunk));
  };
  // Two sweeps over the tiles in order: the lengths' histogram, then the lists
  // (calls that fit one round need no order).
  const bool sorted = count > slots || chunk < whole;
  const float per_part = (float)(kBuckets - 1) / (float)max(1, min(whole, chunk));
  // (a tail's parts come last of all)
  auto place_bucket = [&](int steps, int parts) {
    const int len = parts == 1 ? steps : (int)((float)(steps + parts - 1) / (float)parts);
    const int at = bucket_of(len, per_part);
    return tail > 1 ? (parts > 1 ? kBuckets - 1 : min(at, kBuckets - 2)) : at;
  };
  const bool cuts = tail > 1 || chunk < whole;
  const bool placed = ranked != 0 && !cuts;  // the histogram is there already
  if (sorted && !placed) {
    if (tid < kBuckets) hist[tid] = 0;
    __syncthreads();
  }
  uint32_t items = placed ? tiles : 0, split_sums = 0;
  for (int sweep = sorted && !placed ? 0 : 1; sweep < 2; ++sweep) {
    uint32_t seen = 0;
    for (int i0 = 0; i0 < tiles; i0 += kThreads) {
      const int i = i0 + tid;
      const int steps = i < tiles ? steps_at(i) : 0;
      uint32_t cut_before = 0;
      if (tail > 1) {
        const uint32_t flag = i < tiles && bucket(steps) == cut_at;
        cut_before = seen + group_scan<kThreads>(flag, scan_lds, &total) - flag;
        seen += total;
      }
      const int parts = i < tiles ? parts_of(steps, cut_before) : 0;
      if (sweep == 0) {
        if (parts > 0) atomicAdd(&hist[place_bucket(steps, parts)], parts);
        continue;
      }
      const bool split = parts > 1;
      int place = 0;
      if (sorted) {
        if (parts > 0) place = atomicAdd(&hist[place_bucket(steps, parts)], parts);
      } else {
        place = (int)(items + group_scan<kThreads>((uint32_t)parts, scan_lds, &total)) - parts;
        items += total;
      }
      // Slots and split tiles in tile order: 16 bits each.
      uint32_t at = 0;
      if (cuts) {
        const uint32_t own = split ? (uint32_t)parts << 16 | 1u : 0u;
        at = split_sums + group_scan<kThreads>(own, scan_lds, &total) - own;
        split_sums += total;
      }
      if (parts == 0) continue;
      Item it = {};
      it.request = find(i);
      const Sequence s = seq_of(it.request);
      it.q0 = s.q0; it.n = s.n; it.k0 = s.k0; it.m = s.m;
      it.tile = i - base[it.request];
      it.parts = parts;
      const int slot0 = (int)(at >> 16), split0 = (int)(at & 0xffff);
      if (split && split0 < p.max_splits) {
        it.slot = slot0;
        p.splits[split0] = it;
      }
      if (parts > kManyParts && i < kLdsTiles) {
        const int n = atomicAdd(&many_count, 1);
        many[0][n] = i; many[1][n] = place; many[2][n] = slot0;
        tile_steps[i] = steps;
        continue;
      }
      const Cut cut(steps, parts);
      for (int j = 0; j < parts; ++j) {
        it.s0 = cut.from(j);
        it.s1 = cut.from(j + 1);
        it.slot = split ? slot0 + j : -1;
        if (place + j < p.max_items) p.items[place + j] = it;
      }
    }
    if (sweep == 0) {
      __syncthreads();
      const uint32_t own = tid < kBuckets ? hist[tid] : 0;
      const uint32_t upto = group_scan<kThreads>(own, scan_lds, &total);
      items = total;
      if (tid < kBuckets) hist[tid] = (int)(upto - own);
      // By head groups: whole tiles before a tail, else those of more than half
      // the longest's length; a call that cuts more evens out as one list.
      const int edge = tail > 1 ? kBuckets - 2 : kBuckets / 2;
      if (tid == edge) grouped_lds = chunk < whole || count <= slots ? 0 : (int)upto;
      __syncthreads();
    }
  }
  if (tid == 0) {
    p.counts[0] = (int)min(items, (uint32_t)p.max_items);
    p.counts[1] = (int)min(split_sums & 0xffff, (uint32_t)p.max_splits);
    p.counts[2] = min(grouped_lds, p.counts[0]);
  }
  __syncthreads();
  for (int n = 0; n < many_count; ++n) {
    const int i = many[0][n], steps = tile_steps[i];
    const int parts = parts_of(steps, 0);  // (tails have at most kManyParts)
    Item it = {};
    it.request = find(i);
    const Sequence s = seq_of(it.request);
    it.q0 = s.q0; it.n = s.n; it.k0 = s.k0; it.m = s.m;
    it.tile = i - base[it.request];
    it.parts = parts;
    const Cut cut(steps, parts);
    for (int j = tid; j < parts; j += kThreads) {
      it.s0 = cut.from(j);
      it.s1 = cut.from(j + 1);
      it.slot = many[2][n] + j;
      if (many[1][n] + j < p.max_items) p.items[many[1][n] + j] = it;
    }
  }
}

namespace {

size_t round256(size_t bytes) { return (bytes + 255) & ~(size_t)255; }

// Shape of a call's schedule, from what the host knows of it.
struct Plan {
  bool narrow, merge, unlisted;
  int tile_rows, step_keys, min_chunk, slots;
  int64_t max_tiles, max_items, max_splits, max_slots;
  size_t counts, chains, base, items, splits, parts, bytes;
};

// Calls of at most 16 rows (tokens x heads of a group) per sequence on average,
// decoding steps, run 16-row tiles.  32 requests of 8,000 tokens, 8 key heads: 8
// and 16 rows 172 us on 16-row tiles and 212 on 128-row ones, 24 and 32 rows (two
// 16-row tiles) 365 and 212 us, 64 rows 716 and 213.
Plan make_plan(int64_t q_rows, int64_t requests, int group, int kv_heads, int head_dim,
               int64_t max_keys) {
  Plan s;
  s.narrow = q_rows * group <= 16 * requests;
  s.tile_rows = s.narrow ? kNarrowRows : kWideRows;
  s.step_keys = s.narrow ? kNarrowKeys : kWideKeys;
  s.slots = s.narrow ? kNarrowSlots : kWideSlots;
  s.min_chunk = s.narrow ? 1 : 2;
  s.max_tiles = std::max<int64_t>(1, q_rows * group / s.tile_rows + requests);
  // Of one key head: no more than 2 `slots` partials over all of them.  Tiles cut
  // at a slot's share of the work keep to that by themselves: each has more than
  // one whole chunk, of which the work of all heads holds `slots`.
  // Few keys are not cut: the join's launch costs what it saves.  Cut against whole,
  // 8 key heads: 16-row tiles of 4 requests, 1,024 keys 15.9 / 13.1 us (the host's
  // time), 1,536 keys 16.0 / 18.2; 128-row tiles of 2 requests, 512 keys 17.5 / 16.9,
  // 768 keys 19.3 / 21.7, 1,536 keys 22.7 / 36.1.
  s.merge = max_keys > (s.narrow ? 1024 : 640) && s.slots >= kv_heads;
  s.max_slots = s.merge ? 2 * s.slots / kv_heads : 0;
  s.max_splits = std::min(s.max_tiles, s.max_slots / 2);
  s.max_items = s.max_tiles + s.max_slots;
  // A call whose tiles all run at once, few enough for the lanes of a wave, works
  // its items out by itself; 128-row tiles of long walks are better listed, for the
  // list may cut them into more than one round of parts.  (16 tiles x 8 key heads,
  // listed against not: 4,096 keys 59 / 54 us, 16,384 keys 146 / 143, 32,768 keys
  // 272 / 294.)
  s.unlisted = requests <= 64 && s.max_tiles <= 64 && s.max_tiles * kv_heads <= s.slots &&
               (s.narrow || s.max_tiles * kv_heads * std::min<int64_t>(max_keys, kMaxKeys) <=
                                80 * (int64_t)s.slots * s.step_keys);
  const int dim = head_dim <= 64 ? 64 : 128;
  s.counts = 0;
  s.chains = 256;
  s.base = s.chains + kMaxChains * sizeof(int32_t);
  s.items = s.base + round256((size_t)(requests + 1) * sizeof(int32_t));
  s.splits = s.items + (size_t)s.max_items * sizeof(Item);
  s.parts = s.splits + round256((size_t)s.max_splits * sizeof(Item));
  s.bytes = s.parts + (size_t)s.max_slots * kv_heads * part_floats(s.tile_rows, dim) * sizeof(float);
  return s;
}

constexpr int64_t kMaxItems = (1 << 21) - 1;

// Checks what both entry points share, lays out the workspace and launches.
int run(Params p, int32_t dtype, bool paged, int64_t max_keys, float scale, void* workspace,
        size_t workspace_bytes, hipStream_t stream, const char* who) {
  const bool keys = paged ? p.pages > 0 && p.table_width > 0 : p.k_rows > 0;
  if (!p.q || !p.o || !p.q_start || (keys && (!p.k || !p.v)))
    return dsa::set_error(DSA_EINVAL, "%s: null pointer", who);
  if (dtype != DSA_BF16 && dtype != DSA_F16)
    return dsa::set_error(DSA_EUNSUPPORTED, "%s: dtype %d (bf16 or fp16)", who, dtype);
  if (p.heads <= 0 || p.kv_heads <= 0 || p.heads % p.kv_heads != 0)
    return dsa::set_error(DSA_EINVAL, "%s: %d heads do not share %d key/value heads", who, p.heads,
                          p.kv_heads);
  if (p.head_dim <= 0 || p.head_dim > 128 || p.head_dim % 8 != 0)
    return dsa::set_error(DSA_EUNSUPPORTED, "%s: head_dim %d (a multiple of 8 up to 128)", who,
                          p.head_dim);
  if (p.requests < 0 || p.q_rows < 0 || p.k_rows < 0)
    return dsa::set_error(DSA_EINVAL, "%s: negative size", who);
  if ((p.causal != 0 && p.causal != 1) || (p.fill != 0 && p.fill != 1))
    return dsa::set_error(DSA_EINVAL, "%s: causal and fill are 0 or 1", who);
  // (the softmax runs in base 2: a scale whose product with log2(e) is infinite would
  // make NaN of a score of 0)
  if (!(scale > 0.f) || scale > 2.3e38f)
    return dsa::set_error(DSA_EINVAL, "%s: scale must be positive and finite, up to 2.3e38", who);
  const int64_t strides[] = {p.q_st, p.q_sh, p.o_st, p.o_sh, p.k_sp, p.k_st, p.k_sh,
                             p.v_sp, p.v_st, p.v_sh};
  for (int64_t s : strides)
    if (s % 8 != 0 || s < 0) return dsa::set_error(DSA_EINVAL, "%s: strides must be multiples of 8", who);
  // 16 staged rows are addressed by 32-bit byte offsets, pages by 32 bits of 16 bytes.
  if (std::max(p.k_st, p.v_st) > (int64_t)1 << 25)
    return dsa::set_error(DSA_EUNSUPPORTED, "%s: token stride above 2^25 elements", who);
  if (p.pages > 1 && std::max(p.k_sp, p.v_sp) >= (int64_t)1 << 35)
    return dsa::set_error(DSA_EUNSUPPORTED, "%s: page stride of 2^35 elements or more", who);
  const void* const pointers[] = {p.q, p.k, p.v, p.o, workspace};
  for (const void* ptr : pointers)
    if (reinterpret_cast<uintptr_t>(ptr) & 15)
      return dsa::set_error(DSA_EINVAL, "%s: pointers must be 16-byte aligned", who);
  p.group = p.heads / p.kv_heads;
  if ((int64_t)p.q_rows * p.group > 0x7fffff00)
    return dsa::set_error(DSA_EUNSUPPORTED, "%s: more than 2^31 query rows per key head", who);
  if (p.q_rows == 0) return DSA_OK;
  const Plan s = make_plan(p.q_rows, p.requests, p.group, p.kv_heads, p.head_dim, max_keys);
  // (a launch counts its threads, 256 for each item and key head, in 32 bits)
  if (s.max_items > kMaxItems || (!s.narrow && s.max_items * p.kv_heads >= 1 << 24))
    return dsa::set_error(DSA_EUNSUPPORTED, "%s: too many query tiles (%lld)", who,
                          (long long)s.max_items);
  if (!workspace || workspace_bytes < s.bytes)
    return dsa::set_error(DSA_EINVAL, "%s: workspace of %zu bytes, %zu needed", who,
                          workspace ? workspace_bytes : (size_t)0, s.bytes);
  unsigned char* const ws = static_cast<unsigned char*>(workspace);
  p.scale_log2 = scale * 1.4426950408889634f;
  p.tile_shift = __builtin_ctz(s.tile_rows);
  p.step_shift = __builtin_ctz(s.step_keys);
  p.min_chunk = s.min_chunk;
  p.slots = s.slots;
  auto shares = [](const void* at, int64_t head_stride) {
    return head_stride % 64 != 0 || (reinterpret_cast<uintptr_t>(at) & 127) != 0;
  };
  p.shared_lines = s.narrow && p.kv_heads > 1 && (shares(p.k, p.k_sh) || shares(p.v, p.v_sh));
  p.max_tiles = (int32_t)s.max_tiles;
  p.max_items = (int32_t)s.max_items;
  p.max_splits = (int32_t)s.max_splits;
  p.max_slots = (int32_t)s.max_slots;
  // In key steps: what an item costs beside its keys, what a partial adds, and
  // its share of the join.
  p.item_cost = 2.0f;
  p.part_cost = s.narrow ? 0.25f : 2.5f;
  p.merge_cost = s.narrow ? 0.0005f : 0.011f;
  p.counts = reinterpret_cast<int32_t*>(ws + s.counts);
  p.chain_start = reinterpret_cast<int32_t*>(ws + s.chains);
  p.tile_base = reinterpret_cast<int32_t*>(ws + s.base);
  p.items = reinterpret_cast<Item*>(ws + s.items);
  p.splits = reinterpret_cast<Item*>(ws + s.splits);
  p.part = reinterpret_cast<float*>(ws + s.parts);
  dsa::clear_error();
  p.unlisted = s.unlisted;
  // Workgroups for the rows outside every sequence, beside those with items.
  const int outside =
      p.fill || p.lse ? (int)std::min<int64_t>(64, (p.q_rows + 3) / 4) : 0;
  int groups = (int)(s.max_items * p.kv_heads);
  if (s.unlisted) {
    groups = (s.merge ? s.slots : (int)s.max_tiles * p.kv_heads) + outside;
  } else {
    const bool small = s.max_tiles <= 512 && p.requests <= 512;
    const dim3 lists((unsigned)(1 + outside)), threads(small ? 256 : 1024);
    auto schedule = [&](auto kernel) { hipLaunchKernelGGL(kernel, lists, threads, 0, stream, p); };
    if (s.narrow) {
      groups = std::max(1, kNarrowSlots / p.kv_heads) * p.kv_heads;
      small ? schedule(seq_schedule_kernel<256, true>) : schedule(seq_schedule_kernel<1024, true>);
    } else {
      small ? schedule(seq_schedule_kernel<256, false>) : schedule(seq_schedule_kernel<1024, false>);
    }
  }
  return dtype == DSA_BF16
             ? launch_typed<__bf16>(p, paged, s.narrow, groups, s.merge, stream, who)
             : seq_launch_f16(p, paged, s.narrow, groups, s.merge, stream, who);
}

}  // namespace
}  // namespace seq

extern "C" size_t dsa_seq_attention_workspace_bytes(int32_t q_rows, int32_t requests, int32_t heads,
                                                    int32_t kv_heads, int32_t head_dim,
                                                    int64_t max_keys) {
  if (q_rows <= 0 || requests < 0 || kv_heads <= 0 || heads <= 0 || heads % kv_heads != 0 ||
      head_dim <= 0 || max_keys < 0)
    return 0;
  return seq::make_plan(q_rows, requests, heads / kv_heads, kv_heads, head_dim, max_keys).bytes;
}

extern "C" int dsa_packed_attention(const void* q, const void* k, const void* v, void* o,
                                    int32_t dtype, const int64_t* strides, int32_t q_rows,
                                    int32_t k_rows, int32_t requests, int32_t heads,
                                    int32_t kv_heads, int32_t head_dim, const int32_t* q_start,
                                    const int32_t* k_start, float scale, int32_t causal,
                                    int32_t fill, float* lse, void* workspace,
                                    size_t workspace_bytes, hipStream_t stream) {
  if (!strides) return dsa::set_error(DSA_EINVAL, "dsa_packed_attention: null strides");
  seq::Params p = {};
  p.q = q; p.k = k; p.v = v; p.o = o; p.lse = lse;
  p.q_st = strides[0]; p.q_sh = strides[1];
  p.k_st = strides[2]; p.k_sh = strides[3];
  p.v_st = strides[4]; p.v_sh = strides[5];
  p.o_st = strides[6]; p.o_sh = strides[7];
  p.q_start = q_start;
  p.k_start = k_start ? k_start : q_start;
  p.q_rows = q_rows; p.k_rows = k_rows; p.requests = requests;
  p.heads = heads; p.kv_heads = kv_heads; p.head_dim = head_dim;
  p.causal = causal; p.fill = fill;
  return seq::run(p, dtype, false, k_rows, scale, workspace, workspace_bytes, stream,
                  "dsa_packed_attention");
}

extern "C" int dsa_paged_attention(const void* q, const void* k_cache, const void* v_cache, void* o,
                                   int32_t dtype, const int64_t* strides, int32_t q_rows,
                                   int32_t requests, int32_t heads, int32_t kv_heads,
                                   int32_t head_dim, int32_t pages, int32_t page_size,
                                   const int32_t* table, int64_t table_stride, int32_t table_width,
                                   const int32_t* kv_lens, const int32_t* q_start, float scale,
                                   int32_t causal, int32_t fill, float* lse, void* workspace,
                                   size_t workspace_bytes, hipStream_t stream) {
  const char* const who = "dsa_paged_attention";
  if (!strides) return dsa::set_error(DSA_EINVAL, "%s: null strides", who);
  if (page_size < 16 || (page_size & (page_size - 1)) != 0)
    return dsa::set_error(DSA_EUNSUPPORTED, "%s: page_size %d (a power of two from 16)", who,
                          page_size);
  if (pages < 0 || table_width < 0 || table_stride < table_width)
    return dsa::set_error(DSA_EINVAL, "%s: bad table or page count", who);
  if (requests > 0 && (!kv_lens || (!table && table_width > 0)))
    return dsa::set_error(DSA_EINVAL, "%s: null block table or lengths", who);
  const int64_t max_keys = (int64_t)table_width * page_size;
  seq::Params p = {};
  p.q = q; p.k = k_cache; p.v = v_cache; p.o = o; p.lse = lse;
  p.q_st = strides[0]; p.q_sh = strides[1];
  p.k_sp = strides[2]; p.k_st = strides[3]; p.k_sh = strides[4];
  p.v_sp = strides[5]; p.v_st = strides[6]; p.v_sh = strides[7];
  p.o_st = strides[8]; p.o_sh = strides[9];
  p.q_start = q_start; p.kv_lens = kv_lens;
  p.table = table; p.table_stride = table_stride; p.table_width = table_width;
  p.pages = pages; p.page_shift = __builtin_ctz(page_size);
  p.q_rows = q_rows; p.requests = requests;
  p.heads = heads; p.kv_heads = kv_heads; p.head_dim = head_dim;
  p.causal = causal; p.fill = fill;
  return seq::run(p, dtype, true, max_keys, scale, workspace, workspace_bytes, stream, who);
}
