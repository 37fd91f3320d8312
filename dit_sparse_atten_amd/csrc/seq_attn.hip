// Attention of packed sequences and of new tokens over a paged cache: the
// schedule kernel, the bf16 instances and the C-ABI entry points (seq_attn.h
// has the kernels).
#include "seq_launch.h"

namespace seq {

constexpr int kScheduleThreads = 1024;
constexpr int kLdsRequests = 4096;  // sequences whose tile counts the schedule keeps in LDS
constexpr int kBuckets = 256;       // item lengths are ordered to 1/256 of the longest

// Inclusive sum over the workgroup, `total` for every thread.  `lds` holds 16.
__device__ __forceinline__ uint64_t group_scan(uint64_t v, uint64_t* lds, uint64_t* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint64_t other = (uint64_t)__shfl_up((unsigned long long)v, d);
    if (lane >= d) v += other;
  }
  dsa::lds_barrier();  // the last scan's reads are done
  if (lane == 63) lds[wave] = v;
  dsa::lds_barrier();
  uint64_t before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < kScheduleThreads / 64; ++i) {
    if (i < wave) before += lds[i];
    all += lds[i];
  }
  *total = all;
  return before + v;
}

struct Sequence {
  int32_t q0, n, k0, m;
};

// Sequence r, whatever the arrays hold: rows and keys within the tensors.
__device__ __forceinline__ Sequence sequence(const Params& p, int r) {
  Sequence s;
  s.q0 = min(max(p.q_start[r], 0), p.q_rows);
  s.n = min(max(p.q_start[r + 1], s.q0), p.q_rows) - s.q0;
  if (p.kv_lens) {
    s.k0 = 0;
    const int64_t room = (int64_t)p.table_width << p.page_shift;
    s.m = (int32_t)min((int64_t)max(p.kv_lens[r], 0), room);
  } else {
    s.k0 = min(max(p.k_start[r], 0), p.k_rows);
    s.m = min(max(p.k_start[r + 1], s.k0), p.k_rows) - s.k0;
  }
  return s;
}

__device__ __forceinline__ int tiles_of(const Params& p, const Sequence& s) {
  return (s.n * p.group + p.tile_rows - 1) / p.tile_rows;
}

// Key steps of a tile: up to the last key its last row sees.
__device__ __forceinline__ int steps_of(const Params& p, const Sequence& s, int tile) {
  int end = s.m;
  if (p.causal) {
    const int last = min((tile + 1) * p.tile_rows, s.n * p.group) - 1;
    end = max(0, min(s.m, s.m - s.n + last / p.group + 1));
  }
  return (end + p.step_keys - 1) / p.step_keys;
}

// Workgroup 0 lists the call's items and split tiles; the others give the rows
// that belong to no sequence their values (O 0 with p.fill, LSE -inf).  Parts: a tile longer than `chunk` steps
// is cut into near-equal parts of at most that, with chunk = the whole work /
// p.target, so that `target` workgroups share it evenly.  A call of more items
// than that is ordered longest first, by a counting sort of the lengths (the
// order inside a bucket is that of the atomics; no result depends on it).
__global__ void __launch_bounds__(kScheduleThreads) seq_schedule_kernel(Params p, int esize) {
  const int tid = threadIdx.x;
  if (blockIdx.x > 0) {
    const int first = min(max(p.q_start[0], 0), p.q_rows);
    const int last = min(max(p.q_start[p.requests], first), p.q_rows);
    const int chunks = p.head_dim / 8 * p.heads;  // 16-byte chunks of a row
    const int empty = first + p.q_rows - last;
    const dsa_u32x4 zero = {0u, 0u, 0u, 0u};
    for (int i = blockIdx.x - 1; i < empty; i += gridDim.x - 1) {
      const int row = i < first ? i : last + i - first;
      for (int c = tid; p.fill && c < chunks; c += kScheduleThreads) {
        const int head = c / (p.head_dim / 8), d = c % (p.head_dim / 8) * 8;
        *reinterpret_cast<dsa_u32x4*>(static_cast<unsigned char*>(p.o) +
                                      ((int64_t)row * p.o_st + head * p.o_sh + d) * esize) = zero;
      }
      if (p.lse)
        for (int head = tid; head < p.heads; head += kScheduleThreads)
          p.lse[(int64_t)head * p.q_rows + row] = -INFINITY;
    }
    return;
  }
  __shared__ uint64_t scan_lds[kScheduleThreads / 64];
  __shared__ int base_lds[kLdsRequests + 1];
  __shared__ int hist[kBuckets];
  __shared__ unsigned long long work_lds;
  __shared__ int longest_lds;
  int* const base = p.requests <= kLdsRequests ? base_lds : p.tile_base;
  if (tid == 0) {
    work_lds = 0;
    longest_lds = 0;
  }
  // Tiles before each sequence.
  uint64_t total = 0, before = 0;
  for (int r0 = 0; r0 < p.requests; r0 += kScheduleThreads) {
    const int r = r0 + tid;
    const int tiles = r < p.requests ? tiles_of(p, sequence(p, r)) : 0;
    const uint64_t upto = group_scan((uint64_t)tiles, scan_lds, &total);
    if (r < p.requests) base[r] = (int)(before + upto - tiles);
    before += total;
  }
  // (starts that overlap list more tiles than the lists have room for)
  const int tiles = (int)min(before, (uint64_t)p.max_items);
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
  // The work, in key steps of one key head, and the longest tile.
  uint64_t mine = 0;
  int longest = 0;
  for (int i = tid; i < tiles; i += kScheduleThreads) {
    const int r = find(i);
    const int steps = steps_of(p, sequence(p, r), i - base[r]);
    mine += steps;
    longest = max(longest, steps);
  }
  atomicAdd(&work_lds, (unsigned long long)mine);
  atomicMax(&longest_lds, longest);
  __syncthreads();
  const uint64_t work = work_lds * (uint64_t)p.kv_heads;
  const int chunk =
      (int)max((work + p.target - 1) / (uint64_t)p.target, (uint64_t)p.min_chunk);
  const int longest_part = min(longest_lds, chunk);
  auto parts_of = [&](int steps) { return max(1, (steps + chunk - 1) / chunk); };
  // Calls of more than one round of workgroups list the longest first.
  const bool sorted = (int64_t)tiles * p.kv_heads > p.target;
  auto bucket = [&](int length) {
    return longest_part > 0 ? (kBuckets - 1) - (int)((int64_t)length * (kBuckets - 1) / longest_part)
                            : 0;
  };
  if (sorted) {
    if (tid < kBuckets) hist[tid] = 0;
    __syncthreads();
    for (int i = tid; i < tiles; i += kScheduleThreads) {
      const int r = find(i);
      const int steps = steps_of(p, sequence(p, r), i - base[r]);
      const int parts = parts_of(steps);
      atomicAdd(&hist[bucket((steps + parts - 1) / parts)], parts);
    }
    __syncthreads();
    const int count = tid < kBuckets ? hist[tid] : 0;
    const uint64_t upto = group_scan((uint64_t)count, scan_lds, &total);
    __syncthreads();
    if (tid < kBuckets) hist[tid] = (int)upto - count;
    __syncthreads();
  }
  // Items, split tiles and partial slots, in tile order: 21 bits each.
  uint64_t sums = 0;
  for (int i0 = 0; i0 < tiles; i0 += kScheduleThreads) {
    const int i = i0 + tid;
    Item it = {};
    int steps = 0, parts = 0;
    if (i < tiles) {
      it.request = find(i);
      const Sequence s = sequence(p, it.request);
      it.q0 = s.q0; it.n = s.n; it.k0 = s.k0; it.m = s.m;
      it.tile = i - base[it.request];
      steps = steps_of(p, s, it.tile);
      parts = parts_of(steps);
    }
    const bool split = parts > 1;
    const uint64_t own = (uint64_t)parts | (uint64_t)(split ? parts : 0) << 21 |
                         (uint64_t)(split ? 1 : 0) << 42;
    const uint64_t at = sums + group_scan(own, scan_lds, &total) - own;
    sums += total;
    const int item0 = (int)(at & 0x1fffff), slot0 = (int)(at >> 21 & 0x1fffff),
              split0 = (int)(at >> 42);
    it.parts = parts;
    if (split && split0 < p.max_splits) {
      it.slot = slot0;
      p.splits[split0] = it;
    }
    const int place = sorted && parts > 0
                          ? atomicAdd(&hist[bucket((steps + parts - 1) / parts)], parts)
                          : item0;
    for (int j = 0; j < parts; ++j) {
      it.s0 = (int)((int64_t)steps * j / parts);
      it.s1 = (int)((int64_t)steps * (j + 1) / parts);
      it.slot = split ? slot0 + j : -1;
      if (place + j < p.max_items) p.items[place + j] = it;
    }
  }
  if (tid == 0) {
    p.counts[0] = (int)min(sums & 0x1fffff, (uint64_t)p.max_items);
    p.counts[1] = (int)min(sums >> 42, (uint64_t)p.max_splits);
  }
}

namespace {

size_t round256(size_t bytes) { return (bytes + 255) & ~(size_t)255; }

// Shape of a call's schedule, from what the host knows of it.
struct Plan {
  bool narrow, merge;
  int tile_rows, step_keys, min_chunk, target;
  int64_t max_items, max_splits, max_slots;
  size_t counts, base, items, splits, parts, bytes;
};

// Few rows per sequence (decoding steps) run 16-row tiles.
Plan make_plan(int64_t q_rows, int64_t requests, int group, int kv_heads, int head_dim,
               int64_t max_keys) {
  Plan s;
  s.narrow = q_rows * group <= 16 * requests;
  s.tile_rows = s.narrow ? kNarrowRows : kWideRows;
  s.step_keys = s.narrow ? kNarrowKeys : kWideKeys;
  s.target = s.narrow ? 256 : 512;
  s.min_chunk = s.narrow ? 2 : 4;
  const int64_t tiles = q_rows * group / s.tile_rows + requests;
  // Every part but a tile's last is a whole chunk, of which the work of all key
  // heads holds at most `target`; a split tile has at least one whole chunk.
  const int64_t chunks = s.target / kv_heads;
  s.merge = max_keys > (int64_t)s.min_chunk * s.step_keys && chunks > 0;
  s.max_items = std::max<int64_t>(1, tiles + (s.merge ? chunks : 0));
  s.max_splits = s.merge ? std::min(tiles, chunks) : 0;
  s.max_slots = s.merge ? 2 * s.target / kv_heads : 0;
  const int dim = head_dim <= 64 ? 64 : 128;
  s.counts = 0;
  s.base = 256;
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
  if (!(scale > 0.f) || scale > 3e38f)
    return dsa::set_error(DSA_EINVAL, "%s: scale must be positive and finite", who);
  const int64_t strides[] = {p.q_st, p.q_sh, p.o_st, p.o_sh, p.k_sp, p.k_st, p.k_sh,
                             p.v_sp, p.v_st, p.v_sh};
  for (int64_t s : strides)
    if (s % 8 != 0 || s < 0) return dsa::set_error(DSA_EINVAL, "%s: strides must be multiples of 8", who);
  // 16 staged rows are addressed by 32-bit byte offsets.
  if (std::max(p.k_st, p.v_st) > (int64_t)1 << 25)
    return dsa::set_error(DSA_EUNSUPPORTED, "%s: token stride above 2^25 elements", who);
  const void* const pointers[] = {p.q, p.k, p.v, p.o, workspace};
  for (const void* ptr : pointers)
    if (reinterpret_cast<uintptr_t>(ptr) & 15)
      return dsa::set_error(DSA_EINVAL, "%s: pointers must be 16-byte aligned", who);
  p.group = p.heads / p.kv_heads;
  if ((int64_t)p.q_rows * p.group > 0x7fffff00)
    return dsa::set_error(DSA_EUNSUPPORTED, "%s: more than 2^31 query rows per key head", who);
  if (p.q_rows == 0) return DSA_OK;
  const Plan s = make_plan(p.q_rows, p.requests, p.group, p.kv_heads, p.head_dim, max_keys);
  if (s.max_items > kMaxItems || s.max_items * p.kv_heads > 0x7fffffff)
    return dsa::set_error(DSA_EUNSUPPORTED, "%s: too many query tiles (%lld)", who,
                          (long long)s.max_items);
  if (!workspace || workspace_bytes < s.bytes)
    return dsa::set_error(DSA_EINVAL, "%s: workspace of %zu bytes, %zu needed", who,
                          workspace ? workspace_bytes : (size_t)0, s.bytes);
  unsigned char* const ws = static_cast<unsigned char*>(workspace);
  p.scale_log2 = scale * 1.4426950408889634f;
  p.tile_rows = s.tile_rows;
  p.step_keys = s.step_keys;
  p.min_chunk = s.merge ? s.min_chunk : 0x7fffffff;
  p.target = s.target;
  p.max_items = (int32_t)s.max_items;
  p.max_splits = (int32_t)s.max_splits;
  p.max_slots = (int32_t)s.max_slots;
  p.counts = reinterpret_cast<int32_t*>(ws + s.counts);
  p.tile_base = reinterpret_cast<int32_t*>(ws + s.base);
  p.items = reinterpret_cast<Item*>(ws + s.items);
  p.splits = reinterpret_cast<Item*>(ws + s.splits);
  p.part = reinterpret_cast<float*>(ws + s.parts);
  dsa::clear_error();
  hipLaunchKernelGGL(seq_schedule_kernel, dim3(p.fill || p.lse ? 65 : 1), dim3(kScheduleThreads), 0, stream,
                     p, 2);
  const int groups = (int)(s.max_items * p.kv_heads);
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
  if (!kv_lens || (!table && table_width > 0))
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
