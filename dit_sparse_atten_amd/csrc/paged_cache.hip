// Book-keeping of a paged key/value cache (gfx950): the plan of a step (where
// every new token goes) and the write of its keys and values.
#include <algorithm>

#include "dsa_common.h"

namespace {

constexpr int kThreads = 512;
constexpr int kMaxRequests = 8192;  // two prefix arrays of a call in LDS: 64 KB

struct PlanParams {
  const int32_t* cached;
  const int32_t* fresh;
  int32_t* table;
  const int32_t* free_pages;
  const int32_t* free_start;  // pages of the list given out before, or null
  int32_t* q_start;
  int32_t* kv_lens;
  int64_t* slots;
  int32_t* status;
  int64_t table_stride;
  int32_t requests, table_width, free_count, page_shift, tokens;
};

__device__ __forceinline__ int pages_for(int64_t tokens, int shift) {
  return (int)((tokens + (1 << shift) - 1) >> shift);
}

// Pages request r holds before the step and after it (of at most table_width).
struct Need {
  int cached, fresh, held, want;
};
__device__ __forceinline__ Need need_of(const PlanParams& p, int r) {
  Need n;
  n.cached = max(p.cached[r], 0);
  // (lengths past 2^31 tokens in all are cut there)
  n.fresh = min(max(p.fresh[r], 0), 0x7fffffff - n.cached);
  n.held = min(pages_for(n.cached, p.page_shift), p.table_width);
  n.want = min(pages_for((int64_t)n.cached + n.fresh, p.page_shift), p.table_width);
  return n;
}

// Latency-bound: a few hundred lengths in, a slot per token out.  Every
// workgroup scans all lengths into LDS (token starts and, of the free list, page
// starts), so none waits for another, then fills its share of the slots and of
// the new table entries, finding each one's request by bisection; workgroup 0
// also writes the starts, lengths and status.  A slot of a token's page comes
// from the table where the page was held before and from the free list where it
// is new, so no workgroup reads what another writes.
__global__ void __launch_bounds__(kThreads) paged_plan_kernel(PlanParams p) {
  __shared__ int start[kMaxRequests + 1];  // tokens before each request
  __shared__ int first[kMaxRequests + 1];  // new pages before each request
  __shared__ int wave_sum[2][kThreads / 64];
  __shared__ unsigned long long lost_lds;  // tokens without a slot
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const bool lead = blockIdx.x == 0;
  // What is left of the free list (a count that leaves it, negative ones of a sum past
  // 2^31 among them: nothing).
  int given = p.free_start ? p.free_start[0] : 0;
  if (given < 0) given = p.free_count;
  given = min(given, p.free_count);
  const int32_t* const free_pages = p.free_pages + given;
  const int free_count = p.free_count - given;
  if (tid == 0) lost_lds = 0;
  int tokens = 0, pages = 0;  // before these requests
  for (int r0 = 0; r0 < p.requests; r0 += kThreads) {
    const int r = r0 + tid;
    Need n = {0, 0, 0, 0};
    if (r < p.requests) n = need_of(p, r);
    // The page that the first new tokens share with cached ones, as the table has it
    // (no page: a step that ran out of pages left it so).
    const int partial = n.cached & ((1 << p.page_shift) - 1);
    const bool shares = lead && n.fresh > 0 && partial != 0 &&
                        (n.cached >> p.page_shift) < n.held;
    const int shared =
        shares ? p.table[r * p.table_stride + (n.cached >> p.page_shift)] : 0;
    int a = n.fresh, b = n.want - n.held;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int ua = __shfl_up(a, d), ub = __shfl_up(b, d);
      if (lane >= d) {
        a = (int)min((int64_t)a + ua, (int64_t)0x7fffffff);
        b = (int)min((int64_t)b + ub, (int64_t)0x7fffffff);
      }
    }
    dsa::lds_barrier();
    if (lane == 63) {
      wave_sum[0][wave] = a;
      wave_sum[1][wave] = b;
    }
    dsa::lds_barrier();
    int64_t before_a = tokens, before_b = pages, all_a = tokens, all_b = pages;
#pragma unroll
    for (int i = 0; i < kThreads / 64; ++i) {
      if (i < wave) {
        before_a += wave_sum[0][i];
        before_b += wave_sum[1][i];
      }
      all_a += wave_sum[0][i];
      all_b += wave_sum[1][i];
    }
    const int64_t top = 0x7fffffff;
    const int upto_a = (int)min(before_a + a, top), upto_b = (int)min(before_b + b, top);
    const int ahead = __shfl_up(a, 1);
    const int64_t from_a = min(before_a + (lane > 0 ? ahead : 0), top);
    if (r < p.requests) {
      start[r + 1] = upto_a;
      first[r + 1] = upto_b;
      if (lead) {
        p.q_start[r + 1] = upto_a;
        p.kv_lens[r] = n.cached + n.fresh;
        // Lost at the end: tokens past the last page the request got, or behind the
        // slot map; at the start: those in a shared page that is none.
        const int from = upto_b - (n.want - n.held);
        const int granted = max(0, min(free_count - from, n.want - n.held));
        const int64_t fresh = n.fresh, cached = n.cached;
        const int64_t room = (int64_t)(n.held + granted) << p.page_shift;
        const int64_t past = cached + fresh - max(room, cached);
        const int64_t behind = fresh - min(max(p.tokens - from_a, (int64_t)0), fresh);
        const int64_t head = shared < 0 ? (1 << p.page_shift) - partial : 0;
        const int64_t lost = min(max(past, behind) + head, fresh);
        if (lost > 0) atomicAdd(&lost_lds, (unsigned long long)lost);
      }
    }
    tokens = (int)min(all_a, top);
    pages = (int)min(all_b, top);
  }
  if (tid == 0) {
    start[0] = 0;
    first[0] = 0;
  }
  dsa::lds_barrier();
  auto find = [&](const int* before, int i) -> int {  // the last request with before <= i
    int lo = 0, hi = p.requests;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (before[mid] <= i) lo = mid;
      else hi = mid;
    }
    return lo;
  };
  if (lead) {
    // Tokens whose page would be an entry of the free list that is none.
    const int granted = min(pages, free_count);
    for (int i = tid; i < granted; i += kThreads) {
      if (free_pages[i] >= 0) continue;
      const int r = find(first, i);
      const Need n = need_of(p, r);
      const int64_t begin = (int64_t)(n.held + (i - first[r])) << p.page_shift;
      const int64_t upto = n.cached + min((int64_t)n.fresh, max(p.tokens - (int64_t)start[r],
                                                                (int64_t)0));
      const int64_t lost = min(begin + (1 << p.page_shift), upto) - max(begin, (int64_t)n.cached);
      if (lost > 0) atomicAdd(&lost_lds, (unsigned long long)lost);
    }
    dsa::lds_barrier();
    if (tid == 0) {
      p.q_start[0] = 0;
      p.status[0] = pages;
      p.status[1] = (int)min(lost_lds, 0x7fffffffull);
    }
  }
  const int at = blockIdx.x * kThreads + tid, all = gridDim.x * kThreads;
  const int mask = (1 << p.page_shift) - 1;
  for (int64_t t = at; t < p.tokens; t += all) {
    int64_t slot = -1;
    if (t < tokens) {
      const int r = find(start, (int)t);
      const Need n = need_of(p, r);
      const int64_t position = (int64_t)n.cached + (t - start[r]);
      const int64_t index = position >> p.page_shift;
      int page = -1;
      if (index < n.held) {
        page = p.table[r * p.table_stride + index];
      } else if (index < n.want) {
        const int64_t from = first[r] + index - n.held;
        if (from < free_count) page = free_pages[from];
      }
      if (page >= 0) slot = ((int64_t)page << p.page_shift) + (position & mask);
    }
    p.slots[t] = slot;
  }
  for (int64_t i = at; i < pages; i += all) {
    const int r = find(first, (int)i);
    const Need n = need_of(p, r);
    const int64_t index = n.held + (i - first[r]);
    if (index < n.want)
      p.table[r * p.table_stride + index] = i < free_count ? free_pages[i] : -1;
  }
}

struct WriteParams {
  const unsigned char* src[2];  // k, v
  unsigned char* dst[2];        // k_cache, v_cache
  int64_t src_st[2], src_sh[2];               // bytes
  int64_t dst_sp[2], dst_st[2], dst_sh[2];
  const int64_t* slots;
  int64_t total;                   // slots of the cache
  int32_t tokens, row, chunks;     // 16-byte chunks per token of one tensor, per head
  uint32_t row_magic, chunk_magic; // of quotient() by row and by chunks
  int32_t group_tokens;            // tokens of a workgroup
  int32_t page_shift;
};

// i / d by a multiplication, exact for 1 <= d < 2^15 and i < 2^15: the magic is
// (2^31 + e) / d with e < d, so i magic / 2^31 exceeds i / d by i e / (d 2^31) < 1 / d,
// which reaches no further quotient.  (2^32 in its place would leave 32 bits at d = 1.)
uint32_t quotient_magic(uint32_t d) { return (uint32_t)(((1ull << 31) + d - 1) / d); }
__device__ __forceinline__ uint32_t quotient(uint32_t i, uint32_t magic) {
  return __umulhi(2 * i, magic);
}

// Moves 16 bytes per thread and turn, bound by memory on long calls.  A workgroup
// takes `group_tokens` tokens of one tensor (y), their chunks to consecutive
// threads; every thread has all its loads on their way before its first store.
// 57,600 tokens x 12 heads x 128 (708 MB): 137 us, 5.2 TB/s, against 198 us with
// 64-bit indexes and four turns; a plain copy of as much takes 126 us, one past the
// caches 109.  Rows are read once (non-temporal) but stored through the caches, where
// the attention that follows finds them: with non-temporal stores the write alone took
// 130 us, but 131,072 tokens x 8 heads with a decoding step behind them 327 us against
// 299.
// Indexes are divided by quotient(): a workgroup has fewer than 2^15 chunks.
constexpr int kWriteTurns = 8;
constexpr int kWriteChunks = 256 * kWriteTurns;  // at most, of a workgroup
__global__ void __launch_bounds__(256) paged_write_kernel(WriteParams p) {
  const int which = blockIdx.y;
  const int first = blockIdx.x * p.group_tokens;
  const uint32_t count = (uint32_t)min(p.group_tokens, p.tokens - first) * (uint32_t)p.row;
  const unsigned char* const src = p.src[which];
  for (uint32_t i0 = threadIdx.x; i0 < count; i0 += kWriteChunks) {
    dsa_u32x4 x[kWriteTurns];
    int64_t slot[kWriteTurns];
    uint32_t head[kWriteTurns], at[kWriteTurns];
#pragma unroll
    for (int u = 0; u < kWriteTurns; ++u) {
      const uint32_t i = i0 + u * 256;
      slot[u] = -1;
      if (i >= count) continue;
      const uint32_t t = quotient(i, p.row_magic), c = i - t * p.row;
      head[u] = quotient(c, p.chunk_magic);
      at[u] = (c - head[u] * p.chunks) * 16;
      slot[u] = p.slots[first + t];
      x[u] = __builtin_nontemporal_load(reinterpret_cast<const dsa_u32x4*>(
          src + (int64_t)(first + t) * p.src_st[which] + head[u] * p.src_sh[which] + at[u]));
    }
#pragma unroll
    for (int u = 0; u < kWriteTurns; ++u) {
      if (slot[u] < 0 || slot[u] >= p.total) continue;
      const int64_t page = slot[u] >> p.page_shift, row = slot[u] & ((1 << p.page_shift) - 1);
      *reinterpret_cast<dsa_u32x4*>(p.dst[which] + page * p.dst_sp[which] +
                                    row * p.dst_st[which] + head[u] * p.dst_sh[which] + at[u]) =
          x[u];
    }
  }
}

bool bad_page_size(int32_t size) { return size < 16 || (size & (size - 1)) != 0; }

}  // namespace

extern "C" int dsa_paged_plan(const int32_t* cached, const int32_t* fresh, int32_t requests,
                              int32_t* table, int64_t table_stride, int32_t table_width,
                              const int32_t* free_pages, int32_t free_count, int32_t page_size,
                              int32_t tokens, int32_t* q_start, int32_t* kv_lens, int64_t* slots,
                              int32_t* status, hipStream_t stream) {
  return dsa_paged_plan_from(cached, fresh, requests, table, table_stride, table_width, free_pages,
                             free_count, nullptr, page_size, tokens, q_start, kv_lens, slots,
                             status, stream);
}

extern "C" int dsa_paged_plan_from(const int32_t* cached, const int32_t* fresh, int32_t requests,
                                   int32_t* table, int64_t table_stride, int32_t table_width,
                                   const int32_t* free_pages, int32_t free_count,
                                   const int32_t* free_start, int32_t page_size, int32_t tokens,
                                   int32_t* q_start, int32_t* kv_lens, int64_t* slots,
                                   int32_t* status, hipStream_t stream) {
  const char* const who = "dsa_paged_plan";
  if (requests < 0 || tokens < 0 || free_count < 0 || table_width < 0 || table_stride < table_width)
    return dsa::set_error(DSA_EINVAL, "%s: negative size or table rows that overlap", who);
  if (!q_start || !status || (requests > 0 && (!cached || !fresh || !kv_lens)) ||
      (tokens > 0 && !slots) || (free_count > 0 && !free_pages) ||
      (requests > 0 && table_width > 0 && !table))
    return dsa::set_error(DSA_EINVAL, "%s: null pointer", who);
  if (requests > kMaxRequests)
    return dsa::set_error(DSA_EUNSUPPORTED, "%s: %d requests (up to %d)", who, requests,
                          kMaxRequests);
  if (bad_page_size(page_size))
    return dsa::set_error(DSA_EUNSUPPORTED, "%s: page_size %d (a power of two from 16)", who,
                          page_size);
  PlanParams p;
  p.cached = cached; p.fresh = fresh; p.table = table; p.free_pages = free_pages;
  p.free_start = free_start;
  p.q_start = q_start; p.kv_lens = kv_lens; p.slots = slots; p.status = status;
  p.table_stride = table_stride;
  p.requests = requests; p.table_width = table_width; p.free_count = free_count;
  p.page_shift = __builtin_ctz(page_size);
  p.tokens = tokens;
  dsa::clear_error();
  const int64_t groups = ((int64_t)tokens + kThreads - 1) / kThreads;
  hipLaunchKernelGGL(paged_plan_kernel, dim3((unsigned)std::clamp<int64_t>(groups, 1, 256)),
                     dim3(kThreads), 0, stream, p);
  return dsa::check_launch(who);
}

extern "C" int dsa_paged_write(const void* k, const void* v, void* k_cache, void* v_cache,
                               const int64_t* strides, int32_t tokens, int32_t heads,
                               int32_t row_bytes, int32_t pages, int32_t page_size,
                               const int64_t* slots, hipStream_t stream) {
  const char* const who = "dsa_paged_write";
  if (!strides || tokens < 0 || heads <= 0 || row_bytes <= 0 || pages < 0)
    return dsa::set_error(DSA_EINVAL, "%s: bad size or null strides", who);
  if (bad_page_size(page_size))
    return dsa::set_error(DSA_EUNSUPPORTED, "%s: page_size %d (a power of two from 16)", who,
                          page_size);
  if (row_bytes % 16 != 0)
    return dsa::set_error(DSA_EUNSUPPORTED, "%s: rows must be a multiple of 16 bytes", who);
  for (int i = 0; i < 10; ++i)
    if (strides[i] % 16 != 0 || strides[i] < 0)
      return dsa::set_error(DSA_EINVAL, "%s: strides must be multiples of 16 bytes", who);
  if (tokens == 0 || pages == 0) return DSA_OK;
  if (!k || !v || !k_cache || !v_cache || !slots)
    return dsa::set_error(DSA_EINVAL, "%s: null pointer", who);
  const void* const pointers[] = {k, v, k_cache, v_cache};
  for (const void* ptr : pointers)
    if (reinterpret_cast<uintptr_t>(ptr) & 15)
      return dsa::set_error(DSA_EINVAL, "%s: pointers must be 16-byte aligned", who);
  const int32_t chunks = row_bytes / 16;
  const int64_t row = (int64_t)heads * chunks;
  if (row > 0x7fff)
    return dsa::set_error(DSA_EUNSUPPORTED, "%s: tokens of more than 512 KB", who);
  WriteParams p;
  p.src[0] = static_cast<const unsigned char*>(k);
  p.src[1] = static_cast<const unsigned char*>(v);
  p.dst[0] = static_cast<unsigned char*>(k_cache);
  p.dst[1] = static_cast<unsigned char*>(v_cache);
  for (int i = 0; i < 2; ++i) {
    p.src_st[i] = strides[2 * i];
    p.src_sh[i] = strides[2 * i + 1];
    p.dst_sp[i] = strides[4 + 3 * i];
    p.dst_st[i] = strides[5 + 3 * i];
    p.dst_sh[i] = strides[6 + 3 * i];
  }
  p.slots = slots;
  p.total = (int64_t)pages * page_size;
  p.tokens = tokens; p.row = (int32_t)row; p.chunks = chunks;
  p.row_magic = quotient_magic((uint32_t)row);
  p.chunk_magic = quotient_magic((uint32_t)chunks);
  p.group_tokens = (int32_t)std::max<int64_t>(1, kWriteChunks / row);
  p.page_shift = __builtin_ctz(page_size);
  const int64_t groups = ((int64_t)tokens + p.group_tokens - 1) / p.group_tokens;
  // (a launch counts its threads, 256 for each, in 32 bits)
  if (groups >= 1 << 24)
    return dsa::set_error(DSA_EUNSUPPORTED,
                          "%s: %d tokens of %d bytes (up to %d a workgroup, 2^24 - 1 workgroups)",
                          who, tokens, (int)row * 16, p.group_tokens);
  dsa::clear_error();
  hipLaunchKernelGGL(paged_write_kernel, dim3((unsigned)groups, 2), dim3(256), 0, stream, p);
  return dsa::check_launch(who);
}
