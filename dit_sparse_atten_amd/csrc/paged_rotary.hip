// Writes into a paged key/value cache that turn keys (and queries) with their
// positions on the way (gfx950), 16-bit caches and caches of 4-bit elements, and the
// read of a 4-bit cache as 16-bit values.
//
// The rotation of token t, with (c_i, s_i) = cos_sin[positions[t]][i]:
//   pair i = (a, b) -> (a c_i - b s_i, b c_i + a s_i),
// pairs of neighbouring dims (2 i, 2 i + 1), or of dims (i, i + rot / 2) ("halves").
//
// A 4-bit group's exponent is the smallest e with max|x| <= 7 2^e, so that its largest
// element rounds to 6 at most: of the rules by powers of two this one errs least (normal
// values by 11.2% of their norm; with 6 or 8 in place of 7 by 11.6 and 11.5%).
#include <algorithm>
#include <type_traits>

#include "fp4.h"
#include "paged_rows.h"

namespace {

constexpr int kThreads = 256;
constexpr int kMaxBatch = 8;   // heads that a workgroup walks
// Heads whose loads are on their way at a time: of 16-bit rows, and of rows to 4 bits,
// whose loads (non-temporal) are followed by more work.  (57,600 tokens x 12 heads to 4
// bits: two 94 us, 4.9 TB/s, four 95, six and eight 102 and 104; kept loads 97.)
constexpr int kHeadTurns = 4;
constexpr int kPackTurns = 2;

enum Rows { kQ = 0, kK = 1, kV = 2 };

struct TurnParams {
  const uint16_t* src[3];        // q, k, v
  uint16_t* dst[3];              // q_out; k_cache, v_cache (16-bit caches)
  int64_t src_st[3], src_sh[3];  // elements
  int64_t dst_sp[3], dst_st[3], dst_sh[3];
  unsigned char* cache;          // 4-bit caches
  int64_t cache_sp, cache_sh;    // bytes
  const int64_t* slots;
  const int32_t* positions;
  const float* cos_sin;          // [max_positions, rot / 2, 2]
  int64_t total;                 // slots of the cache
  int32_t tokens, heads, kv_heads, head_dim, rot, max_positions, page_shift;
  int32_t batch, q_batches, kv_batches;  // heads of a workgroup, workgroups over heads
  int32_t low, high;             // exponents of a 4-bit group
};

__device__ __forceinline__ void load8(const float* at, float* to) {
  const dsa_f32x4 a = *reinterpret_cast<const dsa_f32x4*>(at);
  const dsa_f32x4 b = *reinterpret_cast<const dsa_f32x4*>(at + 4);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    to[e] = a[e];
    to[4 + e] = b[e];
  }
}

// Token t's slot, -1 where it has none in the cache, or no angles.
__device__ __forceinline__ int64_t slot_of(const TurnParams& p, int t, int position) {
  const int64_t slot = p.slots[t];
  const bool angles = p.rot == 0 || (unsigned)position < (unsigned)p.max_positions;
  return slot >= 0 && slot < p.total && angles ? slot : -1;
}

// 16-bit rows to 16-bit rows, bound by memory: 57,600 tokens x 12 query and key heads x
// 128 (1.09 GB) 218 us, 5.0 TB/s, the rate of a large copy (with non-temporal loads 225,
// stores 240).  A thread takes 16-byte chunks of a row in pairs (c, c +
// rot / 16): with halves a pair's elements turn with each other, so that a row may be
// turned in place.  Chunks behind the turned ones go in neighbouring pairs.  The thread
// keeps its angles and walks the heads of the workgroup's batch.
template <typename T, bool kHalves>
__device__ __forceinline__ void turn_rows(const TurnParams& p, int which, int head0, int heads) {
  typedef typename dsa::Elem<T>::x8 x8;
  const int turned = which == kV ? 0 : p.rot / 16;  // pairs of chunks that turn
  const int chunks = p.head_dim / 8;
  const int units = (chunks + 1) / 2, per_group = kThreads / units;
  const int local = threadIdx.x / units, u = threadIdx.x - local * units;
  const int t = paged::token_of(blockIdx.x, per_group, local, p.tokens);
  if (t < 0) return;
  bool turn = u < turned;
  const int c0 = turn ? u : 2 * u;  // 2 turned + 2 (u - turned)
  const int c1 = turn ? u + turned : c0 + 1;
  const bool second = c1 < chunks;
  const int position = p.rot > 0 ? p.positions[t] : 0;
  int64_t out;
  if (which == kQ) {
    out = t * p.dst_st[kQ];
    if ((unsigned)position >= (unsigned)p.max_positions) turn = false;
  } else {
    const int64_t slot = slot_of(p, t, position);
    if (slot < 0) return;
    out = (slot >> p.page_shift) * p.dst_sp[which] +
          (slot & ((1 << p.page_shift) - 1)) * p.dst_st[which];
  }
  float cs[16];  // of c0's and c1's pairs, or of the pairs between them
  if (turn) {
    const float* const row = p.cos_sin + (int64_t)position * p.rot;
    load8(row + (kHalves ? 16 * u : 8 * c0), cs);
    load8(row + (kHalves ? 16 * u + 8 : 8 * c1), cs + 8);
  }
  const uint16_t* const src = p.src[which] + t * p.src_st[which] + head0 * p.src_sh[which];
  uint16_t* const dst = p.dst[which] + out + head0 * p.dst_sh[which];
#pragma unroll 1
  for (int h0 = 0; h0 < heads; h0 += kHeadTurns) {
    x8 x[kHeadTurns][2];
#pragma unroll
    for (int i = 0; i < kHeadTurns; ++i) {
      if (h0 + i >= heads) continue;
      const uint16_t* const at = src + (h0 + i) * p.src_sh[which];
      x[i][0] = *reinterpret_cast<const x8*>(at + c0 * 8);
      if (second) x[i][1] = *reinterpret_cast<const x8*>(at + c1 * 8);
    }
#pragma unroll
    for (int i = 0; i < kHeadTurns; ++i) {
      if (h0 + i >= heads) continue;
      if (turn) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          // Pair e of 8: across the chunks, or the four of each.
          constexpr bool across = kHalves;
          const int ca = across ? 0 : e / 4, cb = across ? 1 : e / 4;
          const int ea = across ? e : e % 4 * 2, eb = across ? e : e % 4 * 2 + 1;
          const float a = (float)x[i][ca][ea], b = (float)x[i][cb][eb];
          // To float32 and from there to 16 bits, in every turn of the loops alike: left to
          // itself the compiler fuses the last step in some of them.
          float ya = fmaf(a, cs[2 * e], -(b * cs[2 * e + 1]));
          float yb = fmaf(b, cs[2 * e], a * cs[2 * e + 1]);
          asm("" : "+v"(ya), "+v"(yb));
          x[i][ca][ea] = (T)ya;
          x[i][cb][eb] = (T)yb;
        }
      }
      uint16_t* const at = dst + (h0 + i) * p.dst_sh[which];
      *reinterpret_cast<x8*>(at + c0 * 8) = x[i][0];
      if (second) *reinterpret_cast<x8*>(at + c1 * 8) = x[i][1];
    }
  }
}

// The workgroup's heads [*head0, *head0 + return) of one of q, k and v (y).
__device__ __forceinline__ int batch_of(const TurnParams& p, int* which, int* head0) {
  const int y = blockIdx.y;
  *which = y < p.q_batches ? kQ : y < p.q_batches + p.kv_batches ? kK : kV;
  const int first = *which == kQ ? 0 : *which == kK ? p.q_batches : p.q_batches + p.kv_batches;
  *head0 = (y - first) * p.batch;
  return min(p.batch, (*which == kQ ? p.heads : p.kv_heads) - *head0);
}

template <typename T, bool kHalves>
__global__ void __launch_bounds__(kThreads) paged_write_rotary_kernel(TurnParams p) {
  int which, head0;
  const int heads = batch_of(p, &which, &head0);
  turn_rows<T, kHalves>(p, which, head0, heads);
}

// 16-bit rows to 4-bit rows, bound by memory (57,600 tokens x 12 heads x 128, 447 MB: 86
// to 94 us).  A thread takes a chunk of 8 dims, four neighbours a group;
// with halves it reads the chunk that its own turns with too.  A code may hang on the
// last bit of what it rounds, so the turned element does not depend on what the compiler
// fuses: in 64 bits the products of a 16-bit and a 32-bit float are exact, and so their
// sum in 64 bits, which is then rounded to float32, is the same either way.
template <typename T, bool kHalves>
__device__ __forceinline__ void pack_rows(const TurnParams& p, int which, int head0, int heads) {
  typedef typename dsa::Elem<T>::x8 x8;
  const int groups = fp4::groups_of(p.head_dim);
  const int lanes = 4 * groups;  // of a row
  const int per_group = kThreads / lanes;
  const int local = threadIdx.x / lanes, c = threadIdx.x - local * lanes;
  const int t = paged::token_of(blockIdx.x, per_group, local, p.tokens);
  if (t < 0) return;  // (whole quads)
  const bool real = c < p.head_dim / 8;
  const bool turn = which == kK && c < p.rot / 8;
  const int position = p.rot > 0 ? p.positions[t] : 0;
  const int64_t slot = slot_of(p, t, position);
  if (slot < 0) return;
  const bool lower = c < p.rot / 16;
  const int pair = lower ? c + p.rot / 16 : c - p.rot / 16;  // the chunk that c turns with
  float cs[16];
  if (turn) {
    const float* const row = p.cos_sin + (int64_t)position * p.rot;
    load8(row + (kHalves ? 16 * (lower ? c : pair) : 8 * c), cs);
    if (kHalves) load8(row + 16 * (lower ? c : pair) + 8, cs + 8);
    // (an upper element: b c + a s = b c - a (-s))
    if (kHalves && !lower) {
#pragma unroll
      for (int e = 0; e < 8; ++e) cs[2 * e + 1] = -cs[2 * e + 1];
    }
  }
  const uint16_t* const src = p.src[which] + t * p.src_st[which] + head0 * p.src_sh[which];
  const fp4::Layout at(groups, p.page_shift);
  const int row = (int)(slot & ((1 << p.page_shift) - 1));
  unsigned char* const dst = p.cache + (slot >> p.page_shift) * p.cache_sp + head0 * p.cache_sh;
  unsigned char* const codes = dst + (which == kV ? at.v_codes : 0) + row * at.code_row + 4 * c;
  unsigned char* const scales = dst + (which == kV ? at.v_scales : at.k_scales) + 4 * row + c / 4;
#pragma unroll 1
  for (int h0 = 0; h0 < heads; h0 += kPackTurns) {
    x8 x[kPackTurns], y[kPackTurns];
#pragma unroll
    for (int i = 0; i < kPackTurns; ++i) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[i][e] = (T)0.f;
      if (h0 + i >= heads || !real) continue;
      const uint16_t* const from = src + (h0 + i) * p.src_sh[which];
      x[i] = __builtin_nontemporal_load(reinterpret_cast<const x8*>(from + 8 * c));
      if (kHalves && turn) y[i] = *reinterpret_cast<const x8*>(from + 8 * pair);
    }
#pragma unroll
    for (int i = 0; i < kPackTurns; ++i) {
      if (h0 + i >= heads) continue;
      float f[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = (float)x[i][e];
      if (turn) {
        if (kHalves) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            f[e] = (float)((double)f[e] * cs[2 * e] - (double)(float)y[i][e] * cs[2 * e + 1]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            const double a = f[e], b = f[e + 1], co = cs[e], si = cs[e + 1];
            f[e] = (float)(a * co - b * si);
            f[e + 1] = (float)(b * co + a * si);
          }
        }
      }
      // The group's largest magnitude, as bits (those of a NaN are the largest).
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(f[e]) & 0x7fffffffu);
      top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xF, 0xF, false));
      top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xF, 0xF, false));
      // 1.75 2^2 = 7.
      int e = (int)(top >> 23) - 129 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
      e = min(max(e, p.low), p.high);
      const bool bad = top >= 0x7f800000u;
      const float scale = fp4::scale_of(e + 127);
      uint32_t code = 0;
      code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, f[0], f[1], scale, 0);
      code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, f[2], f[3], scale, 1);
      code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, f[4], f[5], scale, 2);
      code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, f[6], f[7], scale, 3);
      *reinterpret_cast<uint32_t*>(codes + (h0 + i) * p.cache_sh) = bad ? 0u : code;
      if ((c & 3) == 0) scales[(h0 + i) * p.cache_sh] = (unsigned char)(bad ? 255 : e + 127);
    }
  }
}

template <typename T, bool kHalves>
__global__ void __launch_bounds__(kThreads) paged_write_fp4_kernel(TurnParams p) {
  int which, head0;
  const int heads = batch_of(p, &which, &head0);
  if (which == kQ) turn_rows<T, kHalves>(p, which, head0, heads);
  else pack_rows<T, kHalves>(p, which, head0, heads);
}

struct ReadParams {
  const unsigned char* cache;
  int64_t cache_sp, cache_sh;
  void* dst[2];            // [count, page_size, kv_heads, head_dim]
  const int32_t* list;     // pages, or null: all of them
  uint32_t units;          // of 16 tokens and a head (up to 2^29, by the launch's bound)
  int32_t pages, kv_heads, head_dim, page_shift;
};

// Rows of a 4-bit cache, keys or values (y): a lane to 8 dims, four bytes in and 16 out.
// 16 tokens of a head (1 KB of codes in a row) at a time, the heads of the same tokens
// one after the other, which together fill the memory that they go to.  Bound by memory:
// 57,600 tokens x 12 heads x 128 (447 MB) 100 us, 4.5 TB/s, a large copy 5.0.
//
// kOnce: the values go past the caches, in reads of 192 MB and more of them, which the
// 256 MB cache would not keep for whoever takes them up.  (Read alone, and with a
// paged_write of all of them behind it, kept / past: 101 MB 22.7 / 20.6 and 54.0 / 55.3
// us, 201 MB 40.6 / 39.8 and 110.6 / 100.4, 403 MB 96.9 / 75.5 and 239.6 / 241.4, 805 MB
// 190 / 148 and 478 / 494.)
constexpr int64_t kOnceBytes = (int64_t)192 << 20;
constexpr int kReadTurns = 8;
constexpr int kReadRows = 16;
__host__ __device__ constexpr int read_units(int groups) {  // that a workgroup reads at a time
  return kThreads / (kReadRows * 4 * groups);
}
template <typename T, bool kOnce>
__global__ void __launch_bounds__(kThreads) paged_read_fp4_kernel(ReadParams p) {
  const int which = blockIdx.y;
  const int groups = fp4::groups_of(p.head_dim);
  const int lanes = 4 * groups, each = read_units(groups);
  const int local = threadIdx.x / lanes, c = threadIdx.x - local * lanes;
  const int unit0 = local / kReadRows, in_unit = local % kReadRows;
  if (unit0 >= each || c >= p.head_dim / 8) return;
  const fp4::Layout at(groups, p.page_shift);
  const int per_page = p.page_shift - 4;  // log2 of the 16-token units of a page
  uint32_t code[kReadTurns], scale[kReadTurns];
  int64_t to[kReadTurns];
#pragma unroll
  for (int i = 0; i < kReadTurns; ++i) {
    const uint32_t unit = (blockIdx.x * kReadTurns + i) * each + unit0;
    code[i] = scale[i] = 0;
    to[i] = -1;
    if (unit >= p.units) continue;
    const uint32_t tokens = unit / (uint32_t)p.kv_heads;  // 16 of a listed page's
    const int head = (int)(unit - tokens * (uint32_t)p.kv_heads);
    const int64_t index = tokens >> per_page;
    const int row = (int)(tokens & ((1u << per_page) - 1)) * kReadRows + in_unit;
    to[i] = (((index << p.page_shift) + row) * p.kv_heads + head) * p.head_dim + 8 * c;
    const int64_t page = p.list ? p.list[index] : index;
    if (page < 0 || page >= p.pages) continue;  // (zeros)
    const unsigned char* const from = p.cache + page * p.cache_sp + head * p.cache_sh;
    code[i] = *reinterpret_cast<const uint32_t*>(from + (which ? at.v_codes : 0) +
                                                 row * at.code_row + 4 * c);
    scale[i] = from[(which ? at.v_scales : at.k_scales) + 4 * row + c / 4];
  }
#pragma unroll
  for (int i = 0; i < kReadTurns; ++i) {
    if (to[i] < 0) continue;
    typedef typename dsa::Elem<T>::x8 x8;
    const x8 y = fp4::expand(code[i], fp4::scale_of(scale[i]), T());
    x8* const at_y = reinterpret_cast<x8*>(static_cast<T*>(p.dst[which]) + to[i]);
    if (kOnce) __builtin_nontemporal_store(y, at_y);
    else *at_y = y;
  }
}

bool bad_page_size(int32_t size) { return size < 16 || (size & (size - 1)) != 0; }
bool aligned(const void* at, int bytes) {
  return (reinterpret_cast<uintptr_t>(at) & (bytes - 1)) == 0;
}

// Checks what both writes share and completes their parameters but for the caches.
// strides: q, q_out, k, v (token, head).
int prepare(TurnParams* p, const char* who, const void* q, void* q_out, const void* k,
            const void* v, int32_t dtype, const int64_t* strides, int caches, int32_t tokens,
            int32_t heads, int32_t kv_heads, int32_t head_dim, int32_t rot_dim, int32_t halves,
            int32_t pages, int32_t page_size, const int64_t* slots, const int32_t* positions,
            const float* cos_sin, int32_t max_positions) {
  if (!strides || tokens < 0 || heads < 0 || kv_heads <= 0 || pages < 0 || max_positions < 0)
    return dsa::set_error(DSA_EINVAL, "%s: bad size or null strides", who);
  if (dtype != DSA_BF16 && dtype != DSA_F16)
    return dsa::set_error(DSA_EUNSUPPORTED, "%s: dtype %d (bf16 or fp16)", who, dtype);
  if (head_dim <= 0 || head_dim > 128 || head_dim % 8 != 0)
    return dsa::set_error(DSA_EUNSUPPORTED, "%s: head_dim %d (a multiple of 8 up to 128)", who,
                          head_dim);
  if (rot_dim < 0 || rot_dim > head_dim || rot_dim % 16 != 0)
    return dsa::set_error(DSA_EUNSUPPORTED, "%s: rot_dim %d (a multiple of 16 up to head_dim)",
                          who, rot_dim);
  if (halves != 0 && halves != 1)
    return dsa::set_error(DSA_EINVAL, "%s: halves is 0 or 1", who);
  if (bad_page_size(page_size))
    return dsa::set_error(DSA_EUNSUPPORTED, "%s: page_size %d (a power of two from 16)", who,
                          page_size);
  for (int i = 0; i < 8 + caches; ++i)
    if (strides[i] % 8 != 0 || strides[i] < 0)
      return dsa::set_error(DSA_EINVAL, "%s: strides must be multiples of 8", who);
  // (a launch counts its workgroups along y in 16 bits)
  if (heads > 4096 || kv_heads > 4096)
    return dsa::set_error(DSA_EUNSUPPORTED, "%s: more than 4,096 heads", who);
  if (tokens == 0) return DSA_OK;
  if ((heads > 0 && (!q || !q_out)) || !k || !v || !slots ||
      (rot_dim > 0 && (!positions || (max_positions > 0 && !cos_sin))))
    return dsa::set_error(DSA_EINVAL, "%s: null pointer", who);
  const void* const pointers[] = {q, q_out, k, v, cos_sin};
  for (const void* ptr : pointers)
    if (!aligned(ptr, 16))
      return dsa::set_error(DSA_EINVAL, "%s: pointers must be 16-byte aligned", who);
  const void* const from[3] = {q, k, v};
  for (int i = 0; i < 3; ++i) {
    const int at = i == 0 ? 0 : 2 + 2 * i;
    p->src[i] = static_cast<const uint16_t*>(from[i]);
    p->src_st[i] = strides[at];
    p->src_sh[i] = strides[at + 1];
  }
  p->dst[kQ] = static_cast<uint16_t*>(q_out);
  p->dst_st[kQ] = strides[2];
  p->dst_sh[kQ] = strides[3];
  p->slots = slots;
  p->positions = positions;
  p->cos_sin = cos_sin;
  p->total = (int64_t)pages * page_size;
  p->tokens = tokens; p->heads = heads; p->kv_heads = kv_heads; p->head_dim = head_dim;
  p->rot = rot_dim; p->max_positions = max_positions;
  p->page_shift = __builtin_ctz(page_size);
  p->low = dtype == DSA_BF16 ? fp4::kLowBf16 : fp4::kLowF16;
  p->high = dtype == DSA_BF16 ? fp4::kHighBf16 : fp4::kHighF16;
  return DSA_OK;
}

// Workgroups: token groups of at least `per_group` tokens by batches of heads, small
// ones in calls that would not fill the chip.
dim3 grid_of(TurnParams* p, int per_group) {
  const int64_t groups = ((int64_t)p->tokens + per_group - 1) / per_group;
  const int64_t rows = groups * (p->heads + 2 * p->kv_heads);
  p->batch = (int32_t)std::clamp<int64_t>(rows / 1024, 1, kMaxBatch);
  p->q_batches = (p->heads + p->batch - 1) / p->batch;
  p->kv_batches = (p->kv_heads + p->batch - 1) / p->batch;
  return dim3((unsigned)groups, (unsigned)(p->q_batches + 2 * p->kv_batches));
}

int check_groups(const dim3& grid, const char* who) {
  // (a launch counts its threads along x in 32 bits)
  if (grid.x >= 1 << 24) return dsa::set_error(DSA_EUNSUPPORTED, "%s: too many tokens", who);
  return DSA_OK;
}

// kernel(type, halves) for a call's type and pairs.
template <typename F>
void with_types(int32_t dtype, int32_t halves, F launch) {
  if (dtype == DSA_BF16) {
    if (halves) launch(__bf16(), std::true_type());
    else launch(__bf16(), std::false_type());
  } else {
    if (halves) launch(_Float16(), std::true_type());
    else launch(_Float16(), std::false_type());
  }
}

}  // namespace

extern "C" int dsa_paged_write_rotary(const void* q, void* q_out, const void* k, const void* v,
                                      void* k_cache, void* v_cache, int32_t dtype,
                                      const int64_t* strides, int32_t tokens, int32_t heads,
                                      int32_t kv_heads, int32_t head_dim, int32_t rot_dim,
                                      int32_t halves, int32_t pages, int32_t page_size,
                                      const int64_t* slots, const int32_t* positions,
                                      const float* cos_sin, int32_t max_positions,
                                      hipStream_t stream) {
  const char* const who = "dsa_paged_write_rotary";
  TurnParams p = {};
  const int status =
      prepare(&p, who, q, q_out, k, v, dtype, strides, 6, tokens, heads, kv_heads, head_dim,
              rot_dim, halves, pages, page_size, slots, positions, cos_sin, max_positions);
  if (status != DSA_OK || tokens == 0) return status;
  if (pages > 0 && (!k_cache || !v_cache))
    return dsa::set_error(DSA_EINVAL, "%s: null pointer", who);
  if (!aligned(k_cache, 16) || !aligned(v_cache, 16))
    return dsa::set_error(DSA_EINVAL, "%s: pointers must be 16-byte aligned", who);
  p.dst[kK] = static_cast<uint16_t*>(k_cache);
  p.dst[kV] = static_cast<uint16_t*>(v_cache);
  for (int i = 0; i < 2; ++i) {
    p.dst_sp[kK + i] = strides[8 + 3 * i];
    p.dst_st[kK + i] = strides[9 + 3 * i];
    p.dst_sh[kK + i] = strides[10 + 3 * i];
  }
  const dim3 grid = grid_of(&p, kThreads / ((head_dim / 8 + 1) / 2));
  if (const int bad = check_groups(grid, who)) return bad;
  dsa::clear_error();
  with_types(dtype, halves, [&](auto type, auto half) {
    hipLaunchKernelGGL((paged_write_rotary_kernel<decltype(type), decltype(half)::value>), grid,
                       dim3(kThreads), 0, stream, p);
  });
  return dsa::check_launch(who);
}

namespace {

int check_cache(const void* cache, int64_t sp, int64_t sh, int32_t pages, int32_t page_size,
                const char* who) {
  if (fp4::bad_page_size(page_size))
    return dsa::set_error(DSA_EUNSUPPORTED, "%s: page_size %d (a power of two, 16 to %d)", who,
                          page_size, fp4::kMaxPage);
  if (sp % 16 != 0 || sh % 16 != 0 || sp < 0 || sh < 0)
    return dsa::set_error(DSA_EINVAL, "%s: cache strides must be multiples of 16 bytes", who);
  if (pages > 0 && !cache) return dsa::set_error(DSA_EINVAL, "%s: null pointer", who);
  if (!aligned(cache, 16))
    return dsa::set_error(DSA_EINVAL, "%s: pointers must be 16-byte aligned", who);
  return DSA_OK;
}

}  // namespace

extern "C" int dsa_paged_write_fp4(const void* q, void* q_out, const void* k, const void* v,
                                   void* cache, int32_t dtype, const int64_t* strides,
                                   int32_t tokens, int32_t heads, int32_t kv_heads,
                                   int32_t head_dim, int32_t rot_dim, int32_t halves, int32_t pages,
                                   int32_t page_size, const int64_t* slots,
                                   const int32_t* positions, const float* cos_sin,
                                   int32_t max_positions, hipStream_t stream) {
  const char* const who = "dsa_paged_write_fp4";
  TurnParams p = {};
  int status = prepare(&p, who, q, q_out, k, v, dtype, strides, 0, tokens, heads, kv_heads,
                       head_dim, rot_dim, halves, pages, page_size, slots, positions, cos_sin,
                       max_positions);
  if (status != DSA_OK) return status;
  status = check_cache(cache, strides[8], strides[9], pages, page_size, who);
  if (status != DSA_OK || tokens == 0) return status;
  p.cache = static_cast<unsigned char*>(cache);
  p.cache_sp = strides[8];
  p.cache_sh = strides[9];
  const dim3 grid = grid_of(&p, kThreads / (4 * fp4::groups_of(head_dim)));
  if (const int bad = check_groups(grid, who)) return bad;
  dsa::clear_error();
  with_types(dtype, halves, [&](auto type, auto half) {
    hipLaunchKernelGGL((paged_write_fp4_kernel<decltype(type), decltype(half)::value>), grid,
                       dim3(kThreads), 0, stream, p);
  });
  return dsa::check_launch(who);
}

extern "C" int dsa_paged_read_fp4(const void* cache, const int64_t* strides, void* k, void* v,
                                  int32_t dtype, int32_t pages, int32_t page_size,
                                  int32_t kv_heads, int32_t head_dim, const int32_t* list,
                                  int32_t count, hipStream_t stream) {
  const char* const who = "dsa_paged_read_fp4";
  if (!strides || pages < 0 || kv_heads <= 0 || count < 0)
    return dsa::set_error(DSA_EINVAL, "%s: bad size or null strides", who);
  if (dtype != DSA_BF16 && dtype != DSA_F16)
    return dsa::set_error(DSA_EUNSUPPORTED, "%s: dtype %d (bf16 or fp16)", who, dtype);
  if (head_dim <= 0 || head_dim > 128 || head_dim % 8 != 0)
    return dsa::set_error(DSA_EUNSUPPORTED, "%s: head_dim %d (a multiple of 8 up to 128)", who,
                          head_dim);
  if (!list && count > pages)
    return dsa::set_error(DSA_EINVAL, "%s: %d of %d pages", who, count, pages);
  const int status = check_cache(cache, strides[0], strides[1], pages, page_size, who);
  if (status != DSA_OK) return status;
  if (count == 0) return DSA_OK;
  if (!k || !v) return dsa::set_error(DSA_EINVAL, "%s: null pointer", who);
  if (!aligned(k, 16) || !aligned(v, 16))
    return dsa::set_error(DSA_EINVAL, "%s: pointers must be 16-byte aligned", who);
  ReadParams p;
  p.cache = static_cast<const unsigned char*>(cache);
  p.cache_sp = strides[0];
  p.cache_sh = strides[1];
  p.dst[0] = k;
  p.dst[1] = v;
  p.list = list;
  const int64_t units = (int64_t)count * kv_heads * (page_size / kReadRows);
  p.pages = pages; p.kv_heads = kv_heads; p.head_dim = head_dim;
  p.page_shift = __builtin_ctz(page_size);
  const int64_t each = kReadTurns * read_units(fp4::groups_of(head_dim));
  const int64_t groups = (units + each - 1) / each;
  if (groups >= 1 << 24) return dsa::set_error(DSA_EUNSUPPORTED, "%s: too many rows", who);
  p.units = (uint32_t)units;
  dsa::clear_error();
  const dim3 grid((unsigned)groups, 2);
  const bool once = units * kReadRows * head_dim * 4 >= kOnceBytes;  // keys and values
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, stream, p);
  };
  if (dtype == DSA_BF16)
    once ? launch(paged_read_fp4_kernel<__bf16, true>) : launch(paged_read_fp4_kernel<__bf16, false>);
  else
    once ? launch(paged_read_fp4_kernel<_Float16, true>)
         : launch(paged_read_fp4_kernel<_Float16, false>);
  return dsa::check_launch(who);
}
