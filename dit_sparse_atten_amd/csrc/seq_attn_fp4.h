// Attention of new tokens over a paged cache of 4-bit elements (fp4.h has its layout),
// bf16 or fp16 in and out, fp32 softmax: the walks of seq_attn.h, whose schedule, items
// and joins these kernels share, over keys and values of 32-dim groups with a scale.
//
// Keys and values are expanded to 16 bits (exactly: the conversion takes the scale), keys in
// registers or on the way into LDS, values on the way into LDS, and the products are those
// of a 16-bit cache: S = K Q^T, exact products summed in fp32, and O^T = V^T P^T, P rounded
// to the input type (the matrix operand's; by at most 2^-8 of a weight in bf16, below the
// cache's own error).  Against 64 bits the outputs of normal values are off by 0.0023 of
// their norm in bf16 and 0.00029 in fp16 (0.0017 and 0.00021 with fp32 throughout, the
// output rounded).  The scaled matrix instructions would take the codes as they lie in
// memory, against 8-bit terms of the queries, in 4 to 12% less time for bf16 chunks and 1 to
// 5% less for single tokens, but they cut a product that lies 2^-13 below the largest of
// eight neighbours: with one outlier dim a score was off by up to 100 times its fp32 bound.
//
// A value group that is not of the type's numbers (kLargestScale) enters as zeros, for 0 times
// it would reach rows that do not see its key, and the rows that do are set to NaN at the
// end (unfinite_groups).
#pragma once

#include "fp4.h"
#include "seq_attn.h"

namespace seq {

// The largest scale byte of a group of numbers: every group past it (255, or in fp16 one of a
// cache written from bf16) holds elements that the type has not.
template <typename T>
constexpr uint32_t kLargestScale = (__is_same(T, _Float16) ? fp4::kHighF16 : fp4::kHighBf16) + 127;

// 8 dims from `d` of a query row, zeros past head_dim.
template <typename T>
__device__ __forceinline__ typename dsa::Elem<T>::x8 query_dims(const T* row, int d, int head_dim) {
  typename dsa::Elem<T>::x8 y;
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = (T)0.f;
  if (d < head_dim) y = *reinterpret_cast<const typename dsa::Elem<T>::x8*>(row + d);
  return y;
}

// A wave's groups of values that are not numbers of type T: bit g of the result where a key of [lo,
// hi) that the lane's row sees (those below `lim`) has such a group g.
template <typename T>
__device__ __forceinline__ uint32_t unfinite_groups(LateParams p, const Item& it, int h, int lo,
                                                    int hi, int lim) {
  const int groups = fp4::groups_of(p->head_dim);
  const fp4::Layout at(groups, p->page_shift);
  uint32_t found = 0;
  for (int key0 = lo; key0 < hi; key0 += 64) {
    const int key = key0 + (int)(threadIdx.x & 63);
    uint32_t mine = 0;
    if (key < hi) {
      const int page = p->table[(int64_t)it.request * p->table_stride + (key >> p->page_shift)];
      if ((unsigned)page < (unsigned)p->pages) {
        const uint32_t four = *reinterpret_cast<const uint32_t*>(
            static_cast<const unsigned char*>(p->k) + page * p->k_sp + h * p->k_sh + at.v_scales +
            4 * (key & ((1 << p->page_shift) - 1)));
#pragma unroll
        for (int g = 0; g < 4; ++g)
          if (g < groups && (four >> (8 * g) & 255) > kLargestScale<T>) mine |= 1u << g;
      }
    }
    uint64_t left = __ballot(mine != 0);
    while (left != 0) {
      const int l = (int)__builtin_ctzll(left);
      left &= left - 1;
      const uint32_t theirs = (uint32_t)__builtin_amdgcn_readlane((int)mine, l);
      if (key0 + l < lim) found |= theirs;
    }
  }
  return found;
}

// LDS serves a wave's operations in order; this keeps the compiler from reordering the
// writes of some lanes and the reads of others.
__device__ __forceinline__ void own_lds_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}

// One page and key head of the cache; no bytes, and so zeros, where `any` is false.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t fp4_rsrc(const Params& p, uint32_t page, int h,
                                                           int bytes, bool any) {
  return make_rsrc(static_cast<const unsigned char*>(p.k) + (uint64_t)page * (uint64_t)p.k_sp +
                       (uint64_t)h * (uint64_t)p.k_sh,
                   any ? (uint32_t)bytes : 0u);
}

// 16 rows x the item's keys: kWaves waves, 64 keys at a time each (wave w those from 64 w,
// 64 (w + kWaves), ..), joined at the end.  Bound by the reads of the cache: codes and
// scales go to registers a turn ahead, 70 KB on their way on a compute unit, by eight waves
// of one workgroup or four each of two.  (64 requests of 1,000 to 16,000 tokens, 8 key
// heads: D = 128 167 us, 5.9 TB/s, of 7.0 for a plain streaming read.  64 of 12,000, D = 64:
// 93 us, 4.5 TB/s; 10 us of each are the schedule, the join and their launches, and with
// half the bytes a turn waits a quarter of its time for data and a third to be issued.)
// Lane (q4, c16) =
// (lane / 16, lane % 16) holds the dims kD / 4 q4 .. of the keys 16 i + c16, row c16's scores
// of the keys 16 i + 4 q4 + r and, of O, the dims 16 dt + 4 q4 + r.
constexpr int kFp4Keys = 64;  // of a wave's turn

// A lane's codes of a key: 32, or 16 where kD = 64.
template <int kBytes>
struct Codes;
template <>
struct Codes<16> {
  typedef dsa_u32x4 type;
  static __device__ __forceinline__ type load(__amdgpu_buffer_rsrc_t rsrc, uint32_t at, int from) {
    return __builtin_amdgcn_raw_buffer_load_b128(rsrc, at, from, 2);
  }
};
template <>
struct Codes<8> {
  typedef dsa_u32x2 type;
  static __device__ __forceinline__ type load(__amdgpu_buffer_rsrc_t rsrc, uint32_t at, int from) {
    return __builtin_amdgcn_raw_buffer_load_b64(rsrc, at, from, 2);
  }
};

template <typename T, int kD, int kWaves>
__global__ void __launch_bounds__(kWaves * 64, 1) seq_narrow_fp4_kernel(Params p) {
  typedef dsa::Elem<T> E;
  typedef typename E::x8 x8;
  constexpr int kRow = kD * 2;
  constexpr int kTurn = kWaves * kFp4Keys;  // keys of the workgroup's turn
  constexpr int kStage = kFp4Keys * kRow;  // a wave's values of a turn, expanded
  constexpr int kDt = kD / 16;
  constexpr int kLaneDims = kD / 4;
  typedef Codes<kLaneDims / 2> C;
  __shared__ __attribute__((aligned(1024))) unsigned char lds_v[kWaves * kStage];
  __shared__ float join_ml[2][kWaves][16];
  __shared__ int join_row[2][16];  // token and head
  constexpr int kJoinRow = kD + 4;  // floats
  static_assert(kNarrowRows * kJoinRow * 4 <= kStage, "a wave joins through its own stage");
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int q4 = lane >> 4, c16 = lane & 15;
  const int groups = fp4::groups_of(p.head_dim);
  const fp4::Layout at(groups, p.page_shift);
  const int block_bytes = fp4::row_bytes(groups) << p.page_shift;
  const int group_of = q4 * kLaneDims / 32;
  const uint32_t dead = group_of < groups ? 0u : dsa::kDeadChunk;
  const uint32_t code_at = (uint32_t)(c16 * at.code_row + q4 * kLaneDims / 2) | dead;
  const uint32_t scale_at = (uint32_t)(c16 * 4 + group_of) | dead;

  auto run = [&](const Item& it, const int h) __attribute__((always_inline)) {
  const int rows = it.n * p.group;
  const int row_c = min(it.tile * kNarrowRows + c16, rows - 1);
  const int token = (int)((uint32_t)row_c / (uint32_t)p.group);
  const int head = h * p.group + row_c - token * p.group;
  const int lim = p.causal ? max(0, min(it.m, it.m - it.n + token + 1)) : it.m;
  const int lim_first = __builtin_amdgcn_readlane(lim, 0);
  const int kend = min(__builtin_amdgcn_readlane(lim, 15), it.s1 * kNarrowKeys);
  const int key_first = it.s0 * kNarrowKeys + wave * kFp4Keys;

  // The row's query, of the dims whose codes the lane holds.
  x8 qf[kLaneDims / 8];
  {
    const T* qrow = static_cast<const T*>(p.q) + (int64_t)(it.q0 + token) * p.q_st +
                    head * p.q_sh;
#pragma unroll
    for (int j = 0; j < kLaneDims / 8; ++j)
      qf[j] = query_dims<T>(qrow, kLaneDims * q4 + 8 * j, p.head_dim);
  }

  // Pages of a window of 16 turns: lane l holds granule l & 3 of turn l / 4.
  auto window_ids = [&](int window) -> int {
    const int key = key_first + (window * 16 + (lane >> 2)) * kTurn + (lane & 3) * 16;
    return key < kend ? page_at(p, it.request, key) : -1;
  };
  int ids = window_ids(0), ids_next = window_ids(1);
  uint64_t bad_ids = __ballot((unsigned)ids >= (unsigned)p.pages);

  struct Turn {
    typename C::type k[4], v[4];
    uint32_t ks[4], vs[4];
    int bad;  // granules (bits 0..3) that take no part
  };
  auto load = [&](int turn, Turn& t) __attribute__((always_inline)) {
    if ((turn & 15) == 0 && turn > 0) {
      ids = ids_next;
      bad_ids = __ballot((unsigned)ids >= (unsigned)p.pages);
      ids_next = window_ids((turn >> 4) + 1);
    }
    t.bad = (int)(bad_ids >> ((turn & 15) * 4)) & 15;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int key = key_first + turn * kTurn + 16 * i;
      const int row = key & ((1 << p.page_shift) - 1);
      const uint32_t page = (uint32_t)__builtin_amdgcn_readlane(ids, (turn & 15) * 4 + i);
      const __amdgpu_buffer_rsrc_t rsrc =
          fp4_rsrc(p, page, h, block_bytes, page < (uint32_t)p.pages);
      t.k[i] = C::load(rsrc, code_at, row * at.code_row);
      t.ks[i] = __builtin_amdgcn_raw_buffer_load_b8(rsrc, scale_at, at.k_scales + 4 * row, 2);
      t.v[i] = C::load(rsrc, code_at, at.v_codes + row * at.code_row);
      t.vs[i] = __builtin_amdgcn_raw_buffer_load_b8(rsrc, scale_at, at.v_scales + 4 * row, 2);
    }
  };

  // Two turns' registers in turn: one on its way, one at work.  (Loads past the last key
  // have no bytes.  They go out all the same: the wait for a turn counts those behind it,
  // and where some paths have none it would wait for them too.)
  Turn even, odd;
  load(0, even);
  __builtin_amdgcn_sched_barrier(0);
  float m_run = -INFINITY, l_run = 0.f;
  dsa_f32x4 oacc[kDt];
#pragma unroll
  for (int dt = 0; dt < kDt; ++dt) oacc[dt] = dsa_f32x4{0.f, 0.f, 0.f, 0.f};
  bool unfinite = false;  // a group of values that is not of the type's numbers
  // V chunk c of row r sits at c ^ (2 (r & 3) + (r / 4 & 1)): eight rows of a chunk, as
  // eight lanes write them, and four rows of two chunks, as 16 lanes read them, lie in
  // distinct banks.
  auto v_swz = [](int r, int c) { return c ^ (2 * (r & 3) + (r >> 2 & 1)); };
  const int vr_row = 4 * q4 + (c16 >> 2);
  unsigned char* const stage = lds_v + wave * kStage;

  auto compute = [&](const Turn& t, int key0) __attribute__((always_inline)) {
    dsa_f32x4 s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s[i] = dsa_f32x4{0.f, 0.f, 0.f, 0.f};
      const float scale = fp4::scale_of(t.ks[i]);
#pragma unroll
      for (int j = 0; j < kLaneDims / 8; ++j)
        s[i] = E::mfma16(fp4::expand(t.k[i][j], scale, T()), qf[j], s[i]);
    }
    // (the values' way into LDS covers the products' latency)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool held = key0 + 16 * i + c16 < kend;
      const bool number = t.vs[i] <= kLargestScale<T>;
      unfinite |= held && !number;
      const float scale = fp4::scale_of(held && number ? t.vs[i] : 0u);
#pragma unroll
      for (int j = 0; j < kLaneDims / 8; ++j)
        *reinterpret_cast<x8*>(stage + (16 * i + c16) * kRow +
                               v_swz(c16, kLaneDims / 8 * q4 + j) * 16) =
            fp4::expand(t.v[i][j], scale, T());
    }
    own_lds_order();
    if (key0 + kFp4Keys > lim_first) {
      const int bound = min(lim, kend) - key0 - 4 * q4;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (16 * i + r >= bound) s[i][r] = -INFINITY;
    }
    if (t.bad != 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (t.bad & (1 << i)) s[i][r] = -INFINITY;
    }
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[i][r]);
    // The reference moves only where a lane's own scores call for it: the row's largest is
    // not needed before.
    if (__any(mx * p.scale_log2 > m_run + kRescaleLog2)) {
      mx = fmaxf(mx, __shfl_xor(mx, 16));
      const float mx2 = dsa::pair32_max(mx) * p.scale_log2;
      const bool up = mx2 > m_run + kRescaleLog2;
      const float m_new = up ? mx2 : m_run;
      const float alpha = up ? __builtin_amdgcn_exp2f(m_run - m_new) : 1.0f;
      m_run = m_new;
      l_run *= alpha;
#pragma unroll
      for (int dt = 0; dt < kDt; ++dt) oacc[dt] *= alpha;
    }
    const float m_use = m_run == -INFINITY ? 0.f : m_run;
    x8 pf[2];
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int r = 0; r < 4; r += 2) {
        const float p0 = __builtin_amdgcn_exp2f(fmaf(s[i][r], p.scale_log2, -m_use));
        const float p1 = __builtin_amdgcn_exp2f(fmaf(s[i][r + 1], p.scale_log2, -m_use));
        const dsa_f32x2 two = {p0, p1};
        const typename E::x2 pb = __builtin_convertvector(two, typename E::x2);
        sum += p0 + p1;
        pf[i >> 1][4 * (i & 1) + r] = pb[0];
        pf[i >> 1][4 * (i & 1) + r + 1] = pb[1];
      }
    l_run += sum;
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int dt = 0; dt < kDt; ++dt) {
        const int pos = v_swz(vr_row, 2 * dt + ((c16 & 3) >> 1));
        const unsigned char* from =
            stage + (32 * half + vr_row) * kRow + pos * 16 + (c16 & 1) * 8;
        const typename E::x4 lo = read_tr<T>(from);
        const typename E::x4 hi = read_tr<T>(from + 16 * kRow);
        const x8 a = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        oacc[dt] = E::mfma16(a, pf[half], oacc[dt]);
      }
    own_lds_order();
  };
  if (key_first < kend) {
#pragma unroll 1
    for (int turn = 0;; turn += 2) {
      const int key0 = key_first + turn * kTurn;
      load(turn + 1, odd);
      __builtin_amdgcn_sched_barrier(0);
      compute(even, key0);
      if (key0 + kTurn >= kend) break;
      load(turn + 2, even);
      __builtin_amdgcn_sched_barrier(0);
      compute(odd, key0 + kTurn);
      if (key0 + 2 * kTurn >= kend) break;
    }
  }

  const LateParams late = late_params();
  if (__builtin_expect(__any(unfinite), 0)) {
    // (the wave's own keys alone would do; this is all of the item's)
    const uint32_t found = unfinite_groups<T>(late, it, h, it.s0 * kNarrowKeys, kend, lim);
#pragma unroll
    for (int dt = 0; dt < kDt; ++dt)
      if (found >> (dt / 2) & 1) oacc[dt] = dsa_f32x4{NAN, NAN, NAN, NAN};
  }
  // Join the waves: their O, m and l through the stages, rows of kD + 4 floats (16 bytes
  // from bank to bank between them).
  l_run += __shfl_xor(l_run, 16);
  const float l_wave = dsa::pair32_sum(l_run);
  float* const mine = reinterpret_cast<float*>(stage);
#pragma unroll
  for (int dt = 0; dt < kDt; ++dt)
    *reinterpret_cast<dsa_f32x4*>(mine + c16 * kJoinRow + 16 * dt + 4 * q4) = oacc[dt];
  if (q4 == 0) {
    join_ml[0][wave][c16] = m_run;
    join_ml[1][wave][c16] = l_wave;
    if (wave == 0) {
      join_row[0][c16] = it.q0 + token;
      join_row[1][c16] = head;
    }
  }
  dsa::lds_barrier();
  // Thread (r, c): row r and those kWaves * 256 / kD further on, dims 4 c .. 4 c + 3.
  const int d0 = tid % (kD / 4) * 4;
#pragma unroll
  for (int r = tid / (kD / 4); r < kNarrowRows; r += kWaves * 64 / (kD / 4)) {
    const int out_row = it.tile * kNarrowRows + r;
    if (out_row >= rows) break;
    float m_all = -INFINITY, l_all = 0.f, w[kWaves], m[kWaves], l[kWaves];
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      m[i] = join_ml[0][i][r];
      l[i] = join_ml[1][i][r];
      m_all = fmaxf(m_all, m[i]);
    }
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      // (no finite score: l is 0, or NaN from NaN scores)
      w[i] = m[i] == -INFINITY ? l[i] : __builtin_amdgcn_exp2f(m[i] - m_all);
      l_all = fmaf(w[i], l[i], l_all);
    }
    dsa_f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      const dsa_f32x4 x = *reinterpret_cast<const dsa_f32x4*>(
          reinterpret_cast<const float*>(lds_v + i * kStage) + r * kJoinRow + d0);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = fmaf(w[i], x[e], acc[e]);
    }
    if (it.slot >= 0) {
      float* po =
          late->part + ((int64_t)it.slot * late->kv_heads + h) * part_floats(kNarrowRows, kD);
      *reinterpret_cast<dsa_f32x4*>(po + r * kD + d0) = acc;
      if (d0 == 0) {
        po[kNarrowRows * kD + r] = m_all;
        po[kNarrowRows * (kD + 1) + r] = l_all;
      }
    } else {
      const int out_token = join_row[0][r], out_head = join_row[1][r];
      const float inv = l_all > 0.f ? 1.f / l_all : (l_all == 0.f ? 0.f : l_all);
      if (d0 < late->head_dim) {
        typename E::x4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = (T)(acc[e] * inv);
        *reinterpret_cast<typename E::x4*>(static_cast<T*>(late->o) +
                                           (int64_t)out_token * late->o_st +
                                           out_head * late->o_sh + d0) = y;
      }
      if (late->lse && d0 == 0)
        late->lse[(int64_t)out_head * late->q_rows + out_token] =
            l_all == 0.f ? -INFINITY : m_all * kLn2 + logf(l_all);
    }
  }
  };

  // An unlisted call gives the workgroup one item, a listed one its chain.
  Item it;
  int h;
  if (p.unlisted) {
    if (own_item(p, (int)blockIdx.x, &it, &h)) run(it, h);
    return;
  }
  const int chain = (int)blockIdx.x / p.kv_heads;
  h = (int)blockIdx.x - chain * p.kv_heads;
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

// 128 rows x the item's keys, bound by the matrix instructions: four waves of 32 rows,
// 64 keys a step, as seq_wide_kernel walks a 16-bit cache.  Keys and values are expanded into
// LDS by the thread that loaded their codes, a step ahead.  (3,600 rows over 57,600 keys, 40
// heads, D = 128: 3,840 to 3,960 us, 1.07 to 1.11 PFLOP/s, of 1.36 to 1.39 in a library
// product; a 16-bit cache 3,930.  Keys expanded by every wave for itself, from codes in
// LDS: 4,000 to 4,200.  The chip is at its power limit.  With fewer dims the exponentials
// weigh more: D = 96 1.00, D = 64 0.80 PFLOP/s.)  Lane (g, qi) = (lane / 32, lane % 32)
// holds row qi's scores of the keys 32 kt + 8 (r / 4) + 4 g + r % 4 and, of O, the dims
// 32 dt + 8 (r / 4) + 4 g + r % 4.
template <typename T, int kD, int kUse>
__global__ void __launch_bounds__(256, 2) seq_wide_fp4_kernel(Params p) {
  typedef dsa::Elem<T> E;
  typedef typename E::x8 x8;
  constexpr int kRow = kD * 2;               // bytes of an expanded row
  constexpr int kStage = kWideKeys * kRow;
  constexpr int kDt = kUse / 32;
  constexpr int kChunks = kD / 8;
  __shared__ __attribute__((aligned(1024))) unsigned char lds_k[2 * kStage];
  __shared__ __attribute__((aligned(1024))) unsigned char lds_v[2 * kStage];

  Item it;
  int h;
  if (!take_item(p, &it, &h)) return;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 5, qi = lane & 31;
  const int rows = it.n * p.group;
  // Of a tile of up to 64 rows two waves take each 32 rows, 32 of a step's keys each, and
  // join at the end.  (32 requests of 8,000 tokens, 8 key heads, 64 rows each: 126 us with
  // two of the waves idle, 108 so; 16 of 4,000, 40 key heads, 150 rows: 308 and 289.)
  const bool half = rows - it.tile * kWideRows <= kWideRows / 2;
  const int wave_row = (half ? wave & 1 : wave) * 32;
  const int local = wave_row + qi;
  const int row = it.tile * kWideRows + local;
  const bool row_ok = row < rows;
  const int row_c = min(row, rows - 1);
  const int token = row_c / p.group;
  const int head = h * p.group + row_c - token * p.group;
  // Keys [0, lim) are visible to the lane's row.
  const int lim = p.causal ? max(0, min(it.m, it.m - it.n + token + 1)) : it.m;
  const bool wave_active = it.tile * kWideRows + wave_row < rows;
  const int lim_first = __builtin_amdgcn_readlane(lim, 0);
  const int lim_last = __builtin_amdgcn_readlane(lim, 31);
  // Keys the tile's last row sees.
  const int last_row = min(it.tile * kWideRows + kWideRows, rows) - 1;
  const int kend =
      p.causal ? max(0, min(it.m, it.m - it.n + last_row / p.group + 1)) : it.m;
  const int groups = fp4::groups_of(p.head_dim);
  const fp4::Layout at(groups, p.page_shift);
  const int block_bytes = fp4::row_bytes(groups) << p.page_shift;

  x8 qf[kUse / 16];  // the row's query: dims 16 i + 8 g ..
  {
    const T* qrow = static_cast<const T*>(p.q) + (int64_t)(it.q0 + token) * p.q_st +
                    head * p.q_sh;
#pragma unroll
    for (int i = 0; i < kUse / 16; ++i) qf[i] = query_dims<T>(qrow, 16 * i + 8 * g, p.head_dim);
  }

  // Wave w stages the keys 16 w .. 16 w + 15 of a step, one page: lane (r, c) = (lane / 4,
  // lane % 4) row r's group c, 16 bytes of codes and a scale byte, of keys and of values.
  const int own_row = lane >> 2, own_group = lane & 3;
  const uint32_t code_at = own_group < groups ? (uint32_t)(own_row * at.code_row + own_group * 16)
                                              : dsa::kDeadChunk;
  const uint32_t scale_at = own_group < groups ? (uint32_t)(own_row * 4 + own_group)
                                               : dsa::kDeadChunk;
  // K chunk c of row r sits at c ^ (c / 8) ^ (2 (r & 3) + (r / 4 & 1)): two rows of four chunks
  // 4 apart, as eight lanes write them, and eight rows of a chunk, as eight lanes read
  // them, lie in distinct banks.
  auto k_swz = [](int r, int c) { return c ^ (c >> 3) ^ (2 * (r & 3) + (r >> 2 & 1)); };
  // V chunk c of row r sits at c ^ (c / 8) ^ 2 (r & 3): two rows of four chunks 4 apart,
  // as eight lanes write them, and four rows of two chunks, as 16 lanes read them, lie in
  // distinct banks.
  auto v_swz = [](int r, int c) { return c ^ (c >> 3) ^ (2 * (r & 3)); };
  int vfrag[kDt];
  {
    const int lam = lane & 15, r = lam >> 2, c = lam & 3;
    const int vrow = 4 * g + r;
    const int sub = 2 * ((lane >> 4) & 1) + (c >> 1);
#pragma unroll
    for (int dt = 0; dt < kDt; ++dt)
      vfrag[dt] = vrow * kRow + v_swz(vrow, 4 * dt + sub) * 16 + (c & 1) * 8;
  }

  // Pages of a 1,024-key window, one 16-key granule per lane; the next window's are
  // loaded a window ahead.
  auto window_ids = [&](int window) -> int {
    const int key = window * 1024 + lane * 16;
    return key < kend ? page_at(p, it.request, key) : -1;
  };
  int ids = window_ids(it.s0 >> 4), ids_next = window_ids((it.s0 >> 4) + 1);
  uint64_t bad_ids = __ballot((unsigned)ids >= (unsigned)p.pages);
  if ((it.s0 & 15) == 0) ids_next = ids;  // locate() takes it up
  // Where step s of this wave's keys lies: its page, its first row in there.
  __amdgpu_buffer_rsrc_t rsrc;
  int at_row = 0, bad_next = 0;
  auto locate = [&](int s) __attribute__((always_inline)) {
    if ((s & 15) == 0) {  // the next window (step s0's is there already)
      ids = ids_next;
      bad_ids = __ballot((unsigned)ids >= (unsigned)p.pages);
      ids_next = window_ids((s >> 4) + 1);
    }
    const uint32_t page = (uint32_t)__builtin_amdgcn_readlane(ids, (s & 15) * 4 + wave);
    bad_next = (int)(bad_ids >> ((s & 15) * 4)) & 15;
    at_row = (s * kWideKeys + wave * 16) & ((1 << p.page_shift) - 1);
    rsrc = fp4_rsrc(p, page, h, block_bytes, page < (uint32_t)p.pages);
  };
  dsa_u32x4 k_codes, v_codes;
  uint32_t k_scale = 0, v_scale = 0;
  auto issue = [&]() __attribute__((always_inline)) {
    k_codes = __builtin_amdgcn_raw_buffer_load_b128(rsrc, code_at, at_row * at.code_row, 0);
    k_scale = __builtin_amdgcn_raw_buffer_load_b8(rsrc, scale_at, at.k_scales + 4 * at_row, 0);
    v_codes = __builtin_amdgcn_raw_buffer_load_b128(rsrc, code_at,
                                                    at.v_codes + at_row * at.code_row, 0);
    v_scale = __builtin_amdgcn_raw_buffer_load_b8(rsrc, scale_at, at.v_scales + 4 * at_row, 0);
  };
  uint32_t unfinite = 0;  // 1 where a group of values is not of the type's numbers
  // The keys and values of step s, on their way since issue(), into their stage.
  auto expand = [&](int s, int to) __attribute__((always_inline)) {
    const bool held = s * kWideKeys + wave * 16 + own_row < kend;
    const bool number = v_scale <= kLargestScale<T>;
    unfinite |= held && !number ? 1u : 0u;
    const float k_by = fp4::scale_of(k_scale);
    const float v_by = fp4::scale_of(held && number ? v_scale : 0u);
    const int r = wave * 16 + own_row;
    if (kD == 128 || own_group < 2) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<x8*>(lds_k + to * kStage + r * kRow + k_swz(r, 4 * own_group + j) * 16) =
            fp4::expand(k_codes[j], k_by, T());
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<x8*>(lds_v + to * kStage + r * kRow + v_swz(r, 4 * own_group + j) * 16) =
            fp4::expand(v_codes[j], v_by, T());
    }
  };

  float m_run = -INFINITY, l_run = 0.f;
  dsa_f32x16 oacc[kDt];
#pragma unroll
  for (int dt = 0; dt < kDt; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) oacc[dt][r] = 0.f;

  // Step s from stage `from`, the wave's 32 or 64 keys of it; the keys and values of step
  // s + 1 go to the other stage meanwhile.
  auto compute = [&](auto tiles, int from, int s, int bad) __attribute__((always_inline)) {
    constexpr int kKt = decltype(tiles)::value;  // tiles of 32 keys
    const int row0 = kKt == 2 ? 0 : (wave >> 1) * 32;
    const int key0 = s * kWideKeys + row0;
    const unsigned char* const k_lds = lds_k + from * kStage + row0 * kRow;
    const unsigned char* const v_lds = lds_v + from * kStage + row0 * kRow;
    __builtin_amdgcn_s_setprio(0);
    dsa_f32x16 sacc[kKt];
    // The values' fragments of 16 keys (two reads each), read 16 keys ahead.
    typename E::x4 vf[2][kDt][2];
    auto read_values = [&](int j) __attribute__((always_inline)) {
#pragma unroll
      for (int dt = 0; dt < kDt; ++dt) {
        // Key rows 16 j + 4 g + r (slots 0..3) and 16 j + 8 + 4 g + r (4..7).
        const unsigned char* const at_v = v_lds + vfrag[dt] + j * 16 * kRow;
        vf[j & 1][dt][0] = read_tr<T>(at_v);
        vf[j & 1][dt][1] = read_tr<T>(at_v + 8 * kRow);
      }
    };
#pragma unroll
    for (int kt = 0; kt < kKt; ++kt) {
#pragma unroll
      for (int r = 0; r < 16; ++r) sacc[kt][r] = 0.f;
#pragma unroll
      for (int i = 0; i < kUse / 16; ++i)
        sacc[kt] = E::mfma32(*reinterpret_cast<const x8*>(k_lds + (kt * 32 + qi) * kRow +
                                                          k_swz(qi, 2 * i + g) * 16),
                             qf[i], sacc[kt]);
    }
    expand(s + 1, from ^ 1);
    asm volatile("" : "+v"(unfinite));  // (here, so that the scales' register is free)
    __builtin_amdgcn_sched_barrier(0);
    issue();
    read_values(0);
    if (key0 + 32 * kKt > lim_first) {
      const int bound = lim - key0 - 4 * g;
#pragma unroll
      for (int kt = 0; kt < kKt; ++kt)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (kt * 32 + 8 * (r >> 2) + (r & 3) >= bound) sacc[kt][r] = -INFINITY;
    }
    bad >>= row0 / 16;
    if (bad != 0) {
#pragma unroll
      for (int kt = 0; kt < kKt; ++kt)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (bad & (1 << (2 * kt + (r >> 3)))) sacc[kt][r] = -INFINITY;
    }
    float mx = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < kKt; ++kt)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, sacc[kt][r]);
    // The reference moves only where a lane's own scores call for it: the row's largest is
    // not needed before.
    if (__any(mx * p.scale_log2 > m_run + kRescaleLog2)) {
      const float mx2 = dsa::pair32_max(mx) * p.scale_log2;
      const bool up = mx2 > m_run + kRescaleLog2;
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
    x8 pf[2];
    float sum0 = 0.f, sum1 = 0.f;
    auto weigh = [&](int j) __attribute__((always_inline)) {
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
        pf[j & 1][t] = pb[0];
        pf[j & 1][t + 1] = pb[1];
      }
    };
    // 16 keys' products with the next 16 keys' exponentials and reads between them.
    weigh(0);
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int j = 0; j < 2 * kKt; ++j) {
      if (j < 2 * kKt - 1) {
        read_values(j + 1);
        weigh(j + 1);
      }
#pragma unroll
      for (int dt = 0; dt < kDt; ++dt) {
        const typename E::x4 lo = vf[j & 1][dt][0], hi = vf[j & 1][dt][1];
        const x8 a = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        oacc[dt] = E::mfma32(a, pf[j & 1], oacc[dt]);
      }
      if (j < 2 * kKt - 1) {
#pragma unroll
        for (int dt = 0; dt < kDt; ++dt) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
          __builtin_amdgcn_sched_group_barrier(0x002, 7, 0);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    l_run += sum0 + sum1;
  };
  // Step s, of stage i: behind the barrier its keys and values are there; those of step
  // s + 1, in registers by then, go to the other stage, and the loads of step s + 2 go out.
  int bad_cur = 0;
  auto step = [&](auto tiles, int s, int i) __attribute__((always_inline)) {
    dsa::lds_barrier();
    const int bad_then = bad_next;
    locate(s + 2);  // (past the last key: no bytes)
    // (a wave whose rows see none of the step's keys only stages)
    if (wave_active && s * kWideKeys < lim_last) {
      compute(tiles, i, s, bad_cur);
    } else {
      expand(s + 1, i ^ 1);
      issue();
    }
    bad_cur = bad_then;
  };
  if (it.s0 < it.s1) {
    locate(it.s0);
    bad_cur = bad_next;
    issue();
    expand(it.s0, 0);
    locate(it.s0 + 1);
    issue();
    auto walk = [&](auto tiles) __attribute__((always_inline)) {
      for (int s = it.s0; s < it.s1; s += 2) {
        step(tiles, s, 0);
        if (s + 1 >= it.s1) break;
        step(tiles, s + 1, 1);
      }
    };
    if (half) walk(std::integral_constant<int, 1>());
    else walk(std::integral_constant<int, 2>());
  }

  const LateParams late = late_params();
  float l_tot = dsa::pair32_sum(l_run);
  if (__syncthreads_or((int)unfinite)) {
    const uint32_t found = unfinite_groups<T>(late, it, h, it.s0 * kWideKeys,
                                              min(it.s1 * kWideKeys, kend), lim);
#pragma unroll
    for (int dt = 0; dt < kDt; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (found >> dt & 1) oacc[dt][r] = NAN;
  }
  if (half) {
    // Waves 2 and 3 hand theirs to waves 0 and 1 (every wave is past its reads of the
    // stages), which go on with the rows.
    float* const theirs = reinterpret_cast<float*>(lds_v + (wave & 1) * 64 * kRow) + lane;
    float* const stats = reinterpret_cast<float*>(lds_k) + (wave & 1) * 128 + lane;
    if (wave >= 2) {
#pragma unroll
      for (int dt = 0; dt < kDt; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) theirs[(dt * 16 + r) * 64] = oacc[dt][r];
      stats[0] = m_run;
      stats[64] = l_tot;
    }
    dsa::lds_barrier();
    if (wave >= 2) return;
    const float m_they = stats[0], l_they = stats[64], m_all = fmaxf(m_run, m_they);
    // (no finite score: l is 0, or NaN from NaN scores)
    const float w = m_run == -INFINITY ? l_tot : __builtin_amdgcn_exp2f(m_run - m_all);
    const float w_they = m_they == -INFINITY ? l_they : __builtin_amdgcn_exp2f(m_they - m_all);
    l_tot = fmaf(w, l_tot, w_they * l_they);
    m_run = m_all;
#pragma unroll
    for (int dt = 0; dt < kDt; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float x = theirs[(dt * 16 + r) * 64];
        oacc[dt][r] = fmaf(w_they, x, w * oacc[dt][r]);
      }
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
  // O goes out through the value stages (every wave is past its reads of them: the
  // barrier of __syncthreads_or), row by row as 16-byte chunks, whole rows to a store.
  const float inv = l_tot > 0.f ? 1.f / l_tot : (l_tot == 0.f ? 0.f : l_tot);
  unsigned char* const mine = lds_v + wave * (half ? 64 : 32) * kRow;
  auto o_swz = [](int r, int c) { return kD == 128 ? c ^ (r & 15) : c ^ ((r >> 1) & 7); };
#pragma unroll
  for (int dt = 0; dt < kDt; ++dt)
#pragma unroll
    for (int rr = 0; rr < 4; ++rr) {
      typename E::x4 v4;
#pragma unroll
      for (int e = 0; e < 4; ++e) v4[e] = (T)(oacc[dt][rr * 4 + e] * inv);
      *reinterpret_cast<typename E::x4*>(mine + qi * kRow + o_swz(qi, dt * 4 + rr) * 16 + g * 8) =
          v4;
    }
  __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
  __builtin_amdgcn_wave_barrier();
  const int64_t o_at = row_ok ? (int64_t)(it.q0 + token) * late->o_st + head * late->o_sh : -1;
  constexpr int kRowsPer = 64 / kChunks;
#pragma unroll
  for (int i = 0; i < kD / 16; ++i) {
    const int r = i * kRowsPer + lane / kChunks, c = lane % kChunks;
    const x8 y = *reinterpret_cast<const x8*>(mine + r * kRow + o_swz(r, c) * 16);
    const int64_t o_row = __shfl(o_at, r);
    if (o_row >= 0 && c * 8 < late->head_dim)
      *reinterpret_cast<x8*>(static_cast<T*>(late->o) + o_row + c * 8) = y;
  }
}

}  // namespace seq
