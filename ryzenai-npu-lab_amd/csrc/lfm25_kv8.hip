// The paged 8-bit KV cache on gfx950: pages and slots for a pass (k_kv8_plan,
// k_kv8_slots), the quantizing append (k_kv8_append) and causal attention over
// the pages (k_kv8_attend_narrow for few columns, k_kv8_attend_both for prompt
// chunks and few columns beside them, k_kv8_combine).
//
// Layout: a pool of pages of `page` positions. Keys [pages][kv][page][dim],
// values [pages][kv][dim][page] (a value row of one dimension is contiguous
// along the positions, which is the order the matrix cores read it in), one
// byte each (int8 or FP8 e4m3), and one FP32 scale per page and KV head for
// keys and for values. A value stands for code * scale.
#include <algorithm>
#include <cmath>

#include "lfm25_host.h"
#include "lfm25_device.h"

namespace lfm25 {
namespace {

constexpr int kMaxRequests = LFM25_KV8_MAX_REQUESTS;
constexpr int kStatusPage = 1;  // attention: a table entry outside the pool, or a position past the table
constexpr int kStatusRows = 2;  // attention: row offsets outside the rows, or more rows than max_rows

// ------------------------------------------------------------------ plan
//
// With P the page size: held = ceil(past / P), after = ceil((past + count) /
// P), need = after - held; an exclusive sum of the needs indexes the free
// ring. Requests up to four to a thread, rows and pages one to a thread, each
// finding its request by bisection of the sums in LDS. The sums saturate at
// 2^31 - 1, which no request that is served comes near.
//
// Many rows are divided among blocks, each of which makes the sums for itself
// (a thousand lengths and a dozen lane moves; what blocks write, none reads:
// the ring's entries before the cursor's second counter are not given again,
// and a request's new pages are read from the ring). Not where the cursor is
// (or `holds`) updated in place, which some block may still have to read: then one block,
// and a second launch for the slots of more rows than kPlanRows (14,459 rows
// of 1,000 requests: 8.5 + 4.2 us, in blocks of 512 threads 8.1, of 1,024
// 8.7, of 256 9.8).
constexpr int kPlanRows = 8192, kPlanBlocks = 256;

// Inclusive sums over the wave's lanes.
template <int kCtrl, int kRows>
__device__ __forceinline__ int dpp_add_sat(int v) {
  return __builtin_elementwise_add_sat(v, __builtin_amdgcn_update_dpp(0, v, kCtrl, kRows, 0xf, false));
}
__device__ __forceinline__ int wave_sums(int v) {
  v = dpp_add_sat<0x111, 0xf>(v);  // within a row of 16 lanes: from 1, 2, 4, 8 lanes below
  v = dpp_add_sat<0x112, 0xf>(v);
  v = dpp_add_sat<0x114, 0xf>(v);
  v = dpp_add_sat<0x118, 0xf>(v);
  v = dpp_add_sat<0x142, 0xa>(v);  // the last lane of rows 0 and 2 to rows 1 and 3
  return dpp_add_sat<0x143, 0xc>(v);  // lane 31 to rows 2 and 3
}

// The last index i of at[0 .. n] with at[i] <= x (at[0] = 0 <= x).
__device__ __forceinline__ int last_not_above(const int* at, int n, int x) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (at[mid] <= x) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

template <int kMost>
struct PlanShared {
  int waves[2][16];
  int taken, given;
  int starts[kMost + 1];  // first row of each request
  int takes[kMost + 1];   // pages taken before each request
  int gives[kMost + 1];   // pages given back before each request
  int past[kMost];
  int held[kMost];  // pages of its row (where they are given)
  uint8_t status[kMost];
};

__device__ __forceinline__ int clamp_int(int64_t v) { return v > INT32_MAX ? INT32_MAX : (int)v; }

// Exclusive sum over the block's threads; *total = the whole sum.
template <int kThreads>
__device__ __forceinline__ int block_sums(int v, int* waves, int& total) {
  const int upto = wave_sums(v);
  // the lane below's, not upto - v: the sum may have saturated
  const int below = __builtin_amdgcn_update_dpp(0, upto, 0x138, 0xf, 0xf, false);
  if (kThreads == kWave) {
    total = __builtin_amdgcn_readlane(upto, kWave - 1);
    return below;
  }
  if (lane_id() == kWave - 1) waves[wave_id()] = upto;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kThreads / kWave; ++w) {
    if (w == wave_id()) before = all;
    all = __builtin_elementwise_add_sat(all, waves[w]);
  }
  total = all;
  return __builtin_elementwise_add_sat(before, below);
}

// kThreads threads, requests up to kEach a thread. kPages, the form of
// lfm25_kv8_plan_with() (without it 1,000 requests take 8.2 us, with the tests
// for null pointers in it 8.6): `shared`, pages at each request's beginning that
// are not its own (null: none); `holds`, pages in each request's row (null: what
// its length takes), updated in place, so that one block has to do it all.
template <int kThreads, int kEach, bool kPages>
__global__ void __launch_bounds__(kThreads) k_kv8_plan(const int* __restrict__ past, const int* __restrict__ counts, int n,
                                                       int* table, int width, int* ring, int ring_n, const int64_t* cursor,
                                                       int* __restrict__ row_starts, int* __restrict__ slots, int rows,
                                                       int64_t* next_cursor, int* __restrict__ status, int shift,
                                                       const int* __restrict__ shared_or_null, int* holds_or_null) {
  const int* const shared = kPages ? shared_or_null : nullptr;
  int* const holds = kPages ? holds_or_null : nullptr;
  extern __shared__ uint4 dynamic[];
  PlanShared<kThreads * kEach>& sh = *reinterpret_cast<PlanShared<kThreads * kEach>*>(dynamic);
  const int t = threadIdx.x, page = 1 << shift, everyone = (int)gridDim.x * kThreads, me = (int)blockIdx.x * kThreads + t;
  const bool first_block = blockIdx.x == 0;
  int p[kEach], c[kEach], others[kEach], had[kEach];
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const int b = t * kEach + j;
    p[j] = b < n ? past[b] : 0;
    c[j] = b < n ? counts[b] : 0;
    others[j] = shared && b < n ? shared[b] : 0;
    had[j] = holds && b < n ? holds[b] : 0;
  }
  const int64_t taken = cursor[0], given = cursor[1];
  const int64_t window = given - taken;
  const bool sound_ring = taken >= 0 && window >= 0 && window <= ring_n;
  const int free = sound_ring ? (int)window : 0;
  int v = 0, all_rows, total;
#pragma unroll
  for (int j = 0; j < kEach; ++j) v = __builtin_elementwise_add_sat(v, max(c[j], 0));
  if (t == 0) sh.taken = sh.given = 0;
  int row = block_sums<kThreads>(v, sh.waves[0], all_rows);
  // What each request asks for; the row offsets decide which fit the rows. (As
  // one expression each: carried through branches, the arrays were compiled to
  // registers that other branches had overwritten.)
  int need[kEach], give[kEach], why[kEach], needs = 0, gifts = 0;
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const int b = t * kEach + j;
    if (b < n) {
      sh.starts[b] = row;
      sh.past[b] = p[j];
    }
    row = __builtin_elementwise_add_sat(row, max(c[j], 0));
    const int64_t least = ((int64_t)p[j] + page - 1) >> shift, after = ((int64_t)p[j] + max(c[j], 0) + page - 1) >> shift;
    const int64_t held = holds ? had[j] : least;
    if (holds && b < n) sh.held[b] = had[j];
    const bool length = p[j] < 0 || held < least || held > width || others[j] < 0 || others[j] > width || (c[j] > 0 && p[j] >> shift < others[j]);
    why[j] = length                       ? LFM25_KV8_LENGTH
             : c[j] < 0                   ? 0
             : after > width              ? LFM25_KV8_TABLE
             : c[j] > 0 && row > rows     ? LFM25_KV8_ROWS
                                          : 0;
    need[j] = why[j] == 0 && c[j] > 0 ? max((int)(after - held), 0) : 0;
    give[j] = why[j] == 0 && c[j] < 0 ? max((int)held - others[j], 0) : 0;
    needs = __builtin_elementwise_add_sat(needs, need[j]);
    gifts = __builtin_elementwise_add_sat(gifts, give[j]);
  }
  int take = block_sums<kThreads>(needs, sh.waves[1], total);
  if (t == 0) sh.takes[n] = total, sh.starts[n] = all_rows;
  if (t == 0 && first_block) row_starts[n] = all_rows;
  int back = block_sums<kThreads>(gifts, sh.waves[0], total);  // (everyone has read its sums of rows)
  if (t == 0) sh.gives[n] = total;
  // The sums only grow, so every request after the first that the pool cannot
  // serve is refused too, if it needs a page: the pages up to the last one
  // served go to the requests served, in order.
  int last_take = 0, last_back = 0;
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const int b = t * kEach + j;
    if (b < n) sh.takes[b] = take, sh.gives[b] = back;
    take = __builtin_elementwise_add_sat(take, need[j]);
    back = __builtin_elementwise_add_sat(back, give[j]);
    const bool takes = need[j] > 0, gives = give[j] > 0;
    const bool no = (takes && take > free) || (gives && (!sound_ring || (int64_t)free + back > ring_n));
    last_take = takes && !no ? take : last_take;
    last_back = gives && !no ? back : last_back;
    const int reason = no ? LFM25_KV8_POOL : why[j];
    if (b < n) sh.status[b] = (uint8_t)reason;
    if (b < n && first_block) status[b] = reason, row_starts[b] = sh.starts[b];
    if (holds && b < n && reason == 0) holds[b] = c[j] < 0 ? 0 : had[j] + need[j];
  }
  if (last_take > 0) atomicMax(&sh.taken, last_take);
  if (last_back > 0) atomicMax(&sh.given, last_back);
  __syncthreads();
  const int mine = sh.taken, returned = sh.given;
  const auto place = [&](int64_t at) {  // ring entry of a counter
    return at <= INT32_MAX ? (int)((uint32_t)at % (uint32_t)ring_n) : (int)(at % ring_n);
  };
  const int head = sound_ring ? place(taken) : 0, tail = sound_ring ? place(given) : 0;
  const auto at = [&](int from, int k) {  // ring entry k past `from`, k <= ring_n
    const int64_t i = (int64_t)from + k;
    return (int)(i >= ring_n ? i - ring_n : i);
  };
  const auto held_by = [&](int b) { return holds ? sh.held[b] : (int)(((int64_t)sh.past[b] + page - 1) >> shift); };
  for (int k = me; k < mine; k += everyone) {
    const int b = last_not_above(sh.takes, n, k);
    table[(size_t)b * width + held_by(b) + (k - sh.takes[b])] = ring[at(head, k)];
  }
  for (int k = me; k < returned; k += everyone) {
    const int b = last_not_above(sh.gives, n, k);
    ring[at(tail, k)] = table[(size_t)b * width + (shared ? shared[b] : 0) + (k - sh.gives[b])];
  }
  if (rows <= kPlanRows || gridDim.x > 1) {
    // Four rows at a time, their page numbers asked for together. (From the
    // ring where they are new: another thread may not have put them into the
    // table yet.)
    constexpr int kAhead = 4;
    for (int64_t r0 = me; r0 < rows; r0 += (int64_t)kAhead * everyone) {
      int id[kAhead], in_page[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int r = clamp_int(r0 + (int64_t)i * everyone);
        id[i] = -1;
        if (r < min(rows, all_rows)) {
          const int b = last_not_above(sh.starts, n, r);
          if (b < n && !sh.status[b]) {
            const int pos = sh.past[b] + (r - sh.starts[b]), held = held_by(b), e = pos >> shift;
            in_page[i] = pos & (page - 1);
            id[i] = e < held ? table[(size_t)b * width + e] : ring[at(head, sh.takes[b] + e - held)];
          }
        }
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int r = clamp_int(r0 + (int64_t)i * everyone);
        if (r < rows) slots[r] = id[i] >= 0 && id[i] <= (INT32_MAX >> shift) ? id[i] * page + in_page[i] : -1;
      }
    }
  }
  if (t == 0 && first_block) {
    next_cursor[0] = taken + mine;
    next_cursor[1] = given + returned;
  }
}

// Slots of many rows, from what k_kv8_plan wrote, a row a thread.
constexpr int kSlotThreads = 256;

__global__ void __launch_bounds__(kSlotThreads) k_kv8_slots(const int* __restrict__ past, int n, const int* __restrict__ table,
                                                            int width, const int* __restrict__ row_starts,
                                                            const int* __restrict__ status, int* __restrict__ slots, int rows,
                                                            int shift) {
  __shared__ int starts[kMaxRequests + 1];
  for (int i = threadIdx.x; i <= n; i += kSlotThreads) starts[i] = row_starts[i];
  __syncthreads();
  const int r = blockIdx.x * kSlotThreads + threadIdx.x;
  if (r >= rows) return;
  int slot = -1;
  const int b = last_not_above(starts, n, r);
  if (b < n) {
    const int refused = status[b], first = past[b];
    if (!refused) {
      const int pos = first + (r - starts[b]), id = table[(size_t)b * width + (pos >> shift)];
      if (id >= 0 && id <= (INT32_MAX >> shift)) slot = (id << shift) + (pos & ((1 << shift) - 1));
    }
  }
  slots[r] = slot;
}

// ------------------------------------------------------------------ 8-bit codes

template <bool kFp8>
struct Code;

// int8: -127 .. 127 (kMost), to the nearest, ties to even.
template <>
struct Code<false> {
  static constexpr int kMostExponent = 6;     // 127 = 1.984375 * 2^6
  static constexpr uint32_t kMostMantissa = 0x7eu;  // the BF16 mantissa bits of 1.984375
  // (of values in -kMost .. kMost: 1.5 * 2^23 + v has the rounded v, modulo
  // 256, in its last byte)
  __device__ static __forceinline__ uint32_t rounded(float v) { return __float_as_uint(v + 0x1.8p23f); }
  __device__ static __forceinline__ uint32_t four(float a, float b, float c, float d) {
    const uint32_t lo = __builtin_amdgcn_perm(rounded(b), rounded(a), 0x0c0c0400u);
    const uint32_t hi = __builtin_amdgcn_perm(rounded(d), rounded(c), 0x0c0c0400u);
    return __builtin_amdgcn_perm(hi, lo, 0x05040100u);
  }
  __device__ static __forceinline__ void values(uint32_t w, float (&f)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = (float)(int8_t)(w >> (8 * i));
  }
  // four codes as BF16 pairs; every code is a BF16 number, so the upper half
  // of its FP32 form is exact
  __device__ static __forceinline__ void pairs(uint32_t w, uint32_t& lo, uint32_t& hi) {
    float f[4];
    values(w, f);
    lo = __builtin_amdgcn_perm(__float_as_uint(f[1]), __float_as_uint(f[0]), 0x07060302u);
    hi = __builtin_amdgcn_perm(__float_as_uint(f[3]), __float_as_uint(f[2]), 0x07060302u);
  }
};

// FP8 e4m3 (finite values up to kMost, 448), to the nearest, ties to even.
template <>
struct Code<true> {
  static constexpr int kMostExponent = 8;     // 448 = 1.75 * 2^8
  static constexpr uint32_t kMostMantissa = 0x60u;  // the BF16 mantissa bits of 1.75
  __device__ static __forceinline__ uint32_t four(float a, float b, float c, float d) {
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false), true);
  }
  __device__ static __forceinline__ void values(uint32_t w, float (&f)[4]) {
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    f[0] = a[0], f[1] = a[1], f[2] = b[0], f[3] = b[1];
  }
  __device__ static __forceinline__ void pairs(uint32_t w, uint32_t& lo, uint32_t& hi) {
    lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, 1.0f, false));
    hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, 1.0f, true));
  }
};

// ------------------------------------------------------------------ append
//
// A page's rows of one KV head, all its dimensions, are one scale: the largest
// magnitude first (a pass over the new rows, kept in registers), then the
// codes. Keys are stored as they come, values turned (positions of a dimension
// lie together). Few bytes move (4,096 rows, 8 heads of 64: 13 MB in 6.0 us,
// 2.1 TB/s, of which launch and slots are 2.6): what bounds it is the chain of
// slots, rows and, in a page that was begun before, scale and old codes. Of
// 3,181 rows of 7 requests, 128 dims, 12.4 us, the longest block takes 10.7:
// it finds five runs that begin in its rows. Runs each to a wave where there
// are several shorten that (11.8) and lengthen all else by 4 to 10%.

struct Append {
  const uint16_t* x[2];  // keys, values: rows of kv * dim BF16 values
  int64_t stride[2];     // elements between rows
  uint8_t* cache[2];
  float* scales[2];
  const int* slots;
  int rows, kv, pages, shift, chunk;
};

constexpr int kAppendThreads = 256;
constexpr float kLargest = 0x1.ep127f;  // 1.875 * 2^127: its code times its scale is finite in both formats
constexpr int kSmallestScale = -120;

// The smallest power of two s with largest <= kMost * s, from the largest
// value's BF16 magnitude bits (its exponent, plus one where its mantissa is
// past kMost's). An FP8 code keeps its 3 mantissa bits at any such s, and
// both formats move to a larger s by an exact power of two, so that what is
// stored does not depend on how rows were divided among calls but for the
// rounding of what falls off the end (at most one step in all, 1/2 + 1/4 + ..).
template <bool kFp8>
__device__ __forceinline__ float scale_for(uint32_t largest) {
  int e = (int)(largest >> 7) - 127 - Code<kFp8>::kMostExponent + ((largest & 0x7fu) > Code<kFp8>::kMostMantissa ? 1 : 0);
  if (e < kSmallestScale) e = kSmallestScale;
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

struct AppendShared {
  int largest[kAppendThreads / kWave];
};

__device__ __forceinline__ int wave_max_int(int v) {
  v = max(v, __builtin_amdgcn_mov_dpp(v, kDppQuadXor1, 0xf, 0xf, true));
  v = max(v, __builtin_amdgcn_mov_dpp(v, kDppQuadXor2, 0xf, 0xf, true));
  v = max(v, __builtin_amdgcn_mov_dpp(v, kDppRowHalfMirror, 0xf, 0xf, true));
  v = max(v, __builtin_amdgcn_mov_dpp(v, kDppRowMirror, 0xf, 0xf, true));
  return max(max(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16)),
             max(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48)));
}

// A page's scale after a run came into it. value() is bf16 / scale (0 in a
// page that is lost), rounded once: the product with the reciprocal and one
// correction by the exact remainder (Markstein), three operations instead of
// the ten of a division (for a power of two the first is exact already).
struct PageScale {
  float scale, inv, ratio;
  bool grows;
  __device__ __forceinline__ float value(uint32_t bits16) const {
    const float v = __builtin_amdgcn_fmed3f(bf16_to_f32(bits16), -kLargest, kLargest);
    const float q = v * inv;
    return fmaf(fmaf(-q, scale, v), inv, q);
  }
};

// `largest`: this thread's largest magnitude, as BF16 bits (which order as the
// values do; what is not finite is past 0x7f80). Teams of four waves meet here.
template <bool kFp8, int kTeam>
__device__ __forceinline__ PageScale page_scale(AppendShared& sh, int tid, uint32_t largest, float old, int off, float* scale_at) {
  int most = wave_max_int((int)largest);
  if (kTeam > 1) {
    if (lane_id() == 0) sh.largest[tid / kWave] = most;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kTeam; ++i) most = max(most, sh.largest[i]);
    __syncthreads();  // read before the next run writes
  }
  const bool lost = most >= 0x7f80 || old != old;  // not finite, or the page was lost before
  PageScale p;
  p.scale = lost ? 0.0f : fmaxf(old, scale_for<kFp8>((uint32_t)most));
  p.inv = lost ? 0.0f : 1.0f / p.scale;
  p.grows = !lost && off > 0 && p.scale > old;
  p.ratio = p.grows ? old * p.inv : 1.0f;
  if (tid == 0 && (off == 0 || lost || p.grows)) *scale_at = lost ? __uint_as_float(0x7fc00000u) : p.scale;
  return p;
}

template <bool kFp8>
__device__ __forceinline__ uint32_t moved(uint32_t w, float ratio) {
  float f[4];
  Code<kFp8>::values(w, f);
  return Code<kFp8>::four(f[0] * ratio, f[1] * ratio, f[2] * ratio, f[3] * ratio);
}

__device__ __forceinline__ uint32_t largest_of(uint32_t w, uint32_t so_far) {
  return max(so_far, max(w & 0x7fffu, (w >> 16) & 0x7fffu));
}

// A run: rows [r0, r0 + len), at positions off .. off + len of page id.
struct Run {
  int r0, len, id, off;
};

// A run's keys of KV head h by kTeam waves: 8 dimensions of a row a thread
// and unit; the first kKept units' values stay in registers between the
// maximum and the codes, the others are read again.
template <int D, bool kFp8, int kTeam>
__device__ __forceinline__ void append_keys(const Append& a, AppendShared& sh, int h, const Run& run, int tid) {
  constexpr int kPer = D / 8, kThreads = kTeam * kWave, kKept = 4;
  uint8_t* const cache = a.cache[0] + (((size_t)run.id * a.kv + h) * (size_t)D << a.shift);
  float* const scale_at = a.scales[0] + (size_t)run.id * a.kv + h;
  const int64_t stride = a.stride[0];
  const uint16_t* const x = a.x[0] + (size_t)run.r0 * stride + (size_t)h * D;
  const int units = run.len * kPer;
  const auto read = [&](int u) { return load8(x + (u / kPer) * stride + 8 * (u % kPer)); };
  Pack8 kept[kKept];
#pragma unroll
  for (int i = 0; i < kKept; ++i) kept[i] = read(min(tid + i * kThreads, units - 1));
  const float old = run.off > 0 ? *scale_at : 0.0f;
  uint32_t largest = 0;
#pragma unroll
  for (int i = 0; i < kKept; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) largest = largest_of(kept[i].w[k], largest);
  for (int u = tid + kKept * kThreads; u < units; u += kThreads) {
    const Pack8 w = read(u);
#pragma unroll
    for (int k = 0; k < 4; ++k) largest = largest_of(w.w[k], largest);
  }
  const PageScale p = page_scale<kFp8, kTeam>(sh, tid, largest, old, run.off, scale_at);
  const auto write = [&](int u, const Pack8& w) {
    uint2 c;
    c.x = Code<kFp8>::four(p.value(w.w[0] & 0xffffu), p.value(w.w[0] >> 16), p.value(w.w[1] & 0xffffu), p.value(w.w[1] >> 16));
    c.y = Code<kFp8>::four(p.value(w.w[2] & 0xffffu), p.value(w.w[2] >> 16), p.value(w.w[3] & 0xffffu), p.value(w.w[3] >> 16));
    *reinterpret_cast<uint2*>(cache + (size_t)run.off * D + 8 * u) = c;
  };
#pragma unroll
  for (int i = 0; i < kKept; ++i)
    if (tid + i * kThreads < units) write(tid + i * kThreads, kept[i]);
  for (int u = tid + kKept * kThreads; u < units; u += kThreads) write(u, read(u));
  if (p.grows) {
    for (int u = tid; u < run.off * (D / 16); u += kThreads) {
      uint4 w = *reinterpret_cast<const uint4*>(cache + (size_t)u * 16);
      w.x = moved<kFp8>(w.x, p.ratio), w.y = moved<kFp8>(w.y, p.ratio), w.z = moved<kFp8>(w.z, p.ratio), w.w = moved<kFp8>(w.w, p.ratio);
      *reinterpret_cast<uint4*>(cache + (size_t)u * 16) = w;
    }
  }
}

// A run's values: two dimensions of 8 positions a thread and unit, since a
// dimension's positions are contiguous in the cache. No byte has two writers:
// whole new units and changed old ones are stored as 8 bytes, a few new
// positions as bytes.
template <int D, bool kFp8, int kTeam>
__device__ __forceinline__ void append_values(const Append& a, AppendShared& sh, int h, const Run& run, int tid) {
  constexpr int kPer = D / 2, kThreads = kTeam * kWave, kKept = 2;
  uint8_t* const cache = a.cache[1] + (((size_t)run.id * a.kv + h) * (size_t)D << a.shift);
  float* const scale_at = a.scales[1] + (size_t)run.id * a.kv + h;
  const int64_t stride = a.stride[1];
  const uint16_t* const x = a.x[1] + (size_t)run.r0 * stride + (size_t)h * D;
  const int off = run.off, to = run.off + run.len, b0 = off >> 3, units = (((to + 7) >> 3) - b0) * kPer;
  struct Words {
    uint32_t w[8];
  };
  // (positions outside the run repeat its first or last row: no larger, and not written)
  const auto read = [&](int u) {
    const int d = 2 * (u % kPer), r = 8 * (b0 + u / kPer) - off;
    Words w;
#pragma unroll
    for (int i = 0; i < 8; ++i) w.w[i] = *reinterpret_cast<const uint32_t*>(x + min(max(r + i, 0), run.len - 1) * stride + d);
    return w;
  };
  Words kept[kKept];
#pragma unroll
  for (int i = 0; i < kKept; ++i) kept[i] = read(min(tid + i * kThreads, units - 1));
  const float old = off > 0 ? *scale_at : 0.0f;
  uint32_t largest = 0;
#pragma unroll
  for (int i = 0; i < kKept; ++i)
#pragma unroll
    for (int k = 0; k < 8; ++k) largest = largest_of(kept[i].w[k], largest);
  for (int u = tid + kKept * kThreads; u < units; u += kThreads) {
    const Words w = read(u);
#pragma unroll
    for (int k = 0; k < 8; ++k) largest = largest_of(w.w[k], largest);
  }
  const PageScale p = page_scale<kFp8, kTeam>(sh, tid, largest, old, off, scale_at);
  const auto write = [&](int u, const Words& w) {
    const int d = 2 * (u % kPer), p0 = 8 * (b0 + u / kPer);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      uint8_t* const at = cache + ((size_t)(d + k) << a.shift) + p0;
      uint32_t c[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float f[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = p.value(k ? w.w[4 * i + j] >> 16 : w.w[4 * i + j] & 0xffffu);
        c[i] = Code<kFp8>::four(f[0], f[1], f[2], f[3]);
      }
      if (p0 >= off && p0 + 8 <= to) {
        *reinterpret_cast<uint2*>(at) = uint2{c[0], c[1]};
      } else if (p.grows && p0 < off) {  // old positions before `off`, the run's behind them
        const uint2 was = *reinterpret_cast<const uint2*>(at);
        const uint32_t o[2] = {was.x, was.y};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t m = moved<kFp8>(o[i], p.ratio);
          uint32_t r = 0;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int pos = p0 + 4 * i + j;
            r |= (pos < off ? m : pos < to ? c[i] : o[i]) & (0xffu << (8 * j));
          }
          c[i] = r;
        }
        *reinterpret_cast<uint2*>(at) = uint2{c[0], c[1]};
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (p0 + i >= off && p0 + i < to) at[i] = (uint8_t)(c[i / 4] >> (8 * (i % 4)));
      }
    }
  };
#pragma unroll
  for (int i = 0; i < kKept; ++i)
    if (tid + i * kThreads < units) write(tid + i * kThreads, kept[i]);
  for (int u = tid + kKept * kThreads; u < units; u += kThreads) write(u, read(u));
  if (p.grows) {  // the units before the run's
    for (int u = tid; u < b0 * D; u += kThreads) {
      uint8_t* const at = cache + ((size_t)(u % D) << a.shift) + 8 * (u / D);
      uint2 w = *reinterpret_cast<const uint2*>(at);
      w.x = moved<kFp8>(w.x, p.ratio), w.y = moved<kFp8>(w.y, p.ratio);
      *reinterpret_cast<uint2*>(at) = w;
    }
  }
}

// A run is consecutive rows whose slots follow one another within one page;
// each is handled whole, where it begins, so that its page's scale has one
// writer. Block (c, h, k): the runs that begin in rows [chunk c, chunk (c +
// 1)) of KV head h, keys (k = 0) or values; a long run by the block's four
// waves, a short one by one of them.
template <int D, bool kFp8>
__global__ void __launch_bounds__(kAppendThreads, 6) k_kv8_append(const Append a) {
  __shared__ AppendShared sh;
  const int h = blockIdx.y, w = wave_id(), l = lane_id(), page = 1 << a.shift;
  const int most = a.pages << a.shift;  // (the host checks that it is an int)
  const int c0 = blockIdx.x * a.chunk;
  // lane l: the slot of row c0 + l
  const int slot = c0 + l < a.rows ? a.slots[c0 + l] : -1;
  int before = __shfl_up(slot, 1, kWave);
  if (l == 0) before = c0 > 0 ? a.slots[c0 - 1] : -1;
  const bool begins = slot >= 0 && slot < most && l < a.chunk && !((slot & (page - 1)) != 0 && before == slot - 1);
  int turn = 0;
  for (uint64_t heads = __ballot(begins); heads; heads &= heads - 1) {
    const int at = __builtin_ctzll(heads), first = __builtin_amdgcn_readlane(slot, at);
    Run run;
    run.r0 = c0 + at;
    run.id = first >> a.shift;
    run.off = first & (page - 1);
    const uint64_t on = __ballot(l > at && slot == first + (l - at) && run.off + (l - at) < page);
    run.len = 1 + __builtin_ctzll(~(on >> at >> 1));
    if (at + run.len == kWave) {  // it may go on behind the rows that were looked at
      while (true) {
        const int k = run.len + l;
        const bool more = run.off + k < page && run.r0 + k < a.rows && a.slots[min(run.r0 + k, a.rows - 1)] == first + k;
        const uint64_t stop = ~__ballot(more);
        run.len += stop ? __builtin_ctzll(stop) : kWave;
        if (stop) break;
      }
    }
    if (run.len >= 8) {
      if (blockIdx.z == 0) append_keys<D, kFp8, 4>(a, sh, h, run, threadIdx.x);
      else append_values<D, kFp8, 4>(a, sh, h, run, threadIdx.x);
    } else {
      if ((turn & 3) == w) {
        if (blockIdx.z == 0) append_keys<D, kFp8, 1>(a, sh, h, run, l);
        else append_values<D, kFp8, 1>(a, sh, h, run, l);
      }
      ++turn;
    }
  }
}

// ------------------------------------------------------------------ attention
//
// Row i of request b stands at position past[b] + i and attends to positions
// 0 .. past[b] + i: out = sum_j p_j v_j vs_j / sum_j p_j with p_j = e^(c ks_j
// q . k_j - m). One pass over the keys with the running maximum m (in units
// of log2) and sum in FP32. The scores are formed transposed (keys are the
// products' rows, queries the columns), so that a lane's scores are
// consecutive keys of one query and become the second operand of the value
// product where they are, without a move between lanes: the rows of the key
// operand are assigned to positions so that it comes out that way.
//
// A unit is 64 positions: four segments of 16, each within one page (pages
// are multiples of 16 positions), so a segment has one key and value scale.
// Neither costs an operation per score: the key scale is the factor of the
// exponent's one fused multiply-add, the value scale its addend as a logarithm,
// and the sum of a segment's probabilities takes that factor back out in FP32,
// one operation a segment.
constexpr int kUnit = 64;

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

struct Attend {
  const uint16_t* q;
  int64_t q_stride;  // elements between rows
  const uint8_t* k;
  const uint8_t* v;
  const float* ks;
  const float* vs;
  const int* table;
  const int* past;
  const int* starts;
  uint16_t* out;
  float* part;      // results of parts: [narrow part][16 columns][D], [wide part][128 columns][D]
  float2* part_ml;  // and their maxima and sums
  int* status;
  int width, rows, kv, group, pages, shift, requests, max_rows;
  int narrow_share;  // parts that the narrow requests together are divided into, beside one each; 0: not divided
  int narrow_least;  // least units of a part
  int wide_splits, wide_blocks, early_blocks, narrow_blocks;
  int narrow_items;     // of a block, beside wide tiles
  int narrow_columns;   // a request of at most so many is narrow
  size_t narrow_parts;  // columns of the narrow parts in `part`
  float scale;  // log2(e) * the softmax scale
};

__device__ __forceinline__ void raise(int* status, int bit) {
  if (status != nullptr) atomicOr(status, bit);
}

// A request as the attention takes it.
struct Request {
  int row0, count, past;
  int cap;  // positions that may be attended to
  int len;  // positions that its last row sees, at most cap
  bool narrow;
};

// Positions that are attended to, of those that a table's row can stand for:
// what the kernels look ahead of a position (a few rounds of units) is an int
// too, and must not come out negative.
constexpr int kMostPositions = INT32_MAX - 65535;
__device__ __forceinline__ int positions_of(const Attend& a) {
  return (int)min((int64_t)a.width << a.shift, (int64_t)kMostPositions);
}

__device__ __forceinline__ bool request_at(const Attend& a, int b, Request& r) {
  const int s0 = a.starts[b], s1 = a.starts[b + 1];
  r.past = a.past[b];
  if (s1 == s0) return false;
  if (s0 < 0 || s1 < s0 || s1 > a.rows || s1 - s0 > a.max_rows) {
    raise(a.status, kStatusRows);
    return false;
  }
  r.row0 = s0;
  r.count = s1 - s0;
  r.cap = positions_of(a);
  const int64_t len = (int64_t)r.past + r.count;
  r.past = min(r.past, INT32_MAX - r.count);  // (past any table either way; positions stay ints)
  r.len = len < 0 ? 0 : len > r.cap ? r.cap : (int)len;
  r.narrow = (int64_t)r.count * a.group <= a.narrow_columns;
  if (len > r.cap) raise(a.status, kStatusPage);
  return true;
}

__device__ __forceinline__ float across_max16(float v) {  // over lanes l, l ^ 16, l ^ 32, l ^ 48
  const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
  const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(y[0]), __uint_as_float(y[1]));
}
__device__ __forceinline__ float across_sum16(float v) {
  const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(x[0]) + __uint_as_float(x[1]);
  const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(y[0]) + __uint_as_float(y[1]);
}
__device__ __forceinline__ float across_max32(float v) {  // over lanes l, l ^ 32
  const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(y[0]), __uint_as_float(y[1]));
}
__device__ __forceinline__ float across_sum32(float v) {
  const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(y[0]) + __uint_as_float(y[1]);
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  bf16x2 r;
  r[0] = (__bf16)a;
  r[1] = (__bf16)b;
  return __builtin_bit_cast(uint32_t, r);
}

template <bool kFp8>
__device__ __forceinline__ bf16x8 codes8(uint32_t a, uint32_t b) {
  uint4 r;
  Code<kFp8>::pairs(a, r.x, r.y);
  Code<kFp8>::pairs(b, r.z, r.w);
  return __builtin_bit_cast(bf16x8, r);
}

// The largest of three, one instruction; NaN if one is (the column is NaN
// then in any case), so that no operand has to be quieted first, as fmaxf()
// does with the matrix cores' results.
__device__ __forceinline__ float largest(float a, float b, float c) {
  return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c);
}
__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float nan_of() { return __uint_as_float(0x7fc00000u); }

// log2 of a value scale, whole for a power of two; kNoValue for 0 (below any
// scale's, subnormal ones included, and a number, so that nothing below has to
// tell it from the others), NaN for one that is not finite or is negative.
constexpr float kNoValue = -150.0f;
__device__ __forceinline__ float scale_log2(float s) {
  if (__float_as_uint(s) > 0x7f7fffffu) return s == 0.0f ? kNoValue : nan_of();
  const float m = __builtin_amdgcn_frexp_mantf(s);  // in [1/2, 1), of subnormals too; 0 for 0
  return fmaxf((float)__builtin_amdgcn_frexp_expf(s) + (m == 0.5f ? -1.0f : __builtin_amdgcn_logf(m)), kNoValue);
}

// A segment's scales as the kernels use them. A page that cannot be read, or
// a value scale that is not a number, has to be NaN to the rows that attend
// to it and nothing to the others: the key scale carries it, since masked
// scores are replaced, and its values count as 0.
struct Scales {
  float ks;  // key scale * log2(e) * softmax scale
  float lv;  // log2 of the value scale; kNoValue: the values count as 0
};

// The sum of two BF16 numbers and an FP32 one.
__device__ __forceinline__ float add2(uint32_t p, float sum) {
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, p), __builtin_bit_cast(bf16x2, 0x3f803f80u), sum, false);
}

// The running statistics of a column (a query), all its own. With t a score
// and lv the log2 of its position's value scale: m is the largest t and `top`
// the largest t + lv that it sees (kLowest, a number, before it sees any). The
// value product's weights are e = 2^(t + lv - top), so that none is above 1 and
// the largest is 1, whatever the scales; the probabilities of the sum are 2^(t
// - m) = e 2^(top - m - lv), one factor for a segment's.
//
// Where that factor is past 2^64 (a page whose scale is that far below what
// the others make of the row; 2^-120 is that of a page of zeros) the weights
// would lose what the sum needs: then it takes exponentials of its own.
//
// Both maxima move only when they are passed by more than 2^8: that leaves
// every weight below 2^8 and their ratios as they are.
constexpr float kLowest = -0x1.fffffep127f, kSlack = 8.0f, kMostBack = 64.0f;

// 2^(top - m) as two factors, since it may be smaller than FP32's smallest normal number.
struct Unit {
  float a, b;
};
__device__ __forceinline__ Unit unit_of(float top, float m) {
  const float x = fmaxf(top - m, -400.0f), h = __builtin_rintf(0.5f * x);  // (whole, if x is)
  return Unit{exp2_of(h), exp2_of(x - h)};
}

constexpr int kMostNarrowParts = 64;  // of one request

// A part's share of a whole: its sum against the common maximum (0 for a part
// that saw nothing).
__device__ __forceinline__ float part_weight(float m, float all, float sum) { return exp2_of(m - all) * sum; }

__device__ __forceinline__ int uniform_of(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
__device__ __forceinline__ float uniform_of(float v, int lane) {
  return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), lane));
}

// ---- few columns: single tokens
//
// Up to 16 columns (rows x query heads of one KV head) of one request. Each
// wave takes every kWaves-th unit of the block's range and reads keys and
// values from the cache straight into the operands' registers, the next
// unit's while this one is computed (and the page numbers of the one after):
// no LDS, no barrier until the waves' sums are joined.
//
// Where the requests fill the chip, its memory bounds it (64 requests of
// 3,100 to 4,100 positions, 8 KV heads of 64, int8: 237 MB in 50 us, 4.7
// TB/s). Below that it is one wave's chain: about 1.7 us a unit, half of it
// the 192 instructions that make BF16 of int8 codes (FP8: 64), behind 3 us
// to the first keys (lengths, page numbers, data) and 1.4 for the join. So
// blocks have eight waves (4 to 8: 64 requests 57 -> 51 us, 8 x 8,192
// positions of 128 dims 41 -> 31; 16: no better), and few requests are
// divided into parts of as little as one unit a wave (4,096 positions: 10.9
// us; two units a wave 12.9).
template <int D>
struct NarrowUnit {
  uint4 k[4][D / 64];
  uint4 v[D / 16];
  float ks, vs;  // of this lane's segment, l / 16
  bool bad;
};
struct NarrowIds {
  int k, v;  // this lane's pages, as the table has them
};

// The pages of unit u: keys' rows are positions 16 (r / 4) + 4 t + r % 4 of
// operand row r = l % 16, values segment l / 16. Past the last position: 0.
__device__ __forceinline__ NarrowIds narrow_ids(const Attend& a, const int* row, int len, int u) {
  const int l = lane_id(), at_k = u * kUnit + 16 * ((l & 15) >> 2), at_v = u * kUnit + 16 * (l >> 4);
  NarrowIds x{0, 0};
  if (at_k < len) x.k = row[at_k >> a.shift];
  if (at_v < len) x.v = row[at_v >> a.shift];
  return x;
}

template <int D>
__device__ __forceinline__ void narrow_load(const Attend& a, int h, int u, const NarrowIds& id, NarrowUnit<D>& x) {
  const int l = lane_id(), r = l & 15, g = l >> 4, page = 1 << a.shift;
  const int at_k = u * kUnit + 16 * (r >> 2), at_v = u * kUnit + 16 * g;
  const uint32_t id_k = (uint32_t)id.k < (uint32_t)a.pages ? id.k : 0, id_v = (uint32_t)id.v < (uint32_t)a.pages ? id.v : 0;
  x.bad = (uint32_t)id.v >= (uint32_t)a.pages;
  const uint32_t page_bytes = (uint32_t)((a.kv << a.shift) * D), head_bytes = (uint32_t)((h << a.shift) * D);
  const uint8_t* k = a.k + ((size_t)id_k * page_bytes + (head_bytes + (uint32_t)(((at_k & (page - 1)) + (r & 3)) * D + g * (D / 4))));
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int c = 0; c < D / 64; ++c) x.k[t][c] = *reinterpret_cast<const uint4*>(k + (4 * t) * D + 16 * c);
  const uint8_t* v = a.v + ((size_t)id_v * page_bytes + (head_bytes + (uint32_t)((r << a.shift) + (at_v & (page - 1)))));
#pragma unroll
  for (int t = 0; t < D / 16; ++t) x.v[t] = *reinterpret_cast<const uint4*>(v + ((16 * t) << a.shift));
  const size_t head = (size_t)id_v * (uint32_t)a.kv + h;
  x.ks = a.ks[head];
  x.vs = a.vs[head];
}

template <int D, int kWaves>
struct NarrowShared {
  float m[kWaves][16], l[kWaves][16];
  float o[kWaves][16][D + 4];
};

// The narrow requests' division into parts of `per` units, found by each wave
// from the lengths: as many parts as fill the chip, whoever's keys they are,
// since lengths in a batch differ as they like (a request of 100,000
// positions beside one of 2,000: 44 us with the same number of parts for
// each, 35 with parts of the same length).
constexpr int kDivided = 256;  // requests, at most four a lane; more are not divided (see splits_for)
struct NarrowPart {
  int b, sp;    // request and which of its parts
  int first;    // its first part among all
  int parts;    // how many it has
  int per;
};

__device__ __forceinline__ uint32_t narrow_units(const Attend& a, int b, Request& rq) {
  if (b >= a.requests || !request_at(a, b, rq) || !rq.narrow) return 0;
  return max(1u, (uint32_t)(rq.len + kUnit - 1) / kUnit);
}

// Part number `at` (kPart) or the first part of request `at`, and the request;
// false if there is none.
template <bool kPart>
__device__ __forceinline__ bool narrow_find(const Attend& a, int at, NarrowPart& x, Request& rq) {
  constexpr int kEach = kDivided / kWave;
  // Parts a little longer until there are no more than wanted (each request's
  // last is shorter); with any length from the first on there are at most
  // a.requests more.
  constexpr int kTurns = 6;
  const int l = lane_id();
  const auto per_of = [&](uint32_t total, uint32_t most) {
    total = (uint32_t)uniform_of(wave_sums((int)total), kWave - 1);
    // (rounded to FP32: a bound for the combination's parts, 63 or 64)
    const uint32_t bound = (uint32_t)__builtin_amdgcn_readfirstlane((int)wave_max((float)most)) / (kMostNarrowParts - 1) + 1;
    return max(max((uint32_t)a.narrow_least, (total + a.narrow_share - 1) / a.narrow_share), bound);
  };
  if (a.requests <= kWave) {  // a lane each: no second look at the lengths
    Request my;
    const uint32_t units = narrow_units(a, l, my);
    uint32_t per = per_of(units, units), mine;
    int upto;
    for (int turn = 0;; ++turn) {
      mine = (units + per - 1) / per;
      upto = wave_sums((int)mine);
      if (turn == kTurns || uniform_of(upto, kWave - 1) <= a.narrow_share) break;
      per += per / 16 + 1;
    }
    x.per = (int)per;
    if (kPart) {
      const uint64_t reach = __ballot(upto > at);
      if (reach == 0) return false;
      x.b = __builtin_ctzll(reach);
    } else {
      x.b = at;
    }
    x.first = uniform_of(upto - (int)mine, x.b);
    x.parts = uniform_of((int)mine, x.b);
    x.sp = kPart ? at - x.first : 0;
    rq.row0 = uniform_of(my.row0, x.b), rq.count = uniform_of(my.count, x.b), rq.past = uniform_of(my.past, x.b);
    rq.len = uniform_of(my.len, x.b), rq.cap = positions_of(a);
    return x.parts > 0;
  }
  const int each = (a.requests + kWave - 1) / kWave, b0 = l * each;
  uint32_t units[kEach], total = 0, most = 0;
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    Request my;
    units[j] = j < each ? narrow_units(a, b0 + j, my) : 0;
    total += units[j];
    most = max(most, units[j]);
  }
  uint32_t per = per_of(total, most), parts[kEach];
  int mine, upto;
  for (int turn = 0;; ++turn) {
    mine = 0;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      parts[j] = j < each ? (units[j] + per - 1) / per : 0;
      mine += (int)parts[j];
    }
    upto = wave_sums(mine);
    if (turn == kTurns || uniform_of(upto, kWave - 1) <= a.narrow_share) break;
    per += per / 16 + 1;
  }
  int lane = at / each;
  if (kPart) {
    const uint64_t reach = __ballot(upto > at);
    if (reach == 0) return false;
    lane = __builtin_ctzll(reach);
  }
  x.per = (int)per;
  x.b = lane * each;
  x.first = uniform_of(upto - mine, lane);
  x.parts = uniform_of((int)parts[0], lane);
#pragma unroll
  for (int j = 1; j < kEach; ++j)
    if (j < each && (kPart ? at >= x.first + x.parts : x.b < at)) {
      ++x.b;
      x.first += x.parts;
      x.parts = uniform_of((int)parts[j], lane);
    }
  x.sp = kPart ? at - x.first : 0;
  return x.parts > 0 && request_at(a, x.b, rq);
}

// Item `index` (part, KV head) by kWaves waves, this one number w. A block's
// items, if it has several, meet at its barrier.
template <int D, bool kFp8, int kWaves, bool kAlone, bool kParts>
__device__ __forceinline__ void narrow_block(const Attend& a, int index, int w, NarrowShared<D, kWaves>& sh) {
  const int h = index % a.kv;
  NarrowPart part{index / a.kv, 0, 0, 1, INT32_MAX / 2};
  Request rq;
  bool some;
  if (kParts && a.narrow_share > 0) some = narrow_find<true>(a, part.b, part, rq);
  else some = part.b < a.requests && request_at(a, part.b, rq) && rq.narrow;
  if (!some) {
    if (kAlone) return;
    rq.len = rq.count = 0;
    part.b = 0;
  }
  const int b = __builtin_amdgcn_readfirstlane(part.b);
  rq.row0 = __builtin_amdgcn_readfirstlane(rq.row0), rq.count = __builtin_amdgcn_readfirstlane(rq.count);
  rq.past = __builtin_amdgcn_readfirstlane(rq.past), rq.len = __builtin_amdgcn_readfirstlane(rq.len);
  const int units = (rq.len + kUnit - 1) / kUnit;
  const int u0 = part.sp * part.per, u1 = min(units, u0 + part.per);
  const int l = lane_id(), r = l & 15, g = l >> 4;
  const int* row = a.table + (size_t)b * a.width;
  const int columns = rq.count * a.group;
  // this lane's column: query row i, query head j of the KV head
  const int ci = r / a.group, cj = r - ci * a.group;
  const bool live = r < columns;
  const int pos = live ? rq.past + ci : -1;
  NarrowUnit<D> next;
  int u = u0 + w;
  NarrowIds ids = narrow_ids(a, row, rq.len, u);
  if (u < u1) narrow_load<D>(a, h, u, ids, next);
  ids = narrow_ids(a, row, rq.len, u + kWaves);
  bf16x8 q[D / 32];
  if (kAlone || columns > 0) {
    const uint16_t* src = a.q + (size_t)(rq.row0 + (live ? ci : 0)) * a.q_stride + (size_t)(h * a.group + (live ? cj : 0)) * D + g * (D / 4);
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      Pack8 x = load8(src + 8 * c);
#pragma unroll
      for (int i = 0; i < 4; ++i) x.w[i] = !live ? 0u : pos >= rq.cap ? 0x7fc07fc0u : x.w[i];  // past the table: NaN
      q[c] = __builtin_bit_cast(bf16x8, x);
    }
  }
  float m = kLowest, top = kLowest, sum = 0.0f;
  f32x4 o[D / 16];
#pragma unroll
  for (int t = 0; t < D / 16; ++t) o[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  for (; u < u1; u += kWaves) {
    NarrowUnit<D> x = next;
    if (u + kWaves < u1) narrow_load<D>(a, h, u + kWaves, ids, next);
    ids = narrow_ids(a, row, rq.len, u + 2 * kWaves);
    f32x4 s[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      s[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        const uint4 k = x.k[t][c / 2];
        s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(c & 1 ? codes8<kFp8>(k.z, k.w) : codes8<kFp8>(k.x, k.y), q[c], s[t], 0, 0, 0);
      }
    }
    const int at = u * kUnit + 16 * g;  // this lane's first position
    const bool inside = at < rq.len;
    Scales sc{x.ks * a.scale, scale_log2(x.vs)};
    if (x.bad) raise(a.status, kStatusPage);
    if (x.bad || sc.lv != sc.lv) sc = Scales{nan_of(), kNoValue};
    const bool none = sc.lv == kNoValue;  // the segment's values count as 0
    if (!inside) sc.lv = 0.0f;
    const bool whole = u * kUnit + kUnit - 1 <= rq.past && __ballot(none) == 0;  // seen by every column
    if (!whole) {
      // values behind the last position may be anything
      const int left = none ? 0 : rq.len - at;
#pragma unroll
      for (int t = 0; t < D / 16; ++t) {
        uint32_t* const v = reinterpret_cast<uint32_t*>(&x.v[t]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int n = left - 4 * i;
          v[i] &= n >= 4 ? 0xffffffffu : n <= 0 ? 0u : (1u << (8 * n)) - 1u;
        }
      }
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (at + 4 * t + i > pos) s[t][i] = -INFINITY;
    }
    float most = -INFINITY;
#pragma unroll
    for (int t = 0; t < 4; ++t) most = largest(most, s[t][0], largest(s[t][1], s[t][2], s[t][3]));
    // (a segment that the column sees nothing of has -inf here, whatever its scale)
    most = most == -INFINITY ? most : most * sc.ks;
    const float most_top = across_max16(most + sc.lv);
    most = across_max16(most);
    bool far = false;  // the sum has taken exponentials of its own
    if (__ballot(most > m + kSlack || most_top > top + kSlack || top - m - sc.lv > kMostBack) != 0) {
      const float m_new = fmaxf(m, most), top_new = fmaxf(top, most_top);
      const float shrink = exp2_of(top - top_new);
      sum *= exp2_of(m - m_new);
#pragma unroll
      for (int t = 0; t < D / 16; ++t) o[t] *= shrink;
      m = m_new;
      top = top_new;
      far = __ballot(top - m - sc.lv > kMostBack) != 0;
      if (far) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float e = exp2_of(fmaf(s[t][i], sc.ks, -m));
            sum += !whole && at + 4 * t + i > pos ? 0.0f : e;
          }
      }
    }
    const float add = sc.lv - top;
    float part = 0.0f;  // the sum of the segment's weights
    // The weights are rounded to BF16, the value product's operand type: up to
    // 2^-8 of each, the same rounded ones in the sum. (FP16 has the bits but
    // not the range: beside a weight of 1 whose value is 0, 2^-50 still counts.)
    bf16x8 p[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      uint32_t pk[4];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        float e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          e[i] = exp2_of(fmaf(s[2 * c + t][i], sc.ks, add));
          if (!whole && at + 4 * (2 * c + t) + i > pos) e[i] = 0.0f;
        }
        pk[2 * t] = pack_bf16(e[0], e[1]);
        pk[2 * t + 1] = pack_bf16(e[2], e[3]);
        part = add2(pk[2 * t], part);
        part = add2(pk[2 * t + 1], part);
      }
      p[c] = __builtin_bit_cast(bf16x8, uint4{pk[0], pk[1], pk[2], pk[3]});
    }
    if (!far) sum = fmaf(part, exp2_of(top - m - sc.lv), sum);
#pragma unroll
    for (int t = 0; t < D / 16; ++t) {
      o[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(codes8<kFp8>(x.v[t].x, x.v[t].y), p[0], o[t], 0, 0, 0);
      o[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(codes8<kFp8>(x.v[t].z, x.v[t].w), p[1], o[t], 0, 0, 0);
    }
  }
  // Join the waves, each as its own result (so that nothing passes the range
  // of the values): o of this lane is column r, dimensions 16 t + 4 g + i.
  sum = across_sum16(sum);
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  const Unit unit = unit_of(top, m);
  if (g == 0) {
    sh.m[w][r] = m;
    sh.l[w][r] = sum;
  }
#pragma unroll
  for (int t = 0; t < D / 16; ++t)
    *reinterpret_cast<f32x4*>(&sh.o[w][r][16 * t + 4 * g]) = o[t] * inv * unit.a * unit.b;
  __syncthreads();
  const int heads = a.kv * a.group;
  for (int e = w * kWave + l; e < columns * (D / 4); e += kWaves * kWave) {
    const int c = e / (D / 4), d = 4 * (e % (D / 4));
    float all = -INFINITY;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) all = fmaxf(all, sh.m[i][c]);
    float share[kWaves], total = 0.0f;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) total += share[i] = part_weight(sh.m[i][c], all, sh.l[i][c]);
    f32x4 acc{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < kWaves; ++i) acc += (share[i] / total) * *reinterpret_cast<const f32x4*>(&sh.o[i][c][d]);
    const int i = c / a.group, j = c - i * a.group;
    const size_t at = (size_t)(rq.row0 + i) * heads + h * a.group + j;
    if (part.parts == 1) {
      uint2 y{0, 0};
      if (rq.past + i >= 0) y = uint2{pack_bf16(acc[0], acc[1]), pack_bf16(acc[2], acc[3])};
      *reinterpret_cast<uint2*>(a.out + at * D + d) = y;
    } else {
      const size_t to = (size_t)index * 16 + c;
      if (total == 0.0f) acc = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      *reinterpret_cast<f32x4*>(a.part + to * D + d) = acc;
      if (d == 0) a.part_ml[to] = float2{all, total};
    }
  }
}

template <int D, bool kFp8, int kWaves, bool kParts>
__global__ void __launch_bounds__(kWaves* kWave, D == 64 ? 4 : 2) k_kv8_attend_narrow(const Attend a) {
  extern __shared__ uint4 dynamic[];
  narrow_block<D, kFp8, kWaves, true, kParts>(a, blockIdx.x, wave_id(), *reinterpret_cast<NarrowShared<D, kWaves>*>(dynamic));
}

// ---- many columns: prompt chunks
//
// Tiles of 128 columns of one request and KV head, a wave for 32 of them
// (v_mfma_f32_32x32x16_bf16); a unit's keys and values are converted to BF16
// once for four waves. Groups of four waves share a tile, each with stages of
// its own and every third (dim 64) or second (128) unit.
//
// What bounds it is the vector work around the products (about 280
// instructions a unit and wave: 73,000 of a SIMD's 156,000 cycles at 3,900
// rows x 16 heads of 64, the matrix cores busy for 32,000) and, in what is
// left, the latency of one wave's chain, 2.3 us a round, and 7 us a block for
// its beginning and its end: one tile's longest chain of units decides how
// long a chip that holds about two tiles a CU takes. Hence the groups (one
// group: 77 us, two: 67, three: 67 when that was measured; 60 now), the
// halves of a round (below), and per-segment work moved out of the unit:
// pages and scales of 64 rounds looked up at once, a lane for each (107 -> 84
// us together with 32-bit offsets), nothing per score but the multiply-add,
// the exponential, half a maximum, half a conversion and half a dot product
// (a whole maximum: 2% more). Two scores' buffers in turn, two blocks of six
// waves a CU (80 or 128 registers spill), four groups, and ranges of equal
// length across the tiles of a batch were no faster.
constexpr int kWideWaves = 4, kWideColumns = 32 * kWideWaves;
template <int D>
struct Wide {
  static constexpr int kGroups = D == 64 ? 3 : 2, kWaves = kGroups * kWideWaves, kThreads = kWaves * kWave;
};

struct Found {
  int request, tile;  // request -1: none
  int waves[16], few[16];
};
template <int D>
struct WideStages {
  uint4 k[2][kUnit * (D / 8)];  // [position][dim], rows of D / 8 16-byte slots
  uint4 v[D * (kUnit / 8)];     // [dim][position]
  Scales s[4];                  // the segments'
};
template <int D>
struct WideShared {
  union {
    WideStages<D> group[Wide<D>::kGroups];
    f32x4 o[Wide<D>::kGroups - 1][kWideColumns][D / 4 + 1];  // the groups' results, to be joined
  };
  float2 ml[Wide<D>::kGroups - 1][kWideColumns];
  Found found;
};

// 16 rows read at one slot number spread over all 64 banks (two 128-byte rows
// or one 256-byte row make a round of the banks).
template <int kSlots>
__device__ __forceinline__ int slot_of(int row, int c) {
  return row * kSlots + (c ^ (kSlots == 8 ? (row >> 1) & 7 : row & 15));
}

// A wave's share of a unit's staging: segment w, so that its page and scales
// are the wave's and not each lane's. Keys: position 16 w + l / 4, 16
// dimensions at 16 (l % 4) (and 64 more); values: dimension l (and 64 + l),
// the segment's 16 positions. Keys run a unit ahead of values.
//
// The pages and scales of the wave's segments in the next 64 rounds, a lane
// for each, looked up and made ready together.
struct WideTable {
  int id;     // page that may be read
  Scales s;
};
struct WideEntry {  // as read
  int id;
  bool inside, bad;
  float ks, vs;
};

__device__ __forceinline__ WideEntry wide_entry(const Attend& a, const int* row, int h, int64_t at, int end) {
  WideEntry e;
  e.inside = at < end;
  e.id = e.inside ? row[at >> a.shift] : 0;
  e.bad = (uint32_t)e.id >= (uint32_t)a.pages;
  e.id = e.bad ? 0 : e.id;
  const size_t head = (size_t)e.id * a.kv + h;
  e.ks = a.ks[head];
  e.vs = a.vs[head];
  return e;
}
__device__ __forceinline__ WideTable wide_table(const Attend& a, const WideEntry& e) {
  if (e.bad && e.inside) raise(a.status, kStatusPage);
  WideTable x;
  x.id = e.id;
  x.s = Scales{e.ks * a.scale, scale_log2(e.vs)};
  if (!e.inside) x.s = Scales{0.0f, 0.0f};  // (seen by no column)
  else if (e.bad || x.s.lv != x.s.lv) x.s = Scales{nan_of(), kNoValue};
  return x;
}

// A segment of this wave: where its page's head begins in either cache, its
// scales, its first position.
struct Segment {
  size_t region;
  Scales s;
  int at;
};

template <int D>
struct WideUnit {
  uint4 k[D / 64], v[D / 64];
  Segment of_k, of_v;
};

template <int D, bool kFp8>
__device__ __forceinline__ void store_keys(WideStages<D>& sh, int w, int stage, const WideUnit<D>& x) {
  const int l = lane_id();
#pragma unroll
  for (int c = 0; c < D / 64; ++c) {
    const int row = 16 * w + (l >> 2), at = 8 * c + 2 * (l & 3);
    // at is even, so the two slots differ in their last bit
    const int s = slot_of<D / 8>(row, at);
    sh.k[stage][s] = __builtin_bit_cast(uint4, codes8<kFp8>(x.k[c].x, x.k[c].y));
    sh.k[stage][s ^ 1] = __builtin_bit_cast(uint4, codes8<kFp8>(x.k[c].z, x.k[c].w));
  }
}

template <int D, bool kFp8>
__device__ __forceinline__ void store_values(WideStages<D>& sh, int w, int end, WideUnit<D>& x) {
  const int l = lane_id();
  sh.s[w] = x.of_v.s;  // (every lane the same)
  const int left = end - x.of_v.at;
  if (left < 16 || x.of_v.s.lv == kNoValue) {
    // What lies behind the last position may be anything, and the values of
    // a page or scale that is no number count as 0.
    const int keep = x.of_v.s.lv == kNoValue ? 0 : left;
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
      uint32_t* const v = reinterpret_cast<uint32_t*>(&x.v[c]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int n = keep - 4 * i;
        v[i] &= n >= 4 ? 0xffffffffu : n <= 0 ? 0u : (1u << (8 * n)) - 1u;
      }
    }
  }
#pragma unroll
  for (int c = 0; c < D / 64; ++c) {
    const int at = slot_of<8>(l + 64 * c, 2 * w);
    sh.v[at] = __builtin_bit_cast(uint4, codes8<kFp8>(x.v[c].x, x.v[c].y));
    sh.v[at ^ 1] = __builtin_bit_cast(uint4, codes8<kFp8>(x.v[c].z, x.v[c].w));
  }
}

// A wave's columns and their running results.
template <int D>
struct WideState {
  bf16x8 q[D / 16];
  f32x16 o[D / 32];
  float m, top, sum;
  float m_past, top_past, top_m;  // m + kSlack, top + kSlack, top - m
};
struct WideScores {
  f32x16 t[2];  // positions 32 t ..
};

// The scores of one unit for one wave.
template <int D>
__device__ __forceinline__ void wide_scores(const WideStages<D>& sh, int stage, const WideState<D>& x, WideScores& s) {
  const int l = lane_id(), half = l >> 5;
  // operand row l % 32 of a key tile is position rho with bits 2 and 3
  // exchanged: the results of lane half `half`, i = 0 .. 15, are then
  // positions 16 (i / 8) + 8 half + i % 8
  const int rho = (l & 0x13) | ((l & 4) << 1) | ((l & 8) >> 1);
#pragma unroll
  for (int c = 0; c < D / 16; ++c)
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const bf16x8 k = __builtin_bit_cast(bf16x8, sh.k[stage][slot_of<D / 8>(32 * t + rho, 2 * c + half)]);
      if (c == 0) s.t[t] = f32x16{};
      s.t[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k, x.q[c], s.t[t], 0, 0, 0);
    }
}

// Those scores into the running results; kMasked: some column does not see
// all of the unit.
template <int D, bool kMasked>
__device__ __forceinline__ void wide_unit(const WideStages<D>& sh, int first, int pos, bool one_page, WideScores& s,
                                          WideState<D>& x) {
  const int l = lane_id(), half = l >> 5;
  Scales sc[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) sc[i] = sh.s[i];
  const int behind = pos - first - 8 * half;  // positions 32 t + 16 e + i past this are masked
  if (kMasked) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (32 * t + 16 * (i / 8) + i % 8 > behind) s.t[t][i] = -INFINITY;
  }
  float each[4];  // the segments' largest
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const auto at = [&](int k) { return s.t[i / 2][8 * (i % 2) + k]; };
    each[i] = largest(largest(at(0), at(1), at(2)), largest(at(3), at(4), at(5)), __builtin_elementwise_maximum(at(6), at(7)));
  }
  // (what the column sees nothing of is -inf, whatever its scale)
  const auto scaled = [&](float v, float ks) { return kMasked && v == -INFINITY ? v : v * ks; };
  float most, most_top, least;
  if (one_page) {
    most = across_max32(scaled(fmaxf(fmaxf(each[0], each[1]), fmaxf(each[2], each[3])), sc[0].ks));
    most_top = most + sc[0].lv;
    least = sc[0].lv;
  } else {
    float top[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      each[i] = scaled(each[i], sc[i].ks);
      top[i] = each[i] + sc[i].lv;
    }
    most = across_max32(fmaxf(fmaxf(each[0], each[1]), fmaxf(each[2], each[3])));
    most_top = across_max32(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])));
    least = fminf(fminf(sc[0].lv, sc[1].lv), fminf(sc[2].lv, sc[3].lv));
  }
  bool far = false;  // the sum has taken exponentials of its own
  if (__ballot(most > x.m_past || most_top > x.top_past || x.top_m - least > kMostBack) != 0) {
    const float m_new = fmaxf(x.m, most), top_new = fmaxf(x.top, most_top);
    const float shrink = exp2_of(x.top - top_new);
    x.sum *= exp2_of(x.m - m_new);
#pragma unroll
    for (int t = 0; t < D / 32; ++t) x.o[t] *= shrink;
    x.m = m_new, x.m_past = m_new + kSlack;
    x.top = top_new, x.top_past = top_new + kSlack;
    x.top_m = top_new - m_new;
    far = __ballot(x.top_m - least > kMostBack) != 0;
    if (far) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float f = exp2_of(fmaf(s.t[t][i], sc[2 * t + i / 8].ks, -x.m));
          x.sum += kMasked && 32 * t + 16 * (i / 8) + i % 8 > behind ? 0.0f : f;
        }
    }
  }
  const float of = far ? kLowest : x.top_m;  // (every factor 0)
  float add[4], back[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    add[i] = sc[i].lv - x.top;
    back[i] = exp2_of(of - sc[i].lv);
  }
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float f[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        f[i] = exp2_of(fmaf(s.t[t][8 * e + i], sc[2 * t + e].ks, add[2 * t + e]));
        if (kMasked && 32 * t + 16 * e + i > behind) f[i] = 0.0f;
      }
      // (rounded to BF16 as in the narrow form)
      const uint4 pk{pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7])};
      x.sum = fmaf(add2(pk.w, add2(pk.z, add2(pk.y, add2(pk.x, 0.0f)))), back[2 * t + e], x.sum);
      const bf16x8 p = __builtin_bit_cast(bf16x8, pk);
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        const bf16x8 v = __builtin_bit_cast(bf16x8, sh.v[slot_of<8>(32 * c + (l & 31), 4 * t + 2 * e + half)]);
        x.o[c] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, p, x.o[c], 0, 0, 0);
      }
    }
}

// The wide requests' tiles in order, each request's longest first, each in
// `splits` parts of its keys. Where there is more than one request the host
// cannot know how many tiles there are; the parts are then as many as fill
// what the narrow requests leave of the chip, at most a.wide_splits.
constexpr int kWideParts = 256, kLeastPart = 4;  // blocks that parts are made for; units in a part
struct WideItem {
  int b, tile, sp, splits, part;  // part: number of this part in the workspace
};

__device__ __forceinline__ int wide_per(int units, int splits) { return max((units + splits - 1) / splits, kLeastPart); }

// How many parts each tile is divided into, with `tiles` of them and `others`
// narrow requests.
__device__ __forceinline__ int wide_splits(const Attend& a, int tiles, int others) {
  if (a.requests == 1) return a.wide_splits;
  const int free = kWideParts - (int)min((int64_t)kWideParts, ((int64_t)others + a.narrow_share) * a.kv / a.narrow_items);
  return max(1, min(a.wide_splits, free / max(1, tiles * a.kv)));
}

// Item `index` (head first) of the block, b < 0 if there is none. Up to 64
// requests are a lane's each, and every wave finds the item for itself;
// more are looked through by the whole block.
template <int kThreads>
__device__ __forceinline__ WideItem wide_find(const Attend& a, int index, bool whole_tiles, Request& rq, Found& sh) {
  const int h = index % a.kv, item = index / a.kv;
  WideItem x;
  if (a.requests <= kWave) {
    Request my;
    const bool here = lane_id() < a.requests && request_at(a, lane_id(), my);
    const int n = here && !my.narrow ? (my.count * a.group + kWideColumns - 1) / kWideColumns : 0;
    const int upto = wave_sums(n), total = uniform_of(upto, kWave - 1);
    x.splits = wide_splits(a, total, __builtin_popcountll(__ballot(n == 0 && lane_id() < a.requests)));
    const int rank = whole_tiles ? item : item / x.splits;
    x.sp = whole_tiles ? 0 : item - rank * x.splits;
    x.part = (rank * a.kv + h) * x.splits + x.sp;
    const uint64_t reach = __ballot(upto > rank);
    x.b = reach ? __builtin_ctzll(reach) : -1;
    const int lane = max(x.b, 0);
    x.tile = uniform_of(upto, lane) - 1 - rank;
    rq.row0 = uniform_of(my.row0, lane), rq.count = uniform_of(my.count, lane), rq.past = uniform_of(my.past, lane);
    rq.len = uniform_of(my.len, lane), rq.cap = positions_of(a);
    return x;
  }
  const int each = (a.requests + kThreads - 1) / kThreads, b0 = threadIdx.x * each;
  const int l = lane_id(), w = wave_id();
  const auto tiles_of = [&](int b) {
    if (b >= a.requests) return 0;
    const int s0 = a.starts[b], s1 = a.starts[b + 1];
    if (s0 < 0 || s1 <= s0 || s1 > a.rows || s1 - s0 > a.max_rows || (int64_t)(s1 - s0) * a.group <= a.narrow_columns) return 0;
    return (int)(((int64_t)(s1 - s0) * a.group + kWideColumns - 1) / kWideColumns);
  };
  int mine = 0, few = 0;  // tiles, and requests that have none
  for (int j = 0; j < each; ++j) {
    const int n = tiles_of(b0 + j);
    mine += n;
    few += n == 0 && b0 + j < a.requests;
  }
  int upto = wave_sums(mine);
  const int few_upto = wave_sums(few);
  if (l == kWave - 1) sh.waves[w] = upto, sh.few[w] = few_upto;
  if (threadIdx.x == 0) sh.request = -1;
  __syncthreads();
  int total = 0, others = 0;
#pragma unroll
  for (int i = 0; i < kThreads / kWave; ++i) {
    if (i == w) upto += total;
    total += sh.waves[i];
    others += sh.few[i];
  }
  x.splits = wide_splits(a, total, others);
  const int rank = whole_tiles ? item : item / x.splits;
  x.sp = whole_tiles ? 0 : item - rank * x.splits;
  x.part = (rank * a.kv + h) * x.splits + x.sp;
  int first = upto - mine;
  if (rank >= first && rank < upto) {
    for (int j = 0; j < each; ++j) {
      const int n = tiles_of(b0 + j);
      if (rank >= first && rank < first + n) {
        sh.request = b0 + j;
        sh.tile = n - 1 - (rank - first);
      }
      first += n;
    }
  }
  __syncthreads();
  x.b = __builtin_amdgcn_readfirstlane(sh.request);
  x.tile = __builtin_amdgcn_readfirstlane(sh.tile);
  if (x.b >= 0) request_at(a, x.b, rq);
  return x;
}

// Positions that a tile of columns from c0 on sees, and its last query row.
__device__ __forceinline__ int wide_end(const Attend& a, const Request& rq, int c0) {
  const int last = (min(c0 + kWideColumns, rq.count * a.group) - 1) / a.group;
  const int64_t end = (int64_t)rq.past + last + 1;
  return end < 0 ? 0 : end > rq.cap ? rq.cap : (int)end;
}

template <int D, bool kFp8>
__device__ __forceinline__ void wide_block(const Attend& a, int index, WideShared<D>& sh) {
  const int h = index % a.kv, w = wave_id(), l = lane_id();
  Request rq;
  const WideItem item = wide_find<Wide<D>::kThreads>(a, index, false, rq, sh.found);
  if (item.b < 0) return;
  const int* row = a.table + (size_t)item.b * a.width;
  const int columns = rq.count * a.group, c0 = item.tile * kWideColumns, end = wide_end(a, rq, c0);
  const int units = (rq.len + kUnit - 1) / kUnit, per = wide_per(units, item.splits);
  const int u0 = item.sp * per, u1 = min((end + kUnit - 1) / kUnit, u0 + per);
  if (item.sp > 0 && u0 >= u1) return;
  constexpr int kGroups = Wide<D>::kGroups;
  const int group = w / kWideWaves, w4 = w % kWideWaves;
  WideStages<D>& mine = sh.group[group];
  constexpr int kRound = kGroups * kUnit;            // positions of a round
  const int first = (u0 + group) * kUnit + 16 * w4;  // this wave's first segment to stage
  const uint32_t page_bytes = (uint32_t)((a.kv << a.shift) * D), head_bytes = (uint32_t)((h << a.shift) * D);
  const uint32_t k_lane = (uint32_t)((l >> 2) * D + 16 * (l & 3)), v_lane = (uint32_t)(l << a.shift);
  const int in_page = (1 << a.shift) - 1;
  const WideEntry entry = wide_entry(a, row, h, (int64_t)first + kRound * l, end);
  WideTable table;
  table.id = entry.id;
  WideUnit<D> now, next;
  // Loads are made for rounds past the last too (of page 0; never used).
  const auto load_keys = [&](int i, WideUnit<D>& x) {
    x.of_k.region = (size_t)(uint32_t)uniform_of(table.id, i % kWave) * page_bytes + head_bytes;
    x.of_k.at = first + kRound * i;
    const uint8_t* const k = a.k + (x.of_k.region + (uint32_t)(x.of_k.at & in_page) * D);
#pragma unroll
    for (int c = 0; c < D / 64; ++c) x.k[c] = *reinterpret_cast<const uint4*>(k + (k_lane + 64 * c));
  };
  const auto scale_keys = [&](int i, WideUnit<D>& x) {
    x.of_k.s = Scales{uniform_of(table.s.ks, i % kWave), uniform_of(table.s.lv, i % kWave)};
  };
  const auto load_values = [&] {
    const uint8_t* const v = a.v + (next.of_v.region + (uint32_t)(next.of_v.at & in_page));
#pragma unroll
    for (int c = 0; c < D / 64; ++c) next.v[c] = *reinterpret_cast<const uint4*>(v + (v_lane + (uint32_t)((64 * c) << a.shift)));
  };
  // all that the first round needs, before anything is waited for
  load_keys(0, now);
  load_keys(1, next);
  next.of_v = now.of_k;
  load_values();
  const int half = l >> 5;
  const int column = c0 + 32 * w4 + (l & 31);
  const bool live = column < columns;
  const int ci = live ? column / a.group : 0, cj = live ? column - ci * a.group : 0;
  const int pos = live ? rq.past + ci : -1;
  WideState<D> x;
  {
    const uint16_t* src = a.q + (size_t)(rq.row0 + ci) * a.q_stride + (size_t)(h * a.group + cj) * D + 8 * half;
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      Pack8 y = load8(src + 16 * c);
#pragma unroll
      for (int i = 0; i < 4; ++i) y.w[i] = !live ? 0u : pos >= rq.cap ? 0x7fc07fc0u : y.w[i];
      x.q[c] = __builtin_bit_cast(bf16x8, y);
    }
  }
  x.m = x.top = x.m_past = x.top_past = kLowest;
  x.top_m = 0.0f;
  x.sum = 0.0f;
#pragma unroll
  for (int t = 0; t < D / 32; ++t) x.o[t] = f32x16{};
  // Rounds (a unit for each group) that every column sees whole, then the
  // others (the masks' registers are not held through the first loop).
  const int wave_last = rq.past + min((c0 + 32 * w4 + 31) / a.group, rq.count - 1);  // the last position that the wave sees
  const bool wave_live = c0 + 32 * w4 < columns;
  const int seen = max(0, rq.past + c0 / a.group + 1) / kUnit;
  const int rounds = (u1 - u0 + kGroups - 1) / kGroups, whole = max(0, (min(u1, seen) - u0) / kGroups);
  const bool large = a.shift >= 6;
  // A group's round is two halves: the unit's probabilities and value product
  // (vector work), and the next unit's scores with the staging of what follows
  // (matrix and LDS work): one group is in the first half while the other is
  // in the second, a barrier apart. Keys are staged a round ahead of values.
  const auto load = [&](int i) {  // keys of round i + 1, values of round i
    ++i;
    if (i % kWave == 0) table = wide_table(a, wide_entry(a, row, h, (int64_t)first + (int64_t)kRound * (i + l), end));
    next.of_v = next.of_k;
    load_keys(i, next);
    scale_keys(i, next);
    load_values();
  };
  const auto store = [&](int i) {
    store_keys<D, kFp8>(mine, w4, (i + 1) & 1, next);
    store_values<D, kFp8>(mine, w4, end, next);
  };
  WideScores s;
  const auto stage = [&](int i) {
    lds_barrier();
    wide_scores<D>(mine, (i + 1) & 1, x, s);
    store(i + 1);
    load(i + 2);
    lds_barrier();
  };
  table = wide_table(a, entry);
  scale_keys(0, now);
  next.of_v.s = now.of_k.s;
  scale_keys(1, next);
  store_keys<D, kFp8>(mine, w4, 0, now);
  if (group & 1) lds_barrier();
  stage(-1);
  int i = 0;
  for (; i < whole; ++i) {
    if (wave_live) wide_unit<D, false>(mine, 0, 0, large, s, x);
    stage(i);
  }
  for (; i < rounds; ++i) {
    const int at = (u0 + kGroups * i + group) * kUnit;
    if (wave_live && at <= wave_last && at < u1 * kUnit) wide_unit<D, true>(mine, at, pos, large && at + kUnit <= end, s, x);
    stage(i);
  }
  if (!(group & 1)) lds_barrier();
  // join the groups, each as its own result
  x.sum = across_sum32(x.sum);
  const float inv = x.sum == 0.0f ? 0.0f : 1.0f / x.sum;
  const Unit unit = unit_of(x.top, x.m);
  const int c = 32 * w4 + (l & 31);
  if (group) {
#pragma unroll
    for (int t = 0; t < D / 32; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        sh.o[group - 1][c][8 * t + 2 * i + half] = f32x4{x.o[t][4 * i], x.o[t][4 * i + 1], x.o[t][4 * i + 2], x.o[t][4 * i + 3]} * inv * unit.a * unit.b;
    if (half == 0) sh.ml[group - 1][c] = float2{x.m, x.sum};
  }
  __syncthreads();
  if (group || !live) return;
  float all = x.m;
#pragma unroll
  for (int g = 1; g < kGroups; ++g) all = fmaxf(all, sh.ml[g - 1][c].x);
  float share[kGroups], total = share[0] = part_weight(x.m, all, x.sum);
#pragma unroll
  for (int g = 1; g < kGroups; ++g) total += share[g] = part_weight(sh.ml[g - 1][c].x, all, sh.ml[g - 1][c].y);
  const bool single = item.splits == 1, none = !single && total == 0.0f;
#pragma unroll
  for (int g = 0; g < kGroups; ++g) share[g] = none ? 0.0f : share[g] / total;
  const int heads = a.kv * a.group;
  const size_t at = (size_t)(rq.row0 + ci) * heads + h * a.group + cj;
  const size_t part = a.narrow_parts + (size_t)item.part * kWideColumns + c;  // (narrow parts come first)
#pragma unroll
  for (int t = 0; t < D / 32; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = 32 * t + 8 * i + 4 * half;
      f32x4 y = f32x4{x.o[t][4 * i], x.o[t][4 * i + 1], x.o[t][4 * i + 2], x.o[t][4 * i + 3]} * (share[0] * inv) * unit.a * unit.b;
#pragma unroll
      for (int g = 1; g < kGroups; ++g) y += sh.o[g - 1][c][8 * t + 2 * i + half] * share[g];
      if (single) {
        uint2 z{0, 0};
        if (pos >= 0) z = uint2{pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3])};
        *reinterpret_cast<uint2*>(a.out + at * D + d) = z;
      } else {
        *reinterpret_cast<f32x4*>(a.part + part * D + d) = y;
      }
    }
  if (!single && half == 0) a.part_ml[part] = float2{all, total};
}

// Tiles and narrow requests in one launch. kItems: narrow items of a block, 0
// for a launch without any (one request), 1 where there are few of them (each
// then has all of the block's waves: 40 rows beside 5 requests on 2,048
// positions 35.6 -> 21 us). LDS as dynamic memory: a static array past half of
// a CU's makes the compiler plan for 512 registers and move results between
// their two halves.
template <int D, int kItems>
union BothShared {
  WideShared<D> wide;
  NarrowShared<D, kItems == 1 ? Wide<D>::kWaves : 4> narrow[kItems > 0 ? kItems : 1];
};

template <int D, bool kFp8, int kItems>
__global__ void __launch_bounds__(Wide<D>::kThreads, Wide<D>::kWaves / 4) k_kv8_attend_both(const Attend a) {
  extern __shared__ uint4 dynamic[];
  BothShared<D, kItems>& sh = *reinterpret_cast<BothShared<D, kItems>*>(dynamic);
  if constexpr (kItems == 0) {
    wide_block<D, kFp8>(a, blockIdx.x, sh.wide);
    return;
  }
  // The first `early_blocks` are tiles, since they take longest; those past
  // the first round of the chip, which may be none, come behind the narrow
  // requests. (Divided tiles are short: then the narrow requests come first.)
  int i = blockIdx.x;
  if (i >= a.early_blocks) i = i < a.early_blocks + a.narrow_blocks ? i + (a.wide_blocks - a.early_blocks) : i - a.narrow_blocks;
  if (i < a.wide_blocks) {
    wide_block<D, kFp8>(a, i, sh.wide);
  } else if constexpr (kItems == 1) {
    narrow_block<D, kFp8, Wide<D>::kWaves, true, true>(a, i - a.wide_blocks, wave_id(), sh.narrow[0]);
  } else {
    const int w = wave_id();
    narrow_block<D, kFp8, 4, false, true>(a, (i - a.wide_blocks) * kItems + w / 4, w % 4, sh.narrow[w / 4]);
  }
}

// ---- the parts of a split range of keys joined, in the parts' order
//
// Blocks for the columns of a request and KV head, or for a part of a wide
// tile's, more where there are few of either (a tile's 4 to 8: 64 rows on
// 8,000 positions 24.6 -> 22.5 us in all, but 22.5 -> 23.4 with 128 tiles;
// columns of a narrow block 4 to 2: 3 rows on 100,001 positions 34.4 -> 32.5).
// 4 to 6 us, of which the launch and two dependent loads are most, so the
// parts' values are asked for before their shares are known (0.3 us) and
// threads that the columns leave over take parts of their own (63 parts of 15
// columns: 11 -> 8 us with blocks of four).
constexpr int kCombineThreads = 256, kMostShares = 512;  // parts x columns: 64 x 4, 16 x 32

struct CombineSplit {
  int wide_blocks, wide_shift;        // log2 of the blocks of a tile
  int narrow_shift, narrow_columns;   // of a request and KV head; columns of one
};

struct CombineShared {
  Found found;
  float share[kMostShares];
  f32x4 sums[kCombineThreads];
};

// Sum or maximum over a lane's group of 16 or of all 64.
template <bool kAll>
__device__ __forceinline__ float lanes_max(float v) { return kAll ? wave_max(v) : row16_max(v); }
template <bool kAll>
__device__ __forceinline__ float lanes_sum(float v) { return kAll ? wave_sum(v) : row16_sum(v); }

// Each part's share of its column, a lane for each part.
template <bool kAll>
__device__ __forceinline__ void combine_shares(const float2* ml, size_t stride, int parts, int columns, float* share) {
  constexpr int kLanes = kAll ? kWave : 16;
  const int p = threadIdx.x % kLanes;
  for (int c = threadIdx.x / kLanes; c < columns; c += kCombineThreads / kLanes) {
    float2 x{-INFINITY, 0.0f};
    if (p < parts) x = ml[p * stride + c];
    const float s = part_weight(x.x, lanes_max<kAll>(x.x), x.y);
    const float of = s / lanes_sum<kAll>(s);
    if (p < parts) share[p * columns + c] = of;
  }
}

template <int D>
__global__ void __launch_bounds__(kCombineThreads) k_kv8_combine(const Attend a, const CombineSplit split) {
  __shared__ CombineShared sh;
  const bool wide = (int)blockIdx.x < split.wide_blocks;
  const int block = (int)blockIdx.x - (wide ? 0 : split.wide_blocks), shift = wide ? split.wide_shift : split.narrow_shift;
  const int index = block >> shift, piece = block & ((1 << shift) - 1), h = index % a.kv;
  Request rq;
  int parts, columns, c0 = 0, stride;  // columns of the item, the first of this block's
  size_t from;  // column 0 of part 0
  if (wide) {
    const WideItem item = wide_find<kCombineThreads>(a, index, true, rq, sh.found);
    if (item.b < 0 || item.splits == 1) return;
    c0 = item.tile * kWideColumns;
    columns = min(kWideColumns, rq.count * a.group - c0);
    const int units = (rq.len + kUnit - 1) / kUnit, per = wide_per(units, item.splits);
    parts = max(1, ((wide_end(a, rq, c0) + kUnit - 1) / kUnit + per - 1) / per);
    from = a.narrow_parts + (size_t)item.part * kWideColumns;
    stride = kWideColumns;
  } else {
    NarrowPart part;
    if (!narrow_find<false>(a, index / a.kv, part, rq) || part.parts == 1) return;
    columns = rq.count * a.group;
    parts = part.parts;
    from = ((size_t)part.first * a.kv + h) * 16;
    stride = 16 * a.kv;
  }
  const int mine = wide ? kWideColumns >> shift : split.narrow_columns;
  from += piece * mine;
  columns = min(columns - piece * mine, mine);
  c0 += piece * mine;
  if (columns <= 0) return;
  // Where the columns leave threads over, those take a share of the parts
  // each, so that a part's load does not wait for the one eight before it. The
  // first loads are on their way while the shares are made.
  const int t = threadIdx.x, slots = columns * (D / 4), groups = max(1, kCombineThreads / slots), g = groups == 1 ? 0 : t / slots;
  constexpr int kAhead = 8;
  const auto fetch = [&](int e, int p0, f32x4 (&y)[kAhead]) {
    const float* const x = a.part + (from + e / (D / 4)) * D + 4 * (e % (D / 4));
#pragma unroll
    for (int i = 0; i < kAhead; ++i) y[i] = *reinterpret_cast<const f32x4*>(x + (size_t)min(p0 + i * groups, parts - 1) * stride * D);
  };
  const int e0 = t - g * slots;
  f32x4 ready[kAhead];
  fetch(min(e0, slots - 1), min(g, parts - 1), ready);
  if (parts <= 16) combine_shares<false>(a.part_ml + from, stride, parts, columns, sh.share);
  else combine_shares<true>(a.part_ml + from, stride, parts, columns, sh.share);
  __syncthreads();
  const auto joined = [&](int e, f32x4 (&y)[kAhead]) {
    const float* const share = sh.share + e / (D / 4);
    f32x4 acc{0.0f, 0.0f, 0.0f, 0.0f};
    for (int p0 = g; p0 < parts; p0 += kAhead * groups) {
      if (p0 != g) fetch(e, p0, y);
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        if (p0 + i * groups < parts) acc += share[(p0 + i * groups) * columns] * y[i];
    }
    return acc;
  };
  const auto store = [&](int e, const f32x4& acc) {
    const int c = c0 + e / (D / 4), i = c / a.group, j = c - i * a.group;
    uint2 y{0, 0};
    if (rq.past + i >= 0) y = uint2{pack_bf16(acc[0], acc[1]), pack_bf16(acc[2], acc[3])};
    *reinterpret_cast<uint2*>(a.out + ((size_t)(rq.row0 + i) * (a.kv * a.group) + h * a.group + j) * D + 4 * (e % (D / 4))) = y;
  };
  if (groups == 1) {
    for (int e = t; e < slots; e += kCombineThreads) {
      if (e != t) fetch(e, 0, ready);
      store(e, joined(e, ready));
    }
    return;
  }
  if (g < groups) sh.sums[t] = joined(e0, ready);
  __syncthreads();
  if (t >= slots) return;
  f32x4 acc = sh.sums[t];
  for (int i = 1; i < groups; ++i) acc += sh.sums[t + i * slots];
  store(t, acc);
}

// ------------------------------------------------------------------ host

int page_shift(int32_t page) {
  for (int s = 4; s <= 8; ++s)
    if (page == 1 << s) return s;
  return -1;
}

bool cache_shape(int32_t pages, int32_t page, int32_t kv, int32_t dim, int32_t format) {
  if (page_shift(page) < 0) return set_error(LFM25_EINVAL, "page must be 16, 32, 64, 128 or 256"), false;
  if (pages < 1 || (int64_t)pages * page > INT32_MAX) return set_error(LFM25_EINVAL, "pages * page must be in [1, 2^31)"), false;
  if (kv < 1 || kv > 256) return set_error(LFM25_EINVAL, "kv_heads must be in [1, 256]"), false;
  if (dim != 64 && dim != 128) return set_error(LFM25_EINVAL, "head_dim must be 64 or 128"), false;
  if (format != LFM25_KV8_INT8 && format != LFM25_KV8_FP8) return set_error(LFM25_EINVAL, "unknown 8-bit format %d", format), false;
  return true;
}

bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }
bool aligned8(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 7u) == 0; }

struct Splits {
  int share, least;     // of the narrow requests' division; 0: not divided
  int waves;            // of a narrow part
  int items;            // of a block beside tiles; 0: one request, wide whatever it brings
  int64_t narrow;       // most narrow parts, of all requests
  int wide;             // parts of a wide tile
  int64_t wide_tiles;   // most tiles that the rows can make
  int64_t wide_blocks;  // and blocks for them
  bool has_wide;
  bool few_tiles;       // about half as many as the chip has room for, or fewer
};
constexpr int kMostWideParts = 16;

// Waves of a block and parts of a request's keys, from what the host knows
// (the lengths are on the device; the table's width bounds them).
Splits splits_for(int32_t rows, int32_t requests, int32_t kv, int32_t group, int32_t max_rows, int32_t width, int32_t page,
                  int32_t dim) {
  Splits s{0, 0, 4, 1, requests, 1, 0, 0, false, false};
  const int64_t positions = std::min<int64_t>((int64_t)width * page, INT32_MAX), units = (positions + kUnit - 1) / kUnit;
  const auto parts = [&](int64_t wanted, int64_t blocks, int64_t least) {
    return (int)std::max<int64_t>(1, std::min({wanted / blocks, positions / least, (int64_t)kWave}));
  };
  const int64_t blocks = (int64_t)std::min(requests, rows) * kv;
  // a chip holds 4,096 waves of dim 64, 2,048 of dim 128
  constexpr int most = 8;
  const int64_t full = dim == 64 ? 4096 : 2048;
  while (s.waves < most && units >= 2 * s.waves && blocks * s.waves < full) s.waves *= 2;
  s.has_wide = (int64_t)max_rows * group > 16;
  if (s.has_wide) {
    s.waves = 4;  // beside wide tiles
    const int64_t columns = (int64_t)rows * group;
    s.wide_tiles = requests == 1 ? (columns + kWideColumns - 1) / kWideColumns
                                 : columns / kWideColumns + std::min<int64_t>(requests, columns / 17 + 1);
    s.few_tiles = columns * kv <= (int64_t)kWideParts / 2 * kWideColumns;  // about; less than half a chip
    // A tile takes 7 us and 0.8 for each unit, parts and their combination 5
    // (one tile a head: 13.9 us whole and 16.4 in parts over 512 positions,
    // 19.7 and 16.8 over 1,024; 21.2 and 17.6 beside single tokens).
    if (s.few_tiles && units >= 16) {
      s.wide = requests == 1 ? parts(kWideParts, s.wide_tiles * kv, kLeastPart * kUnit) : (int)(units / kLeastPart);
      s.wide = std::min(s.wide, kMostWideParts);
    }
    s.wide_blocks = s.wide_tiles * kv;
    if (s.wide > 1) s.wide_blocks = requests == 1 ? s.wide_blocks * s.wide : std::max<int64_t>(s.wide_blocks, kWideParts);
    s.items = requests == 1 ? 0 : s.few_tiles && requests * kv <= 128 ? 1 : (dim == 64 ? Wide<64>::kWaves : Wide<128>::kWaves) / 4;
  }
  // Single tokens: a unit takes one block 0.2 us (dim 64), and the chip's
  // memory 0.0016 for each block; parts and their combination 4. Whole and in
  // parts, dim 64, lengths alike (us):
  //   blocks     1,536      2,048      2,560      4,096      5,760 positions
  //        8  10.8 10.7  13.0 10.7  15.0 10.7  21.3 10.7  28.1 10.8
  //       32  11.0 10.8  13.1 10.8  15.1 10.9  22.2 12.9  29.1 15.5
  //       64  11.6 11.6  14.2 12.7  16.2 15.1  22.4 16.6  29.1 19.0
  //       96  12.3 14.9  14.4 15.5  16.5 16.0  22.6 19.5  29.3 22.5
  //      112  12.4 15.2  14.6 15.9  16.7 18.1  22.7 21.5  29.3 24.2
  // and 24 requests of 8 heads, 4,096 positions, 24.6 and 29.2. The border
  // that is taken, units * (120 - blocks) = 2,400 and none from 120 blocks on,
  // is on the side of no parts (and of no workspace): 0 to 1.5 us at 64
  // blocks, up to 7 at 96. Where the memory bounds it, still in parts over
  // long contexts, since a batch's lengths may differ. More than kDivided
  // requests are not divided at all: 256 of 1,000 positions beside one of
  // 100,000 take 120 us, one more 559 (300 and 1,290 beside a prompt of 40).
  const int64_t target = s.has_wide ? kWideParts : full / s.waves;
  const bool many = blocks > target / 2;
  s.least = s.has_wide ? 32 : many ? 128 : s.waves;
  const int64_t from = s.has_wide ? 96 : many ? 256 : units * (dim / 64) * (120 - blocks) >= 2400 ? 2 * s.least : 96;
  if ((!s.has_wide || requests > 1) && requests <= kDivided && units >= from && requests * units <= 1 << 30) {
    s.share = (int)std::max<int64_t>(1, target / kv);
    s.narrow = std::min<int64_t>(requests + s.share, requests * ((units + s.least - 1) / s.least));
  }
  return s;
}

// Columns of the narrow and of the wide parts in the workspace.
size_t narrow_columns(const Splits& s, int64_t kv) { return s.share > 0 ? (size_t)(s.narrow * kv * 16) : 0; }
size_t wide_columns(const Splits& s) { return s.has_wide && s.wide > 1 ? (size_t)kWideParts * kWideColumns : 0; }

template <int kThreads, int kEach>
void plan(const lfm25_kv8_plan_call& c, const lfm25_kv8_plan_pages& pages, int blocks, int shift, hipStream_t stream) {
  const auto kernel = pages.shared || pages.held ? k_kv8_plan<kThreads, kEach, true> : k_kv8_plan<kThreads, kEach, false>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(kThreads), sizeof(PlanShared<kThreads * kEach>), stream, c.past,
                     c.counts, c.requests, c.block_table, c.width, c.free_pages, c.ring, c.cursor, c.row_starts, c.slots, c.rows,
                     c.next_cursor, c.status, shift, pages.shared, pages.held);
}

template <int D, bool kFp8, int kWaves>
void attend_narrow(const Attend& a, int64_t blocks, hipStream_t stream) {
  const dim3 grid((unsigned)blocks), block(kWaves * kWave);
  const size_t lds = sizeof(NarrowShared<D, kWaves>);
  if (a.narrow_share > 0) hipLaunchKernelGGL((k_kv8_attend_narrow<D, kFp8, kWaves, true>), grid, block, lds, stream, a);
  else hipLaunchKernelGGL((k_kv8_attend_narrow<D, kFp8, kWaves, false>), grid, block, lds, stream, a);
}

template <int D, bool kFp8, int kItems>
void attend_both(const Attend& a, hipStream_t stream) {
  hipLaunchKernelGGL((k_kv8_attend_both<D, kFp8, kItems>), dim3((unsigned)(a.wide_blocks + a.narrow_blocks)), dim3(Wide<D>::kThreads),
                     sizeof(BothShared<D, kItems>), stream, a);
}

template <int D, bool kFp8>
int attend(const Attend& a, const Splits& s, hipStream_t stream) {
  const int64_t narrow = s.narrow * a.kv;
  if (s.has_wide) {
    if (s.items == 0) attend_both<D, kFp8, 0>(a, stream);
    else if (s.items == 1) attend_both<D, kFp8, 1>(a, stream);
    else attend_both<D, kFp8, Wide<D>::kWaves / 4>(a, stream);
  } else if (s.waves == 4) {
    attend_narrow<D, kFp8, 4>(a, narrow, stream);
  } else {
    attend_narrow<D, kFp8, 8>(a, narrow, stream);
  }
  if (s.share > 0 || (s.has_wide && s.wide > 1)) {
    CombineSplit c{};
    if (s.has_wide && s.wide > 1) {  // (a tile in parts is one of at most kWideParts / 2)
      const int items = (int)std::min<int64_t>(kWideParts / 2, s.wide_tiles * a.kv);
      c.wide_shift = items <= 64 ? 3 : 2;
      c.wide_blocks = items << c.wide_shift;
    }
    int narrow_blocks = 0;
    if (s.share > 0) {
      const int64_t columns = std::min<int64_t>(16, (int64_t)a.max_rows * a.group), items = (int64_t)a.requests * a.kv;
      c.narrow_columns = columns > 4 && items * columns <= 512 ? 2 : 4;
      while ((c.narrow_columns << c.narrow_shift) < columns) ++c.narrow_shift;
      narrow_blocks = (int)(items << c.narrow_shift);
    }
    hipLaunchKernelGGL((k_kv8_combine<D>), dim3((unsigned)(c.wide_blocks + narrow_blocks)), dim3(kCombineThreads), 0, stream, a, c);
  }
  return check_launch("lfm25_kv8_attention");
}

}  // namespace
}  // namespace lfm25

using namespace lfm25;

extern "C" int lfm25_kv8_plan(const lfm25_kv8_plan_call* call, lfm25_stream_t stream) {
  const lfm25_kv8_plan_pages none{};
  return lfm25_kv8_plan_with(call, &none, stream);
}

extern "C" int lfm25_kv8_plan_with(const lfm25_kv8_plan_call* call, const lfm25_kv8_plan_pages* pages, lfm25_stream_t stream) {
  LFM25_REQUIRE(call && pages, "lfm25_kv8_plan: null pointer");
  const lfm25_kv8_plan_call& c = *call;
  LFM25_REQUIRE(c.past && c.counts && c.block_table && c.free_pages && c.cursor && c.row_starts && c.slots && c.next_cursor && c.status,
                "lfm25_kv8_plan: null pointer");
  LFM25_REQUIRE(page_shift(c.page) >= 0, "lfm25_kv8_plan: page must be 16, 32, 64, 128 or 256");
  LFM25_REQUIRE(c.requests >= 1 && c.requests <= kMaxRequests, "lfm25_kv8_plan: requests must be in [1, %d]", kMaxRequests);
  LFM25_REQUIRE(c.width >= 1 && (int64_t)c.width * c.page <= INT32_MAX, "lfm25_kv8_plan: width * page must be in [1, 2^31)");
  LFM25_REQUIRE(c.ring >= 1 && c.rows >= 1, "lfm25_kv8_plan: an empty ring or no rows");
  LFM25_REQUIRE(aligned4(c.past) && aligned4(c.counts) && aligned4(c.block_table) && aligned4(c.free_pages) && aligned4(c.row_starts) &&
                    aligned4(c.slots) && aligned4(c.status) && aligned8(c.cursor) && aligned8(c.next_cursor) && aligned4(pages->shared) &&
                    aligned4(pages->held),
                "lfm25_kv8_plan: misaligned pointer");
  const int shift = page_shift(c.page);
  // small passes with few waves to wait for one another, large ones with as
  // many threads as a block has
  const uint64_t apart = c.cursor < c.next_cursor ? (uintptr_t)c.next_cursor - (uintptr_t)c.cursor
                                                  : (uintptr_t)c.cursor - (uintptr_t)c.next_cursor;
  const bool in_place = apart < 2 * sizeof(int64_t) || pages->held;
  const auto blocks = [&](int threads) {
    return in_place ? 1 : (int)std::min<int64_t>(kPlanBlocks, (c.rows + (int64_t)threads - 1) / threads);
  };
  if (c.requests <= 64 && c.rows <= 256) plan<64, 1>(c, *pages, 1, shift, stream);
  else if (c.requests <= 256 && (c.rows <= 1024 || !in_place)) plan<256, 1>(c, *pages, blocks(256), shift, stream);
  else if (c.requests <= 1024 && !in_place) plan<512, 2>(c, *pages, blocks(512), shift, stream);
  else if (c.requests <= 1024) plan<1024, 1>(c, *pages, 1, shift, stream);
  else plan<1024, 4>(c, *pages, blocks(1024), shift, stream);
  if (c.rows > kPlanRows && in_place)
    hipLaunchKernelGGL(k_kv8_slots, dim3((unsigned)((c.rows + (int64_t)kSlotThreads - 1) / kSlotThreads)), dim3(kSlotThreads), 0, stream,
                       c.past, c.requests, c.block_table, c.width, c.row_starts, c.status, c.slots, c.rows, shift);
  return check_launch("lfm25_kv8_plan");
}

extern "C" int lfm25_kv8_append(const lfm25_kv8_append_call* call, lfm25_stream_t stream) {
  LFM25_REQUIRE(call, "lfm25_kv8_append: null pointer");
  const lfm25_kv8_append_call& c = *call;
  LFM25_REQUIRE(c.keys && c.values && c.slots && c.key_cache && c.value_cache && c.key_scales && c.value_scales,
                "lfm25_kv8_append: null pointer");
  if (!cache_shape(c.pages, c.page, c.kv_heads, c.head_dim, c.format)) return LFM25_EINVAL;
  LFM25_REQUIRE(c.rows >= 1, "lfm25_kv8_append: no rows");
  const int64_t row = (int64_t)c.kv_heads * c.head_dim;
  LFM25_REQUIRE(c.key_stride >= row && c.value_stride >= row && c.key_stride % 8 == 0 && c.value_stride % 8 == 0,
                "lfm25_kv8_append: row strides must be multiples of 8 of at least kv_heads * head_dim");
  LFM25_REQUIRE(aligned16(c.keys) && aligned16(c.values) && aligned16(c.key_cache) && aligned16(c.value_cache),
                "lfm25_kv8_append: keys, values and caches must be 16-byte aligned");
  LFM25_REQUIRE(aligned4(c.slots) && aligned4(c.key_scales) && aligned4(c.value_scales), "lfm25_kv8_append: misaligned pointer");
  Append a{};
  a.x[0] = c.keys, a.x[1] = c.values;
  a.stride[0] = c.key_stride, a.stride[1] = c.value_stride;
  a.cache[0] = static_cast<uint8_t*>(c.key_cache), a.cache[1] = static_cast<uint8_t*>(c.value_cache);
  a.scales[0] = c.key_scales, a.scales[1] = c.value_scales;
  a.slots = c.slots;
  a.rows = c.rows, a.kv = c.kv_heads, a.pages = c.pages, a.shift = page_shift(c.page);
  // Few rows: a single token of a request for each wave. Many: a page's worth,
  // since a block that finds no run to begin costs as much to start as any
  // (4,096 rows in pages of 64: 19.7 us with 16 rows a block, 7.8 with 64).
  a.chunk = c.rows <= 512 ? 4 : std::min(c.page, kWave);
  const dim3 grid((unsigned)((c.rows + (int64_t)a.chunk - 1) / a.chunk), (unsigned)c.kv_heads, 2), block(kAppendThreads);
  if (c.head_dim == 64) {
    if (c.format == LFM25_KV8_FP8) hipLaunchKernelGGL((k_kv8_append<64, true>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((k_kv8_append<64, false>), grid, block, 0, stream, a);
  } else {
    if (c.format == LFM25_KV8_FP8) hipLaunchKernelGGL((k_kv8_append<128, true>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((k_kv8_append<128, false>), grid, block, 0, stream, a);
  }
  return check_launch("lfm25_kv8_append");
}

static bool attend_shape(int32_t rows, int32_t heads, int32_t kv_heads, int32_t requests, int32_t max_rows, int32_t width, int32_t page) {
  if (kv_heads < 1 || heads < 1 || heads % kv_heads != 0 || heads / kv_heads > 16)
    return set_error(LFM25_EINVAL, "heads must be a multiple of kv_heads, at most 16 times it"), false;
  if (rows < 1 || (int64_t)rows * heads > INT32_MAX) return set_error(LFM25_EINVAL, "rows * heads must be in [1, 2^31)"), false;
  if (requests < 1 || requests > kMaxRequests) return set_error(LFM25_EINVAL, "requests must be in [1, %d]", kMaxRequests), false;
  if (max_rows < 1) return set_error(LFM25_EINVAL, "max_rows must be positive"), false;
  if (width < 1 || (int64_t)width * page > INT32_MAX) return set_error(LFM25_EINVAL, "width * page must be in [1, 2^31)"), false;
  return true;
}

extern "C" size_t lfm25_kv8_attention_workspace_bytes(int32_t rows, int32_t heads, int32_t kv_heads, int32_t head_dim,
                                                      int32_t requests, int32_t max_rows, int32_t width, int32_t page) {
  if (page_shift(page) < 0 || (head_dim != 64 && head_dim != 128) ||
      !attend_shape(rows, heads, kv_heads, requests, max_rows, width, page))
    return 0;
  const Splits s = splits_for(rows, requests, kv_heads, heads / kv_heads, std::min(max_rows, rows), width, page, head_dim);
  return 4 * (narrow_columns(s, kv_heads) + wide_columns(s)) * (head_dim + 2);
}

extern "C" int lfm25_kv8_attention(const lfm25_kv8_attention_call* call, lfm25_stream_t stream) {
  LFM25_REQUIRE(call, "lfm25_kv8_attention: null pointer");
  const lfm25_kv8_attention_call& c = *call;
  LFM25_REQUIRE(c.query && c.key_cache && c.value_cache && c.key_scales && c.value_scales && c.block_table && c.past && c.row_starts &&
                    c.output,
                "lfm25_kv8_attention: null pointer");
  if (!cache_shape(c.pages, c.page, c.kv_heads, c.head_dim, c.format)) return LFM25_EINVAL;
  if (!attend_shape(c.rows, c.heads, c.kv_heads, c.requests, c.max_rows, c.width, c.page)) return LFM25_EINVAL;
  LFM25_REQUIRE(c.query_stride >= (int64_t)c.heads * c.head_dim && c.query_stride % 8 == 0,
                "lfm25_kv8_attention: the query's row stride must be a multiple of 8 of at least heads * head_dim");
  LFM25_REQUIRE(aligned16(c.query) && aligned16(c.key_cache) && aligned16(c.value_cache) && aligned16(c.output),
                "lfm25_kv8_attention: query, output and caches must be 16-byte aligned");
  LFM25_REQUIRE(aligned4(c.key_scales) && aligned4(c.value_scales) && aligned4(c.block_table) && aligned4(c.past) &&
                    aligned4(c.row_starts) && aligned4(c.status),
                "lfm25_kv8_attention: misaligned pointer");
  LFM25_REQUIRE(std::isfinite(c.scale) && c.scale >= 0.0f, "lfm25_kv8_attention: scale must be finite and not negative");
  LFM25_REQUIRE(c.reserved == 0, "lfm25_kv8_attention: reserved must be 0");
  const int group = c.heads / c.kv_heads, max_rows = std::min(c.max_rows, c.rows);
  const Splits s = splits_for(c.rows, c.requests, c.kv_heads, group, max_rows, c.width, c.page, c.head_dim);
  const size_t columns = narrow_columns(s, c.kv_heads) + wide_columns(s);
  LFM25_REQUIRE(columns == 0 || (c.workspace != nullptr && aligned16(c.workspace)),
                "lfm25_kv8_attention: needs a 16-byte aligned workspace of lfm25_kv8_attention_workspace_bytes()");
  Attend a{};
  a.q = c.query, a.q_stride = c.query_stride;
  a.k = static_cast<const uint8_t*>(c.key_cache), a.v = static_cast<const uint8_t*>(c.value_cache);
  a.ks = c.key_scales, a.vs = c.value_scales;
  a.table = c.block_table, a.past = c.past, a.starts = c.row_starts;
  a.out = c.output;
  a.part = static_cast<float*>(c.workspace);
  a.part_ml = reinterpret_cast<float2*>(a.part + columns * c.head_dim);
  a.narrow_parts = narrow_columns(s, c.kv_heads);
  a.status = c.status;
  a.width = c.width, a.rows = c.rows, a.kv = c.kv_heads, a.group = group, a.pages = c.pages, a.shift = page_shift(c.page);
  a.requests = c.requests, a.max_rows = max_rows;
  a.narrow_share = s.share, a.narrow_least = s.least, a.wide_splits = s.wide;
  a.wide_blocks = (int)s.wide_blocks;
  a.early_blocks = s.wide > 1 && s.few_tiles ? 0 : std::min(a.wide_blocks, kWideParts);
  a.narrow_items = std::max(1, s.items);
  a.narrow_blocks = s.items == 0 ? 0 : (int)((s.narrow * c.kv_heads + s.items - 1) / s.items);
  a.narrow_columns = s.has_wide && s.items == 0 ? 0 : 16;
  a.scale = c.scale * 1.4426950408889634f;
  if (c.head_dim == 64) return c.format == LFM25_KV8_FP8 ? attend<64, true>(a, s, stream) : attend<64, false>(a, s, stream);
  return c.format == LFM25_KV8_FP8 ? attend<128, true>(a, s, stream) : attend<128, false>(a, s, stream);
}
