// Attention whose scores follow a rule besides the dot product, and its gradients.
//
// Score of query row i and key j (of query head h, whose keys are those of key head h / rep), with d = i + q_start - j:
//   s = sm_scale q.k;  with a cap c: s = c tanh(s / c);  s -= slopes[h] |d|;  s += table[buckets[clamp(d, -R, R) + R]][h]
// i sees j where from[b][j] <= i < until[b][j] (one interval of rows for each key) and where a block mask keeps
// (i / 64, j / 64). out = softmax(s) v, lse the rows' log2-sum-exp2, and for the gradient do of out:
//   P = exp2(s log2(e) - lse),  dP = do v^T,  dS = P (dP - delta),  delta = rowsum(do out)
//   dtable[n][h] = sum of dS over the pairs of bucket n;  dC = dS (1 - tanh^2)
//   dq = sm_scale dC k,  dk = sm_scale dC^T q,  dv = P^T do  (dk and dv summed over a key head's query heads)
//
// Which 64 x 64 blocks hold a pair that is seen, and which of these hold one that is not (they are cut: only there
// the intervals are looked at), is written down once per call for both sides (scored_lists_kernel), from the
// smallest and largest bounds of each key block.
// The passes themselves are in attn_scored_pass.h.
#include <math.h>

#include <algorithm>
#include <climits>
#include <cmath>

#include "attn_scored_pass.h"

namespace {

using namespace sa_scored;

// ---- What a call's passes read besides its operands.

// {smallest from, largest until} of the keys of a block that have rows, {largest from, smallest until} of all (a key without
// rows: 0; -1 in the last place: there are rows between the first two that see none of the keys). Key blocks whose bounds say
// that a query block sees none of them are left out.
__device__ inline int4 key_bounds(int2 x) {
  x.x = max(x.x, 0);
  return x.y > x.x ? make_int4(x.x, x.y, x.x, x.y) : make_int4(INT_MAX, 0, INT_MAX, 0);
}
__device__ inline int4 join_bounds(int4 a, int4 b) {
  return make_int4(min(a.x, b.x), max(a.y, b.y), max(a.z, b.z), min(a.w, b.w));
}
__device__ inline int4 no_bounds() { return make_int4(INT_MAX, 0, 0, INT_MAX); }

// Of the block that the wave's lanes have a key of each. Its rows have no gap where each interval that ends before the last one
// does ends within another, mostly the first of those that end last.
__device__ inline int4 wave_bounds(const int2* ranges, int first, int Lk, int lane) {
  int4 r = first + lane < Lk ? key_bounds(ranges[first + lane]) : no_bounds();
  const int from = r.x, until = r.y;  // (of a key without rows: none, 0)
#pragma unroll
  for (int o = 32; o > 0; o >>= 1)
    r = join_bounds(r, make_int4(__shfl_xor(r.x, o), __shfl_xor(r.y, o), __shfl_xor(r.z, o), __shfl_xor(r.w, o)));
  const int last = __ffsll((unsigned long long)__ballot(until == r.y)) - 1;
  const int from_last = __shfl(from, last);
  bool open = until > 0 && until < r.y && from_last > until;
  if (__ballot(open)) {
    for (int i = 0; i < 64; ++i) {
      const int a = __shfl(from, i), z = __shfl(until, i);  // (of all lanes: no short cut)
      open &= a > until || z <= until;
    }
    if (__ballot(open)) r.w = -1;
  }
  return r;
}

// Whether one of the rows r0 .. r1 - 1 sees one of a block's keys.
__device__ inline bool some_seen(const int2* ranges, int first, int Lk, int r0, int r1) {
  bool some = false;
  for (int j = first; j < min(first + kBlk, Lk); ++j) {
    const int4 x = key_bounds(ranges[j]);
    some = some || (x.x < r1 && x.y > r0);
  }
  return some;
}

__global__ __launch_bounds__(256) void scored_bounds_kernel(const int2* ranges, int64_t ranges_sb, int64_t n, int Lk, int nkb,
                                                            int4* bounds) {
  const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (at >= n) return;
  const int lane = threadIdx.x & 63;
  const int4 r = wave_bounds(ranges + at / nkb * ranges_sb, (int)(at % nkb) * kBlk, Lk, lane);
  if (lane == 0) bounds[at] = r;
}


struct ListArgs {
  const int2* ranges;   // nullable
  int64_t ranges_sb;
  const int4* bounds;   // of the ranges; null: taken from them here
  const uint8_t* mask;  // nullable
  int64_t s0, s1, s2, s3;
  int B, H, Hl, Lq, Lk, nqb, nkb;  // Hl: heads that lists are made for, H or 1
  int32_t *kv_idx, *kv_cnt, *q_idx, *q_cnt;  // (q_idx null: not made)
  int list_groups;                           // workgroups that make lists; the others expand the biases
  const void* table;                         // nullable, [n_buckets][H]
  int table_dtype, n_buckets, radius;
  const int32_t* buckets;  // [2 radius + 1]
  float* ebias;            // [H][2 radius + 1 + 2 kPad]
};

// A wave per list: the key blocks of a query block, or the other way round. 64 blocks a turn, kept ones counted by ballots:
// 5 us at 278 x 278 blocks, an empty launch's 3 and a walk's latency.
__global__ __launch_bounds__(256) void scored_lists_kernel(ListArgs a) {
  if ((int)blockIdx.x >= a.list_groups) {
    const int n = 2 * a.radius + 1 + 2 * kPad;
    const int64_t i = ((int64_t)blockIdx.x - a.list_groups) * 256 + threadIdx.x;
    if (i >= (int64_t)a.H * n) return;
    const int h = (int)(i / n), at = min(max((int)(i % n) - kPad, 0), 2 * a.radius);
    const int bucket = min(max(a.buckets[at], 0), a.n_buckets - 1);
    a.ebias[i] = load_as_float(a.table, a.table_dtype, (int64_t)bucket * a.H + h) * kLog2e;
    return;
  }
  int64_t row = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 6;
  const int lane = threadIdx.x & 63;
  const int64_t rows = (int64_t)a.B * a.Hl * a.nqb;
  const bool keys = row >= rows;  // a key block's
  if (keys) row -= rows;
  const int n_own = keys ? a.nkb : a.nqb, n_st = keys ? a.nqb : a.nkb;
  if (keys && (!a.q_idx || row >= (int64_t)a.B * a.Hl * a.nkb)) return;
  const int64_t bl = row / n_own;
  const int own = (int)(row - bl * n_own), b = (int)(bl / a.Hl), h = (int)(bl - (int64_t)b * a.Hl);
  const uint8_t* mask = a.mask ? a.mask + b * a.s0 + h * a.s1 : nullptr;
  const int2* ranges = a.ranges ? a.ranges + b * a.ranges_sb : nullptr;
  const int4* bounds = a.bounds ? a.bounds + (int64_t)b * a.nkb : nullptr;
  int4 x = no_bounds();
  if (ranges && !bounds && keys) x = wave_bounds(ranges, own * kBlk, a.Lk, lane);
  int32_t* out = (keys ? a.q_idx : a.kv_idx) + row * n_st;
  int total = 0;
  for (int n0 = 0; n0 < n_st; n0 += 64) {
    const int n = n0 + lane, qb = keys ? n : own, kb = keys ? own : n;
    bool any = n < n_st, whole = (kb + 1) * kBlk <= a.Lk;
    if (any && ranges) {
      const int r0 = qb * kBlk, r1 = min(r0 + kBlk, a.Lq);
      if (bounds) {
        x = bounds[kb];
      } else if (!keys) {
        x = no_bounds();
#pragma unroll 8
        for (int j = kb * kBlk; j < min((kb + 1) * kBlk, a.Lk); ++j) x = join_bounds(x, key_bounds(ranges[j]));
      }
      any = x.x < r1 && x.y > r0;
      // (intervals that all share a row have no gap; of the others the wave's or the call's bounds say so)
      if (any && (x.w < 0 || (!bounds && !keys && x.z > x.w))) any = some_seen(ranges, kb * kBlk, a.Lk, r0, r1);
      whole = whole && x.z <= r0 && x.w >= r1;
    }
    if (any && mask) any = mask[(int64_t)qb * a.s2 + (int64_t)kb * a.s3] != 0;
    const uint64_t bal = __ballot(any);
    const int pre = __builtin_amdgcn_mbcnt_hi((uint32_t)(bal >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)bal, 0));
    if (any) out[total + pre] = 2 * n + !whole;
    total += __popcll(bal);
  }
  if (lane == 0) (keys ? a.q_cnt : a.kv_cnt)[row] = total;
}

// The units of work of a pass: items whose lists are long for the call are shared by several workgroups, in chunks of at most
// `limit` of their entries. Dealt out longest first, units take about as long as the longest one, or as all of them together on
// the workgroups that an XCD holds at once and one of middling length; each costs some time besides its entries, and one
// of a split item more. The limit with the least such time is taken, of the longest list's fractions.
constexpr int kLimits = 10;
constexpr int kMostItems = 4096;  // of an XCD; with more, what lists' lengths make of the time is little
// Units of the longest list: 1, 2, 3, 4, 6, 8, 12, 16, 32, 64.
__device__ inline int parts_of(int k) { return k < 3 ? k + 1 : (int)(0x4020100c080604ull >> (8 * (k - 3)) & 0xff); }
struct SideArgs {
  const int32_t* cnt;  // lists' lengths; null: n_st each
  int per_head, heads_own, BH_own, rep, n_own, n_st;  // rep: streamed heads of an own one
  int keys, slots, least, max_units, cap, split_cap, sorted;
  // In quarters of an entry: a unit, one of a split item besides; that there are split items, each sum of the longest one.
  int unit_cost, split_cost, merge_cost, part_cost;
  int4 *units, *splits;  // [8][cap], [8][split_cap]
  int32_t *n_units, *n_splits;
};
struct ScheduleArgs {
  SideArgs side[2];
};
constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;

// Sum over the wave, in lane 63 (of data moved between lanes without LDS, which this is short of).
template <int kControl>
__device__ inline int dpp_add(int x) {
  return x + __builtin_amdgcn_update_dpp(0, x, kControl, 0xf, 0xf, true);
}
__device__ inline int sum_to_last(int x) {
  x = dpp_add<0x111>(x);  // row_shr 1, 2, 4, 8
  x = dpp_add<0x112>(x);
  x = dpp_add<0x114>(x);
  x = dpp_add<0x118>(x);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast 15, 31
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);
  return x;
}

// n / d rounded up, for n below 2^30 and inv = 1 / d (the quotient's float is off by one at most below 2^23, where lists end).
__device__ inline int ceil_div(int n, int d, float inv) {
  const int q = (int)((float)n * inv), r = n - q * d;
  return r <= 0 ? (r <= -d ? q - 1 : q) : r <= d ? q + 1 : q + 2;
}

// Units of work from the lists' lengths: of ten limits of a unit's entries the one with the least time by the costs that
// side_plan has, then the units in order, or longest first. A workgroup per XCD and side, 9 to 22 us (278 blocks of 15 heads); it
// is worth that where lists are long or unlike: [2, 12, 4546, 64] in a window, key pass 178 us unsplit, 70 split.
// (Loops are rolled up: the kernel runs once a call, on code that no cache has, and waits for that more than for anything else.)
__global__ __launch_bounds__(kPlanThreads) void scored_schedule_kernel(ScheduleArgs args) {
  __shared__ int lengths[kMostItems], items[kMostItems];  // (length -1: no such item)
  __shared__ uint64_t wave_sums[kPlanWaves];
  __shared__ unsigned long long all_entries;
  __shared__ float times[kLimits];
  __shared__ int most, limits[kLimits];
  __shared__ int4 kept[kPlanThreads];
  __shared__ __attribute__((aligned(16))) uint32_t key[kPlanThreads];
  const SideArgs& a = args.side[blockIdx.x >> 3];
  const int xcd = blockIdx.x & 7, t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int n_seq = xcd_items(a.BH_own, a.n_own);  // at most kMostItems
  if (t == 0) {
    all_entries = 0;
    most = 0;
  }
  __syncthreads();
  int longest = 0, entries = 0;
#pragma unroll 1
  for (int seq = t; seq < n_seq; seq += kPlanThreads) {
    int bh, rank, n = -1;
    if (own_block(xcd, seq, a.BH_own, a.n_own, bh, rank)) {
      const int blk = block_of_rank(a.keys, rank, a.n_own);
      items[seq] = bh * a.n_own + blk;
      n = a.n_st * a.rep;
      if (a.cnt && !a.per_head) n = min(max(a.cnt[bh / a.heads_own * a.n_own + blk], 0), a.n_st) * a.rep;
      if (a.cnt && a.per_head) {
        n = 0;
#pragma unroll 1
        for (int g = 0; g < a.rep; ++g) n += min(max(a.cnt[(bh * a.rep + g) * a.n_own + blk], 0), a.n_st);
      }
    }
    lengths[seq] = n;
    longest = max(longest, n);
    entries += max(n, 0);
  }
  if (wave * 64 < n_seq) {
    entries = sum_to_last(entries);
    if (lane == 63) atomicAdd(&all_entries, (unsigned long long)entries);
    atomicMax(&most, longest);
  }
  __syncthreads();
  longest = most;
  if (wave < kLimits) {  // a wave tries a limit
    const int parts_k = parts_of(wave), limit = max((longest + parts_k - 1) / parts_k, max(a.least, 1));
    const float inv = 1.f / (float)limit;
    int units = 0, of_split = 0;
#pragma unroll 2
    for (int seq = lane; seq < n_seq; seq += 64) {
      const int n = lengths[seq], parts = n > limit ? ceil_div(n, limit, inv) : n >= 0;
      units += parts;
      of_split += parts > 1 ? parts : 0;
    }
    units = sum_to_last(units);
    of_split = sum_to_last(of_split);
    if (lane == 63) {
      const float quarters = 4.f * (float)all_entries;
      const float all = (quarters + (float)units * a.unit_cost + (float)of_split * a.split_cost) * 8.f / a.slots;
      // (units that all run at once end with the longest; of more, the last ones run while others have ended)
      const float tail = 8 * units <= a.slots ? 0.f : quarters / fmaxf((float)units, 1.f);
      const float time = fmaxf(4.f * limit + a.unit_cost + (of_split ? a.split_cost : 0), all + tail) +
                         (of_split ? a.merge_cost + (float)a.part_cost * ((float)longest * inv) : 0.f);
      times[wave] = of_split <= a.max_units ? time : INFINITY;  // (the first splits nothing)
      limits[wave] = limit;
    }
  }
  __syncthreads();
  int limit = limits[0];
  float best = times[0];
#pragma unroll
  for (int k = 1; k < kLimits; ++k)
    if (times[k] < best) {
      best = times[k];
      limit = limits[k];
    }
  const float inv = 1.f / (float)limit;
  int units = 0, splits = 0, places = 0;
  int4* to_units = a.units + (int64_t)xcd * a.cap;
#pragma unroll 1
  for (int s0 = 0; s0 < n_seq; s0 += kPlanThreads) {
    const int seq = s0 + t, n = seq < n_seq ? lengths[seq] : -1, parts = n > limit ? ceil_div(n, limit, inv) : n >= 0;
    const int item = n >= 0 ? items[seq] : 0;
    // Units, split items and their units before this one, 21 bits each.
    const uint64_t mine = (uint64_t)parts | (uint64_t)(parts > 1) << 21 | (uint64_t)(parts > 1 ? parts : 0) << 42;
    uint64_t sum = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint64_t y = __shfl_up((unsigned long long)sum, o);
      if (lane >= o) sum += y;
    }
    __syncthreads();
    if (lane == 63) wave_sums[wave] = sum;
    __syncthreads();
    uint64_t before = sum - mine, all = 0;
#pragma unroll
    for (int i = 0; i < kPlanWaves; ++i) {
      if (i < wave) before += wave_sums[i];
      all += wave_sums[i];
    }
    constexpr int kMask = (1 << 21) - 1;
    const int at = units + (int)(before & kMask), at_split = splits + (int)(before >> 21 & kMask);
    const int place = xcd * a.max_units + places + (int)(before >> 42);
    const int each = parts > 1 ? (int)((float)n / (float)parts) : n, rest = n - each * parts;
    int from = 0;  // (`rest` units, the first or the last ones, have one more or less)
#pragma unroll 1
    for (int p = 0; p < parts; ++p) {
      const int to = p + 1 < parts ? from + each + (p < rest) : n;
      const int4 u = make_int4(item, from, to, parts > 1 ? place + p : -1);
      from = to;
      if (at + p < kPlanThreads) kept[at + p] = u;
      to_units[at + p] = u;
    }
    if (parts > 1) a.splits[(int64_t)xcd * a.split_cap + at_split] = make_int4(item, place, parts, 0);
    units += (int)(all & kMask);
    splits += (int)(all >> 21 & kMask);
    places += (int)(all >> 42);
  }
  if (t == 0) {
    a.n_units[xcd] = units;
    a.n_splits[xcd] = splits;
  }
  // Longest first, where the streamed sides of all the XCD's heads fit its L2, or its workgroups have few units each
  // (and a workgroup here has room for them).
  if (units > (a.sorted ? kPlanThreads : 3 * a.slots / 8) || units > kPlanThreads) return;
  __syncthreads();
  int4 u = make_int4(0, 0, 0, 0);
  uint32_t mine = 0;
  if (t < units) {
    u = kept[t];
    mine = (uint32_t)min(u.z - u.y, (1 << 21) - 1) * kPlanThreads + (kPlanThreads - 1 - t);
  }
  key[t] = mine;
  __syncthreads();
  if (t >= units) return;
  int rank = 0;
#pragma unroll 2
  for (int i = 0; i < units; i += 4) {
    const uint4 y = *reinterpret_cast<const uint4*>(key + i);
    rank += (y.x > mine) + (y.y > mine) + (y.z > mine) + (y.w > mine);
  }
  to_units[rank] = u;
}

// dtable[n][h]: the items' sums by distance, added in order (a workgroup for 64 distances of a head), then those of the
// distances of each bucket (a workgroup per head, a wave per bucket).
constexpr int kSumThreads = 1024;
struct TableArgs {
  const float* far;  // [b * H + h][nqb][n_far]
  float* totals;     // [h][n_far]
  const int32_t* buckets;
  void* dtable;
  int B, H, nqb, n_far, n_buckets, dtype;
};
// The sums of dS by distance over batches and query blocks, in a fixed order: 4 to 5 us, latency.
__global__ __launch_bounds__(kSumThreads) void scored_far_kernel(TableArgs a) {
  __shared__ float part[kSumThreads / 64][64];
  const int h = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = blockIdx.y * 64 + lane;
  float s = 0.f;
  if (i < a.n_far)
    for (int b = 0; b < a.B; ++b) {
      const float* from = a.far + ((int64_t)b * a.H + h) * a.nqb * a.n_far + i;
#pragma unroll 4
      for (int q = wave; q < a.nqb; q += kSumThreads / 64) s += from[(int64_t)q * a.n_far];
    }
  part[wave][lane] = s;
  __syncthreads();
  if (wave != 0 || i >= a.n_far) return;
  s = part[0][lane];
#pragma unroll
  for (int v = 1; v < kSumThreads / 64; ++v) s += part[v][lane];
  a.totals[(int64_t)h * a.n_far + i] = s;
}
// And over a bucket's distances: 4 us at radius 128, 11 at 800.
__global__ __launch_bounds__(kSumThreads) void scored_table_kernel(TableArgs a) {
  __shared__ float total[2 * kMostRadius + 1];
  __shared__ int bucket[2 * kMostRadius + 1];
  const int h = blockIdx.x, lane = threadIdx.x & 63;
  for (int i = threadIdx.x; i < a.n_far; i += kSumThreads) {
    total[i] = a.totals[(int64_t)h * a.n_far + i];
    bucket[i] = min(max(a.buckets[i], 0), a.n_buckets - 1);
  }
  __syncthreads();
  for (int n = threadIdx.x >> 6; n < a.n_buckets; n += kSumThreads / 64) {
    float s = 0.f;
    for (int i = lane; i < a.n_far; i += 64) s += bucket[i] == n ? total[i] : 0.f;
    s = wave_sum(s);
    if (lane != 0) continue;
    const int64_t at = (int64_t)n * a.H + h;
    if (a.dtype == SA_DTYPE_F32) static_cast<float*>(a.dtable)[at] = s;
    else if (a.dtype == SA_DTYPE_F16) static_cast<_Float16*>(a.dtable)[at] = (_Float16)s;
    else static_cast<__bf16*>(a.dtable)[at] = (__bf16)s;
  }
}

// ---- Row intervals of packed documents.

constexpr int kMostDocs = 8192;
constexpr int kRangeKeys = 1024;  // keys of a workgroup, which sums up the sequence's lengths for itself
struct RangeArgs {
  const int32_t *lengths, *prefix;  // [B][n]; prefix may be null
  int n, L, causal, frame, window;
  int2* out;  // [B][L]
};
// A key finds its document by bisection of the lengths' running sum in LDS: 4 to 5 us up to 17776 keys, latency.
__global__ __launch_bounds__(256) void row_ranges_kernel(RangeArgs a) {
  __shared__ int ends[kMostDocs];
  __shared__ int sums[256];
  const int b = blockIdx.y, t = threadIdx.x;
  const int32_t* lengths = a.lengths + (int64_t)b * a.n;
  // Ends of the documents, at most L (adding with that limit is associative).
  auto add = [&](int x, int y) { return (int)min((unsigned)x + (unsigned)y, (unsigned)a.L); };
  const int per = (a.n + 255) / 256, first = t * per, last = min(first + per, a.n);
  int s = 0;
  for (int i = first; i < last; ++i) ends[i] = s = add(s, min(max(lengths[i], 0), a.L));
  sums[t] = s;
  __syncthreads();
  for (int o = 1; o < 256; o <<= 1) {
    const int y = t >= o ? sums[t - o] : 0;
    __syncthreads();
    sums[t] = add(sums[t], y);
    __syncthreads();
  }
  const int before = t > 0 ? sums[t - 1] : 0;
  for (int i = first; i < last; ++i) ends[i] = add(ends[i], before);
  __syncthreads();
  const int key0 = blockIdx.x * kRangeKeys;
  for (int j = key0 + t; j < min(key0 + kRangeKeys, a.L); j += 256) {
    int lo = 0, hi = a.n;  // the first document that ends behind j
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (ends[mid] > j) hi = mid;
      else lo = mid + 1;
    }
    int2 r = make_int2(0, 0);
    if (lo < a.n) {
      const int end = ends[lo], begin = lo > 0 ? ends[lo - 1] : 0;
      const int body = a.prefix ? begin + min(max(a.prefix[(int64_t)b * a.n + lo], 0), end - begin) : begin;
      r = make_int2(begin, end);
      if (j >= body) {
        if (a.causal) r.x = j - (j - body) % a.frame;
        else if (a.window) r.x = max(begin, j - a.window + 1);
        if (a.window) r.y = min((int64_t)end, (int64_t)j + a.window);
      }
    }
    a.out[(int64_t)b * a.L + j] = r;
  }
}

// ---- Host side.

constexpr int kDirect = 32;

// Where both sides have few blocks and there is no block mask, a call walks over all of them, cut ones all.
bool has_lists(const sa_attn_scored& t) {
  return t.mask || (t.ranges && std::max(t.Lq, t.Lk) > 4 * kBlk);
}

struct SidePlan {  // how a side's items are dealt out; byte offsets into a call's plan buffer
  bool scheduled, sorted;
  int slots, least, max_units, cap, split_cap, unit_cost, split_cost, merge_cost, part_cost;
  int64_t units, n_units, splits, n_splits;
};
struct Plan {
  int64_t bounds, ebias, offsets, kv_idx, kv_cnt, q_idx, q_cnt, bytes;
  SidePlan side[2];  // queries, keys
};

// Whether the items of a side are split is decided by the longest list that there can be.
SidePlan side_plan(const sa_attn_scored& t, bool keys) {
  SidePlan p{};
  const bool f32 = t.dtype == SA_DTYPE_F32;
  const int64_t rep = keys ? t.H / t.Hk : 1, BH = (int64_t)t.B * (keys ? t.Hk : t.H);
  const int n_own = sa::cdiv(keys ? t.Lk : t.Lq, kBlk), n_st = sa::cdiv(keys ? t.Lq : t.Lk, kBlk);
  // Workgroups that the card holds at once (waves_per_simd).
  p.slots = kCus * 2 * (f32 ? (t.D == 64 ? 2 : 1) : t.D == 64 ? 3 : 2);
  // In quarters of an entry's time (64 x 64 pairs: about a microsecond of a workgroup's in 16 bits, five in fp32): a unit's own
  // operands and results, its share of a sum (by its bytes; 6 in all cases: key pass of a window's lists 71 + 11 us, not 70 + 5),
  // and the launch that adds them. Where lists are short for that, the launches to split them would take longer than they do.
  p.least = f32 ? 1 : 2;
  p.unit_cost = f32 ? 1 : 4;
  p.split_cost = f32 ? 2 : 6 * (t.D / 64) * (keys ? 2 : 1);
  p.merge_cost = f32 ? 2 : 12;
  p.part_cost = 1;
  const int64_t longest = n_st * rep;
  const int64_t items = xcd_items((int)BH, n_own);
  p.scheduled = longest > (f32 ? 4 : 16) && items <= kMostItems && longest < 1 << 21;
  if (!p.scheduled) return p;
  p.max_units = (int)std::min<int64_t>(p.slots / 4, items * ((longest + p.least - 1) / p.least));
  p.cap = (int)(items + p.max_units);
  p.split_cap = p.max_units / 2 + 1;
  p.sorted = (BH + 7) / 8 * rep * (keys ? t.Lq : t.Lk) * t.D * (f32 ? 4 : 2) * 2 <= 4 << 20;
  return p;
}

struct Buffer {
  int64_t at = 0;
  int64_t take(int64_t bytes) {
    const int64_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  }
};

Plan plan_of(const sa_attn_scored& t) {
  Plan p;
  const int64_t nqb = sa::cdiv(t.Lq, kBlk), nkb = sa::cdiv(t.Lk, kBlk);
  const int64_t lists = has_lists(t) ? (int64_t)t.B * (t.mask ? t.H : 1) : 0;
  const bool keys = t.follow & SA_SCORED_KEYS;
  Buffer buf;
  p.bounds = buf.take(t.ranges && nkb > kDirect ? t.B * nkb * 16 : 0);
  p.ebias = buf.take(t.table ? (int64_t)t.H * (2 * t.radius + 1 + 2 * kPad) * 4 : 0);
  p.offsets = buf.take(t.slopes ? (int64_t)t.B * t.H * nqb * kBlk * 8 : 0);
  p.kv_idx = buf.take(lists * nqb * nkb * 4);
  p.kv_cnt = buf.take(lists * nqb * 4);
  p.q_idx = buf.take(keys ? lists * nqb * nkb * 4 : 0);
  p.q_cnt = buf.take(keys ? lists * nkb * 4 : 0);
  for (int i = 0; i < 2; ++i) {
    SidePlan& s = p.side[i] = i == 0 || keys ? side_plan(t, i == 1) : SidePlan{};
    s.units = buf.take((int64_t)8 * s.cap * 16);
    s.splits = buf.take((int64_t)8 * s.split_cap * 16);
    s.n_units = buf.take(s.scheduled ? 32 : 0);
    s.n_splits = buf.take(s.scheduled ? 32 : 0);
  }
  p.bytes = buf.at;
  return p;
}

struct Work {  // byte offsets into the workspaces of the forward and the backward call
  int64_t fwd_parts, fwd_sums, fwd_bytes;
  int64_t stats, far, part_far, totals, parts, bytes;
};
Work work_of(const sa_attn_scored& t, const Plan& p) {
  const int64_t rows = (int64_t)t.B * t.H * sa::cdiv(t.Lq, kBlk), sums = (int64_t)kBlk * t.D * 4;
  const int64_t q_places = 8 * p.side[0].max_units, k_places = 8 * p.side[1].max_units;
  Work w;
  Buffer fwd, bwd;
  w.fwd_parts = fwd.take(q_places * sums);
  w.fwd_sums = fwd.take(q_places * kBlk * 8);
  w.fwd_bytes = fwd.at;
  w.stats = bwd.take(rows * (t.slopes ? 1024 : 512));
  const bool table = t.follow & SA_SCORED_TABLE;
  const int64_t n_far = 4 * (2 * t.radius + 1);
  w.far = bwd.take(table ? rows * n_far : 0);
  w.part_far = bwd.take(table ? q_places * n_far : 0);
  w.totals = bwd.take(table ? t.H * n_far : 0);
  w.parts = bwd.take(std::max(q_places, 2 * k_places) * sums);  // of one pass after the other
  w.bytes = bwd.at;
  return w;
}

int check_scored(const sa_attn_scored* t, const char* fn) {
  SA_REQUIRE(t, "%s: null call", fn);
  SA_REQUIRE(t->dtype >= SA_DTYPE_BF16 && t->dtype <= SA_DTYPE_F32, "%s: dtype %d", fn, t->dtype);
  SA_REQUIRE(t->B > 0 && t->H > 0 && t->Hk > 0 && t->Lq > 0 && t->Lk > 0, "%s: bad shape B=%d H=%d Hk=%d Lq=%d Lk=%d", fn,
             t->B, t->H, t->Hk, t->Lq, t->Lk);
  SA_REQUIRE(t->H % t->Hk == 0, "%s: %d query heads over %d key heads", fn, t->H, t->Hk);
  if (t->D != 64 && t->D != 128) return sa::fail(SA_ERR_UNSUPPORTED, "%s: head_dim %d (64 or 128)", fn, t->D);
  SA_REQUIRE(t->sm_scale > 0.f && std::isfinite(t->sm_scale), "%s: sm_scale must be positive and finite", fn);
  SA_REQUIRE(t->cap >= 0.f && std::isfinite(t->cap), "%s: cap must be positive and finite, or 0 for none", fn);
  SA_REQUIRE(cap_in_range(t->sm_scale, t->cap), "%s: cap or sm_scale / cap out of range", fn);
  if (t->Lq > 1 << 27 || t->Lk > 1 << 27) return sa::fail(SA_ERR_UNSUPPORTED, "%s: more than 2^27 rows", fn);
  SA_REQUIRE(t->q_start > -(1 << 29) && t->q_start < 1 << 29, "%s: q_start %d", fn, t->q_start);
  if ((int64_t)t->B * t->H * std::max(sa::cdiv(t->Lq, kBlk), sa::cdiv(t->Lk, kBlk)) >= 1LL << 24 || t->H >= 1 << 20)
    return sa::fail(SA_ERR_UNSUPPORTED, "%s: 2^24 blocks or 2^20 heads, or more", fn);  // (grids of fewer than 2^32 threads)
  if (t->table) {
    SA_REQUIRE(t->buckets && t->n_buckets > 0, "%s: table without buckets", fn);
    SA_REQUIRE(t->table_dtype >= SA_DTYPE_BF16 && t->table_dtype <= SA_DTYPE_F32, "%s: table dtype %d", fn, t->table_dtype);
    if (t->radius < 0 || t->radius > kMostRadius)
      return sa::fail(SA_ERR_UNSUPPORTED, "%s: distances up to %d told apart (at most %d)", fn, t->radius, kMostRadius);
  }
  SA_REQUIRE(t->table || !(t->follow & SA_SCORED_TABLE), "%s: a table's gradient without a table", fn);
  return SA_OK;
}

// The operands a pass streams are copied through 32-bit offsets from each head's first row.
int check_operands(const sa_attn_scored* t, const char* fn, int first, int last) {
  const int size = t->dtype == SA_DTYPE_F32 ? 4 : 2, per16 = 16 / size;
  const void* ptrs[8] = {t->q, t->k, t->v, t->out, t->dout, t->dq, t->dk, t->dv};
  const int64_t rows[8] = {t->Lq, t->Lk, t->Lk, t->Lq, t->Lq, t->Lq, t->Lk, t->Lk};
  for (int i = first; i < last; ++i) {
    if (reinterpret_cast<uintptr_t>(ptrs[i]) % 16 != 0)
      return sa::fail(SA_ERR_UNSUPPORTED, "%s: tensor base not 16-byte aligned", fn);
    if (!ptrs[i]) continue;
    for (int j = 0; j < 3; ++j)
      if (t->strides[3 * i + j] % per16 != 0)
        return sa::fail(SA_ERR_UNSUPPORTED, "%s: strides must be multiples of %d elements", fn, per16);
    const int64_t stride = t->strides[3 * i + 2];
    if (stride < 0 || stride > INT_MAX || (rows[i] + kBlk) * stride * size + 2 * t->D > INT_MAX)
      return sa::fail(SA_ERR_UNSUPPORTED, "%s: rows of one head span more than 2 GiB", fn);
  }
  return SA_OK;
}

void launch_pass(int mode, ScoredArgs a, const sa_attn_scored& t, const SidePlan& p, hipStream_t s) {
  const uint8_t* plan = static_cast<const uint8_t*>(t.plan);
  MergeArgs m{};
  if (p.scheduled) {
    a.units = reinterpret_cast<const int4*>(plan + p.units);
    a.n_units = reinterpret_cast<const int32_t*>(plan + p.n_units);
    a.unit_cap = p.cap;
    m.splits = reinterpret_cast<const int4*>(plan + p.splits);
    m.n_splits = reinterpret_cast<const int32_t*>(plan + p.n_splits);
    m.cap = p.split_cap;
    m.heads_own = a.heads_own; m.n_own = a.n_own; m.L_own = a.L_own;
    m.parts = a.parts; m.part_sums = a.part_sums; m.part_far = a.part_far;
    m.grad_a = a.grad_a; m.grad_b = a.grad_b; m.out_lo = a.out_lo;
    m.ga_sb = a.ga_sb; m.ga_sh = a.ga_sh; m.ga_sl = a.ga_sl;
    m.gb_sb = a.gb_sb; m.gb_sh = a.gb_sh; m.gb_sl = a.gb_sl;
    m.sm_scale = a.sm_scale; m.lse = a.lse; m.offsets = a.offsets; m.far = a.far; m.n_far = 2 * a.radius + 1;
  }
  const int cap = !(t.cap > 0) ? kNoCap : cap_of(t.sm_scale, t.cap, t.dtype).fine ? kFineTanh : kTanh;
  PassCall c = {mode, t.D, cap, 8u * (unsigned)(p.scheduled ? p.cap : xcd_items(a.BH_own, a.n_own)), 0, s};
  // (the statistics alone are written by every item's first unit)
  if (p.scheduled && (a.grad_a || a.grad_b || a.far)) c.merge_grid = 8u * (unsigned)p.split_cap;
  if (t.dtype == SA_DTYPE_BF16) launch_pass_bf16(a, m, c);
  else if (t.dtype == SA_DTYPE_F16) launch_pass_f16(a, m, c);
  else launch_pass_f32(a, m, c);
}

Side side_of(const sa_attn_scored& t, const void* p, int i) {
  return Side{p, t.strides[3 * i], t.strides[3 * i + 1], t.strides[3 * i + 2]};
}

ScoredArgs common_args(const sa_attn_scored& t, const Plan& p) {
  ScoredArgs a{};
  a.H = t.H;
  a.rep = t.H / t.Hk;
  a.q_start = t.q_start;
  a.ranges = reinterpret_cast<const int2*>(t.ranges);
  a.ranges_sb = t.ranges_stride;
  a.sm_scale = t.sm_scale;
  a.scale_log2 = t.sm_scale * kLog2e;
  if (t.cap > 0) {
    const Cap c = cap_of(t.sm_scale, t.cap, t.dtype);
    a.cap_in = c.in;
    a.cap_log2 = c.log2;
  }
  a.slopes = t.slopes;
  a.radius = t.table ? t.radius : 0;
  a.per_head = t.mask != nullptr;
  a.lse = t.lse;
  if (t.slopes) a.offsets = reinterpret_cast<float2*>(static_cast<uint8_t*>(t.plan) + p.offsets);
  a.out_lo = t.dtype == SA_DTYPE_F32 ? nullptr : t.out_lo;
  return a;
}

void own_queries(ScoredArgs& a, const sa_attn_scored& t, const Plan& p) {
  const uint8_t* plan = static_cast<const uint8_t*>(t.plan);
  a.heads_own = t.H;
  a.BH_own = t.B * t.H;
  a.L_own = t.Lq; a.L_st = t.Lk;
  a.n_own = sa::cdiv(t.Lq, kBlk); a.n_st = sa::cdiv(t.Lk, kBlk);
  a.own_a = side_of(t, t.q, 0);
  a.st_a = side_of(t, t.k, 1);
  a.st_b = side_of(t, t.v, 2);
  if (has_lists(t)) {
    a.idx = reinterpret_cast<const int32_t*>(plan + p.kv_idx);
    a.cnt = reinterpret_cast<const int32_t*>(plan + p.kv_cnt);
  }
  if (t.table) a.ebias = reinterpret_cast<const float*>(plan + p.ebias);
}

}  // namespace

extern "C" int sa_row_ranges(const int32_t* lengths, const int32_t* prefix, int B, int n, int L, int causal, int frame,
                             int window, int32_t* ranges, void* stream) {
  const char* fn = "sa_row_ranges";
  SA_REQUIRE(lengths && ranges, "%s: null pointer", fn);
  SA_REQUIRE(B > 0 && n > 0 && L > 0, "%s: bad shape B=%d n=%d L=%d", fn, B, n, L);
  SA_REQUIRE(frame > 0 && window >= 0, "%s: frame=%d window=%d", fn, frame, window);
  SA_REQUIRE(causal || frame == 1, "%s: frames without causal", fn);
  if (n > kMostDocs || B > 65535 || L > 1 << 30)
    return sa::fail(SA_ERR_UNSUPPORTED, "%s: B=%d n=%d L=%d (at most 65535, %d, 2^30)", fn, B, n, L, kMostDocs);
  const RangeArgs a = {lengths, prefix, n, L, causal, frame, window, reinterpret_cast<int2*>(ranges)};
  hipLaunchKernelGGL(row_ranges_kernel, dim3((unsigned)sa::cdiv(L, kRangeKeys), (unsigned)B), dim3(256), 0,
                     sa::as_stream(stream), a);
  return sa::check_launch(fn);
}

extern "C" int sa_attn_scored_sizes(const sa_attn_scored* t, int64_t bytes[3]) {
  const char* fn = "sa_attn_scored_sizes";
  SA_REQUIRE(bytes, "%s: null pointer", fn);
  if (int rc = check_scored(t, fn)) return rc;
  const Plan p = plan_of(*t);
  const Work w = work_of(*t, p);
  bytes[0] = p.bytes;
  bytes[1] = w.fwd_bytes;
  bytes[2] = w.bytes;
  return sa::ok();
}

static int check_buffers(const sa_attn_scored* t, const Plan& p, int64_t bytes, const char* fn) {
  SA_REQUIRE(!p.bytes || (t->plan && reinterpret_cast<uintptr_t>(t->plan) % 256 == 0), "%s: plan null or not 256-byte aligned",
             fn);
  SA_REQUIRE(t->plan_bytes >= p.bytes, "%s: plan of %lld bytes < %lld", fn, (long long)t->plan_bytes, (long long)p.bytes);
  SA_REQUIRE(!bytes || (t->workspace && reinterpret_cast<uintptr_t>(t->workspace) % 256 == 0),
             "%s: workspace null or not 256-byte aligned", fn);
  SA_REQUIRE(t->workspace_bytes >= bytes, "%s: workspace of %lld bytes < %lld", fn, (long long)t->workspace_bytes,
             (long long)bytes);
  SA_REQUIRE(reinterpret_cast<uintptr_t>(t->ranges) % 8 == 0, "%s: ranges not 8-byte aligned", fn);
  SA_REQUIRE(reinterpret_cast<uintptr_t>(t->out_lo) % 16 == 0, "%s: out_lo not 16-byte aligned", fn);
  return SA_OK;
}

extern "C" int sa_attn_scored_fwd(const sa_attn_scored* t, void* stream) {
  const char* fn = "sa_attn_scored_fwd";
  if (int rc = check_scored(t, fn)) return rc;
  SA_REQUIRE(t->q && t->k && t->v && t->out && t->lse, "%s: null pointer", fn);
  if (int rc = check_operands(t, fn, 0, 4)) return rc;
  const Plan p = plan_of(*t);
  const Work work = work_of(*t, p);
  if (int rc = check_buffers(t, p, work.fwd_bytes, fn)) return rc;
  hipStream_t s = sa::as_stream(stream);
  uint8_t* plan = static_cast<uint8_t*>(t->plan);
  const int nqb = sa::cdiv(t->Lq, kBlk), nkb = sa::cdiv(t->Lk, kBlk);
  const bool lists = has_lists(*t), keys = t->follow & SA_SCORED_KEYS;
  // Bounds of few key blocks are taken from the ranges where they are needed.
  const int4* bounds = t->ranges && lists && nkb > kDirect ? reinterpret_cast<const int4*>(plan + p.bounds) : nullptr;
  if (bounds) {
    const int64_t n = (int64_t)t->B * nkb;
    hipLaunchKernelGGL(scored_bounds_kernel, dim3((unsigned)((n + 3) / 4)), dim3(256), 0, s,
                       reinterpret_cast<const int2*>(t->ranges), t->ranges_stride, n, t->Lk, nkb, const_cast<int4*>(bounds));
    if (int rc = sa::check_launch(fn)) return rc;
  }
  if (lists || t->table) {
    ListArgs g{};
    g.ranges = reinterpret_cast<const int2*>(t->ranges);
    g.ranges_sb = t->ranges_stride;
    g.bounds = bounds;
    g.mask = t->mask;
    g.s0 = t->mask_strides[0]; g.s1 = t->mask_strides[1]; g.s2 = t->mask_strides[2]; g.s3 = t->mask_strides[3];
    g.B = t->B; g.H = t->H; g.Hl = t->mask ? t->H : 1;
    g.Lq = t->Lq; g.Lk = t->Lk; g.nqb = nqb; g.nkb = nkb;
    g.kv_idx = reinterpret_cast<int32_t*>(plan + p.kv_idx);
    g.kv_cnt = reinterpret_cast<int32_t*>(plan + p.kv_cnt);
    if (keys) {
      g.q_idx = reinterpret_cast<int32_t*>(plan + p.q_idx);
      g.q_cnt = reinterpret_cast<int32_t*>(plan + p.q_cnt);
    }
    const int64_t rows = lists ? (int64_t)g.B * g.Hl * (nqb + (keys ? nkb : 0)) : 0;
    g.list_groups = (int)((rows + 3) / 4);
    g.table = t->table; g.table_dtype = t->table_dtype; g.n_buckets = t->n_buckets; g.radius = t->radius;
    g.buckets = t->buckets;
    g.ebias = reinterpret_cast<float*>(plan + p.ebias);
    const int64_t more = t->table ? ((int64_t)t->H * (2 * t->radius + 1 + 2 * kPad) + 255) / 256 : 0;
    hipLaunchKernelGGL(scored_lists_kernel, dim3((unsigned)(g.list_groups + more)), dim3(256), 0, s, g);
    if (int rc = sa::check_launch(fn)) return rc;
  }
  ScheduleArgs g{};
  int n_sides = 0;
  for (int i = 0; i < 2; ++i) {
    const SidePlan& sp = p.side[i];
    if (!sp.scheduled) continue;
    SideArgs& a = g.side[n_sides++];
    a.cnt = lists ? reinterpret_cast<const int32_t*>(plan + (i ? p.q_cnt : p.kv_cnt)) : nullptr;
    a.per_head = t->mask != nullptr;
    a.heads_own = i ? t->Hk : t->H;
    a.BH_own = t->B * a.heads_own;
    a.rep = i ? t->H / t->Hk : 1;
    a.n_own = i ? nkb : nqb;
    a.n_st = i ? nqb : nkb;
    a.keys = i;
    a.slots = sp.slots; a.least = sp.least; a.max_units = sp.max_units; a.cap = sp.cap; a.split_cap = sp.split_cap;
    a.sorted = sp.sorted; a.unit_cost = sp.unit_cost; a.split_cost = sp.split_cost;
    a.merge_cost = sp.merge_cost; a.part_cost = sp.part_cost;
    a.units = reinterpret_cast<int4*>(plan + sp.units);
    a.splits = reinterpret_cast<int4*>(plan + sp.splits);
    a.n_units = reinterpret_cast<int32_t*>(plan + sp.n_units);
    a.n_splits = reinterpret_cast<int32_t*>(plan + sp.n_splits);
  }
  if (n_sides) {
    hipLaunchKernelGGL(scored_schedule_kernel, dim3(8 * n_sides), dim3(kPlanThreads), 0, s, g);
    if (int rc = sa::check_launch(fn)) return rc;
  }
  ScoredArgs a = common_args(*t, p);
  own_queries(a, *t, p);
  a.grad_a = t->out;
  a.ga_sb = t->strides[9]; a.ga_sh = t->strides[10]; a.ga_sl = t->strides[11];
  uint8_t* ws = static_cast<uint8_t*>(t->workspace);
  a.parts = reinterpret_cast<float*>(ws + work.fwd_parts);
  a.part_sums = reinterpret_cast<float*>(ws + work.fwd_sums);
  launch_pass(kForward, a, *t, p.side[0], s);
  return sa::check_launch(fn);
}

extern "C" int sa_attn_scored_bwd(const sa_attn_scored* t, void* stream) {
  const char* fn = "sa_attn_scored_bwd";
  if (int rc = check_scored(t, fn)) return rc;
  SA_REQUIRE(t->q && t->k && t->v && t->out && t->dout && t->lse, "%s: null pointer", fn);
  if (int rc = check_operands(t, fn, 0, 8)) return rc;
  const bool lists = has_lists(*t), keys = t->dk || t->dv;
  SA_REQUIRE((!keys || (t->follow & SA_SCORED_KEYS)) && (!t->dtable || (t->follow & SA_SCORED_TABLE)),
             "%s: gradients that the plan does not follow", fn);
  const Plan p = plan_of(*t);
  const Work w = work_of(*t, p);
  if (int rc = check_buffers(t, p, w.bytes, fn)) return rc;
  hipStream_t s = sa::as_stream(stream);
  uint8_t* ws = static_cast<uint8_t*>(t->workspace);
  const uint8_t* plan = static_cast<const uint8_t*>(t->plan);
  ScoredArgs a = common_args(*t, p);
  own_queries(a, *t, p);
  a.own_b = side_of(*t, t->dout, 4);
  a.out = side_of(*t, t->out, 3);
  a.grad_a = t->dq;
  a.ga_sb = t->strides[15]; a.ga_sh = t->strides[16]; a.ga_sl = t->strides[17];
  a.stats = reinterpret_cast<float*>(ws + w.stats);
  a.parts = reinterpret_cast<float*>(ws + w.parts);
  if (t->dtable) {
    a.far = reinterpret_cast<float*>(ws + w.far);
    a.part_far = reinterpret_cast<float*>(ws + w.part_far);
  }
  launch_pass(kQueries, a, *t, p.side[0], s);
  if (int rc = sa::check_launch(fn)) return rc;
  if (t->dtable) {
    const TableArgs g = {a.far, reinterpret_cast<float*>(ws + w.totals), t->buckets, t->dtable, t->B, t->H, a.n_own,
                         2 * t->radius + 1, t->n_buckets, t->table_dtype};
    hipLaunchKernelGGL(scored_far_kernel, dim3((unsigned)t->H, (unsigned)sa::cdiv(g.n_far, 64)), dim3(kSumThreads), 0, s, g);
    if (int rc = sa::check_launch(fn)) return rc;
    hipLaunchKernelGGL(scored_table_kernel, dim3((unsigned)t->H), dim3(kSumThreads), 0, s, g);
    if (int rc = sa::check_launch(fn)) return rc;
  }
  if (!keys) return sa::ok();
  a.far = nullptr;
  a.out_lo = nullptr;
  a.own_a = side_of(*t, t->k, 1);
  a.own_b = side_of(*t, t->v, 2);
  a.st_a = side_of(*t, t->q, 0);
  a.st_b = side_of(*t, t->dout, 4);
  a.grad_a = t->dk; a.ga_sb = t->strides[18]; a.ga_sh = t->strides[19]; a.ga_sl = t->strides[20];
  a.grad_b = t->dv; a.gb_sb = t->strides[21]; a.gb_sh = t->strides[22]; a.gb_sl = t->strides[23];
  a.heads_own = t->Hk;
  a.BH_own = t->B * t->Hk;
  std::swap(a.L_own, a.L_st);
  std::swap(a.n_own, a.n_st);
  if (lists) {
    a.idx = reinterpret_cast<const int32_t*>(plan + p.q_idx);
    a.cnt = reinterpret_cast<const int32_t*>(plan + p.q_cnt);
  }
  launch_pass(kKeys, a, *t, p.side[1], s);
  return sa::check_launch(fn);
}
