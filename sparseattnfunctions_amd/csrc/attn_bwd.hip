// Gradients of block-sparse attention (the reference's backward raises NotImplementedError,
// special_attentions/utils/block_sparse_attn_kernel.py:278-281), recomputing the probabilities.
//
// With S = q k^T, lse the rows' log2-sum-exp2 that the forward pass stored, do the gradient of out
// and everything restricted to the listed 64 x 64 blocks:
//   P     = exp2(S * sm_scale * log2(e) [+ bias * log2(e) - offset] - lse)
//   delta = rowsum(do * out),  dP = do v^T,  dS = P * (dP - delta)
//   dq = sm_scale dS k,  dk = sm_scale dS^T q,  dv = P^T do
// Two passes, each over the lists of one side: one per query block for dq (and delta), one per key
// block, over the transposed lists (kv_list.hip), for dk and dv. S and dP are computed in both: seven
// products instead of five, but no score leaves the chip (writing dS would move 16 KB per tile, as
// long as two tiles' products) and no sum is shared by workgroups, so that results do not depend on
// the order in which they run.
//
// Both passes are one kernel: the "own" side is the block whose gradients a workgroup computes, the
// "streamed" side the listed blocks. kKeys: own = (k, v), streamed = (q, do), results (dk, dv); else
// own = (q, do), streamed = (k, v), result dq. A pair of waves shares the streamed rows, 32 at a time
// (a step), in two LDS stages: rows of step i + 1 are copied while step i computes; one barrier per
// step. Each wave owns 32 rows of the block. Its operands stay in registers, the own row is the
// MFMA column, and P and dS come out of the first products in the layout of the second ones' B operand
// (attn_fwd.hip's P^T):
//   S^T-like [streamed][own] = st_a own_a^T,  [streamed][own] dP = st_b own_b^T
//   grad_a^T [d][own] += st_a^T dS,  kKeys: grad_b^T [d][own] += st_b^T P
// with row reads for the first and transposed reads for the second from the same LDS rows. For dk and
// dv the streamed rows' -lse / scale and -delta start the accumulators of S and dP, so that an element
// costs two products, an exp2 and its share of two roundings.
//
// With a key bias a row's offset and its lse, relative to it, come apart: where a row's keys all have a bias of -1e9,
// say, one number for both has no bits for the sum. 32 rows with an offset past kFarOffset among them round a score as the
// forward pass does, the bias times log2(e) and then the sum, and take off the offset and the lse one after the
// other, so that they have the forward pass's probabilities; the others take off both at once (off by 2^-14 of a
// probability at most). Two operations of the VALU more an element: the passes of [2, 12, 1350 x 5626, 64] with 0.3 of
// the blocks take 49 and 62 us, all rows done so 57 and 69.
//
// Bound: the issue of MFMA and VALU, as in the forward pass. [2, 30, 2560, 64] bf16 with every block: query pass
// 177 us (850 TFLOP/s of its three products), key pass 229 us (880 of its four); there the matrix cores work 51 % of
// the cycles at 1.85 GHz under the power limit, the VALU 43 %, LDS 40 % without bank conflicts, and 85 % of the CU
// time has a workgroup. [1, 15, 8229, 128] fp16 with 0.35 of the blocks: 309 and 392 us (885, 930), the matrix cores 55
// %, CUs 87 %; with every block 1 050. Of four parts, wave priorities over the two product phases, and splits of the last
// round nothing was faster (see deal).
#include <math.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

#include "attn_tile.h"
#include "sa_common.h"

namespace {

constexpr int kBlk = 64;   // rows per block of either side
constexpr int kStep = 32;  // streamed rows per step, own rows per wave
constexpr int kMostLast = 128;
// fp16 holds normal numbers from 2^-14, which the probabilities of an even row fall short of over more than 16 384 keys:
// where lists may be that long, P is rounded to the type with this factor, which dv loses at the end, so that they are
// normal down to 2^-26. (dS has the loss's scale.) A product an element: the key pass of [1, 15, 8229, 128] with 0.35 of
// the blocks takes 374 us without and 389 with.
constexpr float kPScale = 4096.f;
constexpr int64_t kPNormalKeys = 16384;
constexpr float kFarOffset = 64.f;  // (in log2 units)

struct BwdArgs {
  const void* own_a;  // k or q
  const void* own_b;  // v or do
  const void* st_a;   // q or k
  const void* st_b;   // do or v
  const void* out;    // for delta (query pass)
  void* grad_a;       // dk or dq; may be null
  void* grad_b;       // dv; may be null
  int64_t oa_sb, oa_sh, oa_sl;
  int64_t ob_sb, ob_sh, ob_sl;
  int64_t sa_sb, sa_sh, sa_sl;
  int64_t sb_sb, sb_sh, sb_sl;
  int64_t o_sb, o_sh, o_sl;
  int64_t ga_sb, ga_sh, ga_sl;
  int64_t gb_sb, gb_sh, gb_sl;
  int H, L_own, L_st, n_own, n_st;  // rows and 64-row blocks of the two sides
  int n_items;                      // B * H * n_own
  const int32_t* order;             // dispatch slot -> item, -1 = idle; may be null
  int n_slots;
  // Item's entries idx[item * max_cnt ..], cnt[item] of them (clamped). Key pass over transposed lists (packed):
  // entries idx[bh * n_st * max_cnt + cnt[bh * (n_own + 1) + block] ..] up to the next block's.
  const int32_t* idx;
  const int32_t* cnt;
  int max_cnt, packed;
  const float* bias;  // [b * bias_sb + h * bias_sh + key]
  int64_t bias_sb, bias_sh;
  float sm_scale;
  float scale_log2;     // sm_scale * log2(e)
  float inv_scale_log2;
  float dv_scale;       // 1 / the factor of P (kPScale or 1)
  const float* lse;     // query pass: [bh][64 * query blocks]
  const float* row_max; // with a bias, alike: the rows' offsets
  // [bh][2 * query blocks][2][32]: per 32 query rows their -lse / scale_log2, then their -delta. With a bias
  // [..][4][32], then their offset and lse, which rows use whose first is NaN (all 32 or none). Written by the query
  // pass, read by the key pass.
  float* stats;
  // More than one split: the items of an XCD's dispatch slots first .. first + n_split - 1 (first < 0: every
  // item, n_split of them) are computed by `splits` workgroups each, on shares of the item's steps, which store
  // their sums to partial[place][split][result][64][kD]; bwd_merge_kernel adds them in order.
  int splits, first, n_split;
  // The items of an XCD's last n_last slots (at most kMostLast; not beside splits) run longest list first; lists
  // below 2^length_bits - 1 entries are told apart.
  int n_last, length_bits;
  float* partial;
};

// The two 16-bit values of a pair as floats.
template <typename T>
__device__ inline float2 unpack2(uint32_t w) {
  if constexpr (std::is_same<T, __bf16>::value)
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  const sa_f16x2 h = __builtin_bit_cast(sa_f16x2, w);
  return make_float2((float)h[0], (float)h[1]);
}

// Slots of an XCD.
__host__ __device__ inline int xcd_slots(int64_t n_slots) { return (int)(((n_slots + 3) / 4 + 7) / 8 * 4); }

// Item of slot `seq` of XCD `xcd` (the work order's slots come in groups of four, group w on XCD w % 8).
__device__ inline int slot_item(const BwdArgs& a, int xcd, int seq) {
  const int slot = 4 * (8 * (seq >> 2) + xcd) + (seq & 3);
  if (slot >= a.n_slots) return -1;
  return a.order ? order_item(a.order, slot) : slot;
}

// Entries of an item's list.
template <bool kKeys>
__device__ inline int list_length(const BwdArgs& a, int item) {
  if (!kKeys || !a.packed) return min(max(a.cnt[item], 0), a.max_cnt);
  const int bh = item / a.n_own;
  const int32_t* beg = a.cnt + item + bh;  // bh * (n_own + 1) + block
  return beg[1] - beg[0];
}

// The item with the t-th longest list (from 0) of the XCD's last slots, the same in every lane: the largest key that
// t + 1 of them reach, bit by bit. Keys are unlike, equal lists in order of their slots.
template <bool kKeys>
__device__ inline int longest_item(const BwdArgs& a, int xcd, int from, int t) {
  constexpr int kPer = kMostLast / 64;
  const int lane = threadIdx.x & 63;
  int item[kPer];
  uint32_t key[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int at = lane + 64 * i;
    item[i] = at < a.n_last ? slot_item(a, xcd, from + at) : -1;
    const bool ok = item[i] >= 0 && item[i] < a.n_items;
    const int n = ok ? min(1 + list_length<kKeys>(a, item[i]), (1 << a.length_bits) - 1) : 0;
    key[i] = at < a.n_last ? (uint32_t)(n * kMostLast + kMostLast - 1 - at) : 0;
  }
  uint32_t found = 0;
  for (uint32_t bit = (uint32_t)kMostLast << a.length_bits >> 1; bit; bit >>= 1) {
    int reach = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) reach += __popcll(__ballot(key[i] >= (found | bit)));
    if (reach > t) found |= bit;
  }
  int r = -1;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const uint64_t m = __ballot(key[i] == found && lane + 64 * i < a.n_last);
    if (m) r = __builtin_amdgcn_readlane(item[i], __ffsll((unsigned long long)m) - 1);
  }
  return r;
}

// Item of a workgroup (-1: none), its split, and the place of its sums (-1: not split). The dispatcher deals
// workgroups out to the XCDs in turn. Where every item is split there are no idle workgroups, which would
// leave CUs out of turn ([1, 1, 64 x 17776, 64] in fp32 ran on a quarter of 32 CUs): item and split count up.
template <bool kKeys, bool kSorted>
__device__ inline int bwd_item(const BwdArgs& a, int x, int& split, int& place) {
  split = 0;
  place = -1;
  if (a.splits > 1 && a.first < 0) {
    split = x % a.splits;
    return place = x / a.splits;
  }
  int seq = x >> 3;
  if (a.splits > 1 && seq >= a.first) {
    const int t = (seq - a.first) / a.splits;
    if (t < a.n_split) {
      split = seq - a.first - t * a.splits;
      place = (x & 7) * a.n_split + t;
      seq = a.first + t;
    } else {
      seq -= a.n_split * (a.splits - 1);
    }
  }
  if constexpr (kSorted) {
    const int from = xcd_slots(a.n_slots) - a.n_last;
    if (seq >= from) return longest_item<kKeys>(a, x & 7, from, seq - from);
  }
  return slot_item(a, x & 7, seq);
}

// The item's list: entries list[0 .. n).
template <bool kKeys>
__device__ inline const __attribute__((address_space(4))) int32_t* bwd_list(const BwdArgs& a, int item, int bh,
                                                                              int blk, int& n) {
  const int32_t* p;
  if (kKeys && a.packed) {
    const int32_t* beg = a.cnt + (int64_t)bh * (a.n_own + 1) + blk;
    p = a.idx + (int64_t)bh * a.n_st * a.max_cnt + beg[0];
    n = beg[1] - beg[0];
  } else {
    p = a.idx + (int64_t)item * a.max_cnt;
    n = min(max(a.cnt[item], 0), a.max_cnt);
  }
  return (const __attribute__((address_space(4))) int32_t*)p;
}

// kParts: pairs per workgroup, each on its share of the item's list; their sums are added in LDS, in
// order, at the end. kScaleP: P has the factor kPScale.
template <bool kKeys, bool kBias, typename T, int kD, int kParts, bool kScaleP = false>
__global__ __launch_bounds__(128 * kParts, kD == 64 ? 3 : 2) void bsa_bwd_kernel(BwdArgs a) {
  typedef Elem<T> E;
  typedef typename E::v8 v8;
  constexpr int kDS = kD / 16;      // 16-wide d steps of the first products
  constexpr int kDC = kD / 32;      // 32-row d chunks of the results
  constexpr int kHalves = kD / 64;  // 128-byte half rows per row
  constexpr int kRowTile = kStep * 128;          // one half of a step's rows
  constexpr int kMat = kHalves * kRowTile;       // a step's rows of one matrix
  constexpr bool kStats = kKeys || kBias;
  constexpr int kRowStats = kBias ? 128 : 64;               // statistics of 32 query rows
  constexpr int kStatTile = kKeys ? kRowStats : 64;         // of a step, or its biases
  constexpr int kAcc = kKeys ? 2 : 1;
  constexpr int kRead = !kKeys && !kBias ? 4 : kKeys && kD == 128 ? 1 : 2;
  constexpr bool kEarly = !kKeys || kD == 64;  // registers for the first transposed reads before the exponentials
  // The two stages are separate objects, so that the compiler's waits tell reads of one from the
  // copies into the other.
  __shared__ __attribute__((aligned(1024))) uint8_t tile0[kParts * 2 * kMat], tile1[kParts * 2 * kMat];
  __shared__ __attribute__((aligned(256))) float stat0[kParts * kStatTile], stat1[kParts * kStatTile];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int part = wave >> 1, w = wave & 1;
  const int col = lane & 31, hh = lane >> 5;
  int split, place;
  const int item = __builtin_amdgcn_readfirstlane(bwd_item<kKeys, true>(a, blockIdx.x, split, place));
  if (item < 0 || item >= a.n_items) return;  // (the whole workgroup)
  const int bh = item / a.n_own;
  const int blk = item - bh * a.n_own;
  const int b = bh / a.H;
  const int h = bh - b * a.H;
  int cnt;
  const auto list = bwd_list<kKeys>(a, item, bh, blk, cnt);

  const uint16_t* oa = static_cast<const uint16_t*>(a.own_a) + b * a.oa_sb + h * a.oa_sh;
  const uint16_t* ob = static_cast<const uint16_t*>(a.own_b) + b * a.ob_sb + h * a.ob_sh;
  const int own_row = blk * kBlk + kStep * w + col;
  const int own_clamped = min(own_row, a.L_own - 1);  // rows past L_own are never stored
  v8 fa[kDS], fb[kDS];
#pragma unroll
  for (int s = 0; s < kDS; ++s) {
    fa[s] = __builtin_bit_cast(v8, *reinterpret_cast<const uint4*>(oa + (int64_t)own_clamped * a.oa_sl + 16 * s + 8 * hh));
    fb[s] = __builtin_bit_cast(v8, *reinterpret_cast<const uint4*>(ob + (int64_t)own_clamped * a.ob_sl + 16 * s + 8 * hh));
  }

  float lse = 0.f, offset = 0.f, delta = 0.f;
  bool far = false;  // query pass with a bias: the wave's rows take off offset and lse one after the other
  if constexpr (!kKeys) {
    const uint16_t* op = static_cast<const uint16_t*>(a.out) + b * a.o_sb + h * a.o_sh + (int64_t)own_clamped * a.o_sl;
#pragma unroll
    for (int s = 0; s < kDS; ++s) {
      const sa_u32x4v x = __builtin_bit_cast(sa_u32x4v, *reinterpret_cast<const uint4*>(op + 16 * s + 8 * hh));
      const sa_u32x4v y = __builtin_bit_cast(sa_u32x4v, fb[s]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 o = unpack2<T>(x[i]), d = unpack2<T>(y[i]);
        delta = fmaf(o.x, d.x, fmaf(o.y, d.y, delta));
      }
    }
    delta = xhalf_sum(delta);
    const int64_t at = ((int64_t)bh * a.n_own + blk) * kBlk + kStep * w + col;
    lse = a.lse[at];
    if constexpr (kBias) {
      offset = a.row_max[at];
      far = __ballot(fabsf(offset) > kFarOffset) != 0;
      if (!far) lse += offset;
    }
    if (part == 0 && split == 0) {
      const bool row_ok = own_row < a.L_own;
      float* st = a.stats + (((int64_t)bh * a.n_own + blk) * 2 + w) * kRowStats;
      const float v = hh == 0 ? -lse * a.inv_scale_log2 : -delta;
      st[lane] = kBias && far && hh == 0 ? NAN : row_ok ? v : hh == 0 ? -INFINITY : 0.f;
      if constexpr (kBias) st[64 + lane] = hh == 0 ? (far ? offset : 0.f) : lse;
    }
    if (!a.grad_a) return;  // only the statistics are wanted
  }
  float own_bias = 0.f;
  const float* bias = kBias ? a.bias + b * a.bias_sb + h * a.bias_sh : nullptr;
  if (kKeys && kBias) own_bias = bias[own_clamped] * kLog2e;

  // Streamed rows: wave 0 of the pair copies st_a's (and the statistics or biases), wave 1 st_b's.
  const uint16_t* st = w == 0 ? static_cast<const uint16_t*>(a.st_a) + b * a.sa_sb + h * a.sa_sh
                              : static_cast<const uint16_t*>(a.st_b) + b * a.sb_sb + h * a.sb_sh;
  const uint32_t row_bytes = (uint32_t)(w == 0 ? a.sa_sl : a.sb_sl) * 2;
  const uint32_t st_bytes = (uint32_t)(a.L_st - 1) * row_bytes + 128;
  uint32_t goff[2];  // lane offsets of the copies of rows 0 .. 7 and 8 .. 15 (and of 16 .. 31 from row 16)
#pragma unroll
  for (int j = 0; j < 2; ++j)
    goff[j] = (8 * j + (lane >> 3)) * row_bytes + 16 * ((lane & 7) ^ swz(8 * j + (lane >> 3)));
  const float* stat_src = kKeys ? a.stats + (int64_t)bh * a.n_st * 2 * kRowStats : bias;
  const uint32_t stat_bytes = kKeys ? (uint32_t)a.n_st * 8 * kRowStats : (uint32_t)a.L_st * 4;

  // The split's share of the 2 cnt steps, of it the part's.
  const int splits = place < 0 ? 1 : a.splits;
  const int per_split = (2 * cnt + splits - 1) / splits;
  const int n_steps = min(2 * cnt, per_split * (split + 1));
  const int per_part = (per_split + kParts - 1) / kParts;
  const int beg = split * per_split + part * per_part;
  auto block_of = [&](int i) -> int {  // the streamed block of the part's i-th step, -1: none
    const int s = beg + i;
    return i < per_part && s < n_steps ? list[s >> 1] : -1;
  };
  // Whether the rows of the part's i-th step take off offset and lse one after the other (a scalar load).
  auto far_of = [&](int rb, int i) __attribute__((always_inline)) -> bool {
    if constexpr (!kKeys || !kBias) return far;
    if ((unsigned)rb >= (unsigned)a.n_st) return false;
    const auto* st = (const __attribute__((address_space(4))) float*)stat_src;
    const float first = st[((int64_t)2 * rb + ((beg + i) & 1)) * kRowStats];
    return first != first;
  };
  // Copies of the part's i-th step. The descriptors begin at the step's rows and end with the head's, so
  // that rows past the last one read as zero and the lane offsets never change.
  auto issue = [&](int rb, int i, lds_u8* tile, lds_u8* stat) __attribute__((always_inline)) {
    if ((unsigned)rb >= (unsigned)a.n_st) return;
    const uint32_t row0 = __builtin_amdgcn_readfirstlane(rb * kBlk + kStep * ((beg + i) & 1));
    lds_u8* dst = tile + (part * 2 + w) * kMat;
#pragma unroll
    for (int r16 = 0; r16 < 2; ++r16) {
      const uint32_t off = min((row0 + 16 * r16) * row_bytes, st_bytes);
      const uint8_t* from = reinterpret_cast<const uint8_t*>(st) + off;
#pragma unroll
      for (int hf = 0; hf < kHalves; ++hf) {
        const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<uint8_t*>(from + 128 * hf), (short)0, (int)(st_bytes - off), 0x00020000);
#pragma unroll
        for (int j = 0; j < 2; ++j)
          __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_u8*)(dst + hf * kRowTile + 2048 * r16 + 1024 * j), 16,
                                                   goff[j], 0, 0, 0);
      }
    }
    if (kStats && w == 0) {
      const uint32_t soff = min(kKeys ? row0 * (kRowStats / 8) : row0 * 4, stat_bytes);
      const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<uint8_t*>(reinterpret_cast<const uint8_t*>(stat_src) + soff), (short)0, (int)(stat_bytes - soff),
          0x00020000);
      lds_u8* to = stat + part * 4 * kStatTile;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, to, 4, 4 * lane, 0, 0, 0);
      if constexpr (kStatTile > 64) __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, to, 4, 4 * lane, 0, 256, 0);
    }
  };

  // Lane constants: row operand reads of chunk s and transposed reads (attn_fwd.hip's kro and vro).
  int ro[4], to[2][2];
#pragma unroll
  for (int s = 0; s < 4; ++s) ro[s] = part * 2 * kMat + 128 * col + 16 * ((2 * s + hh) ^ swz(col));
  {
    const int i = lane & 15, hq = lane >> 5, dg = (lane >> 4) & 1;
#pragma unroll
    for (int dc = 0; dc < 2; ++dc)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int r = 8 * t + 4 * hq + (i >> 2);
        const int chunk = 4 * dc + 2 * dg + ((i & 3) >> 1);
        to[dc][t] = part * 2 * kMat + 128 * r + 16 * (chunk ^ swz(r)) + 8 * (i & 1);
      }
  }

  sa_f32x16 acc[kAcc][kDC];
#pragma unroll
  for (int x = 0; x < kAcc; ++x)
#pragma unroll
    for (int dc = 0; dc < kDC; ++dc) acc[x][dc] = sa_f32x16{};
  sa_f32x16 less_delta;  // query pass: dP's accumulators start at -delta
#pragma unroll
  for (int e = 0; e < 16; ++e) less_delta[e] = -delta;

  auto compute = [&](int cur, int i, bool far_step, const lds_u8* tile, const float* stat) __attribute__((always_inline)) {
    if ((unsigned)cur >= (unsigned)a.n_st) return;
    const float* st_ = stat + part * kStatTile + 4 * hh;
    auto stats = [&](int at) __attribute__((always_inline)) {  // 16 of 32 of the step's statistics or biases
      sa_f32x16 r;
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        const float4 y = *reinterpret_cast<const float4*>(st_ + at + 8 * q4);
        r[4 * q4] = y.x; r[4 * q4 + 1] = y.y; r[4 * q4 + 2] = y.z; r[4 * q4 + 3] = y.w;
      }
      return r;
    };
    sa_f32x16 S = {}, dP = less_delta;
    if constexpr (kKeys) {
      if (!kBias || !far_step) S = stats(0);
      dP = stats(32);
    }
    float scale = a.scale_log2, add = kKeys ? own_bias : -lse;  // (with a bias)
    // Row operands in groups of kRead 16-column steps: a group's reads are issued while the products of
    // the group before run, each of which waits for its own two.
    sa_u32x4v x[kDS], y[kDS];
    auto rows = [&](int s0) __attribute__((always_inline)) {
#pragma unroll
      for (int s = s0; s < s0 + kRead; ++s) {
        x[s] = lds_read_b128(tile + ro[s & 3] + (s >> 2) * kRowTile);
        y[s] = lds_read_b128(tile + ro[s & 3] + (s >> 2) * kRowTile + kMat);
      }
    };
    rows(0);
#pragma unroll
    for (int s0 = 0; s0 < kDS; s0 += kRead) {
      __builtin_amdgcn_sched_barrier(0);
      if (s0 + kRead < kDS) rows(s0 + kRead);
#pragma unroll
      for (int s = s0; s < s0 + kRead; ++s) {
        S = E::mfma(E::as8(x[s]), fa[s], S);
        dP = E::mfma(E::as8(y[s]), fb[s], dP);
      }
    }
    // Transposed operands of 64 columns: r[dc][u], requested before they are needed.
    struct Trans {
      uint2 r[2][2][2];
    };
    auto transposed = [&](int x, int hf) __attribute__((always_inline)) {
      Trans t;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int dc = 0; dc < 2; ++dc)
#pragma unroll
          for (int j = 0; j < 2; ++j) t.r[dc][u][j] = lds_read_tr16(tile + x * kMat + hf * kRowTile + 2048 * u + to[dc][j]);
      return t;
    };
    Trans tr;
    if constexpr (kEarly) {
      tr = transposed(kAcc - 1, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
    // Elements e: streamed row 8 (e / 4) + 4 hh + e % 4 of the step, own row col.
    uint32_t Pp[8], Sp[8];
    if constexpr (kKeys) {
      if constexpr (kBias) {
        if (far_step) {  // S becomes the exponent
#pragma unroll
          for (int e = 0; e < 16; e += 4) {  // four rows' offsets, and sums, at a time, read no earlier (the registers)
            __builtin_amdgcn_sched_barrier(0);
            const float4 off = *reinterpret_cast<const float4*>(st_ + 64 + 2 * e);
            S[e] = fmaf(S[e], scale, add) - off.x;
            S[e + 1] = fmaf(S[e + 1], scale, add) - off.y;
            S[e + 2] = fmaf(S[e + 2], scale, add) - off.z;
            S[e + 3] = fmaf(S[e + 3], scale, add) - off.w;
            __builtin_amdgcn_sched_barrier(0);
            const float4 sum = *reinterpret_cast<const float4*>(st_ + 96 + 2 * e);
            S[e] -= sum.x;
            S[e + 1] -= sum.y;
            S[e + 2] -= sum.z;
            S[e + 3] -= sum.w;
          }
          scale = 1.f;
          add = 0.f;
        }
      }
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        const float p0 = fast_exp2(kBias ? fmaf(S[e], scale, add) : S[e] * a.scale_log2);
        const float p1 = fast_exp2(kBias ? fmaf(S[e + 1], scale, add) : S[e + 1] * a.scale_log2);
        Pp[e >> 1] = kScaleP ? E::pack(p0 * kPScale, p1 * kPScale) : E::pack(p0, p1);
        Sp[e >> 1] = E::pack(p0 * dP[e], p1 * dP[e + 1]);
      }
    } else {
      sa_f32x16 kb2 = {};
      if constexpr (kBias) kb2 = stats(0);
      const int row0 = cur * kBlk + kStep * ((beg + i) & 1);
      if (row0 + kStep > a.L_st) {  // keys past the last one: P = 0
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (row0 + 8 * (e >> 2) + 4 * hh + (e & 3) >= a.L_st) S[e] = -INFINITY;
      }
      if constexpr (kBias) {
        if (far_step) {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            S[e] = fmaf(S[e], scale, kb2[e] * kLog2e) - offset - lse;
            kb2[e] = 0.f;
          }
          scale = 1.f;
          add = 0.f;
        }
      }
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        const float p0 = fast_exp2(kBias ? fmaf(S[e], scale, fmaf(kb2[e], kLog2e, add)) : fmaf(S[e], a.scale_log2, -lse));
        const float p1 = fast_exp2(kBias ? fmaf(S[e + 1], scale, fmaf(kb2[e + 1], kLog2e, add))
                                         : fmaf(S[e + 1], a.scale_log2, -lse));
        Sp[e >> 1] = E::pack(p0 * dP[e], p1 * dP[e + 1]);
      }
    }
    if constexpr (!kEarly) tr = transposed(kAcc - 1, 0);
    // st_b^T P first: P is ready first.
#pragma unroll
    for (int j = 0; j < kAcc * kHalves; ++j) {
      const int x = kAcc - 1 - j / kHalves, hf = j % kHalves;
      const Trans now = tr;
      if (j + 1 < kAcc * kHalves) tr = transposed(kAcc - 1 - (j + 1) / kHalves, (j + 1) % kHalves);
      const uint32_t(&P)[8] = x == 0 ? Sp : Pp;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int dc = 0; dc < 2; ++dc)
          acc[x][2 * hf + dc] = E::mfma(
              E::as8(sa_u32x4v{now.r[dc][u][0].x, now.r[dc][u][0].y, now.r[dc][u][1].x, now.r[dc][u][1].y}),
              E::as8(sa_u32x4v{P[4 * u], P[4 * u + 1], P[4 * u + 2], P[4 * u + 3]}), acc[x][2 * hf + dc]);
    }
  };

  lds_u8* const t0 = (lds_u8*)tile0;
  lds_u8* const t1 = (lds_u8*)tile1;
  int rb = block_of(0);
  issue(rb, 0, t0, (lds_u8*)stat0);
  bool far0 = far_of(rb, 0), far1;
  int rb_next = block_of(1);
  for (int i = 0; i < per_part; i += 2) {
    // This wave's copies of step i have landed, then everyone's; every wave is done with step i - 1 (its reads of LDS have
    // returned), whose stage the copies of step i + 1 overwrite.
    __builtin_amdgcn_s_waitcnt(kWaitVmLgkm0);
    wg_barrier();
    issue(rb_next, i + 1, t1, (lds_u8*)stat1);
    far1 = far_of(rb_next, i + 1);
    compute(rb, i, far0, t0, stat0);
    if (i + 1 >= per_part) break;
    rb = block_of(i + 2);
    __builtin_amdgcn_s_waitcnt(kWaitVmLgkm0);
    wg_barrier();
    issue(rb, i + 2, t0, (lds_u8*)stat0);
    far0 = far_of(rb, i + 2);
    compute(rb_next, i + 1, far1, t1, stat1);
    rb_next = block_of(i + 3);
  }

  // ---- Results: element 4 q4 + j of acc[x][dc] is d = 32 dc + 8 q4 + 4 hh + j of own row col.
#pragma unroll
  for (int x = 0; x < kAcc; ++x) {
    uint16_t* g = static_cast<uint16_t*>(x == 0 ? a.grad_a : a.grad_b);
    const int64_t sb = x == 0 ? a.ga_sb : a.gb_sb, sh = x == 0 ? a.ga_sh : a.gb_sh, sl = x == 0 ? a.ga_sl : a.gb_sl;
    const float f = x == 0 ? a.sm_scale : kScaleP ? a.dv_scale : 1.f;
    if constexpr (kParts == 1) {
      if (g && own_row < a.L_own) {
        uint16_t* p = g + b * sb + h * sh + (int64_t)own_row * sl + 4 * hh;
#pragma unroll
        for (int dc = 0; dc < kDC; ++dc)
#pragma unroll
          for (int q4 = 0; q4 < 4; ++q4) {
            const sa_f32x16& A = acc[x][dc];
            *reinterpret_cast<uint2*>(p + 32 * dc + 8 * q4) =
                make_uint2(E::pack(A[4 * q4] * f, A[4 * q4 + 1] * f), E::pack(A[4 * q4 + 2] * f, A[4 * q4 + 3] * f));
          }
      }
    } else {
      constexpr int kCh = kD / 4;  // 16-byte chunks of a row of sums
      // [part][64 rows][kD] sums, chunks swizzled by the row: the first half of the parts over one stage,
      // the others over the other one.
      auto sums = [&](int p) {
        return reinterpret_cast<float*>(p < kParts / 2 ? tile0 : tile1) + (p % (kParts / 2)) * kBlk * kD;
      };
      static_assert(kParts == 1 || kParts / 2 * kBlk * kD * 4 <= kParts * 2 * kMat, "the sums fit a stage");
      __syncthreads();  // every wave is done with the stages (x = 0) or with the last sums
      float* mine = sums(part) + (kStep * w + col) * kD;
#pragma unroll
      for (int dc = 0; dc < kDC; ++dc)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
          const sa_f32x16& A = acc[x][dc];
          *reinterpret_cast<float4*>(mine + 4 * ((8 * dc + 2 * q4 + hh) ^ (col & (kCh - 1)))) =
              make_float4(A[4 * q4], A[4 * q4 + 1], A[4 * q4 + 2], A[4 * q4 + 3]);
        }
      __syncthreads();
      for (int t = threadIdx.x; t < kBlk * kCh; t += 128 * kParts) {
        const int r = t / kCh, ch = t % kCh;
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int p = 0; p < kParts; ++p) {
          const float4 y = *reinterpret_cast<const float4*>(sums(p) + r * kD + 4 * (ch ^ (r & 31 & (kCh - 1))));
          s.x += y.x;
          s.y += y.y;
          s.z += y.z;
          s.w += y.w;
        }
        if (place >= 0)
          *reinterpret_cast<float4*>(a.partial + ((((int64_t)place * a.splits + split) * kAcc + x) * kBlk + r) * kD +
                                     4 * ch) = s;
        else if (g && blk * kBlk + r < a.L_own)
          *reinterpret_cast<uint2*>(g + b * sb + h * sh + (int64_t)(blk * kBlk + r) * sl + 4 * ch) =
              make_uint2(E::pack(s.x * f, s.y * f), E::pack(s.z * f, s.w * f));
      }
    }
  }
}

// ---- fp32: the same passes on the bf16 matrix core, whose rate is 16 times the fp32 one's: every operand is
// split exactly into three bf16 terms (x = hi + mid + lo, 8 significand bits each) and each product takes the six
// term products down to 2^-18 of the largest (the dropped ones are below 2^-26), smallest first, in fp32 sums.
// Streamed rows are loaded a step ahead into registers, split once per pair of waves and stored to LDS as three
// 16-bit tiles of bsa_bwd_kernel's layout, whose row and transposed reads serve both products; P and dS are split
// where they come out. One stage and two barriers per step (a step's products take 2 304 cycles and more at head
// dim 64).
//
// Bound: the matrix core, beside the splits (11 VALU operations a pair of values) and exp2. [1, 30, 2560, 64] with
// half the blocks: query pass 236 us, key pass 297 (162 and 171 TFLOP/s of fp32 products, six times that in bf16 ones, the
// matrix cores 45 and 48 % of the cycles); with merges and lists 250 and 320, on the fp32 matrix instructions 365 and
// 459. [1, 10, 3500, 128] with 0.4 of them 288 and 388 (410 and 555). Values have to be below 3.39e38, from where
// bf16 rounds to infinity; those below about 1e-33, as of gradients of a loss scaled down so far, lose their low terms.

// The six term products of A and B onto c.
__device__ inline sa_f32x16 mfma_terms(const sa_u32x4v (&A)[3], const sa_bf16x8 (&B)[3], sa_f32x16 c) {
  c = mfma32(as_bf16x8(A[0]), B[2], c);
  c = mfma32(as_bf16x8(A[2]), B[0], c);
  c = mfma32(as_bf16x8(A[1]), B[1], c);
  c = mfma32(as_bf16x8(A[0]), B[1], c);
  c = mfma32(as_bf16x8(A[1]), B[0], c);
  return mfma32(as_bf16x8(A[0]), B[0], c);
}

// Eight fp32 values (two 16-byte loads) as operand terms.
__device__ inline void split8(sa_u32x4v x, sa_u32x4v y, sa_u32x4v (&t)[3]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const sa_u32x4v& z = i < 2 ? x : y;
    uint32_t hi, mid, lo;
    split3(__uint_as_float(z[2 * (i & 1)]), __uint_as_float(z[2 * (i & 1) + 1]), hi, mid, lo);
    t[0][i] = hi;
    t[1][i] = mid;
    t[2][i] = lo;
  }
}

template <bool kKeys, int kD>
__global__ __launch_bounds__(256, kD == 64 ? 2 : 1) void bsa_bwd_f32_kernel(BwdArgs a) {
  constexpr int kParts = 2;
  constexpr int kDS = kD / 16;
  constexpr int kDC = kD / 32;
  constexpr int kHalves = kD / 64;
  constexpr int kAcc = kKeys ? 2 : 1;
  constexpr int kRowTile = kStep * 128;       // one half of a step's rows of one term
  constexpr int kTerm = kHalves * kRowTile;   // a step's rows of one term
  constexpr int kMat = 3 * kTerm;             // of one matrix
  constexpr int kLanes = kD / 8;              // lanes per row of a copy, 8 values each
  constexpr int kPasses = kStep * kLanes / 64;
  __shared__ __attribute__((aligned(1024))) uint8_t tile_lds[kParts * 2 * kMat];
  __shared__ __attribute__((aligned(256))) float stat[kParts * 64];
  // The key pass at two waves per SIMD has no registers for its own v's low terms: with them, [1, 30, 2560, 64] took 348
  // us (key pass, lists and merge), without 325. Four registers are still spilled.
  constexpr bool kLowInLds = kKeys && kD == 64;
  __shared__ sa_u32x4v low[kLowInLds ? 2 * kParts : 1][kLowInLds ? kDS : 1][64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int part = wave >> 1, w = wave & 1;
  const int col = lane & 31, hh = lane >> 5;
  int split, place;
  const int item = __builtin_amdgcn_readfirstlane(bwd_item<kKeys, false>(a, blockIdx.x, split, place));
  if (item < 0 || item >= a.n_items) return;  // (the whole workgroup)
  const int bh = item / a.n_own;
  const int blk = item - bh * a.n_own;
  const int b = bh / a.H;
  const int h = bh - b * a.H;
  int cnt;
  const auto list = bwd_list<kKeys>(a, item, bh, blk, cnt);
  const int own_row = blk * kBlk + kStep * w + col;
  const int own_clamped = min(own_row, a.L_own - 1);  // rows past L_own are never stored
  const float* oa = static_cast<const float*>(a.own_a) + b * a.oa_sb + h * a.oa_sh + (int64_t)own_clamped * a.oa_sl + 8 * hh;
  const float* ob = static_cast<const float*>(a.own_b) + b * a.ob_sb + h * a.ob_sh + (int64_t)own_clamped * a.ob_sl + 8 * hh;
  const float* op = kKeys ? nullptr : static_cast<const float*>(a.out) + b * a.o_sb + h * a.o_sh + (int64_t)own_clamped * a.o_sl + 8 * hh;
  sa_bf16x8 fa[kDS][3], fb[kDS][3];
  float lse = 0.f, delta = 0.f;
#pragma unroll
  for (int s = 0; s < kDS; ++s) {
    sa_u32x4v x[2], y[2], t[3];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      x[i] = *reinterpret_cast<const sa_u32x4v*>(oa + 16 * s + 4 * i);
      y[i] = *reinterpret_cast<const sa_u32x4v*>(ob + 16 * s + 4 * i);
      if constexpr (!kKeys) {
        const float4 o = *reinterpret_cast<const float4*>(op + 16 * s + 4 * i);
        delta = fmaf(o.x, __uint_as_float(y[i][0]), fmaf(o.y, __uint_as_float(y[i][1]),
                fmaf(o.z, __uint_as_float(y[i][2]), fmaf(o.w, __uint_as_float(y[i][3]), delta))));
      }
    }
    split8(x[0], x[1], t);
#pragma unroll
    for (int i = 0; i < 3; ++i) fa[s][i] = as_bf16x8(t[i]);
    split8(y[0], y[1], t);
#pragma unroll
    for (int i = 0; i < 3; ++i)
      if (!kLowInLds || i < 2) fb[s][i] = as_bf16x8(t[i]);
    if constexpr (kLowInLds) low[wave][s][lane] = t[2];  // (read by this lane alone)
  }
  if constexpr (!kKeys) {
    delta = xhalf_sum(delta);
    lse = a.lse[((int64_t)bh * a.n_own + blk) * kBlk + kStep * w + col];
    if (part == 0 && split == 0) {
      const bool row_ok = own_row < a.L_own;
      // (the key pass takes lse as it is here: its element costs a fused multiply-add either way)
      const float v = hh == 0 ? -lse : -delta;
      a.stats[(((int64_t)bh * a.n_own + blk) * 2 + w) * 64 + lane] = row_ok ? v : hh == 0 ? -INFINITY : 0.f;
    }
    if (!a.grad_a) return;
  }

  const float* st = w == 0 ? static_cast<const float*>(a.st_a) + b * a.sa_sb + h * a.sa_sh
                           : static_cast<const float*>(a.st_b) + b * a.sb_sb + h * a.sb_sh;
  const uint32_t row_bytes = (uint32_t)(w == 0 ? a.sa_sl : a.sb_sl) * 4;
  const uint32_t st_bytes = (uint32_t)(a.L_st - 1) * row_bytes + 4 * kD;
  const float* stat_src = a.stats + (int64_t)bh * a.n_st * 128;

  const int splits = place < 0 ? 1 : a.splits;
  const int per_split = (2 * cnt + splits - 1) / splits;
  const int n_steps = min(2 * cnt, per_split * (split + 1));
  const int per_part = (per_split + kParts - 1) / kParts;
  const int beg = split * per_split + part * per_part;
  auto block_of = [&](int i) -> int {  // the streamed block of the part's i-th step, -1: none
    const int s = beg + i;
    const int rb = i < per_part && s < n_steps ? list[s >> 1] : -1;
    return (unsigned)rb < (unsigned)a.n_st ? rb : -1;
  };
  // Rows of the part's i-th step: wave 0 st_a's (and the statistics), wave 1 st_b's. The descriptor begins at the
  // step's rows and ends with the head's, so that rows past the last one read as zero.
  const int r_lane = lane / kLanes, c_lane = lane % kLanes;
  sa_u32x4v pre[kPasses][2];
  float pre_stat = 0.f;
  auto fetch = [&](int rb, int i) __attribute__((always_inline)) {
    if (rb < 0) return;
    const uint32_t row0 = __builtin_amdgcn_readfirstlane(rb * kBlk + kStep * ((beg + i) & 1));
    const uint32_t off = min(row0 * row_bytes, st_bytes);
    const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t*>(reinterpret_cast<const uint8_t*>(st) + off), (short)0, (int)(st_bytes - off), 0x00020000);
#pragma unroll
    for (int j = 0; j < kPasses; ++j) {
      const uint32_t at = (j * (64 / kLanes) + r_lane) * row_bytes + 32 * c_lane;
      pre[j][0] = __builtin_bit_cast(sa_u32x4v, __builtin_amdgcn_raw_buffer_load_b128(rsrc, at, 0, 0));
      pre[j][1] = __builtin_bit_cast(sa_u32x4v, __builtin_amdgcn_raw_buffer_load_b128(rsrc, at + 16, 0, 0));
    }
    if (kKeys && w == 0) pre_stat = stat_src[2 * row0 + lane];
  };
  lds_u8* const tile = (lds_u8*)tile_lds + part * 2 * kMat;
  auto stage = [&](int rb) __attribute__((always_inline)) {
    if (rb < 0) return;
#pragma unroll
    for (int j = 0; j < kPasses; ++j) {
      const int r = j * (64 / kLanes) + r_lane;
      sa_u32x4v t[3];
      split8(pre[j][0], pre[j][1], t);
      lds_u8* q = tile + w * kMat + (c_lane >> 3) * kRowTile + 128 * r + 16 * ((c_lane & 7) ^ swz(r));
#pragma unroll
      for (int i = 0; i < 3; ++i) *reinterpret_cast<__attribute__((address_space(3))) sa_u32x4v*>(q + i * kTerm) = t[i];
    }
    if (kKeys && w == 0) stat[part * 64 + lane] = pre_stat;
  };

  // Lane constants of the reads (as in bsa_bwd_kernel).
  int ro[4], to[2][2];
#pragma unroll
  for (int s = 0; s < 4; ++s) ro[s] = 128 * col + 16 * ((2 * s + hh) ^ swz(col));
  {
    const int i = lane & 15, hq = lane >> 5, dg = (lane >> 4) & 1;
#pragma unroll
    for (int dc = 0; dc < 2; ++dc)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int r = 8 * t + 4 * hq + (i >> 2);
        const int chunk = 4 * dc + 2 * dg + ((i & 3) >> 1);
        to[dc][t] = 128 * r + 16 * (chunk ^ swz(r)) + 8 * (i & 1);
      }
  }

  sa_f32x16 acc[kAcc][kDC];
#pragma unroll
  for (int x = 0; x < kAcc; ++x)
#pragma unroll
    for (int dc = 0; dc < kDC; ++dc) acc[x][dc] = sa_f32x16{};

  auto compute = [&](int cur, int i) __attribute__((always_inline)) {
    const int row0 = cur * kBlk + kStep * ((beg + i) & 1);
    if (cur < 0 || row0 >= a.L_st) return;
    sa_f32x16 S = {}, dP = {};
    const float* st_ = stat + part * 64 + 4 * hh;
#pragma unroll
    for (int e = 0; e < 16; ++e) dP[e] = kKeys ? st_[32 + 8 * (e >> 2) + (e & 3)] : -delta;
    // Operands of st_a and st_b in turn, each requested before the products of the one before it.
    sa_u32x4v x[2][3];
    auto rows = [&](int g) __attribute__((always_inline)) {
      const int s = g >> 1;
#pragma unroll
      for (int t = 0; t < 3; ++t)
        x[g & 1][t] = lds_read_b128(tile + ro[s & 3] + (s >> 2) * kRowTile + t * kTerm + (g & 1) * kMat);
    };
    rows(0);
#pragma unroll
    for (int g = 0; g < 2 * kDS; ++g) {
      __builtin_amdgcn_sched_barrier(0);
      if (g + 1 < 2 * kDS) rows(g + 1);
      if (g & 1) {
        if constexpr (kLowInLds) {
          const sa_bf16x8 B[3] = {fb[g >> 1][0], fb[g >> 1][1], as_bf16x8(low[wave][g >> 1][lane])};
          dP = mfma_terms(x[1], B, dP);
        } else {
          dP = mfma_terms(x[1], fb[g >> 1], dP);
        }
      } else {
        S = mfma_terms(x[0], fa[g >> 1], S);
      }
    }
    // Elements e: streamed row 8 (e / 4) + 4 hh + e % 4 of the step, own row col.
    float p[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) p[e] = fast_exp2(fmaf(S[e], a.scale_log2, kKeys ? st_[8 * (e >> 2) + (e & 3)] : -lse));
    if (!kKeys && row0 + kStep > a.L_st) {  // keys past the last one (the statistics see to queries)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (row0 + 8 * (e >> 2) + 4 * hh + (e & 3) >= a.L_st) p[e] = 0.f;
    }
    // st_b^T P, then st_a^T dS, 16 streamed rows (u) at a time.
#pragma unroll
    for (int z = kAcc - 1; z >= 0; --z)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        sa_u32x4v t[3];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int e = 8 * u + 2 * j;
          const float v0 = z ? p[e] : p[e] * dP[e];
          const float v1 = z ? p[e + 1] : p[e + 1] * dP[e + 1];
          uint32_t hi, mid, lo;
          split3(v0, v1, hi, mid, lo);
          t[0][j] = hi;
          t[1][j] = mid;
          t[2][j] = lo;
        }
        const sa_bf16x8 B[3] = {as_bf16x8(t[0]), as_bf16x8(t[1]), as_bf16x8(t[2])};
#pragma unroll
        for (int dc = 0; dc < kDC; ++dc) {
          sa_u32x4v A[3];
#pragma unroll
          for (int i = 0; i < 3; ++i) {
            const lds_u8* q = tile + z * kMat + i * kTerm + (dc >> 1) * kRowTile + 2048 * u;
            const uint2 lo = lds_read_tr16(q + to[dc & 1][0]), hi = lds_read_tr16(q + to[dc & 1][1]);
            A[i] = sa_u32x4v{lo.x, lo.y, hi.x, hi.y};
          }
          acc[z][dc] = mfma_terms(A, B, acc[z][dc]);
        }
      }
  };

  int rb = block_of(0);
  fetch(rb, 0);
  for (int i = 0; i < per_part; ++i) {
    __syncthreads();  // everyone is done with the step before
    stage(rb);
    __syncthreads();
    const int rb_next = block_of(i + 1);
    fetch(rb_next, i + 1);
    compute(rb, i);
    rb = rb_next;
  }

  // ---- Results: the parts' sums are added in LDS, in order.
  constexpr int kCh = kD / 4;
#pragma unroll
  for (int x = 0; x < kAcc; ++x) {
    float* g = static_cast<float*>(x == 0 ? a.grad_a : a.grad_b);
    const int64_t sb = x == 0 ? a.ga_sb : a.gb_sb, sh = x == 0 ? a.ga_sh : a.gb_sh, sl = x == 0 ? a.ga_sl : a.gb_sl;
    const float f = x == 0 ? a.sm_scale : 1.f;
    constexpr int kSums = kBlk * kD;
    static_assert(kParts * kSums * 4 <= kParts * 2 * kMat, "the sums fit the tiles");
    __syncthreads();
    float* mine = reinterpret_cast<float*>(tile_lds) + part * kSums + (kStep * w + col) * kD;
#pragma unroll
    for (int dc = 0; dc < kDC; ++dc)
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        const sa_f32x16& A = acc[x][dc];
        *reinterpret_cast<float4*>(mine + 4 * ((8 * dc + 2 * q4 + hh) ^ (col & (kCh - 1)))) =
            make_float4(A[4 * q4], A[4 * q4 + 1], A[4 * q4 + 2], A[4 * q4 + 3]);
      }
    __syncthreads();
    for (int t = threadIdx.x; t < kBlk * kCh; t += 256) {
      const int r = t / kCh, ch = t % kCh;
      const int at = r * kD + 4 * (ch ^ (r & 31 & (kCh - 1)));
      const float4 y = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(tile_lds) + at);
      const float4 z = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(tile_lds) + kSums + at);
      const float4 s = make_float4(y.x + z.x, y.y + z.y, y.z + z.z, y.w + z.w);
      const int row = blk * kBlk + r;
      if (place >= 0)
        *reinterpret_cast<float4*>(a.partial + ((((int64_t)place * a.splits + split) * kAcc + x) * kBlk + r) * kD +
                                   4 * ch) = s;
      else if (g && row < a.L_own)
        *reinterpret_cast<float4*>(g + b * sb + h * sh + (int64_t)row * sl + 4 * ch) =
            make_float4(s.x * f, s.y * f, s.z * f, s.w * f);
    }
  }
}

// Gradients from the splits' sums, in order: D / 16 workgroups per split item and result, four values a thread.
template <bool kKeys, typename T>
__global__ __launch_bounds__(256) void bwd_merge_kernel(BwdArgs a, int D) {
  constexpr int kAcc = kKeys ? 2 : 1;
  const int place = blockIdx.x, x = blockIdx.y;
  const int item = a.first < 0 ? place : slot_item(a, place / a.n_split, a.first + place % a.n_split);
  if (item < 0 || item >= a.n_items) return;
  const int bh = item / a.n_own;
  const int blk = item - bh * a.n_own;
  const int b = bh / a.H;
  const int h = bh - b * a.H;
  T* g = static_cast<T*>(x == 0 ? a.grad_a : a.grad_b);
  if (!g) return;
  g += b * (x == 0 ? a.ga_sb : a.gb_sb) + h * (x == 0 ? a.ga_sh : a.gb_sh);
  const int64_t sl = x == 0 ? a.ga_sl : a.gb_sl;
  const float f = x == 0 ? a.sm_scale : a.dv_scale;
  const int64_t n = (int64_t)kBlk * D;
  const float* from = a.partial + ((int64_t)place * a.splits * kAcc + x) * n;
  const int t = blockIdx.z * 256 + threadIdx.x;
  const int r = t / (D / 4), d = 4 * (t % (D / 4));
  if (blk * kBlk + r >= a.L_own) return;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int p = 0; p < a.splits; ++p) {
    const float4 y = *reinterpret_cast<const float4*>(from + (int64_t)p * kAcc * n + 4 * t);
    s.x += y.x;
    s.y += y.y;
    s.z += y.z;
    s.w += y.w;
  }
  T* o = g + (int64_t)(blk * kBlk + r) * sl + d;
  if constexpr (std::is_same<T, float>::value)
    *reinterpret_cast<float4*>(o) = make_float4(s.x * f, s.y * f, s.z * f, s.w * f);
  else
    *reinterpret_cast<uint2*>(o) = make_uint2(Elem<T>::pack(s.x * f, s.y * f), Elem<T>::pack(s.z * f, s.w * f));
}

template <bool kKeys, typename T>
void launch_merge(const BwdArgs& a, int D, hipStream_t s) {
  if (a.splits > 1)
    hipLaunchKernelGGL((bwd_merge_kernel<kKeys, T>), dim3((unsigned)(a.first < 0 ? a.n_items : 8 * a.n_split), kKeys ? 2 : 1, D / 16),
                       dim3(256), 0, s, a, D);
}

unsigned workgroups(const BwdArgs& a) {
  if (a.splits > 1 && a.first < 0) return (unsigned)a.n_items * a.splits;
  return 8u * (xcd_slots(a.n_slots) + (a.splits - 1) * a.n_split);
}

template <bool kKeys, typename T, int kD, int kParts>
void launch_parts(const BwdArgs& a, hipStream_t s) {
  const dim3 grid(workgroups(a)), blk(128 * kParts);
  if constexpr (kKeys && std::is_same<T, _Float16>::value) {
    if (a.dv_scale != 1.f) {
      if (a.bias) hipLaunchKernelGGL((bsa_bwd_kernel<kKeys, true, T, kD, kParts, true>), grid, blk, 0, s, a);
      else hipLaunchKernelGGL((bsa_bwd_kernel<kKeys, false, T, kD, kParts, true>), grid, blk, 0, s, a);
      return;
    }
  }
  if (a.bias) hipLaunchKernelGGL((bsa_bwd_kernel<kKeys, true, T, kD, kParts>), grid, blk, 0, s, a);
  else hipLaunchKernelGGL((bsa_bwd_kernel<kKeys, false, T, kD, kParts>), grid, blk, 0, s, a);
}

// Pairs per item, by the number of items and the lists' width (how many entries they hold the host does
// not know). One or two pairs, us of the query pass (the key pass is alike; four pairs, one workgroup per
// CU: slower in every case but those that splits_of takes):
//   head dim 64, dense lists of 40: 160 items 43 / 24, 320 47 / 32, 1 280 93 / 86, 1 920 141 / 132; of 10:
//     40 items 13.8 / 10.3, 640 20 / 20, 1 500 33 / 36; lists of 5 of 40: 640 items 19 / 17, 1 920 32 / 33, 3 200
//     45 / 51; 28 of 278: 278 items 51 / 30, 2 224 120 / 115;
//   head dim 128, dense lists of 40: 160 items 62 / 41, 320 82 / 59, 640 98 / 100, 1 280 178 / 165, 1 920 239 /
//     245; of 10: 320 27 / 24, 640 34 / 37; 28 of 278: 1 112 139 / 125, 2 224 225 / 232.
// (Lists much longer than the others, of text blocks say, gain further by a second pair: [1, 15, 17776,
// 64] with 4 of 278 blocks dense 449 / 431 us.)
int pairs_per_item(int n_items, int max_cnt, int D) {
  if (D == 64) return n_items > 768 && max_cnt <= 16 ? 1 : 2;
  return n_items <= 512 || (n_items <= 1536 && max_cnt >= 32) ? 2 : 1;
}

// Splits of each item's list over workgroups of two pairs, where the items leave most of the card idle
// and their lists (of up to `width` entries) are long: at least 8 entries each. Without / with, us of the
// query pass of 64 queries and the key pass of 64 keys against 17 776 of the other: one head 93 / 9 and 114 / 10,
// 30 heads 112 / 27 and 120 / 29; [1, 1, 2048, 64], 8 of 32 blocks, 10.3 / 7.0 and 10.9 / 8.0; fp32 [1, 4, 2000, 64], 0.3 of
// 32 blocks, in three or four 32.8 / 29.2 and 55.7 / 49.8. The merge is 4 to 5 us more: two to five splits gain no more than that (160 items with dense
// lists of 40: 24.2 / 21.2 and the merge), but in fp32, whose steps take six times as long.
int splits_of(int64_t n_items, int width, int D, bool f32) {
  if (width < (f32 ? 16 : 32)) return 1;
  const int64_t slots = f32 ? (D == 64 ? 512 : 256) : (D == 64 ? 768 : 512);  // such workgroups on the card
  const int64_t fit = slots / n_items;
  if (fit < (f32 ? 4 : 6)) return 1;
  return (int)std::min<int64_t>({fit, width / 8, 32});
}

// The most text items of an XCD (its items are a contiguous eighth, the first n_text of each n_own text).
int text_slots(int64_t n_items, int n_own, int n_text) {
  n_text = std::min(n_text, n_own);
  auto before = [&](int64_t it) { return it / n_own * n_text + std::min<int64_t>(it % n_own, n_text); };
  int64_t most = 0;
  for (int x = 0; x < 8; ++x) most = std::max(most, before(n_items * (x + 1) / 8) - before(n_items * x / 8));
  return (int)most;
}

// How the items of a pass are dealt out.
struct Deal {
  int parts;                   // pairs of waves per workgroup
  int splits, first, n_split;  // as in BwdArgs
  int n_last, length_bits;
  int64_t places() const { return splits == 1 ? 0 : first < 0 ? n_split : 8 * (int64_t)n_split; }  // items that are split
};

// fp32: the items behind the last full round of an XCD's workgroups are split, by three where lists may be long.
// Whole / split, us of the query and key pass with the merge: [1, 30, 2560, 64] half the blocks 262 / 256 and 353 /
// 330, 0.15 of them 104 / 103 and 153 / 153; [1, 12, 2100, 64], less than a round, 106 / 95 and 142 / 139; [1, 10,
// 3500, 128] 340 / 289 and 447 / 390, [1, 3, 1700, 128] 80 / 51 and 125 / 81; at worst, by two, [2, 10, 1500, 64] 60 / 60
// and 86 / 92. 16-bit steps are too short for it: dense lists of 40 gain 171 / 163 and 229 / 227 (by two 159 and 222),
// the same lists with a fifth of the blocks lose 54 / 61 and 87 / 94, and the host does not know which they are.
//
// 16 bits: text items, several times as long as the others, are split by two where they outlast them: up to one
// round of workgroups over lists of 40 and more, two rounds over 96. Whole / split, us of the query pass, texts of 4
// blocks: [2, 12, 1350 x 5626, 64] with 0.3 of the blocks 59 / 53, [1, 8, 3000, 64] 0.2 of them 31 / 26, [1, 10, 8000, 64]
// 0.1 of them 78 / 59 (more splits: 51, 26, 63 and slower); past those lines [1, 5, 1500, 64] 18 / 20, [1, 24, 4546,
// 64] 89 / 95, [1, 20, 3000, 64] dense 80 / 90, [1, 30, 8000, 64] 136 / 147.
//
// 16 bits, more than one round: the last round's items, which run together in any order, start with the longest lists
// (other orders of all items part neighbours that share keys). Order of the items / longest first, us of both
// passes, random lists: [1, 15, 8229, 128] 0.35 of the blocks 315 / 280 and 411 / 385, [2, 15, 4096, 128] 0.3 of them 139 /
// 126 and 200 / 185, [1, 15, 17776, 64] 0.2 of them 377 / 359 and 511 / 504, [1, 8, 8192, 64] 0.3 of them 80 / 72 and 117 /
// 108; equal or short lists pay one to two us for it: [2, 30, 2560, 64] a fifth of 40 blocks 53 / 54 and 86 / 88.
Deal deal(int64_t n_items, int n_own, int n_text, int width, int D, bool f32) {
  Deal d = {2, splits_of(n_items, width, D, f32), -1, (int)n_items, 0, 1};
  if (d.splits > 1) return d;
  const int slots = xcd_slots(n_items);
  if (f32) {
    const int left = slots % (D == 64 ? 64 : 32);  // (two workgroups, or one, per CU)
    if (left > 0 && width >= 16) d = {2, width >= 32 ? 3 : 2, slots - left, left, 0, 1};
    return d;
  }
  d.parts = pairs_per_item((int)n_items, width, D);
  const int room = 32 * (D == 64 ? 3 : 2);  // of workgroups of two pairs
  if (n_text > 0 && d.parts == 2 && (slots <= room ? width >= 40 : slots <= 2 * room && width >= 96))
    return {2, 2, 0, text_slots(n_items, n_own, n_text), 0, 1};
  const int round = room * 2 / d.parts;
  if (slots > round && round <= kMostLast && width >= (D == 64 ? 64 : 32)) {
    d.n_last = round;
    while (d.length_bits < 22 && (1 << d.length_bits) < width + 3) ++d.length_bits;
  }
  return d;
}

template <bool kKeys, typename T, int kD>
void launch_pass(const BwdArgs& a, int parts, hipStream_t s) {
  if (parts == 2) launch_parts<kKeys, T, kD, 2>(a, s);
  else launch_parts<kKeys, T, kD, 1>(a, s);
  launch_merge<kKeys, T>(a, kD, s);
}

template <bool kKeys>
void launch_pass_f32(const BwdArgs& a, int D, hipStream_t s) {
  const dim3 grid(workgroups(a)), blk(256);
  if (D == 64) hipLaunchKernelGGL((bsa_bwd_f32_kernel<kKeys, 64>), grid, blk, 0, s, a);
  else hipLaunchKernelGGL((bsa_bwd_f32_kernel<kKeys, 128>), grid, blk, 0, s, a);
  launch_merge<kKeys, float>(a, D, s);
}

template <bool kKeys>
void launch_pass_any(BwdArgs& a, int dtype, int D, const Deal& d, hipStream_t s) {
  // (a caller's order may have fewer slots than a plain one)
  a.splits = d.first >= 0 && d.first + d.n_split > xcd_slots(a.n_slots) ? 1 : d.splits;
  a.first = d.first;
  a.n_split = d.n_split;
  a.n_last = a.splits == 1 ? std::min(d.n_last, xcd_slots(a.n_slots)) : 0;
  a.length_bits = d.length_bits;
  if (dtype == SA_DTYPE_F32) return launch_pass_f32<kKeys>(a, D, s);
  if (dtype == SA_DTYPE_F16)
    return D == 64 ? launch_pass<kKeys, _Float16, 64>(a, d.parts, s) : launch_pass<kKeys, _Float16, 128>(a, d.parts, s);
  return D == 64 ? launch_pass<kKeys, __bf16, 64>(a, d.parts, s) : launch_pass<kKeys, __bf16, 128>(a, d.parts, s);
}

int64_t align256(int64_t n) { return (n + 255) / 256 * 256; }

// Workspace of a backward pass: the query rows' statistics, the transposed lists, the splits' sums (of one
// pass at a time).
struct Layout {
  int64_t q_beg, q_idx, partial, bytes;
  Deal q, k;
};

Layout layout(const sa_attn_train& t) {
  const int64_t BH = (int64_t)t.B * t.H, nqb = sa::cdiv(t.Lq, kBlk), nkb = sa::cdiv(t.Lk, kBlk);
  const bool f32 = t.dtype == SA_DTYPE_F32;
  Layout l;
  l.q_beg = align256(BH * nqb * (t.key_bias ? 256 : 128) * (int64_t)sizeof(float));
  l.q_idx = l.q_beg + (t.q_idx ? 0 : align256(BH * (nkb + 1) * (int64_t)sizeof(int32_t)));
  l.partial = l.q_idx + (t.q_idx ? 0 : align256(BH * nqb * t.max_cnt * (int64_t)sizeof(int32_t)));
  // (a list is no longer than the other side has blocks, but for repeated entries)
  l.q = deal(BH * nqb, (int)nqb, t.n_text_blocks, (int)std::min<int64_t>(t.max_cnt, nkb), t.D, f32);
  l.k = deal(BH * nkb, (int)nkb, t.n_text_blocks, (int)nqb, t.D, f32);
  const int64_t tile = (int64_t)kBlk * t.D * sizeof(float);
  l.bytes = l.partial + std::max(l.q.places() * l.q.splits * tile, l.k.places() * l.k.splits * 2 * tile);
  return l;
}

int check_train(const sa_attn_train* t, const char* fn) {
  SA_REQUIRE(t, "%s: null pointer", fn);
  SA_REQUIRE(t->dtype == SA_DTYPE_BF16 || t->dtype == SA_DTYPE_F16 || t->dtype == SA_DTYPE_F32, "%s: dtype %d", fn,
             t->dtype);
  SA_REQUIRE(t->B > 0 && t->H > 0 && t->Lq > 0 && t->Lk > 0, "%s: bad shape B=%d H=%d Lq=%d Lk=%d", fn, t->B, t->H,
             t->Lq, t->Lk);
  if (t->D != 64 && t->D != 128) return sa::fail(SA_ERR_UNSUPPORTED, "%s: head_dim %d (64 or 128)", fn, t->D);
  SA_REQUIRE(t->max_cnt > 0, "%s: max_cnt must be > 0", fn);
  const int64_t nqb = sa::cdiv(t->Lq, kBlk), nkb = sa::cdiv(t->Lk, kBlk), BH = (int64_t)t->B * t->H;
  SA_REQUIRE(BH * nqb < (1LL << 28) && BH * nkb < (1LL << 28), "%s: too many blocks", fn);
  return SA_OK;
}

// What the passes cannot take, of a call whose sizes are right.
int check_limits(const sa_attn_train* t, const char* fn) {
  SA_REQUIRE(std::isfinite(t->sm_scale) && t->sm_scale > 0.f, "%s: sm_scale must be finite and > 0", fn);
  // (the key pass takes the rows' sums in units of the scores, lse / sm_scale)
  if (t->sm_scale < 1e-30f) return sa::fail(SA_ERR_UNSUPPORTED, "%s: sm_scale %g below 1e-30", fn, t->sm_scale);
  if (t->dtype == SA_DTYPE_F32 && t->key_bias) return sa::fail(SA_ERR_UNSUPPORTED, "%s: fp32 with key_bias", fn);
  // Streamed rows are copied through 32-bit buffer offsets relative to each head's first row, and so are the statistics
  // (up to 16 bytes a row; rows may be expanded ones, which take no room).
  if (t->Lq > 1 << 27 || t->Lk > 1 << 27) return sa::fail(SA_ERR_UNSUPPORTED, "%s: more than 2^27 rows", fn);
  const int size = t->dtype == SA_DTYPE_F32 ? 4 : 2;
  const int64_t rows[4] = {t->Lq, t->Lk, t->Lk, t->Lq};
  const int at[4] = {0, 1, 2, 4};
  for (int i = 0; i < 4; ++i) {
    const int64_t stride = t->strides[3 * at[i] + 2];
    if (stride < 0 || stride > INT_MAX || (rows[i] + kBlk) * stride * size + 2 * t->D > INT_MAX)
      return sa::fail(SA_ERR_UNSUPPORTED, "%s: rows of one head span more than 2 GiB", fn);
  }
  // (sa_kv_list_transpose's)
  if ((t->dk || t->dv) && !t->q_idx && (t->max_cnt > 65535 || sa::cdiv(t->Lq, kBlk) * (int64_t)t->max_cnt >= (1LL << 31)))
    return sa::fail(SA_ERR_UNSUPPORTED, "%s: lists of %d entries", fn, t->max_cnt);
  return SA_OK;
}

}  // namespace

extern "C" int sa_block_sparse_bwd_check(const sa_attn_train* t) {
  const char* fn = "sa_block_sparse_bwd_check";
  if (int rc = check_train(t, fn)) return rc;
  if (int rc = check_limits(t, fn)) return rc;
  return sa::ok();
}

extern "C" int sa_block_sparse_bwd_workspace(const sa_attn_train* t, int64_t* bytes) {
  const char* fn = "sa_block_sparse_bwd_workspace";
  SA_REQUIRE(bytes, "%s: null bytes", fn);
  if (int rc = check_train(t, fn)) return rc;
  *bytes = layout(*t).bytes;
  return sa::ok();
}

extern "C" int sa_block_sparse_bwd(const sa_attn_train* t, void* stream) {
  const char* fn = "sa_block_sparse_bwd";
  if (int rc = check_train(t, fn)) return rc;
  const int B = t->B, H = t->H, Lq = t->Lq, Lk = t->Lk, D = t->D;
  SA_REQUIRE(t->q && t->k && t->v && t->out && t->dout && t->lse && t->kv_idx && t->kv_cnt && !t->q_idx == !t->q_cnt,
             "%s: null pointer", fn);
  if (int rc = check_limits(t, fn)) return rc;
  const bool f32 = t->dtype == SA_DTYPE_F32;
  SA_REQUIRE(!t->key_bias || t->row_max, "%s: key_bias without row_max", fn);
  const int nqb = sa::cdiv(Lq, kBlk), nkb = sa::cdiv(Lk, kBlk);
  const int per16 = f32 ? 4 : 8;
  const void* ptrs[8] = {t->q, t->k, t->v, t->out, t->dout, t->dq, t->dk, t->dv};
  const int64_t* strides = t->strides;
  for (int i = 0; i < 8; ++i) {
    if (reinterpret_cast<uintptr_t>(ptrs[i]) % 16 != 0)
      return sa::fail(SA_ERR_UNSUPPORTED, "%s: tensor base not 16-byte aligned", fn);
    for (int j = 0; j < 3; ++j)
      if (ptrs[i] && strides[3 * i + j] % per16 != 0)
        return sa::fail(SA_ERR_UNSUPPORTED, "%s: strides must be multiples of %d elements", fn, per16);
  }
  Layout l = layout(*t);
  SA_REQUIRE(t->workspace && reinterpret_cast<uintptr_t>(t->workspace) % 256 == 0,
             "%s: workspace null or not 256-byte aligned", fn);
  SA_REQUIRE(t->workspace_bytes >= l.bytes, "%s: workspace of %lld bytes < %lld", fn, (long long)t->workspace_bytes,
             (long long)l.bytes);
  SA_REQUIRE((!t->q_order || (t->n_q_slots > 0 && t->n_q_slots % 4 == 0 && t->n_q_slots < (1LL << 30))) &&
                 (!t->k_order || (t->n_k_slots > 0 && t->n_k_slots % 4 == 0 && t->n_k_slots < (1LL << 30))),
             "%s: slots must be a positive multiple of 4", fn);
  uint8_t* ws = static_cast<uint8_t*>(t->workspace);
  int32_t* q_beg = reinterpret_cast<int32_t*>(ws + l.q_beg);
  int32_t* q_idx = reinterpret_cast<int32_t*>(ws + l.q_idx);
  hipStream_t s = sa::as_stream(stream);
  if ((t->dk || t->dv) && !t->q_idx) {
    if (int rc = sa_kv_list_transpose(t->kv_idx, t->kv_cnt, B * H, nqb, nkb, t->max_cnt, q_beg, q_idx, stream)) return rc;
  }
  BwdArgs a;
  a.H = H;
  a.max_cnt = t->max_cnt;
  a.packed = 0;
  a.bias = t->key_bias;
  a.bias_sb = t->key_bias ? t->bias_strides[0] : 0;
  a.bias_sh = t->key_bias ? t->bias_strides[1] : 0;
  a.sm_scale = t->sm_scale;
  a.scale_log2 = t->sm_scale * kLog2e;
  a.inv_scale_log2 = 1.f / a.scale_log2;
  // (a block listed more than once counts as often)
  a.dv_scale = t->dtype == SA_DTYPE_F16 && (int64_t)t->max_cnt * kBlk > kPNormalKeys ? 1.f / kPScale : 1.f;
  a.lse = t->lse;
  a.row_max = t->row_max;
  a.stats = reinterpret_cast<float*>(ws);
  a.partial = reinterpret_cast<float*>(ws + l.partial);
  a.out = t->out;
  a.o_sb = strides[9]; a.o_sh = strides[10]; a.o_sl = strides[11];

  a.own_a = t->q; a.oa_sb = strides[0]; a.oa_sh = strides[1]; a.oa_sl = strides[2];
  a.own_b = t->dout; a.ob_sb = strides[12]; a.ob_sh = strides[13]; a.ob_sl = strides[14];
  a.st_a = t->k; a.sa_sb = strides[3]; a.sa_sh = strides[4]; a.sa_sl = strides[5];
  a.st_b = t->v; a.sb_sb = strides[6]; a.sb_sh = strides[7]; a.sb_sl = strides[8];
  a.grad_a = t->dq; a.ga_sb = strides[15]; a.ga_sh = strides[16]; a.ga_sl = strides[17];
  a.grad_b = nullptr; a.gb_sb = a.gb_sh = a.gb_sl = 0;
  a.L_own = Lq; a.L_st = Lk; a.n_own = nqb; a.n_st = nkb;
  a.n_items = B * H * nqb;
  a.order = t->q_order;
  a.n_slots = (int)(t->q_order ? t->n_q_slots : (a.n_items + 3) / 4 * 4);
  a.idx = t->kv_idx; a.cnt = t->kv_cnt;
  if (!t->dq) l.q.splits = 1;
  launch_pass_any<false>(a, t->dtype, D, l.q, s);
  if (int rc = sa::check_launch(fn)) return rc;
  if (!t->dk && !t->dv) return sa::ok();

  a.own_a = t->k; a.oa_sb = strides[3]; a.oa_sh = strides[4]; a.oa_sl = strides[5];
  a.own_b = t->v; a.ob_sb = strides[6]; a.ob_sh = strides[7]; a.ob_sl = strides[8];
  a.st_a = t->q; a.sa_sb = strides[0]; a.sa_sh = strides[1]; a.sa_sl = strides[2];
  a.st_b = t->dout; a.sb_sb = strides[12]; a.sb_sh = strides[13]; a.sb_sl = strides[14];
  a.grad_a = t->dk; a.ga_sb = strides[18]; a.ga_sh = strides[19]; a.ga_sl = strides[20];
  a.grad_b = t->dv; a.gb_sb = strides[21]; a.gb_sh = strides[22]; a.gb_sl = strides[23];
  a.L_own = Lk; a.L_st = Lq; a.n_own = nkb; a.n_st = nqb;
  a.n_items = B * H * nkb;
  a.order = t->k_order;
  a.n_slots = (int)(t->k_order ? t->n_k_slots : (a.n_items + 3) / 4 * 4);
  a.idx = t->q_idx ? t->q_idx : q_idx;
  a.cnt = t->q_idx ? t->q_cnt : q_beg;
  a.packed = !t->q_idx;
  if (t->q_idx) a.max_cnt = nqb;
  launch_pass_any<true>(a, t->dtype, D, l.k, s);
  return sa::check_launch(fn);
}
