// Kernels of attention with score rules (attn_scored.hip has the mathematics, the plan of a call and its entry points).
//
// All three passes are one kernel, in the manner of attn_bwd.hip: the "own" side is the block whose results a
// workgroup computes, the "streamed" side the listed blocks, 32 rows of it at a time (a step) in two LDS stages that
// a pair of waves shares: rows of step i + 1 are copied while step i computes. Each wave owns 32 rows of the block,
// whose operands stay in registers; the own row is the MFMA column:
//   kForward  own q,        streamed k, v    S^T = k q^T; out^T += v^T P
//   kQueries  own q, do     streamed k, v    S^T, dP^T = v do^T; dq^T += k^T dC
//   kKeys     own k, v      streamed q, do   S, dP = do v^T; dv^T += do^T P; dk^T += q^T dC
// P and dC come out of the first products in the layout of the second ones' B operand. No sum is shared by
// workgroups: results do not depend on the order in which they run.
//
// Bound: the matrix instructions and the vector ones beside them, at the clock that the power limit leaves. An element
// of a tile takes 3 D (forward: 2 D, and D for P's second term), 3 D and 4 D products, and an exp2, a scaling, a sum, a
// rounding or two: at [1, 15, 17776, 64] by frames of 1350 the matrix units are busy for 51, 57 and 57 % of the
// three passes' cycles and vector instructions issue in 77, 51 and 50 %, at 1.8 GHz; LDS has no bank conflicts. Shorter or
// capped calls have neither unit busy (25 to 40 %, 30 to 58 %): with two or three waves a SIMD each step waits for its copies, a
// barrier and the chains of its products. The query and key passes spill registers where there is a cap besides slopes or a
// bias, the key pass at head dim 128 always (8 to 48 of them).
// Measured, us of forward, query and key pass (TFLOP/s of the products done), of 50 passes without a pause: 1010, 930, 1225
// (970, 1050, 1065) there; seven documents in a row of [1, 15 of 5 key heads, 8229, 128] fp16 with a cap 123, 132, 175 (its tanh is
// an exp2, a reciprocal and three more an element); [2, 30, 2560, 64] with a bias 193, 205, 222 (780, 740, 910).
// Tiles of 32 own rows a wave: 64 would halve the LDS reads, which are not the bound, for twice the registers.
#pragma once

#include <math.h>

#include <climits>
#include <type_traits>

#include "attn_score.h"

namespace sa_scored {

constexpr int kBlk = 64;
constexpr int kCus = 256;
enum { kForward = 0, kQueries = 1, kKeys = 2 };
enum { kPlain = 0, kSlopes = 1, kTable = 2 };  // (both: 3)
// How scores are capped (bend). A choice of kernels: with both ways in one, registers that fit are spilled (query pass with
// slopes at head dim 64 20 bytes a lane, 36 so).
enum { kNoCap = 0, kTanh = 1, kFineTanh = 2 };
// fp16 holds normal numbers from 2^-14, which the probabilities of an even row fall short of over more than 16 384
// keys: P is rounded to the type with this factor (one product an element), which dv loses at the end.
constexpr float kPScale = 4096.f;

// Distances past the radius that the expanded biases repeat on each side, so that the 95 distances of a step and a block
// are next to each other wherever one of them is not past it.
constexpr int kPad = 96;
constexpr int kWindow = 128;
constexpr int kDiagonals = 8 * 64;  // floats of a wave in which dS is summed by distance (16 * 64: a workgroup less on a CU)

struct Side {
  const void* p;
  int64_t sb, sh, sl;  // elements
};

struct ScoredArgs {
  Side own_a, own_b, st_a, st_b, out;  // out: for delta
  void *grad_a, *grad_b;               // out, dq, or dk and dv
  int64_t ga_sb, ga_sh, ga_sl, gb_sb, gb_sh, gb_sl;
  int heads_own, BH_own;  // key heads in kKeys, else query heads
  int H, rep;             // query heads, and how many share a key head
  int L_own, L_st, n_own, n_st, q_start;
  // Lists of the own blocks: entries (block << 1 | cut) idx[row * width ..], cnt[row] of them, row = ((b or, per_head,
  // b * H + query head) * n_own + block); idx null: every block, all cut if there are ranges.
  const int32_t *idx, *cnt;
  int per_head;
  const int2* ranges;  // [b * ranges_sb + key] = {from, until}; may be null
  int64_t ranges_sb;
  float sm_scale, scale_log2;
  float cap_in, cap_log2;  // 2 log2(e) sm_scale / cap (fine: sm_scale / cap), cap log2(e)
  const float* slopes;     // [H]; may be null
  const float* ebias;      // [H][2 radius + 1 + 2 kPad] biases of distances -radius - kPad .., times log2(e); may be null
  int radius;
  float* lse;              // [b * H + h][64 n]
  float2* offsets;         // with slopes: {offset, log2-sum-exp2 relative to it} of each row, laid out like lse; else null
  // [b * H + h][2 n][2][32]: of 32 query rows their lse, then their delta. With slopes [4][32]: the relative one, delta, the
  // offset, the position p.
  float* stats;
  void* out_lo;            // what out's rounding left out, laid out like it; may be null
  // Units of work of each XCD, {item = (b * heads_own + head) * n_own + block, first entry, behind the last, place of the
  // sums}: units[xcd * unit_cap ..], n_units[xcd] of them (scored_schedule_kernel). Null: items as own_block has them.
  const int4* units;
  const int32_t* n_units;
  int unit_cap;
  float* parts;      // units of split items: [place][result][64][kD]
  float* part_sums;  // kForward: [place][64] {offset, sum}
  float* far;        // kQueries, nullable: [item][2 radius + 1] sums of dS by distance
  float* part_far;   // and [place]
};

// The rule on a tile's products S, but for the slopes: S times what is returned is the score times log2(e). least .. least + 62:
// the wave's distances. window: where the lane's biases lie in LDS, from element 0 (kSign > 0) or element 15 (kSign < 0) on; element
// e is kSign (8 (e / 4) + e % 4) away from element 0. kSlope: slope becomes the cap's derivative. side: whether all pairs of the
// wave are past the radius, 1 above, -1 below, 0 not all.
template <int kSign, int kCap, int kRule, bool kSlope, typename T>
__device__ __forceinline__ float apply_rule(const ScoredArgs& a, float past, float before, int least, const float* window,
                                            sa_f32x16& S, sa_f32x16& slope, int& side) {
  float sc = a.scale_log2;
  if constexpr (kCap) {
    bend_all<kCap == kFineTanh || std::is_same<T, float>::value, kSlope>(a.cap_in, a.cap_log2, S, slope);
    sc = 1.f;
  }
  side = 0;
  if constexpr (kRule & kTable) {
    side = least >= a.radius ? 1 : least + 62 <= -a.radius ? -1 : 0;
    if (side) {
      const float c = side > 0 ? past : before;
#pragma unroll
      for (int e = 0; e < 16; ++e) S[e] = fmaf(S[e], sc, c);
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int c = 8 * (e >> 2) + (e & 3);
        S[e] = fmaf(S[e], sc, window[kSign > 0 ? c : 27 - c]);
      }
    }
    sc = 1.f;
  }
  return sc;
}

// A cut tile of own queries: pairs that are not seen get -inf. row: the lane's query row; key0: its key at element 0. Where
// there are ranges, the step's intervals lie at `intervals` in LDS (keys past the last one: no rows): read from memory here
// they held up the step (seven documents in a row, forward 161 us, not 132).
__device__ __forceinline__ void cut_keys(const ScoredArgs& a, int Lk, int row, int key0, int lane, const lds_u8* intervals,
                                         sa_f32x16& S) {
  if (a.ranges) {
    asm volatile("" : "+v"(lane));  // (the address is worked out here, not kept in a register throughout)
    const lds_u8* p = intervals + (lane & 32);
#pragma unroll
    for (int e = 0; e < 16; e += 2) {
      if (e % 4 == 0) __builtin_amdgcn_sched_barrier(0);  // (all of them at once would take 32 registers)
      const sa_u32x4v r = lds_read_b128(p + 8 * (8 * (e >> 2) + (e & 3)));
      S[e] = (row < (int)r[0]) | (row >= (int)r[1]) ? -INFINITY : S[e];
      S[e + 1] = (row < (int)r[2]) | (row >= (int)r[3]) ? -INFINITY : S[e + 1];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e)
      if (key0 + 8 * (e >> 2) + (e & 3) >= Lk) S[e] = -INFINITY;
  }
}

// Item `seq` of an XCD, to which the dispatcher deals out workgroups in turn: an XCD works on whole heads one after the
// other, so that its L2 holds the streamed side; the heads that are left over go to all XCDs. False: none.
__host__ __device__ inline int xcd_items(int BH, int n) { return (BH >> 3) * n + ((BH & 7) * n + 7) / 8; }
__device__ inline bool own_block(int xcd, int seq, int BH, int n, int& bh, int& rank) {
  const int full = BH >> 3;
  if (seq < full * n) {
    bh = seq / n * 8 + xcd;
    rank = seq % n;
    return true;
  }
  const int rem = BH & 7, t = (seq - full * n) * 8 + xcd;
  if (t >= rem * n) return false;
  bh = full * 8 + t % rem;
  rank = t / rem;
  return true;
}
// Where keys are seen by later rows, the last query blocks and the first key blocks have the longest lists.
__device__ inline int block_of_rank(bool keys, int rank, int n) { return keys ? rank : n - 1 - rank; }

// Four values of a result row, rounded to the type; lo: what the rounding leaves, where it is wanted.
template <typename T>
__device__ __forceinline__ void store_result(uint8_t* row, uint8_t* lo, int at, float4 v) {
  if constexpr (std::is_same<T, float>::value) {
    *reinterpret_cast<float4*>(row + 4 * at) = v;
  } else {
    const uint32_t x = Elem<T>::pack(v.x, v.y), y = Elem<T>::pack(v.z, v.w);
    *reinterpret_cast<uint2*>(row + 2 * at) = make_uint2(x, y);
    if (lo) {
      const float2 p = unpack2<T>(x), q = unpack2<T>(y);
      *reinterpret_cast<uint2*>(lo + 2 * at) = make_uint2(Elem<T>::pack(v.x - p.x, v.y - p.y), Elem<T>::pack(v.z - q.x, v.w - q.y));
    }
  }
}

// A row's log2-sum-exp2 (none: it sees no key), of sum l relative to offset m.
__device__ __forceinline__ void store_sums(float* lse, float2* offsets, int64_t at, bool none, float m, float l) {
  const float log = none ? INFINITY : __builtin_amdgcn_logf(l), off = none ? 0.f : m;
  lse[at] = off + log;
  if (offsets) offsets[at] = make_float2(off, log);
}

__device__ inline float wave_sum(float x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
  return x;
}

template <typename T, int kD>
constexpr int waves_per_simd() {
  return std::is_same<T, float>::value ? (kD == 64 ? 2 : 1) : kD == 64 ? 3 : 2;
}

// The forward pass with a bias would fit four waves a SIMD (125 registers), and is held to the three that a call's plan counts
// with: [2, 30, 2560, 64] 219 us, 237 with four.
template <int kMode, int kRule, typename T, int kD>
constexpr int most_waves() {
  return kMode == kForward && (kRule & kTable) ? waves_per_simd<T, kD>() : 8;
}

template <int kMode, int kCap, int kRule, typename T, int kD>
__global__ __launch_bounds__(128)
__attribute__((amdgpu_waves_per_eu((waves_per_simd<T, kD>()), (most_waves<kMode, kRule, T, kD>()))))
void scored_kernel(ScoredArgs a) {
  constexpr bool kF32 = std::is_same<T, float>::value;
  constexpr int kSize = kF32 ? 4 : 2;
  constexpr int kDS = kD * kSize / 32;      // steps of the first products
  constexpr int kDC = kD / 32;              // 32-row chunks of the results
  constexpr int kHalves = kD * kSize / 128; // 128-byte pieces of a row
  constexpr int kRowTile = kStep * 128;
  constexpr int kMat = kHalves * kRowTile;  // a step's rows of one matrix
  constexpr int kAcc = kMode == kKeys ? 2 : 1;
  // Row operands are read in groups of kRead 16-byte steps, transposed ones 64 columns at a time, each a group ahead of the
  // products; kEarly: the first transposed ones before the exponentials, where there are registers for them (kKeys of
  // [1, 15, 17776, 64] by frames 1 500 us with, 1 375 without; kQueries of a bias at head dim 64 320 and 253).
  constexpr bool kTight = kMode == kQueries && kD == 64 && (kCap || kRule != kPlain);
  constexpr int kRead = kF32 || kTight ? 2 : kMode == kKeys ? 1 : 4;
  constexpr bool kEarly = !kF32 && kMode != kKeys && !kTight;
  __shared__ __attribute__((aligned(1024))) uint8_t tile0[2 * kMat], tile1[2 * kMat];
  constexpr bool kSloped = kRule & kSlopes, kBiased = kRule & kTable;
  constexpr int kRowStats = kSloped ? 128 : 64;  // of 32 query rows
  constexpr int kStat = kMode == kKeys ? kRowStats : 64;
  __shared__ __attribute__((aligned(256))) float stat0[kStat], stat1[kStat];
  __shared__ __attribute__((aligned(256))) float bias0[kBiased ? kWindow : 1], bias1[kBiased ? kWindow : 1];
  extern __shared__ float far_lds[];  // kQueries with far: [wave][8][64] for a quarter of a tile, [wave][2 radius + 1] sums

  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, hh = lane >> 5;
  int bh, blk, first_entry = 0, left = INT_MAX, place = -1;
  if (a.units) {
    const int xcd = blockIdx.x & 7, seq = blockIdx.x >> 3;
    if (seq >= a.n_units[xcd]) return;  // (the whole workgroup)
    const int4 u = a.units[(int64_t)xcd * a.unit_cap + seq];
    const int item = __builtin_amdgcn_readfirstlane(u.x);
    bh = item / a.n_own;
    blk = item - bh * a.n_own;
    first_entry = __builtin_amdgcn_readfirstlane(u.y);
    left = __builtin_amdgcn_readfirstlane(u.z) - first_entry;
    place = __builtin_amdgcn_readfirstlane(u.w);
  } else {
    int rank;
    if (!own_block(blockIdx.x & 7, blockIdx.x >> 3, a.BH_own, a.n_own, bh, rank)) return;
    blk = block_of_rank(kMode == kKeys, rank, a.n_own);
  }
  const int b = bh / a.heads_own, head = bh - b * a.heads_own;
  const int n_heads = kMode == kKeys ? a.rep : 1;  // streamed heads
  const int st_head = kMode == kKeys ? head * a.rep : head / a.rep;

  auto at = [](const Side& s, int b, int h) {
    return static_cast<const uint8_t*>(s.p) + (b * s.sb + h * s.sh) * kSize;
  };
  const int own_row = blk * kBlk + kStep * w + col;
  const int own_clamped = min(own_row, a.L_own - 1);  // rows past L_own are never stored
  sa_u32x4v fa[kDS], fb[kDS];
  {
    const uint8_t* pa = at(a.own_a, b, head) + (int64_t)own_clamped * a.own_a.sl * kSize + 16 * hh;
    const uint8_t* pb = kMode == kForward ? pa : at(a.own_b, b, head) + (int64_t)own_clamped * a.own_b.sl * kSize + 16 * hh;
#pragma unroll
    for (int s = 0; s < kDS; ++s) {
      fa[s] = *reinterpret_cast<const sa_u32x4v*>(pa + 32 * s);
      if constexpr (kMode != kForward) fb[s] = *reinterpret_cast<const sa_u32x4v*>(pb + 32 * s);
    }
  }

  // kQueries: of the row its log2-sum-exp2, with slopes relative to its offset; rowsum(do out).
  float lse = 0.f, row_off = 0.f, delta = 0.f;
  if constexpr (kMode == kQueries) {
    const int64_t at_row = (int64_t)own_clamped * a.out.sl * kSize + 16 * hh;
    const uint8_t* po = at(a.out, b, head) + at_row;
    const uint8_t* pl = static_cast<const uint8_t*>(a.out_lo) + (b * a.out.sb + head * a.out.sh) * kSize + at_row;
#pragma unroll
    for (int s = 0; s < kDS; ++s) {
      delta = dot_chunk<T>(*reinterpret_cast<const sa_u32x4v*>(po + 32 * s), fb[s], delta);
      if (!kF32 && a.out_lo) delta = dot_chunk<T>(*reinterpret_cast<const sa_u32x4v*>(pl + 32 * s), fb[s], delta);
    }
    delta = xhalf_sum(delta);
    const int64_t row = ((int64_t)bh * a.n_own + blk) * kBlk + kStep * w + col;
    if constexpr (kSloped) {
      const float2 x = a.offsets[row];
      row_off = x.x;
      lse = x.y;
    } else {
      lse = a.lse[row];
    }
    if (first_entry == 0) {
      float* to = a.stats + (((int64_t)bh * a.n_own + blk) * 2 + w) * kRowStats + lane;
      to[0] = own_row < a.L_own ? (hh == 0 ? lse : delta) : hh == 0 ? INFINITY : 0.f;
      if constexpr (kSloped) to[64] = hh == 0 ? row_off : (float)min(max(own_row + a.q_start, 0), a.L_st - 1);
    }
    if (!a.grad_a && !a.far) return;  // only the statistics are wanted
    if (kBiased && a.far) {
      for (int i = threadIdx.x; i < 2 * (kDiagonals + 2 * a.radius + 1); i += 128) far_lds[i] = 0.f;
      __syncthreads();
    }
  }
  int from = 0, len = 0;  // kKeys: the own key's interval
  if constexpr (kMode == kKeys) {
    if (a.ranges) {
      const int2 r = a.ranges[b * a.ranges_sb + own_clamped];
      from = max(r.x, 0);
      len = max(r.y, from) - from;
    }
  }

  // The list of the g-th streamed head, and the walk over all of them. An entry is requested a step before it is used, a
  // head's parameters with its first.
  typedef const __attribute__((address_space(4))) int32_t* ListPtr;
  typedef const __attribute__((address_space(4))) float* ConstPtr;
  struct Step {
    int block, cut, half, g;  // block -1: none
    float slope, past, before;  // slopes[h] log2(e), the biases from the radius on and up to minus the radius
  };
  ListPtr list = nullptr;
  int cnt = 0, g = 0, pos = 0, half = 0, ahead = 0;
  float slope_h = 0.f, past = 0.f, before = 0.f;
  auto set_list = [&]() __attribute__((always_inline)) {  // (at entry 0)
    const int hq = kMode == kKeys ? st_head + g : head;
    if (kSloped) slope_h = *(ConstPtr)(a.slopes + hq);
    if (kBiased) {
      const float* eb = a.ebias + (int64_t)hq * (2 * a.radius + 1 + 2 * kPad) + kPad;
      before = *(ConstPtr)eb;
      past = *(ConstPtr)(eb + 2 * a.radius);
    }
    cnt = a.n_st;
    if (a.idx) {
      const int64_t row = ((int64_t)(a.per_head ? b * a.H + hq : b)) * a.n_own + blk;
      list = (ListPtr)(a.idx + row * a.n_st);
      cnt = min(max(*(ListPtr)(a.cnt + row), 0), a.n_st);
      if (cnt > 0) ahead = list[0];
    }
  };
  auto next = [&]() __attribute__((always_inline)) {
    while (pos >= cnt && g + 1 < n_heads) {
      ++g;
      pos = 0;
      set_list();
    }
    Step s = {-1, 0, half, g, slope_h * kLog2e, past, before};
    if (pos < cnt && left > 0) {
      const int e = a.idx ? ahead : 2 * pos + (a.ranges || kBlk * (pos + 1) > a.L_st);
      s.block = e >> 1;
      s.cut = e & 1;
      // (the second half of a block that ends before it is left out)
      if (half == 0 && s.block * kBlk + kStep < a.L_st) {
        half = 1;
      } else {
        half = 0;
        ++pos;
        --left;
        if (a.idx && pos < cnt) ahead = list[pos];
      }
      if ((unsigned)s.block >= (unsigned)a.n_st) s.block = 0, s.cut = 2;  // (no such block: skipped)
    }
    return s;
  };
  set_list();
  for (pos = first_entry; pos >= cnt && g + 1 < n_heads;) {
    const int rest = pos - cnt;
    ++g;
    set_list();
    pos = rest;
  }
  if (a.idx && pos > 0 && pos < cnt) ahead = list[pos];

  // Streamed rows: wave 0 copies st_a's (and the statistics), wave 1 st_b's. The descriptors begin at the step's rows
  // and end with the head's, so that rows past the last one read as zero and the lane offsets never change.
  const Side& side = w == 0 ? a.st_a : a.st_b;
  const uint8_t* st0 = at(side, b, st_head);
  const int64_t st_sh = side.sh * kSize;
  const uint32_t row_bytes = (uint32_t)side.sl * kSize;
  const uint32_t st_bytes = (uint32_t)(a.L_st - 1) * row_bytes + 128;
  uint32_t goff[2];
#pragma unroll
  for (int j = 0; j < 2; ++j)
    goff[j] = (8 * j + (lane >> 3)) * row_bytes + 16 * ((lane & 7) ^ swz(8 * j + (lane >> 3)));
  // The smallest distance of a step's rows and the whole own block (95 of them).
  auto least_of = [&](int row0) { return kMode == kKeys ? row0 + a.q_start - blk * kBlk - 63 : blk * kBlk + a.q_start - row0 - 31; };
  auto issue = [&](const Step& s, lds_u8* tile, lds_u8* stat, lds_u8* bias) __attribute__((always_inline)) {
    const uint32_t row0 = __builtin_amdgcn_readfirstlane(s.block * kBlk + kStep * s.half);
    const uint8_t* st = st0 + (kMode == kKeys ? s.g * st_sh : 0);
#pragma unroll
    for (int r16 = 0; r16 < 2; ++r16) {
      const uint32_t off = min((row0 + 16 * r16) * row_bytes, st_bytes);
#pragma unroll
      for (int hf = 0; hf < kHalves; ++hf) {
        const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<uint8_t*>(st + off + 128 * hf), (short)0, (int)(st_bytes - off), 0x00020000);
#pragma unroll
        for (int j = 0; j < 2; ++j)
          __builtin_amdgcn_raw_ptr_buffer_load_lds(
              rsrc, (lds_u8*)(tile + w * kMat + hf * kRowTile + 2048 * r16 + 1024 * j), 16, goff[j], 0, 0, 0);
      }
    }
    if (kMode == kKeys && w == 0) {
      const float* src = a.stats + ((int64_t)(b * a.H + st_head + s.g) * a.n_st * 2 + 2 * s.block + s.half) * kRowStats;
      const __amdgpu_buffer_rsrc_t rs =
          __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(src), (short)0, 4 * kRowStats, 0x00020000);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, stat, 4, 4 * lane, 0, 0, 0);
      if (kSloped) __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, stat, 4, 4 * lane, 0, 256, 0);
    }
    if (kMode != kKeys && w == 0 && a.ranges && s.cut) {  // the keys' intervals
      const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<int2*>(a.ranges + b * a.ranges_sb + row0), (short)0, 8 * max(a.L_st - (int)row0, 0), 0x00020000);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, stat, 4, 4 * lane, 0, 0, 0);
    }
    if (kBiased && w == 1) {  // (where neither wave's pairs are all past the radius they are in bounds)
      const int least = least_of((int)row0), n = 2 * a.radius + 1 + 2 * kPad;
      const int hq = kMode == kKeys ? st_head + s.g : head;
      if (least < a.radius && least + 94 > -a.radius) {
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<float*>(a.ebias + (int64_t)hq * n), (short)0, 4 * n, 0x00020000);
        const int from = 4 * (least + a.radius + kPad + lane);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, bias, 4, from, 0, 0, 0);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, bias, 4, from, 0, 256, 0);
      }
    }
  };

  const TileReads<T, kD> reads(lane);

  sa_f32x16 acc[kAcc][kDC];
#pragma unroll
  for (int x = 0; x < kAcc; ++x)
#pragma unroll
    for (int dc = 0; dc < kDC; ++dc) acc[x][dc] = sa_f32x16{};
  float m = -INFINITY, l = 0.f;          // kForward: the row's offset, and its sum
  float far_hi = 0.f, far_lo = 0.f;      // kQueries with far: the lane's sums of dS past the radius

  auto compute = [&](const Step& s, const lds_u8* tile, const float* stat, const float* bias) __attribute__((always_inline)) {
    if (s.cut == 2) return;
    const int row0 = s.block * kBlk + kStep * s.half;
    sa_f32x16 S = {}, dP = {}, slope;
    if constexpr (kMode == kQueries) {
#pragma unroll
      for (int e = 0; e < 16; ++e) dP[e] = -delta;
    } else if constexpr (kMode == kKeys) {
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        const float4 y = *reinterpret_cast<const float4*>(stat + 32 + 8 * q4 + 4 * hh);
        dP[4 * q4] = -y.x; dP[4 * q4 + 1] = -y.y; dP[4 * q4 + 2] = -y.z; dP[4 * q4 + 3] = -y.w;
      }
    }
    sa_u32x4v x[kDS], y[kDS];
    auto rows = [&](int c0) __attribute__((always_inline)) {
#pragma unroll
      for (int c = c0; c < c0 + kRead; ++c) {
        x[c] = lds_read_b128(reads.row(tile, c));
        if constexpr (kMode != kForward) y[c] = lds_read_b128(reads.row(tile, c) + kMat);
      }
    };
    rows(0);
#pragma unroll
    for (int c0 = 0; c0 < kDS; c0 += kRead) {
      __builtin_amdgcn_sched_barrier(0);
      if (c0 + kRead < kDS) rows(c0 + kRead);
#pragma unroll
      for (int c = c0; c < c0 + kRead; ++c) {
        S = mfma_chunk<T>(x[c], fa[c], S);
        if constexpr (kMode != kForward) dP = mfma_chunk<T>(y[c], fb[c], dP);
      }
    }
    typename TileReads<T, kD>::Columns tr;
    constexpr int kFirst = kMode == kQueries ? 0 : kMat;  // the matrix of the first second product
    if constexpr (kEarly) {
      tr = reads.columns(tile + kFirst, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
    // Elements e: streamed row row0 + 4 hh + 8 (e / 4) + e % 4 of own row own_row.
    const int first = __builtin_amdgcn_readfirstlane(blk * kBlk + kStep * w);
    const int least = kMode == kKeys ? row0 + a.q_start - first - 31 : first + a.q_start - row0 - 31;
    int side_far;
    const int own = kStep * w + col;
    // With nothing but a cap the key pass keeps the reciprocals r of bend in S: the score is cap - 2 cap r, its derivative 4 (r - r^2).
    // That takes 16 registers less than both, which were spilled (428 us at head dim 128, 401 so).
    constexpr bool kHoldsR = kMode == kKeys && kCap == kTanh && kRule == kPlain && !kF32;
    constexpr float kHidden = kHoldsR ? 1e18f : -INFINITY;  // of pairs that are not seen (2e18 of the least cap, and P is 0)
    float sc = 1.f;
    if constexpr (kHoldsR) {
#pragma unroll
      for (int e = 0; e < 16; ++e) S[e] = bend_r(S[e] * a.cap_in);
    } else {
      sc = apply_rule<kMode == kKeys ? 1 : -1, kCap, kRule, kMode != kForward, T>(
          a, s.past, s.before, least, bias + (kMode == kKeys ? 4 * hh + 63 - own : own + 4 - 4 * hh), S, slope, side_far);
    }
    // Slopes: with the query's position p taken as the nearest of the keys' positions (which leaves out what all of a row's
    // distances have in common), S becomes S - slope |p - j| - ref. ref is close to what the row's nearer keys lose: the row's
    // offset, or where the forward pass has yet to find one as large, what this step's middle key loses. It goes in before S does:
    // of two large numbers that cancel no bits are lost (a row that sees nothing but keys 1e5 away: P off by 4e-3 of itself
    // where it went in last). (Slopes of either sign: |d| is an addition of its own, which takes 2 us of 207.)
    float ref = row_off;
    if constexpr (kSloped) {
      if constexpr (kMode == kKeys) {
        const float* offs = stat + 64 + 4 * hh;
        const float key = (float)own_row;
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
          const float4 y = *reinterpret_cast<const float4*>(offs + 8 * q4), z = *reinterpret_cast<const float4*>(offs + 32 + 8 * q4);
          const float off[4] = {y.x, y.y, y.z, y.w}, p[4] = {z.x, z.y, z.z, z.w};
#pragma unroll
          for (int i = 0; i < 4; ++i)
            S[4 * q4 + i] = fmaf(S[4 * q4 + i], sc, fmaf(-s.slope, fabsf(p[i] - key), -off[i]));
        }
      } else {
        const int p = min(max(own_row + a.q_start, 0), a.L_st - 1) - row0;
        const float d0 = (float)(p - 4 * hh);
        if constexpr (kMode == kForward) ref = fmaxf(m, -s.slope * fabsf((float)(p - kStep / 2)));
#pragma unroll
        for (int e = 0; e < 16; ++e)
          S[e] = fmaf(S[e], sc, fmaf(-s.slope, fabsf(d0 - (float)(8 * (e >> 2) + (e & 3))), -ref));
      }
      sc = 1.f;
    }
    if (s.cut) {
      if constexpr (kMode == kKeys) {
        if (a.ranges) {
          const int t = row0 + 4 * hh - from;
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if ((unsigned)(t + 8 * (e >> 2) + (e & 3)) >= (unsigned)len) S[e] = kHidden;
        }
      } else {
        cut_keys(a, a.L_st, own_row, row0 + 4 * hh, lane, (const lds_u8*)stat, S);
      }
    }
    if constexpr (kMode == kForward) {
      float top = S[0];
#pragma unroll
      for (int e = 1; e < 16; ++e) top = fmaxf(top, S[e]);
      top = xhalf_max(top) * sc;
      if constexpr (kSloped) top += ref;
      if (__ballot(top > m + kAbove<T>)) {
        const float next_m = fmaxf(m, top - kBelow<T>);
        const float f = next_m == m ? 1.f : fast_exp2(m - next_m);
        m = next_m;
        l *= f;
#pragma unroll
        for (int dc = 0; dc < kDC; ++dc)
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[0][dc][e] *= f;
      }
      const float off = m == -INFINITY ? 0.f : kSloped ? m - ref : m;
      Weights<T> P, rest;
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        const float p0 = fast_exp2(fmaf(S[e], sc, -off)), p1 = fast_exp2(fmaf(S[e + 1], sc, -off));
        l += p0 + p1;
        set_two_terms<T>(P, rest, e, p0, p1);
      }
      if constexpr (kF32) {
        reads.product(tile + kMat, P, acc[0]);
      } else {
#pragma unroll
        for (int hf = 0; hf < kHalves; ++hf) {
          const auto now = tr;
          if (hf + 1 < kHalves) tr = reads.columns(tile + kMat, hf + 1);
          reads.product(now, hf, P, acc[0]);
          reads.product(now, hf, rest, acc[0]);
        }
      }
    } else {
      Weights<T> P, dC;
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        float4 off = make_float4(lse, lse, lse, lse);
        if constexpr (kMode == kKeys) off = *reinterpret_cast<const float4*>(stat + 2 * e + 4 * hh);
        if constexpr (kHoldsR) {
          off.x -= a.cap_log2; off.y -= a.cap_log2; off.z -= a.cap_log2; off.w -= a.cap_log2;
          sc = -2.f * a.cap_log2;
        }
        const float p[4] = {fast_exp2(fmaf(S[e], sc, -off.x)), fast_exp2(fmaf(S[e + 1], sc, -off.y)),
                            fast_exp2(fmaf(S[e + 2], sc, -off.z)), fast_exp2(fmaf(S[e + 3], sc, -off.w))};
        if constexpr (kMode == kKeys) {
          constexpr float f = std::is_same<T, _Float16>::value ? kPScale : 1.f;
          P.set(e, p[0] * f, p[1] * f);
          P.set(e + 2, p[2] * f, p[3] * f);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          dP[e + i] *= p[i];
          if constexpr (kHoldsR) dP[e + i] *= 4.f * fmaf(-S[e + i], S[e + i], S[e + i]);
        }
      }
      if constexpr (kMode == kQueries && kBiased) {
        if (a.far) {
          if (side_far) {
            float t = 0.f;
#pragma unroll
            for (int e = 0; e < 16; ++e) t += dP[e];
            if (side_far > 0) far_hi += t;
            else far_lo += t;
          } else {
            // Sums along the tile's diagonals, 8 of its keys j at a time: row j of the wave's 64 columns holds the values at
            // column col - j + 31, which are all written each time, and zeros, so that column x sums up a distance.
            const int at = 64 * 4 * hh + col - 4 * hh + 31;
            float* sums = far_lds + 2 * kDiagonals + w * (2 * a.radius + 1) + a.radius;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              float* mine = far_lds + w * kDiagonals;
#pragma unroll
              for (int e = 0; e < 4; ++e) mine[at + 63 * e] = dP[4 * u + e];
              float t = 0.f;
#pragma unroll
              for (int j = 0; j < 8; ++j) t += mine[64 * j + lane];
              const int d = least + lane - 8 * u;  // (lane 63 and columns that no pair has: zeros)
              if (d >= a.radius) far_hi += t;
              else if (d <= -a.radius) far_lo += t;
              else sums[d] += t;
            }
          }
        }
      }
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        if constexpr (kCap && !kHoldsR) dC.set(e, dP[e] * slope[e], dP[e + 1] * slope[e + 1]);
        else dC.set(e, dP[e], dP[e + 1]);
      }
      if constexpr (kF32) {
        if constexpr (kMode == kKeys) reads.product(tile + kMat, P, acc[1]);
        reads.product(tile, dC, acc[0]);
      } else {
        if constexpr (!kEarly) tr = reads.columns(tile + kFirst, 0);
#pragma unroll
        for (int j = 0; j < kAcc * kHalves; ++j) {  // (P is ready first)
          const int x = kAcc - 1 - j / kHalves, hf = j % kHalves;
          const auto now = tr;
          if (j + 1 < kAcc * kHalves) tr = reads.columns(tile + (kAcc - 1 - (j + 1) / kHalves) * kMat, (j + 1) % kHalves);
          reads.product(now, hf, x == 0 ? dC : P, acc[x]);
        }
      }
    }
  };

  lds_u8* const t0 = (lds_u8*)tile0;
  lds_u8* const t1 = (lds_u8*)tile1;
  Step s0 = next(), s1;
  if (s0.block >= 0) issue(s0, t0, (lds_u8*)stat0, (lds_u8*)bias0);
  while (s0.block >= 0) {
    // This wave's copies of the step have landed, then everyone's; every wave is done with the step before (its reads of
    // LDS have returned), whose stage the copies of the next step overwrite.
    __builtin_amdgcn_s_waitcnt(kWaitVmLgkm0);
    wg_barrier();
    s1 = next();
    if (s1.block >= 0) issue(s1, t1, (lds_u8*)stat1, (lds_u8*)bias1);
    compute(s0, t0, stat0, bias0);
    if (s1.block < 0) break;
    __builtin_amdgcn_s_waitcnt(kWaitVmLgkm0);
    wg_barrier();
    s0 = next();
    if (s0.block >= 0) issue(s0, t0, (lds_u8*)stat0, (lds_u8*)bias0);
    compute(s1, t1, stat1, bias1);
  }

  // ---- Results: element 4 q4 + j of acc[x][dc] is d = 32 dc + 8 q4 + 4 hh + j of own row own_row.
  if constexpr (kMode == kForward) l = xhalf_sum(l);
  if constexpr (kMode == kQueries && kBiased) {
    if (a.far) {
      far_hi = wave_sum(far_hi);
      far_lo = wave_sum(far_lo);
      const int n_far = 2 * a.radius + 1;
      float* sums = far_lds + 2 * kDiagonals;
      if (lane == 0) {
        sums[w * n_far + 2 * a.radius] += far_hi;
        sums[w * n_far] += far_lo;
      }
      __syncthreads();
      float* to = place < 0 ? a.far + ((int64_t)bh * a.n_own + blk) * n_far : a.part_far + (int64_t)place * n_far;
      for (int i = threadIdx.x; i < n_far; i += 128) to[i] = sums[i] + sums[n_far + i];
    }
  }
  if (place >= 0) {
    const int r = kStep * w + col;
    if (kMode == kForward && hh == 0)
      *reinterpret_cast<float2*>(a.part_sums + ((int64_t)place * kBlk + r) * 2) = make_float2(m, l);
#pragma unroll
    for (int x = 0; x < kAcc; ++x) {
      float* p = a.parts + (((int64_t)place * kAcc + x) * kBlk + r) * kD + 4 * hh;
#pragma unroll
      for (int dc = 0; dc < kDC; ++dc)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
          const sa_f32x16& A = acc[x][dc];
          *reinterpret_cast<float4*>(p + 32 * dc + 8 * q4) =
              make_float4(A[4 * q4], A[4 * q4 + 1], A[4 * q4 + 2], A[4 * q4 + 3]);
        }
    }
    return;
  }
  float f_a = a.sm_scale;
  if constexpr (kMode == kForward) {
    f_a = l == 0.f ? 0.f : 1.f / l;
    if (hh == 0)
      store_sums(a.lse, a.offsets, ((int64_t)bh * a.n_own + blk) * kBlk + kStep * w + col, own_row >= a.L_own || l == 0.f, m, l);
  }
#pragma unroll
  for (int x = 0; x < kAcc; ++x) {
    uint8_t* grad = static_cast<uint8_t*>(x == 0 ? a.grad_a : a.grad_b);
    if (!grad || own_row >= a.L_own) continue;
    const int64_t sb = x == 0 ? a.ga_sb : a.gb_sb, sh = x == 0 ? a.ga_sh : a.gb_sh, sl = x == 0 ? a.ga_sl : a.gb_sl;
    const int64_t at_row = (b * sb + head * sh + own_row * sl + 4 * hh) * kSize;
    uint8_t* lo = kMode == kForward && a.out_lo ? static_cast<uint8_t*>(a.out_lo) + at_row : nullptr;
    const float f = x == 0 ? f_a : std::is_same<T, _Float16>::value ? 1.f / kPScale : 1.f;
#pragma unroll
    for (int dc = 0; dc < kDC; ++dc)
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        const sa_f32x16& A = acc[x][dc];
        store_result<T>(grad + at_row, lo, 32 * dc + 8 * q4,
                        make_float4(A[4 * q4] * f, A[4 * q4 + 1] * f, A[4 * q4 + 2] * f, A[4 * q4 + 3] * f));
      }
  }
}

// Split items: their units' sums, added in order. A workgroup per split item: 4 to 8 us, the latency of a launch and of two
// reads after each other, and for many long ones HBM (1500 units of [64][128] twice: 24 us, 4 TB/s).
struct MergeArgs {
  const int4* splits;  // [xcd * cap ..] {item, first place, units}
  const int32_t* n_splits;
  int cap, heads_own, n_own, L_own, n_far;
  const float *parts, *part_sums, *part_far;
  void *grad_a, *grad_b, *out_lo;
  int64_t ga_sb, ga_sh, ga_sl, gb_sb, gb_sh, gb_sl;
  float sm_scale;
  float *lse, *far;
  float2* offsets;
};

constexpr int kMergeThreads = 1024;  // (a unit's sums are a load of each thread's: latency)
template <int kMode, typename T, int kD>
__global__ __launch_bounds__(kMergeThreads) void scored_merge_kernel(MergeArgs a) {
  constexpr int kAcc = kMode == kKeys ? 2 : 1, kCh = kD / 4;
  const int xcd = blockIdx.x & 7, seq = blockIdx.x >> 3;
  if (seq >= a.n_splits[xcd]) return;
  const int4 u = a.splits[(int64_t)xcd * a.cap + seq];
  const int bh = u.x / a.n_own, blk = u.x - bh * a.n_own, b = bh / a.heads_own, head = bh - b * a.heads_own;
  if (kMode == kQueries && a.far) {
    for (int i = threadIdx.x; i < a.n_far; i += kMergeThreads) {
      float s = 0.f;
      for (int p = 0; p < u.z; ++p) s += a.part_far[(int64_t)(u.y + p) * a.n_far + i];
      a.far[(int64_t)u.x * a.n_far + i] = s;
    }
  }
  for (int t = threadIdx.x; t < kAcc * kBlk * kCh; t += kMergeThreads) {
    const int x = t / (kBlk * kCh), r = t / kCh % kBlk, ch = t % kCh, row = blk * kBlk + r;
    const float* parts = a.parts + (((int64_t)u.y * kAcc + x) * kBlk + r) * kD + 4 * ch;
    const float* sums = a.part_sums + ((int64_t)u.y * kBlk + r) * 2;
    float top = -INFINITY, l = 0.f;
    if constexpr (kMode == kForward)
#pragma unroll 8
      for (int p = 0; p < u.z; ++p) top = fmaxf(top, sums[(int64_t)p * kBlk * 2]);
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int p = 0; p < u.z; ++p) {
      const float4 y = *reinterpret_cast<const float4*>(parts + (int64_t)p * kAcc * kBlk * kD);
      float f = 1.f;
      if constexpr (kMode == kForward) {
        const float2 z = *reinterpret_cast<const float2*>(sums + (int64_t)p * kBlk * 2);
        f = z.x == top ? 1.f : fast_exp2(z.x - top);
        l = fmaf(z.y, f, l);
      }
      s.x = fmaf(y.x, f, s.x);
      s.y = fmaf(y.y, f, s.y);
      s.z = fmaf(y.z, f, s.z);
      s.w = fmaf(y.w, f, s.w);
    }
    float f = x == 0 ? a.sm_scale : std::is_same<T, _Float16>::value ? 1.f / kPScale : 1.f;
    if constexpr (kMode == kForward) {
      f = l == 0.f ? 0.f : 1.f / l;
      if (ch == 0)
        store_sums(a.lse, a.offsets, (int64_t)u.x * kBlk + r, row >= a.L_own || l == 0.f, top, l);
    }
    uint8_t* grad = static_cast<uint8_t*>(x == 0 ? a.grad_a : a.grad_b);
    if (!grad || row >= a.L_own) continue;
    const int64_t sb = x == 0 ? a.ga_sb : a.gb_sb, sh = x == 0 ? a.ga_sh : a.gb_sh, sl = x == 0 ? a.ga_sl : a.gb_sl;
    const int64_t at_row = (b * sb + head * sh + row * sl) * (int64_t)sizeof(T);
    uint8_t* lo = kMode == kForward && a.out_lo ? static_cast<uint8_t*>(a.out_lo) + at_row : nullptr;
    store_result<T>(grad + at_row, lo, 4 * ch, make_float4(s.x * f, s.y * f, s.z * f, s.w * f));
  }
}

// ---- Launches of a pass. Each element type's kernels are compiled by themselves (attn_scored_*.hip).
struct PassCall {
  int mode, D;
  int cap;  // kNoCap, kTanh or kFineTanh
  unsigned grid, merge_grid;  // merge_grid 0: no item is split
  hipStream_t stream;
};

template <int kMode, int kCap, int kRule, typename T, int kD>
void launch_kernels(const ScoredArgs& a, const MergeArgs& m, const PassCall& c) {
  const size_t lds = kMode == kQueries && (kRule & kTable) && a.far ? 2 * (kDiagonals + 2 * a.radius + 1) * sizeof(float) : 0;
  hipLaunchKernelGGL((scored_kernel<kMode, kCap, kRule, T, kD>), dim3(c.grid), dim3(128), lds, c.stream, a);
  if (c.merge_grid)
    hipLaunchKernelGGL((scored_merge_kernel<kMode, T, kD>), dim3(c.merge_grid), dim3(kMergeThreads), 0, c.stream, m);
}

template <typename T>
void launch_pass_of(const ScoredArgs& a, const MergeArgs& m, const PassCall& c) {
  auto dim = [&](auto mode, auto cap, auto rule) {
    constexpr int kMode = decltype(mode)::value, kRule = decltype(rule)::value;
    constexpr int kCap = decltype(cap)::value;
    if (c.D == 64) launch_kernels<kMode, kCap, kRule, T, 64>(a, m, c);
    else launch_kernels<kMode, kCap, kRule, T, 128>(a, m, c);
  };
  auto rule = [&](auto mode, auto cap) {
    if (a.ebias && a.slopes) dim(mode, cap, std::integral_constant<int, kTable | kSlopes>());
    else if (a.ebias) dim(mode, cap, std::integral_constant<int, kTable>());
    else if (a.slopes) dim(mode, cap, std::integral_constant<int, kSlopes>());
    else dim(mode, cap, std::integral_constant<int, kPlain>());
  };
  auto cap = [&](auto mode) {
    if (c.cap == kNoCap) return rule(mode, std::integral_constant<int, kNoCap>());
    if constexpr (!std::is_same<T, float>::value)
      if (c.cap == kTanh) return rule(mode, std::integral_constant<int, kTanh>());
    rule(mode, std::integral_constant<int, kFineTanh>());
  };
  if (c.mode == kForward) cap(std::integral_constant<int, kForward>());
  else if (c.mode == kQueries) cap(std::integral_constant<int, kQueries>());
  else cap(std::integral_constant<int, kKeys>());
}

void launch_pass_bf16(const ScoredArgs& a, const MergeArgs& m, const PassCall& c);
void launch_pass_f16(const ScoredArgs& a, const MergeArgs& m, const PassCall& c);
void launch_pass_f32(const ScoredArgs& a, const MergeArgs& m, const PassCall& c);

}  // namespace sa_scored
