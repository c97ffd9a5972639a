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
#include <math.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

#include "attn_score.h"

namespace {

constexpr int kBlk = 64;
enum { kForward = 0, kQueries = 1, kKeys = 2 };
// fp16 holds normal numbers from 2^-14, which the probabilities of an even row fall short of over more than 16 384
// keys: P is rounded to the type with this factor (one product an element), which dv loses at the end.
constexpr float kPScale = 4096.f;

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
  // b * H + query head) * n_own + block); idx null: every block.
  const int32_t *idx, *cnt;
  int per_head;
  const int2* ranges;  // [b * ranges_sb + key] = {from, until}; may be null
  int64_t ranges_sb;
  float sm_scale, scale_log2;
  float cap_in, cap_log2;  // 2 log2(e) sm_scale / cap (fp32: sm_scale / cap), cap log2(e)
  const float* slopes;     // [H]; may be null
  const float* ebias;      // [H][2 radius + 1], times log2(e); may be null
  int radius;
  float* lse;              // [b * H + h][64 n]
  float* stats;            // [b * H + h][2 n][2][32]: of 32 query rows their lse, then their delta
  void* out_lo;            // what out's rounding left out, laid out like it; may be null
  // Units of work of each XCD, {item = (b * heads_own + head) * n_own + block, first entry, behind the last, place of the
  // sums}: units[xcd * unit_cap ..], n_units[xcd] of them (scored_schedule_kernel). Null: items as own_block has them.
  const int4* units;
  const int32_t* n_units;
  int unit_cap;
  float* parts;      // units of split items: [place][result][64][kD]
  float* part_sums;  // kForward: [place][64] {offset, sum}
  float* far;        // kQueries, nullable: [item] {sums of dS at distances from the radius on, up to minus the radius}
  float* part_far;   // and [place]
};

// The rule on a tile's products S: S times what is returned is the score times log2(e). base: the lane's distance at element
// 0, from which element e is kSign (8 (e / 4) + e % 4) away. least .. least + 62: the wave's distances. kSlope: slope becomes
// the cap's derivative. side: whether all pairs of the wave are past the radius, 1 above, -1 below, 0 not all.
template <int kSign, bool kCap, bool kSlope, typename T>
__device__ __forceinline__ float apply_rule(const ScoredArgs& a, int hq, float slope_h, float past, float before, int base,
                                            int least, sa_f32x16& S, sa_f32x16& slope, int& side) {
  float sc = a.scale_log2;
  if constexpr (kCap) {
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      float t = 0.f;
      S[e] = bend<T, kSlope>(S[e] * a.cap_in, t) * a.cap_log2;
      if constexpr (kSlope) slope[e] = t;
    }
    sc = 1.f;
  }
  if (a.slopes) {
    const float f = slope_h * (float)base;
#pragma unroll
    for (int e = 0; e < 16; ++e) S[e] = fmaf(S[e], sc, -fabsf(fmaf(slope_h, (float)(kSign * (8 * (e >> 2) + (e & 3))), f)));
    sc = 1.f;
  }
  side = 0;
  if (a.ebias) {
    side = least >= a.radius ? 1 : least + 62 <= -a.radius ? -1 : 0;
    if (side) {
      const float c = side > 0 ? past : before;
#pragma unroll
      for (int e = 0; e < 16; ++e) S[e] = fmaf(S[e], sc, c);
    } else {
      const float* eb = a.ebias + (int64_t)hq * (2 * a.radius + 1) + a.radius;
#pragma unroll
      for (int e = 0; e < 16; ++e)
        S[e] = fmaf(S[e], sc, eb[min(max(base + kSign * (8 * (e >> 2) + (e & 3)), -a.radius), a.radius)]);
    }
    sc = 1.f;
  }
  return sc;
}

// A cut tile of own queries: pairs that are not seen get -inf. row: the lane's query row; key0: its key at element 0.
__device__ __forceinline__ void cut_keys(const ScoredArgs& a, int b, int Lk, int row, int key0, sa_f32x16& S) {
  if (a.ranges) {  // (keys past the last one: no rows)
    const __amdgpu_buffer_rsrc_t rs =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<int2*>(a.ranges + b * a.ranges_sb), (short)0, Lk * 8, 0x00020000);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const sa_u32x2v r = __builtin_amdgcn_raw_buffer_load_b64(rs, 8 * (key0 + 8 * (e >> 2) + (e & 3)), 0, 0);
      if (row < (int)r[0] || row >= (int)r[1]) S[e] = -INFINITY;
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

__device__ inline float wave_sum(float x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
  return x;
}

template <typename T, int kD>
constexpr int waves_per_simd() {
  return std::is_same<T, float>::value ? (kD == 64 ? 2 : 1) : kD == 64 ? 3 : 2;
}

template <int kMode, bool kCap, typename T, int kD>
__global__ __launch_bounds__(128, (waves_per_simd<T, kD>())) void scored_kernel(ScoredArgs a) {
  constexpr bool kF32 = std::is_same<T, float>::value;
  constexpr int kSize = kF32 ? 4 : 2;
  constexpr int kDS = kD * kSize / 32;      // steps of the first products
  constexpr int kDC = kD / 32;              // 32-row chunks of the results
  constexpr int kHalves = kD * kSize / 128; // 128-byte pieces of a row
  constexpr int kRowTile = kStep * 128;
  constexpr int kMat = kHalves * kRowTile;  // a step's rows of one matrix
  constexpr int kAcc = kMode == kKeys ? 2 : 1;
  __shared__ __attribute__((aligned(1024))) uint8_t tile0[2 * kMat], tile1[2 * kMat];
  __shared__ __attribute__((aligned(256))) float stat0[64], stat1[64];

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

  float lse = 0.f, delta = 0.f;
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
    lse = a.lse[((int64_t)bh * a.n_own + blk) * kBlk + kStep * w + col];
    if (first_entry == 0)
      a.stats[(((int64_t)bh * a.n_own + blk) * 2 + w) * 64 + lane] =
          own_row < a.L_own ? (hh == 0 ? lse : delta) : hh == 0 ? INFINITY : 0.f;
    if (!a.grad_a && !a.far) return;  // only the statistics are wanted
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
    if (a.slopes) slope_h = *(ConstPtr)(a.slopes + hq);
    if (a.ebias) {
      const float* eb = a.ebias + (int64_t)hq * (2 * a.radius + 1);
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
      const int e = a.idx ? ahead : 2 * pos + (kBlk * (pos + 1) > a.L_st);
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
  auto issue = [&](const Step& s, lds_u8* tile, lds_u8* stat) __attribute__((always_inline)) {
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
      const float* src = a.stats + ((int64_t)(b * a.H + st_head + s.g) * a.n_st * 2 + 2 * s.block + s.half) * 64;
      const __amdgpu_buffer_rsrc_t rs =
          __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(src), (short)0, 256, 0x00020000);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, stat, 4, 4 * lane, 0, 0, 0);
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

  auto compute = [&](const Step& s, const lds_u8* tile, const float* stat) __attribute__((always_inline)) {
    if (s.cut == 2) return;
    const int row0 = s.block * kBlk + kStep * s.half;
    const int hq = kMode == kKeys ? st_head + s.g : head;  // the query head
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
#pragma unroll
    for (int c = 0; c < kDS; ++c) {
      const lds_u8* p = reads.row(tile, c);
      S = mfma_chunk<T>(lds_read_b128(p), fa[c], S);
      if constexpr (kMode != kForward) dP = mfma_chunk<T>(lds_read_b128(p + kMat), fb[c], dP);
    }
    // Elements e: streamed row row0 + 4 hh + 8 (e / 4) + e % 4 of own row own_row.
    const int first = __builtin_amdgcn_readfirstlane(blk * kBlk + kStep * w);
    const int base = kMode == kKeys ? row0 + 4 * hh + a.q_start - own_row : own_row + a.q_start - row0 - 4 * hh;
    const int least = kMode == kKeys ? row0 + a.q_start - first - 31 : first + a.q_start - row0 - 31;
    int side_far;
    const float sc = apply_rule<kMode == kKeys ? 1 : -1, kCap, kMode != kForward, T>(a, hq, s.slope, s.past, s.before, base,
                                                                                     least, S, slope, side_far);
    if (s.cut) {
      if constexpr (kMode == kKeys) {
        if (a.ranges) {
          const int t = row0 + 4 * hh - from;
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if ((unsigned)(t + 8 * (e >> 2) + (e & 3)) >= (unsigned)len) S[e] = -INFINITY;
        }
      } else {
        cut_keys(a, b, a.L_st, own_row, row0 + 4 * hh, S);
      }
    }
    if constexpr (kMode == kForward) {
      float top = S[0];
#pragma unroll
      for (int e = 1; e < 16; ++e) top = fmaxf(top, S[e]);
      top = xhalf_max(top) * sc;
      if (__ballot(top > m + kSlack)) {
        const float next_m = fmaxf(m, top);
        const float f = next_m == m ? 1.f : fast_exp2(m - next_m);
        m = next_m;
        l *= f;
#pragma unroll
        for (int dc = 0; dc < kDC; ++dc)
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[0][dc][e] *= f;
      }
      const float off = m == -INFINITY ? 0.f : m;
      Weights<T> P, rest;
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        const float p0 = fast_exp2(fmaf(S[e], sc, -off)), p1 = fast_exp2(fmaf(S[e + 1], sc, -off));
        l += p0 + p1;
        P.set(e, p0, p1);
        if constexpr (!kF32) {
          const float2 hi = unpack2<T>(P.w[e >> 1]);
          rest.set(e, p0 - hi.x, p1 - hi.y);
        }
      }
      reads.product(tile + kMat, P, acc[0]);
      if constexpr (!kF32) reads.product(tile + kMat, rest, acc[0]);
    } else {
      Weights<T> P, dC;
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        float4 off = make_float4(lse, lse, lse, lse);
        if constexpr (kMode == kKeys) off = *reinterpret_cast<const float4*>(stat + 2 * e + 4 * hh);
        const float p[4] = {fast_exp2(fmaf(S[e], sc, -off.x)), fast_exp2(fmaf(S[e + 1], sc, -off.y)),
                            fast_exp2(fmaf(S[e + 2], sc, -off.z)), fast_exp2(fmaf(S[e + 3], sc, -off.w))};
        if constexpr (kMode == kKeys) {
          constexpr float f = std::is_same<T, _Float16>::value ? kPScale : 1.f;
          P.set(e, p[0] * f, p[1] * f);
          P.set(e + 2, p[2] * f, p[3] * f);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) dP[e + i] *= p[i];
      }
      if constexpr (kMode == kQueries) {
        if (a.far && side_far) {  // (the others are scored_diagonal_kernel's)
          float t = 0.f;
#pragma unroll
          for (int e = 0; e < 16; ++e) t += dP[e];
          if (side_far > 0) far_hi += t;
          else far_lo += t;
        }
      }
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        if constexpr (kCap) dC.set(e, dP[e] * slope[e], dP[e + 1] * slope[e + 1]);
        else dC.set(e, dP[e], dP[e + 1]);
      }
      if constexpr (kMode == kKeys) reads.product(tile + kMat, P, acc[1]);
      reads.product(tile, dC, acc[0]);
    }
  };

  lds_u8* const t0 = (lds_u8*)tile0;
  lds_u8* const t1 = (lds_u8*)tile1;
  Step s0 = next(), s1;
  if (s0.block >= 0) issue(s0, t0, (lds_u8*)stat0);
  while (s0.block >= 0) {
    // This wave's copies of the step have landed, then everyone's; every wave is done with the step before (its reads of
    // LDS have returned), whose stage the copies of the next step overwrite.
    __builtin_amdgcn_s_waitcnt(kWaitVmLgkm0);
    wg_barrier();
    s1 = next();
    if (s1.block >= 0) issue(s1, t1, (lds_u8*)stat1);
    compute(s0, t0, stat0);
    if (s1.block < 0) break;
    __builtin_amdgcn_s_waitcnt(kWaitVmLgkm0);
    wg_barrier();
    s0 = next();
    if (s0.block >= 0) issue(s0, t0, (lds_u8*)stat0);
    compute(s1, t1, stat1);
  }

  // ---- Results: element 4 q4 + j of acc[x][dc] is d = 32 dc + 8 q4 + 4 hh + j of own row own_row.
  if constexpr (kMode == kForward) l = xhalf_sum(l);
  if constexpr (kMode == kQueries) {
    if (a.far) {
      far_hi = wave_sum(far_hi);
      far_lo = wave_sum(far_lo);
      if (lane == 0) *reinterpret_cast<float2*>(stat0 + 2 * w) = make_float2(far_hi, far_lo);
      __syncthreads();
      if (threadIdx.x < 2)
        (place < 0 ? a.far + 2 * ((int64_t)bh * a.n_own + blk) : a.part_far + 2 * (int64_t)place)[threadIdx.x] =
            stat0[threadIdx.x] + stat0[2 + threadIdx.x];
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
      a.lse[((int64_t)bh * a.n_own + blk) * kBlk + kStep * w + col] =
          own_row >= a.L_own || l == 0.f ? INFINITY : m + __builtin_amdgcn_logf(l);
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

// Split items: their units' sums, added in order. A workgroup per split item.
struct MergeArgs {
  const int4* splits;  // [xcd * cap ..] {item, first place, units}
  const int32_t* n_splits;
  int cap, heads_own, n_own, L_own;
  const float *parts, *part_sums, *part_far;
  void *grad_a, *grad_b, *out_lo;
  int64_t ga_sb, ga_sh, ga_sl, gb_sb, gb_sh, gb_sl;
  float sm_scale;
  float *lse, *far;
};

template <int kMode, typename T, int kD>
__global__ __launch_bounds__(256) void scored_merge_kernel(MergeArgs a) {
  constexpr int kAcc = kMode == kKeys ? 2 : 1, kCh = kD / 4;
  const int xcd = blockIdx.x & 7, seq = blockIdx.x >> 3;
  if (seq >= a.n_splits[xcd]) return;
  const int4 u = a.splits[(int64_t)xcd * a.cap + seq];
  const int bh = u.x / a.n_own, blk = u.x - bh * a.n_own, b = bh / a.heads_own, head = bh - b * a.heads_own;
  if (kMode == kQueries && a.far && threadIdx.x < 2) {
    float s = 0.f;
    for (int p = 0; p < u.z; ++p) s += a.part_far[2 * (int64_t)(u.y + p) + threadIdx.x];
    a.far[2 * (int64_t)u.x + threadIdx.x] = s;
  }
  for (int t = threadIdx.x; t < kAcc * kBlk * kCh; t += 256) {
    const int x = t / (kBlk * kCh), r = t / kCh % kBlk, ch = t % kCh, row = blk * kBlk + r;
    const float* parts = a.parts + (((int64_t)u.y * kAcc + x) * kBlk + r) * kD + 4 * ch;
    const float* sums = a.part_sums + ((int64_t)u.y * kBlk + r) * 2;
    float top = -INFINITY, l = 0.f;
    if constexpr (kMode == kForward)
      for (int p = 0; p < u.z; ++p) top = fmaxf(top, sums[(int64_t)p * kBlk * 2]);
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
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
        a.lse[(int64_t)u.x * kBlk + r] = row >= a.L_own || l == 0.f ? INFINITY : top + __builtin_amdgcn_logf(l);
    }
    uint8_t* grad = static_cast<uint8_t*>(x == 0 ? a.grad_a : a.grad_b);
    if (!grad || row >= a.L_own) continue;
    const int64_t sb = x == 0 ? a.ga_sb : a.gb_sb, sh = x == 0 ? a.ga_sh : a.gb_sh, sl = x == 0 ? a.ga_sl : a.gb_sl;
    const int64_t at_row = (b * sb + head * sh + row * sl) * (int64_t)sizeof(T);
    uint8_t* lo = kMode == kForward && a.out_lo ? static_cast<uint8_t*>(a.out_lo) + at_row : nullptr;
    store_result<T>(grad + at_row, lo, 4 * ch, make_float4(s.x * f, s.y * f, s.z * f, s.w * f));
  }
}

// dS summed along the diagonals of 32 x 32 tiles that are not past the radius: a wave per head, offset o between the tiles'
// query and key rows (in tiles), and kDiagTiles tiles of it, whose dS it adds up element by element in registers; the
// distances 32 o + q_start - 31 .. + 31 of a unit are told apart once, at its end. S and dP are computed anew, on operands
// straight from memory: the tiles near the diagonal are few, and summing by distance inside kQueries took twice its time.
constexpr int kDiagTiles = 16;
struct DiagonalArgs {
  int Lq, Lk, first_offset, n_offsets, n_chunks;
  const uint8_t* classes;  // nullable [b or b * H + h][query block][key block]: 0 none seen, 1 all, 2 some
  float* sums;             // [b * H + h][offset][chunk][64]
};

template <bool kCap, typename T, int kD>
__global__ __launch_bounds__(256, (waves_per_simd<T, kD>())) void scored_diagonal_kernel(ScoredArgs a, DiagonalArgs g) {
  constexpr int kSize = sizeof(T), kDS = kD * kSize / 32;
  __shared__ float tiles[4][32][33];
  const int lane = threadIdx.x & 63, col = lane & 31, hh = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int64_t unit = (int64_t)blockIdx.x * 4 + w;
  if (unit >= (int64_t)a.BH_own * g.n_offsets * g.n_chunks) return;  // (no barrier below)
  float* to = g.sums + unit * 64;
  const int chunk = (int)(unit % g.n_chunks);
  unit /= g.n_chunks;
  const int o = g.first_offset + (int)(unit % g.n_offsets), bh = (int)(unit / g.n_offsets);
  const int b = bh / a.H, head = bh - b * a.H, kv_head = head / a.rep;
  const int nq = (g.Lq + 31) / 32, nk = (g.Lk + 31) / 32, nqb = (g.Lq + 63) / 64, nkb = (g.Lk + 63) / 64;
  const int q_first = max(0, o) + chunk * kDiagTiles, q_last = min(q_first + kDiagTiles, min(nq, nk + o));
  const uint8_t* classes = g.classes ? g.classes + (int64_t)(a.per_head ? bh : b) * nqb * nkb : nullptr;
  auto at = [&](const Side& s, int h, int row) {
    return static_cast<const uint8_t*>(s.p) + (b * s.sb + h * s.sh + row * s.sl) * kSize + 16 * hh;
  };
  const float slope_h = a.slopes ? a.slopes[head] * kLog2e : 0.f;
  sa_f32x16 sum = {};
  for (int t = q_first; t < q_last; ++t) {
    const int key_tile = t - o;
    int cut = kBlk * (key_tile / 2 + 1) > g.Lk;
    if (classes) {
      const int c = classes[(int64_t)(t >> 1) * nkb + (key_tile >> 1)];
      if (c == 0) continue;
      cut = c == 2;
    }
    const int row = 32 * t + col, row_c = min(row, g.Lq - 1), key_c = min(32 * key_tile + col, g.Lk - 1);
    const uint8_t *pq = at(a.own_a, head, row_c), *pd = at(a.own_b, head, row_c);
    const uint8_t *pk = at(a.st_a, kv_head, key_c), *pv = at(a.st_b, kv_head, key_c);
    const float* st = a.stats + ((int64_t)bh * nqb * 2 + t) * 64 + col;
    const float lse = st[0], delta = st[32];
    sa_f32x16 S = {}, dP, slope;
#pragma unroll
    for (int e = 0; e < 16; ++e) dP[e] = -delta;
#pragma unroll
    for (int c = 0; c < kDS; ++c) {
      S = mfma_chunk<T>(*reinterpret_cast<const sa_u32x4v*>(pk + 32 * c), *reinterpret_cast<const sa_u32x4v*>(pq + 32 * c), S);
      dP = mfma_chunk<T>(*reinterpret_cast<const sa_u32x4v*>(pv + 32 * c), *reinterpret_cast<const sa_u32x4v*>(pd + 32 * c), dP);
    }
    int side;
    const float sc = apply_rule<-1, kCap, false, T>(a, head, slope_h, 0.f, 0.f, row + a.q_start - 32 * key_tile - 4 * hh,
                                                    32 * o + a.q_start - 31, S, slope, side);
    if (cut) cut_keys(a, b, g.Lk, row, 32 * key_tile + 4 * hh, S);
#pragma unroll
    for (int e = 0; e < 16; ++e) sum[e] = fmaf(fast_exp2(fmaf(S[e], sc, -lse)), dP[e], sum[e]);
  }
  // Element e is of key 8 (e / 4) + 4 hh + e % 4 and row col of the tile; distance x - 31 of it is lane x's.
#pragma unroll
  for (int e = 0; e < 16; ++e) tiles[w][8 * (e >> 2) + 4 * hh + (e & 3)][col] = sum[e];
  __builtin_amdgcn_s_waitcnt(kWaitLgkm0);
  __builtin_amdgcn_wave_barrier();
  float s = 0.f;
  for (int j = max(0, 31 - lane); j < min(32, 63 - lane); ++j) s += tiles[w][j][j + lane - 31];
  to[lane] = lane < 63 ? s : 0.f;
}

// ---- What a call's passes read besides its operands.

struct PrepareArgs {
  const int2* ranges;  // nullable
  int64_t ranges_sb;
  int B, Lk, nkb;
  int4* bounds;  // [B][nkb]: smallest from and largest until of the keys with rows; largest from, smallest until of all
  const void* table;  // nullable, [n_buckets][H]
  int table_dtype, n_buckets, H, radius;
  const int32_t* buckets;  // [2 radius + 1]
  float* ebias;            // [H][2 radius + 1]
  int bound_groups;        // workgroups of the first kind
};

__global__ __launch_bounds__(256) void scored_prepare_kernel(PrepareArgs a) {
  if ((int)blockIdx.x < a.bound_groups) {  // a wave per key block
    const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (at >= (int64_t)a.B * a.nkb) return;
    const int lane = threadIdx.x & 63, b = (int)(at / a.nkb), key = (int)(at % a.nkb) * kBlk + lane;
    int4 r = make_int4(INT_MAX, 0, 0, INT_MAX);
    if (key < a.Lk) {
      int2 x = a.ranges[b * a.ranges_sb + key];
      x.x = max(x.x, 0);
      if (x.y > x.x) r = make_int4(x.x, x.y, x.x, x.y);
      else r = make_int4(INT_MAX, 0, INT_MAX, 0);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      r.x = min(r.x, __shfl_xor(r.x, o));
      r.y = max(r.y, __shfl_xor(r.y, o));
      r.z = max(r.z, __shfl_xor(r.z, o));
      r.w = min(r.w, __shfl_xor(r.w, o));
    }
    if (lane == 0) a.bounds[at] = r;
    return;
  }
  const int n_far = 2 * a.radius + 1;
  const int64_t i = ((int64_t)blockIdx.x - a.bound_groups) * 256 + threadIdx.x;
  if (i >= (int64_t)a.H * n_far) return;
  const int h = (int)(i / n_far), bucket = min(max(a.buckets[i % n_far], 0), a.n_buckets - 1);
  a.ebias[i] = load_as_float(a.table, a.table_dtype, (int64_t)bucket * a.H + h) * kLog2e;
}

struct ListArgs {
  const int4* bounds;  // nullable
  const uint8_t* mask; // nullable
  int64_t s0, s1, s2, s3;
  int B, H, Hl, Lq, Lk, nqb, nkb;  // Hl: heads that lists are made for, H or 1
  int32_t *kv_idx, *kv_cnt, *q_idx, *q_cnt;  // (q_idx null: not made)
  uint8_t* classes;  // nullable [B * Hl][nqb][nkb]: 0 none seen, 1 all, 2 some
};

// A wave per list: the key blocks of a query block, or the other way round.
__global__ __launch_bounds__(256) void scored_lists_kernel(ListArgs a) {
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
  const int4* bounds = a.bounds ? a.bounds + (int64_t)b * a.nkb : nullptr;
  int32_t* out = (keys ? a.q_idx : a.kv_idx) + row * n_st;
  int total = 0;
  for (int n0 = 0; n0 < n_st; n0 += 64) {
    const int n = n0 + lane, qb = keys ? n : own, kb = keys ? own : n;
    bool any = n < n_st, whole = (kb + 1) * kBlk <= a.Lk;
    if (any && bounds) {
      const int r0 = qb * kBlk, r1 = min(r0 + kBlk, a.Lq);
      const int4 x = bounds[kb];
      any = x.x < r1 && x.y > r0;
      whole = whole && x.z <= r0 && x.w >= r1;
    }
    if (any && mask) any = mask[(int64_t)qb * a.s2 + (int64_t)kb * a.s3] != 0;
    const uint64_t bal = __ballot(any);
    const int pre = __builtin_amdgcn_mbcnt_hi((uint32_t)(bal >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)bal, 0));
    if (any) out[total + pre] = 2 * n + !whole;
    if (a.classes && !keys && n < n_st) a.classes[row * n_st + n] = any ? whole ? 1 : 2 : 0;
    total += __popcll(bal);
  }
  if (lane == 0) (keys ? a.q_cnt : a.kv_cnt)[row] = total;
}

// The units of work of a pass: items whose lists are long for the call are shared by several workgroups, in chunks of
// their entries. A workgroup of XCD x needs about 3/4 of the entries that each of the `slots` workgroups that the card
// holds at once has on average, or `least`, before an item is split.
struct SideArgs {
  const int32_t* cnt;  // lists' lengths; null: n_st each
  int lists, per_head, heads_own, BH_own, rep, n_own, n_st;  // rep: streamed heads of an own one
  int keys, slots, least, max_units, cap, split_cap, sorted;
  int4 *units, *splits;  // [8][cap], [8][split_cap]
  int32_t *n_units, *n_splits;
};
struct ScheduleArgs {
  SideArgs side[2];
};
constexpr int kPlanThreads = 1024;

// Sum over the workgroup; the inclusive sum up to the thread in `upto`.
__device__ inline int group_sum(int x, int* waves, int* upto) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 63) waves[wave] = x;
  __syncthreads();
  int before = 0, all = 0;
  for (int i = 0; i < kPlanThreads / 64; ++i) {
    if (i < wave) before += waves[i];
    all += waves[i];
  }
  if (upto) *upto = before + x;
  return all;
}

__global__ __launch_bounds__(kPlanThreads) void scored_schedule_kernel(ScheduleArgs args) {
  __shared__ int waves[kPlanThreads / 64];
  __shared__ int4 kept[kPlanThreads];
  __shared__ uint32_t key[kPlanThreads];
  const SideArgs& a = args.side[blockIdx.x >> 3];
  const int xcd = blockIdx.x & 7, t = threadIdx.x;
  const int n_seq = xcd_items(a.BH_own, a.n_own);
  auto length = [&](int seq, int& item) {  // entries of an item, -1: none
    int bh, rank;
    if (seq >= n_seq || !own_block(xcd, seq, a.BH_own, a.n_own, bh, rank)) return -1;
    const int blk = block_of_rank(a.keys, rank, a.n_own);
    item = bh * a.n_own + blk;
    if (!a.cnt) return a.n_st * a.rep;
    if (!a.per_head) return min(max(a.cnt[(int64_t)(bh / a.heads_own) * a.n_own + blk], 0), a.n_st) * a.rep;
    int n = 0;
    for (int g = 0; g < a.rep; ++g) n += min(max(a.cnt[((int64_t)bh * a.rep + g) * a.n_own + blk], 0), a.n_st);
    return n;
  };
  // Entries of all items, in units of 64 so that their sum fits.
  int sum = 0;
  if (a.cnt) {
    for (int64_t i = t; i < (int64_t)a.lists * a.n_own; i += kPlanThreads) sum += min(max(a.cnt[i], 0), a.n_st);
  } else {
    for (int64_t i = t; i < (int64_t)a.lists * a.n_own; i += kPlanThreads) sum += a.n_st;
  }
  const int64_t total = (int64_t)group_sum((sum + 63) >> 6, waves, nullptr) * 64 *
                        (a.per_head ? 1 : a.heads_own * a.rep);
  int limit = (int)min(max(total * 3 / (4 * (int64_t)a.slots), (int64_t)a.least), (int64_t)1 << 29);
  for (;;) {  // (ends when no item is longer)
    int more = 0;
    for (int seq = t; seq < n_seq; seq += kPlanThreads) {
      int item;
      const int n = length(seq, item);
      if (n > limit) more += min((n + limit - 1) / limit, a.max_units + 1);
    }
    if (group_sum(min(more, 1 << 20), waves, nullptr) <= a.max_units) break;
    limit += limit / 2 + 1;
  }
  int units = 0, splits = 0, places = 0;
  for (int s0 = 0; s0 < n_seq; s0 += kPlanThreads) {
    int item = -1;
    const int n = length(s0 + t, item), parts = n < 0 ? 0 : n > limit ? (n + limit - 1) / limit : 1;
    int at, at_split, at_place;
    const int more = group_sum(parts, waves, &at);
    const int more_splits = group_sum(parts > 1, waves, &at_split);
    const int more_places = group_sum(parts > 1 ? parts : 0, waves, &at_place);
    at += units - parts;
    at_place += places - (parts > 1 ? parts : 0);
    const int place = xcd * a.max_units + at_place;
    for (int p = 0; p < parts; ++p) {
      const int4 u = make_int4(item, (int)((int64_t)n * p / parts), (int)((int64_t)n * (p + 1) / parts), parts > 1 ? place + p : -1);
      if (a.sorted && at + p < kPlanThreads) kept[at + p] = u;
      a.units[(int64_t)xcd * a.cap + at + p] = u;
    }
    if (parts > 1) a.splits[(int64_t)xcd * a.split_cap + splits + at_split - 1] = make_int4(item, place, parts, 0);
    units += more;
    splits += more_splits;
    places += more_places;
  }
  if (t == 0) {
    a.n_units[xcd] = units;
    a.n_splits[xcd] = splits;
  }
  // Longest first, where the streamed sides of all the XCD's heads fit its L2 and the units a workgroup's registers.
  if (!a.sorted || units > kPlanThreads) return;
  __syncthreads();
  int4 u = make_int4(0, 0, 0, 0);
  if (t < units) {
    u = kept[t];
    key[t] = (uint32_t)min(u.z - u.y, (1 << 21) - 1) * kPlanThreads + (kPlanThreads - 1 - t);
  }
  __syncthreads();
  if (t >= units) return;
  int before = 0;
  for (int i = 0; i < units; ++i) before += key[i] > key[t];
  a.units[(int64_t)xcd * a.cap + before] = u;
}

// dtable[n][h]: the diagonals' sums by distance and the items' sums past the radius, added in order, then the distances
// of each bucket. A workgroup per head.
constexpr int kSumThreads = 1024;
struct TableArgs {
  const float *far, *diagonals;  // [b * H + h][nqb][2]; [b * H + h][offset][chunk][64]
  const int32_t* buckets;
  void* dtable;
  int B, H, nqb, radius, n_buckets, dtype, first_offset, n_offsets, n_chunks, q_start;
};
constexpr int kMostOffsets = (2 * kMostRadius + 62) / 32 + 2;
__global__ __launch_bounds__(kSumThreads) void scored_table_kernel(TableArgs a) {
  __shared__ float sums[kMostOffsets * 64], total[2 * kMostRadius + 1], ends[kSumThreads / 64][2];
  const int h = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = t >> 6, R = a.radius;
  for (int i = t; i < a.n_offsets * 64; i += kSumThreads) {
    float s = 0.f;
    for (int b = 0; b < a.B; ++b) {
      const float* from = a.diagonals + (((int64_t)b * a.H + h) * a.n_offsets + (i >> 6)) * a.n_chunks * 64 + (i & 63);
#pragma unroll 8
      for (int c = 0; c < a.n_chunks; ++c) s += from[(int64_t)c * 64];
    }
    sums[i] = s;
  }
  float hi = 0.f, lo = 0.f;
  for (int i = t; i < a.B * a.nqb; i += kSumThreads) {
    const int b = i / a.nqb;
    const float2 x = *reinterpret_cast<const float2*>(a.far + 2 * (((int64_t)b * a.H + h) * a.nqb + (i - b * a.nqb)));
    hi += x.x;
    lo += x.y;
  }
  hi = wave_sum(hi);
  lo = wave_sum(lo);
  if (lane == 0) {
    ends[wave][0] = hi;
    ends[wave][1] = lo;
  }
  __syncthreads();
  // Value x of offset o is of distance 32 o + q_start + x - 31: a distance inside the radius has two of them at most.
  const int low = 32 * a.first_offset + a.q_start - 31;
  for (int i = t; i <= 2 * R; i += kSumThreads) {
    const bool first = i == 0, last = i == 2 * R;
    float s = 0.f;
    if (first || last)
      for (int v = 0; v < kSumThreads / 64; ++v) s += (last ? ends[v][0] : 0.f) + (first ? ends[v][1] : 0.f);
    // (past an end, all that lie there)
    for (int d = first ? min(low, -R) : i - R; d <= (last ? max(low + 32 * a.n_offsets + 30, R) : i - R); ++d) {
      const int x = d - low, o = x >> 5;
      if (x < 0) continue;
      if (o < a.n_offsets) s += sums[o * 64 + (x & 31)];
      if (o >= 1 && o <= a.n_offsets && (x & 31) < 31) s += sums[(o - 1) * 64 + 32 + (x & 31)];
    }
    total[i] = s;
  }
  __syncthreads();
  for (int n = wave; n < a.n_buckets; n += kSumThreads / 64) {
    float s = 0.f;
    for (int i = lane; i <= 2 * R; i += 64)
      if (min(max(a.buckets[i], 0), a.n_buckets - 1) == n) s += total[i];
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
constexpr int kRangeKeys = 4096;  // keys of a workgroup, which sums up the sequence's lengths for itself
struct RangeArgs {
  const int32_t *lengths, *prefix;  // [B][n]; prefix may be null
  int n, L, causal, frame, window;
  int2* out;  // [B][L]
};
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

constexpr int kCus = 256;

struct SidePlan {  // how a side's items are dealt out; byte offsets into a call's plan buffer
  bool scheduled, sorted;
  int slots, least, max_units, cap, split_cap;
  int64_t units, n_units, splits, n_splits;
};
struct Plan {
  int64_t bounds, ebias, classes, kv_idx, kv_cnt, q_idx, q_cnt, bytes;
  SidePlan side[2];  // queries, keys
};

// Whether and how the items of a side are split: by the longest list that there can be. Without lists, where all are
// alike, the host knows that none is long for the call.
SidePlan side_plan(const sa_attn_scored& t, bool keys) {
  SidePlan p{};
  const bool f32 = t.dtype == SA_DTYPE_F32;
  const int64_t rep = keys ? t.H / t.Hk : 1, BH = (int64_t)t.B * (keys ? t.Hk : t.H);
  const int n_own = sa::cdiv(keys ? t.Lk : t.Lq, kBlk), n_st = sa::cdiv(keys ? t.Lq : t.Lk, kBlk);
  // Workgroups that the card holds at once (waves_per_simd). A 16-bit step takes half a microsecond, of fp32 two to four:
  // units of fewer than 16 and 4 steps would cost more in sums than they save.
  p.slots = kCus * 2 * (f32 ? (t.D == 64 ? 2 : 1) : t.D == 64 ? 3 : 2);
  p.least = f32 ? 2 : 8;
  const int64_t longest = n_st * rep;
  p.scheduled = longest > p.least;
  if (!t.ranges && !t.mask && longest <= std::max<int64_t>(p.least, BH * n_own * longest * 3 / (4 * p.slots))) p.scheduled = false;
  if (!p.scheduled) return p;
  const int64_t items = xcd_items((int)BH, n_own);
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
  const int64_t lists = t.ranges || t.mask ? (int64_t)t.B * (t.mask ? t.H : 1) : 0;
  const bool keys = t.follow & SA_SCORED_KEYS;
  Buffer buf;
  p.bounds = buf.take(t.ranges ? t.B * nkb * 16 : 0);
  p.ebias = buf.take(t.table ? (int64_t)t.H * (2 * t.radius + 1) * 4 : 0);
  p.classes = buf.take(t.follow & SA_SCORED_TABLE ? lists * nqb * nkb : 0);
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

// Offsets o = query tile - key tile (of 32 rows) of the tiles that are not past the radius.
struct Offsets {
  int first, n, chunks;
};
Offsets offsets_of(const sa_attn_scored& t) {
  const int nq = sa::cdiv(t.Lq, kStep), nk = sa::cdiv(t.Lk, kStep);
  // -R - 31 < 32 o + q_start < R + 31
  auto floor32 = [](int64_t x) { return x >= 0 ? x / 32 : -((-x + 31) / 32); };
  const int64_t lo = std::max<int64_t>(floor32((int64_t)-t.radius - 31 - t.q_start) + 1, -(nk - 1));
  const int64_t hi = std::min<int64_t>(floor32((int64_t)t.radius + 30 - t.q_start), nq - 1);
  if (hi < lo) return Offsets{0, 0, 1};
  return Offsets{(int)lo, (int)(hi - lo + 1), sa::cdiv(std::min(nq, nk), kDiagTiles)};
}

struct Work {  // byte offsets into the workspaces of the forward and the backward call
  int64_t fwd_parts, fwd_sums, fwd_bytes;
  int64_t stats, far, part_far, diagonals, parts, bytes;
};
Work work_of(const sa_attn_scored& t, const Plan& p) {
  const int64_t rows = (int64_t)t.B * t.H * sa::cdiv(t.Lq, kBlk), sums = (int64_t)kBlk * t.D * 4;
  const int64_t q_places = 8 * p.side[0].max_units, k_places = 8 * p.side[1].max_units;
  Work w;
  Buffer fwd, bwd;
  w.fwd_parts = fwd.take(q_places * sums);
  w.fwd_sums = fwd.take(q_places * kBlk * 8);
  w.fwd_bytes = fwd.at;
  w.stats = bwd.take(rows * 512);
  const bool table = t.follow & SA_SCORED_TABLE;
  w.far = bwd.take(table ? rows * 8 : 0);
  w.part_far = bwd.take(table ? q_places * 8 : 0);
  const Offsets o = table ? offsets_of(t) : Offsets{};
  w.diagonals = bwd.take((int64_t)t.B * t.H * o.n * o.chunks * 256);
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
  SA_REQUIRE(!t->cap || (t->cap > 1e-30f && std::isfinite(t->sm_scale / t->cap * 3.f) && t->sm_scale / t->cap > 0.f),
             "%s: sm_scale / cap out of range", fn);
  if (t->Lq > 1 << 27 || t->Lk > 1 << 27) return sa::fail(SA_ERR_UNSUPPORTED, "%s: more than 2^27 rows", fn);
  SA_REQUIRE(t->q_start > -(1 << 29) && t->q_start < 1 << 29, "%s: q_start %d", fn, t->q_start);
  if ((int64_t)t->B * t->H * std::max(sa::cdiv(t->Lq, kBlk), sa::cdiv(t->Lk, kBlk)) >= 1LL << 30)
    return sa::fail(SA_ERR_UNSUPPORTED, "%s: more than 2^30 blocks", fn);
  if (t->table) {
    SA_REQUIRE(t->buckets && t->n_buckets > 0, "%s: table without buckets", fn);
    SA_REQUIRE(t->table_dtype >= SA_DTYPE_BF16 && t->table_dtype <= SA_DTYPE_F32, "%s: table dtype %d", fn, t->table_dtype);
    if (t->radius < 0 || t->radius > kMostRadius)
      return sa::fail(SA_ERR_UNSUPPORTED, "%s: distances up to %d told apart (at most %d)", fn, t->radius, kMostRadius);
  }
  SA_REQUIRE(t->table || !(t->follow & SA_SCORED_TABLE), "%s: a table's gradient without a table", fn);
  if (t->follow & SA_SCORED_TABLE) {
    const Offsets o = offsets_of(*t);
    if ((int64_t)t->B * t->H * o.n * o.chunks >= 1LL << 31)
      return sa::fail(SA_ERR_UNSUPPORTED, "%s: more than 2^31 diagonals", fn);
  }
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

template <int kMode, bool kCap, typename T, int kD>
void launch_kernels(const ScoredArgs& a, const SidePlan& p, const MergeArgs& m, hipStream_t s) {
  const unsigned grid = 8u * (unsigned)(p.scheduled ? p.cap : xcd_items(a.BH_own, a.n_own));
  hipLaunchKernelGGL((scored_kernel<kMode, kCap, T, kD>), dim3(grid), dim3(128), 0, s, a);
  // (the statistics alone are written by every unit's first part)
  if (p.scheduled && (a.grad_a || a.grad_b || a.far))
    hipLaunchKernelGGL((scored_merge_kernel<kMode, T, kD>), dim3(8u * (unsigned)p.split_cap), dim3(256), 0, s, m);
}

template <bool kCap, typename T, int kD>
void launch_diagonals(const ScoredArgs& a, const DiagonalArgs& g, hipStream_t s) {
  const int64_t units = (int64_t)a.BH_own * g.n_offsets * g.n_chunks;
  if (units > 0)
    hipLaunchKernelGGL((scored_diagonal_kernel<kCap, T, kD>), dim3((unsigned)((units + 3) / 4)), dim3(256), 0, s, a, g);
}

// f.template operator()<cap, type, head dim>() of a call's.
template <typename F>
void with_kernel(const sa_attn_scored& t, F f) {
  auto dim = [&](auto cap, auto type) {
    if (t.D == 64) f(cap, type, std::integral_constant<int, 64>());
    else f(cap, type, std::integral_constant<int, 128>());
  };
  auto kind = [&](auto cap) {
    if (t.dtype == SA_DTYPE_BF16) dim(cap, __bf16());
    else if (t.dtype == SA_DTYPE_F16) dim(cap, _Float16());
    else dim(cap, float());
  };
  if (t.cap > 0) kind(std::true_type());
  else kind(std::false_type());
}

template <int kMode>
void launch_pass(ScoredArgs a, const sa_attn_scored& t, const SidePlan& p, hipStream_t s) {
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
    m.sm_scale = a.sm_scale; m.lse = a.lse; m.far = a.far;
  }
  with_kernel(t, [&](auto cap, auto type, auto dim) {
    launch_kernels<kMode, decltype(cap)::value, decltype(type), decltype(dim)::value>(a, p, m, s);
  });
}

Side side_of(const sa_attn_scored& t, const void* p, int i) {
  return Side{p, t.strides[3 * i], t.strides[3 * i + 1], t.strides[3 * i + 2]};
}

ScoredArgs common_args(const sa_attn_scored& t) {
  ScoredArgs a{};
  a.H = t.H;
  a.rep = t.H / t.Hk;
  a.q_start = t.q_start;
  a.ranges = reinterpret_cast<const int2*>(t.ranges);
  a.ranges_sb = t.ranges_stride;
  a.sm_scale = t.sm_scale;
  a.scale_log2 = t.sm_scale * kLog2e;
  if (t.cap > 0) {
    a.cap_in = t.sm_scale / t.cap * (t.dtype == SA_DTYPE_F32 ? 1.f : 2.f * kLog2e);
    a.cap_log2 = t.cap * kLog2e;
  }
  a.slopes = t.slopes;
  a.radius = t.table ? t.radius : 0;
  a.per_head = t.mask != nullptr;
  a.lse = t.lse;
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
  if (t.ranges || t.mask) {
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
  const bool lists = t->ranges || t->mask, keys = t->follow & SA_SCORED_KEYS;
  if (t->ranges || t->table) {
    PrepareArgs g{};
    g.ranges = reinterpret_cast<const int2*>(t->ranges);
    g.ranges_sb = t->ranges_stride;
    g.B = t->B; g.Lk = t->Lk; g.nkb = nkb;
    g.bounds = reinterpret_cast<int4*>(plan + p.bounds);
    g.table = t->table; g.table_dtype = t->table_dtype; g.n_buckets = t->n_buckets; g.H = t->H;
    g.radius = t->radius;
    g.buckets = t->buckets;
    g.ebias = reinterpret_cast<float*>(plan + p.ebias);
    g.bound_groups = t->ranges ? (int)(((int64_t)t->B * nkb + 3) / 4) : 0;
    const int64_t more = t->table ? ((int64_t)t->H * (2 * t->radius + 1) + 255) / 256 : 0;
    hipLaunchKernelGGL(scored_prepare_kernel, dim3((unsigned)(g.bound_groups + more)), dim3(256), 0, s, g);
    if (int rc = sa::check_launch(fn)) return rc;
  }
  if (lists) {
    ListArgs g{};
    g.bounds = t->ranges ? reinterpret_cast<const int4*>(plan + p.bounds) : nullptr;
    g.mask = t->mask;
    g.s0 = t->mask_strides[0]; g.s1 = t->mask_strides[1]; g.s2 = t->mask_strides[2]; g.s3 = t->mask_strides[3];
    g.B = t->B; g.H = t->H; g.Hl = t->mask ? t->H : 1;
    g.Lq = t->Lq; g.Lk = t->Lk; g.nqb = nqb; g.nkb = nkb;
    g.kv_idx = reinterpret_cast<int32_t*>(plan + p.kv_idx);
    g.kv_cnt = reinterpret_cast<int32_t*>(plan + p.kv_cnt);
    if (t->follow & SA_SCORED_TABLE) g.classes = plan + p.classes;
    if (keys) {
      g.q_idx = reinterpret_cast<int32_t*>(plan + p.q_idx);
      g.q_cnt = reinterpret_cast<int32_t*>(plan + p.q_cnt);
    }
    const int64_t rows = (int64_t)g.B * g.Hl * (nqb + (keys ? nkb : 0));
    hipLaunchKernelGGL(scored_lists_kernel, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, g);
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
    a.lists = t->B * (t->mask ? t->H : 1);
    a.heads_own = i ? t->Hk : t->H;
    a.BH_own = t->B * a.heads_own;
    a.rep = i ? t->H / t->Hk : 1;
    a.n_own = i ? nkb : nqb;
    a.n_st = i ? nqb : nkb;
    a.keys = i;
    a.slots = sp.slots; a.least = sp.least; a.max_units = sp.max_units; a.cap = sp.cap; a.split_cap = sp.split_cap;
    a.sorted = sp.sorted;
    a.units = reinterpret_cast<int4*>(plan + sp.units);
    a.splits = reinterpret_cast<int4*>(plan + sp.splits);
    a.n_units = reinterpret_cast<int32_t*>(plan + sp.n_units);
    a.n_splits = reinterpret_cast<int32_t*>(plan + sp.n_splits);
  }
  if (n_sides) {
    hipLaunchKernelGGL(scored_schedule_kernel, dim3(8 * n_sides), dim3(kPlanThreads), 0, s, g);
    if (int rc = sa::check_launch(fn)) return rc;
  }
  ScoredArgs a = common_args(*t);
  own_queries(a, *t, p);
  a.grad_a = t->out;
  a.ga_sb = t->strides[9]; a.ga_sh = t->strides[10]; a.ga_sl = t->strides[11];
  uint8_t* ws = static_cast<uint8_t*>(t->workspace);
  a.parts = reinterpret_cast<float*>(ws + work.fwd_parts);
  a.part_sums = reinterpret_cast<float*>(ws + work.fwd_sums);
  launch_pass<kForward>(a, *t, p.side[0], s);
  return sa::check_launch(fn);
}

extern "C" int sa_attn_scored_bwd(const sa_attn_scored* t, void* stream) {
  const char* fn = "sa_attn_scored_bwd";
  if (int rc = check_scored(t, fn)) return rc;
  SA_REQUIRE(t->q && t->k && t->v && t->out && t->dout && t->lse, "%s: null pointer", fn);
  if (int rc = check_operands(t, fn, 0, 8)) return rc;
  const bool lists = t->ranges || t->mask, keys = t->dk || t->dv;
  SA_REQUIRE((!keys || (t->follow & SA_SCORED_KEYS)) && (!t->dtable || (t->follow & SA_SCORED_TABLE)),
             "%s: gradients that the plan does not follow", fn);
  const Plan p = plan_of(*t);
  const Work w = work_of(*t, p);
  if (int rc = check_buffers(t, p, w.bytes, fn)) return rc;
  hipStream_t s = sa::as_stream(stream);
  uint8_t* ws = static_cast<uint8_t*>(t->workspace);
  const uint8_t* plan = static_cast<const uint8_t*>(t->plan);
  ScoredArgs a = common_args(*t);
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
  launch_pass<kQueries>(a, *t, p.side[0], s);
  if (int rc = sa::check_launch(fn)) return rc;
  if (t->dtable) {
    const Offsets o = offsets_of(*t);
    DiagonalArgs d{};
    d.Lq = t->Lq; d.Lk = t->Lk;
    d.first_offset = o.first; d.n_offsets = o.n; d.n_chunks = o.chunks;
    d.classes = lists ? plan + p.classes : nullptr;
    d.sums = reinterpret_cast<float*>(ws + w.diagonals);
    with_kernel(*t, [&](auto cap, auto type, auto dim) {
      launch_diagonals<decltype(cap)::value, decltype(type), decltype(dim)::value>(a, d, s);
    });
    if (int rc = sa::check_launch(fn)) return rc;
    const TableArgs g = {a.far, d.sums, t->buckets, t->dtable, t->B, t->H, a.n_own, t->radius, t->n_buckets, t->table_dtype,
                         o.first, o.n, o.chunks, t->q_start};
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
  launch_pass<kKeys>(a, *t, p.side[1], s);
  return sa::check_launch(fn);
}
