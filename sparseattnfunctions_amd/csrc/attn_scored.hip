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
  float* far_sums;         // kQueries, nullable: [item][2 radius + 1] sums of dS by distance
};

// Own block of a workgroup: workgroups go to the XCDs in turn, and an XCD works on whole heads one after the other, so
// that its L2 holds the streamed side; the heads that are left over go to all XCDs. False: none.
__device__ inline bool own_block(int x, int BH, int n, int& bh, int& rank) {
  const int full = BH >> 3, xcd = x & 7, seq = x >> 3;
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
  extern __shared__ float far_lds[];  // kQueries with far_sums: [wave][hh][2 radius + 1]

  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, hh = lane >> 5;
  int bh, rank;
  if (!own_block(blockIdx.x, a.BH_own, a.n_own, bh, rank)) return;  // (the whole workgroup)
  // Where keys are seen by later rows, the last query blocks and the first key blocks have the longest lists.
  const int blk = kMode == kKeys ? rank : a.n_own - 1 - rank;
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
  const int n_far = 2 * a.radius + 1;
  if constexpr (kMode == kQueries) {
    const uint8_t* po = at(a.out, b, head) + (int64_t)own_clamped * a.out.sl * kSize + 16 * hh;
#pragma unroll
    for (int s = 0; s < kDS; ++s) delta = dot_chunk<T>(*reinterpret_cast<const sa_u32x4v*>(po + 32 * s), fb[s], delta);
    delta = xhalf_sum(delta);
    lse = a.lse[((int64_t)bh * a.n_own + blk) * kBlk + kStep * w + col];
    a.stats[(((int64_t)bh * a.n_own + blk) * 2 + w) * 64 + lane] =
        own_row < a.L_own ? (hh == 0 ? lse : delta) : hh == 0 ? INFINITY : 0.f;
    if (!a.grad_a && !a.far_sums) return;  // only the statistics are wanted
    if (a.far_sums) {
      for (int i = lane; i < 2 * n_far; i += 64) far_lds[w * 2 * n_far + i] = 0.f;
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
  auto set_list = [&]() __attribute__((always_inline)) {
    const int hq = kMode == kKeys ? st_head + g : head;
    if (a.slopes) slope_h = *(ConstPtr)(a.slopes + hq);
    if (a.ebias) {
      before = *(ConstPtr)(a.ebias + (int64_t)hq * n_far);
      past = *(ConstPtr)(a.ebias + (int64_t)hq * n_far + 2 * a.radius);
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
    if (pos < cnt) {
      const int e = a.idx ? ahead : 2 * pos + (kBlk * (pos + 1) > a.L_st);
      s.block = e >> 1;
      s.cut = e & 1;
      // (the second half of a block that ends before it is left out)
      if (half == 0 && s.block * kBlk + kStep < a.L_st) {
        half = 1;
      } else {
        half = 0;
        ++pos;
        if (a.idx && pos < cnt) ahead = list[pos];
      }
      if ((unsigned)s.block >= (unsigned)a.n_st) s.block = 0, s.cut = 2;  // (no such block: skipped)
    }
    return s;
  };
  set_list();

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
  float far_hi = 0.f, far_lo = 0.f;      // kQueries with far_sums: the lane's sums of dS past the radius

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
    // Elements e: streamed row row0 + 4 hh + c_e, c_e = 8 (e / 4) + e % 4, of own row own_row.
    // S sc is the score times log2(e) from here on.
    float sc = a.scale_log2;
    if constexpr (kCap) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        float t = 0.f;
        S[e] = bend<T, kMode != kForward>(S[e] * a.cap_in, t) * a.cap_log2;
        if constexpr (kMode != kForward) slope[e] = t;
      }
      sc = 1.f;
    }
    // Distances: d = base - c_e, or (kKeys) base + c_e.
    const int base = kMode == kKeys ? row0 + 4 * hh + a.q_start - own_row : own_row + a.q_start - row0 - 4 * hh;
    constexpr float kSign = kMode == kKeys ? 1.f : -1.f;
    if (a.slopes) {
      const float f = s.slope, fb_ = f * (float)base;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float c = kSign * (float)(8 * (e >> 2) + (e & 3));
        S[e] = fmaf(S[e], sc, -fabsf(fmaf(f, c, fb_)));
      }
      sc = 1.f;
    }
    // Whether all pairs of the wave are past the radius: 1 above, -1 below, 0 not all.
    int side_far = 0;
    if (a.ebias) {
      const float* eb = a.ebias + (int64_t)hq * n_far;
      const int first = __builtin_amdgcn_readfirstlane(blk * kBlk + kStep * w);
      const int least = kMode == kKeys ? row0 + a.q_start - first - 31 : first + a.q_start - row0 - 31;
      side_far = least >= a.radius ? 1 : least + 62 <= -a.radius ? -1 : 0;
      if (side_far) {
        const float c = side_far > 0 ? s.past : s.before;
#pragma unroll
        for (int e = 0; e < 16; ++e) S[e] = fmaf(S[e], sc, c);
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int c = 8 * (e >> 2) + (e & 3);
          const int d = kMode == kKeys ? base + c : base - c;
          S[e] = fmaf(S[e], sc, eb[min(max(d, -a.radius), a.radius) + a.radius]);
        }
      }
      sc = 1.f;
    }
    if (s.cut) {
      if constexpr (kMode == kKeys) {
        if (a.ranges) {
          const int t = row0 + 4 * hh - from;
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if ((unsigned)(t + 8 * (e >> 2) + (e & 3)) >= (unsigned)len) S[e] = -INFINITY;
        }
      } else if (a.ranges) {  // (keys past the last one: no rows)
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<int2*>(a.ranges + b * a.ranges_sb), (short)0, a.L_st * 8, 0x00020000);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const sa_u32x2v r = __builtin_amdgcn_raw_buffer_load_b64(rs, 8 * (row0 + 4 * hh + 8 * (e >> 2) + (e & 3)), 0, 0);
          if (own_row < (int)r[0] || own_row >= (int)r[1]) S[e] = -INFINITY;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (row0 + 4 * hh + 8 * (e >> 2) + (e & 3) >= a.L_st) S[e] = -INFINITY;
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
      Weights<T> P;
#pragma unroll
      for (int e = 0; e < 16; e += 2) P.set(e, fast_exp2(fmaf(S[e], sc, -off)), fast_exp2(fmaf(S[e + 1], sc, -off)));
      l = P.sum(l);
      reads.product(tile + kMat, P, acc[0]);
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
        if (a.far_sums) {
          if (side_far) {
            float t = 0.f;
#pragma unroll
            for (int e = 0; e < 16; ++e) t += dP[e];
            if (side_far > 0) far_hi += t;
            else far_lo += t;
          } else {
            // Lanes of one instruction and half are at distances of their own (or past the radius, which takes them in
            // the order of the lanes): the sums repeat.
            float* sums = far_lds + (2 * w + hh) * n_far + a.radius;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const int d = base - (8 * (e >> 2) + (e & 3));
              if (d >= a.radius) far_hi += dP[e];
              else if (d <= -a.radius) far_lo += dP[e];
              else __hip_atomic_fetch_add(sums + d, dP[e], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
            }
          }
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
  float f_a = a.sm_scale;
  if constexpr (kMode == kForward) {
    l = xhalf_sum(l);
    f_a = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;  // (NaN stays)
    if (hh == 0)
      a.lse[((int64_t)bh * a.n_own + blk) * kBlk + kStep * w + col] =
          own_row >= a.L_own || l == 0.f ? INFINITY : m + __builtin_amdgcn_logf(l);
  }
#pragma unroll
  for (int x = 0; x < kAcc; ++x) {
    uint8_t* grad = static_cast<uint8_t*>(x == 0 ? a.grad_a : a.grad_b);
    if (!grad || own_row >= a.L_own) continue;
    const int64_t sb = x == 0 ? a.ga_sb : a.gb_sb, sh = x == 0 ? a.ga_sh : a.gb_sh, sl = x == 0 ? a.ga_sl : a.gb_sl;
    const float f = x == 0 ? f_a : std::is_same<T, _Float16>::value ? 1.f / kPScale : 1.f;
    uint8_t* p = grad + (b * sb + head * sh + own_row * sl + 4 * hh) * kSize;
#pragma unroll
    for (int dc = 0; dc < kDC; ++dc)
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        const sa_f32x16& A = acc[x][dc];
        const float r[4] = {A[4 * q4] * f, A[4 * q4 + 1] * f, A[4 * q4 + 2] * f, A[4 * q4 + 3] * f};
        if constexpr (kF32)
          *reinterpret_cast<float4*>(p + 4 * (32 * dc + 8 * q4)) = make_float4(r[0], r[1], r[2], r[3]);
        else
          *reinterpret_cast<uint2*>(p + 2 * (32 * dc + 8 * q4)) =
              make_uint2(Elem<T>::pack(r[0], r[1]), Elem<T>::pack(r[2], r[3]));
      }
  }
  if constexpr (kMode == kQueries) {
    if (a.far_sums) {
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) {
        far_hi += __shfl_xor(far_hi, o);
        far_lo += __shfl_xor(far_lo, o);
      }
      if (lane == 0) {
        float* mine = far_lds + 2 * w * n_far;
        mine[2 * a.radius] = far_hi;
        if (a.radius > 0) mine[0] = far_lo;
        else mine[0] += far_lo;
      }
      __syncthreads();
      float* to = a.far_sums + ((int64_t)bh * a.n_own + blk) * n_far;
      for (int i = threadIdx.x; i < n_far; i += 128)
        to[i] = (far_lds[i] + far_lds[n_far + i]) + (far_lds[2 * n_far + i] + far_lds[3 * n_far + i]);
    }
  }
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
    total += __popcll(bal);
  }
  if (lane == 0) (keys ? a.q_cnt : a.kv_cnt)[row] = total;
}

// dtable[n][h]: the items' sums by distance, added in order, then the distances of each bucket in order. A workgroup
// per head; groups of 256 threads take a share of the items each.
constexpr int kSumThreads = 1024;
struct TableArgs {
  const float* far_sums;  // [b * H + h][nqb][2 radius + 1]
  const int32_t* buckets;
  void* dtable;
  int B, H, nqb, radius, n_buckets, dtype;
};
__global__ __launch_bounds__(kSumThreads) void scored_table_kernel(TableArgs a) {
  __shared__ float part[kSumThreads / 256][256];
  __shared__ float total[2 * kMostRadius + 1];
  const int n_far = 2 * a.radius + 1, h = blockIdx.x;
  const int g = threadIdx.x >> 8, t = threadIdx.x & 255;
  const int items = a.B * a.nqb;
  for (int r0 = 0; r0 < n_far; r0 += 256) {
    float s = 0.f;
    if (r0 + t < n_far)
#pragma unroll 8
      for (int i = g; i < items; i += kSumThreads / 256) {
        const int b = i / a.nqb;
        s += a.far_sums[(((int64_t)b * a.H + h) * a.nqb + (i - b * a.nqb)) * n_far + r0 + t];
      }
    part[g][t] = s;
    __syncthreads();
    if (g == 0 && r0 + t < n_far) total[r0 + t] = (part[0][t] + part[1][t]) + (part[2][t] + part[3][t]);
    __syncthreads();
  }
  for (int n = threadIdx.x; n < a.n_buckets; n += kSumThreads) {
    double s = 0.0;
    for (int r = 0; r < n_far; ++r)
      if (min(max(a.buckets[r], 0), a.n_buckets - 1) == n) s += total[r];
    const int64_t at = (int64_t)n * a.H + h;
    if (a.dtype == SA_DTYPE_F32) static_cast<float*>(a.dtable)[at] = (float)s;
    else if (a.dtype == SA_DTYPE_F16) static_cast<_Float16*>(a.dtable)[at] = (_Float16)(float)s;
    else static_cast<__bf16*>(a.dtable)[at] = (__bf16)(float)s;
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

struct Plan {  // byte offsets into a call's plan buffer
  int64_t bounds, ebias, kv_idx, kv_cnt, q_idx, q_cnt, bytes;
};

Plan plan_of(const sa_attn_scored& t) {
  Plan p;
  const int64_t nqb = sa::cdiv(t.Lq, kBlk), nkb = sa::cdiv(t.Lk, kBlk);
  const int64_t lists = t.ranges || t.mask ? (int64_t)t.B * (t.mask ? t.H : 1) : 0;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  p.bounds = take(t.ranges ? t.B * nkb * 16 : 0);
  p.ebias = take(t.table ? (int64_t)t.H * (2 * t.radius + 1) * 4 : 0);
  p.kv_idx = take(lists * nqb * nkb * 4);
  p.kv_cnt = take(lists * nqb * 4);
  p.q_idx = take(t.key_lists ? lists * nqb * nkb * 4 : 0);
  p.q_cnt = take(t.key_lists ? lists * nkb * 4 : 0);
  p.bytes = at;
  return p;
}

struct Work {  // of the backward call's workspace
  int64_t stats, far_sums, bytes;
};
Work work_of(const sa_attn_scored& t) {
  const int64_t rows = (int64_t)t.B * t.H * sa::cdiv(t.Lq, kBlk);
  Work w;
  w.stats = 0;
  w.far_sums = rows * 512;
  w.bytes = w.far_sums + (t.dtable ? (rows * (2 * t.radius + 1) * 4 + 255) / 256 * 256 : 0);
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
  SA_REQUIRE(!t->dtable || t->table, "%s: dtable without a table", fn);
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

template <int kMode, bool kCap, typename T>
void launch_dim(const ScoredArgs& a, int D, unsigned grid, size_t lds, hipStream_t s) {
  if (D == 64) hipLaunchKernelGGL((scored_kernel<kMode, kCap, T, 64>), dim3(grid), dim3(128), lds, s, a);
  else hipLaunchKernelGGL((scored_kernel<kMode, kCap, T, 128>), dim3(grid), dim3(128), lds, s, a);
}

template <int kMode, typename T>
void launch_type(const ScoredArgs& a, int D, bool cap, size_t lds, hipStream_t s) {
  const int64_t rest = (int64_t)(a.BH_own & 7) * a.n_own;
  const unsigned grid = (unsigned)(8 * ((int64_t)(a.BH_own >> 3) * a.n_own + (rest + 7) / 8));
  if (cap) launch_dim<kMode, true, T>(a, D, grid, lds, s);
  else launch_dim<kMode, false, T>(a, D, grid, lds, s);
}

template <int kMode>
void launch_pass(const ScoredArgs& a, const sa_attn_scored& t, size_t lds, hipStream_t s) {
  if (t.dtype == SA_DTYPE_BF16) launch_type<kMode, __bf16>(a, t.D, t.cap > 0, lds, s);
  else if (t.dtype == SA_DTYPE_F16) launch_type<kMode, _Float16>(a, t.D, t.cap > 0, lds, s);
  else launch_type<kMode, float>(a, t.D, t.cap > 0, lds, s);
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

extern "C" int sa_attn_scored_sizes(const sa_attn_scored* t, int64_t* plan_bytes, int64_t* workspace_bytes) {
  const char* fn = "sa_attn_scored_sizes";
  SA_REQUIRE(plan_bytes && workspace_bytes, "%s: null pointer", fn);
  if (int rc = check_scored(t, fn)) return rc;
  *plan_bytes = plan_of(*t).bytes;
  *workspace_bytes = work_of(*t).bytes;
  return sa::ok();
}

extern "C" int sa_attn_scored_fwd(const sa_attn_scored* t, void* stream) {
  const char* fn = "sa_attn_scored_fwd";
  if (int rc = check_scored(t, fn)) return rc;
  SA_REQUIRE(t->q && t->k && t->v && t->out && t->lse, "%s: null pointer", fn);
  if (int rc = check_operands(t, fn, 0, 4)) return rc;
  const Plan p = plan_of(*t);
  SA_REQUIRE(!p.bytes || (t->plan && reinterpret_cast<uintptr_t>(t->plan) % 256 == 0), "%s: plan null or not 256-byte aligned",
             fn);
  SA_REQUIRE(t->plan_bytes >= p.bytes, "%s: plan of %lld bytes < %lld", fn, (long long)t->plan_bytes, (long long)p.bytes);
  SA_REQUIRE(reinterpret_cast<uintptr_t>(t->ranges) % 8 == 0, "%s: ranges not 8-byte aligned", fn);
  hipStream_t s = sa::as_stream(stream);
  uint8_t* plan = static_cast<uint8_t*>(t->plan);
  const int nqb = sa::cdiv(t->Lq, kBlk), nkb = sa::cdiv(t->Lk, kBlk);
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
  if (t->ranges || t->mask) {
    ListArgs g{};
    g.bounds = t->ranges ? reinterpret_cast<const int4*>(plan + p.bounds) : nullptr;
    g.mask = t->mask;
    g.s0 = t->mask_strides[0]; g.s1 = t->mask_strides[1]; g.s2 = t->mask_strides[2]; g.s3 = t->mask_strides[3];
    g.B = t->B; g.H = t->H; g.Hl = t->mask ? t->H : 1;
    g.Lq = t->Lq; g.Lk = t->Lk; g.nqb = nqb; g.nkb = nkb;
    g.kv_idx = reinterpret_cast<int32_t*>(plan + p.kv_idx);
    g.kv_cnt = reinterpret_cast<int32_t*>(plan + p.kv_cnt);
    if (t->key_lists) {
      g.q_idx = reinterpret_cast<int32_t*>(plan + p.q_idx);
      g.q_cnt = reinterpret_cast<int32_t*>(plan + p.q_cnt);
    }
    const int64_t rows = (int64_t)g.B * g.Hl * (nqb + (t->key_lists ? nkb : 0));
    hipLaunchKernelGGL(scored_lists_kernel, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, g);
    if (int rc = sa::check_launch(fn)) return rc;
  }
  ScoredArgs a = common_args(*t);
  own_queries(a, *t, p);
  a.grad_a = t->out;
  a.ga_sb = t->strides[9]; a.ga_sh = t->strides[10]; a.ga_sl = t->strides[11];
  launch_pass<kForward>(a, *t, 0, s);
  return sa::check_launch(fn);
}

extern "C" int sa_attn_scored_bwd(const sa_attn_scored* t, void* stream) {
  const char* fn = "sa_attn_scored_bwd";
  if (int rc = check_scored(t, fn)) return rc;
  SA_REQUIRE(t->q && t->k && t->v && t->out && t->dout && t->lse, "%s: null pointer", fn);
  if (int rc = check_operands(t, fn, 0, 8)) return rc;
  const bool lists = t->ranges || t->mask, keys = t->dk || t->dv;
  SA_REQUIRE(!keys || !lists || t->key_lists, "%s: dk and dv need the key blocks' lists", fn);
  const Plan p = plan_of(*t);
  SA_REQUIRE(!p.bytes || (t->plan && reinterpret_cast<uintptr_t>(t->plan) % 256 == 0), "%s: plan null or not 256-byte aligned",
             fn);
  SA_REQUIRE(t->plan_bytes >= p.bytes, "%s: plan of %lld bytes < %lld", fn, (long long)t->plan_bytes, (long long)p.bytes);
  SA_REQUIRE(reinterpret_cast<uintptr_t>(t->ranges) % 8 == 0, "%s: ranges not 8-byte aligned", fn);
  const Work w = work_of(*t);
  SA_REQUIRE(t->workspace && reinterpret_cast<uintptr_t>(t->workspace) % 256 == 0,
             "%s: workspace null or not 256-byte aligned", fn);
  SA_REQUIRE(t->workspace_bytes >= w.bytes, "%s: workspace of %lld bytes < %lld", fn, (long long)t->workspace_bytes,
             (long long)w.bytes);
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
  a.far_sums = t->dtable ? reinterpret_cast<float*>(ws + w.far_sums) : nullptr;
  launch_pass<kQueries>(a, *t, t->dtable ? 4 * (2 * t->radius + 1) * sizeof(float) : 0, s);
  if (int rc = sa::check_launch(fn)) return rc;
  if (t->dtable) {
    const TableArgs g = {a.far_sums, t->buckets, t->dtable, t->B, t->H, a.n_own, t->radius, t->n_buckets, t->table_dtype};
    hipLaunchKernelGGL(scored_table_kernel, dim3((unsigned)t->H), dim3(kSumThreads), 0, s, g);
    if (int rc = sa::check_launch(fn)) return rc;
  }
  if (!keys) return sa::ok();
  a.far_sums = nullptr;
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
  launch_pass<kKeys>(a, *t, 0, s);
  return sa::check_launch(fn);
}
