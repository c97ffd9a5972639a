// Attention of a few new tokens of each sequence over its cached keys and values, and over a prefix that all sequences
// share, with the score rule of attn_scored.hip.
//
// Sequence b has lengths[b] cached tokens, of which the last Ln are the new ones; behind the Lp tokens of the shared prefix.
// New token i is the sequence's own token t = lengths[b] - Ln + i, at distance d = t - j from own key j and d = Lp + t - j
// from prefix key j; it sees keys at 0 <= d (< window, if there is one), and none where t < 0.
//
// Reading the cached keys and values is a call's bound (one new token: 2 operations a byte in 16 bits, against the card's 300), so
// the work is dealt out by keys: a sequence's and key head's rows (its query heads' new tokens) share a read of the keys, 32
// rows as the columns of a matrix product, and the keys are split over workgroups and their waves. Every 32 rows read the keys
// again, so that many new tokens (a chunk of a prompt) cost as many reads. The prefix's keys are read once for each 32 rows of
// all sequences together; a short prefix by each sequence, ahead of its own keys. Each wave copies its steps of 32
// keys into LDS stages of its own, with no barrier between steps; a workgroup's waves join their sums in LDS, and
// cached_merge_kernel joins the workgroups', in order: results do not depend on the order in which they run.
//
// Measured (kernel and merge): 8 sequences of 8888 to 17776 keys, 30 heads of 64, bf16: 162 to 169 + 5 us, 5.5 TB/s; 4 of 22552 to
// 45104 keys, 8 heads of 128 read by 48, 4 tokens each, fp16: 118 to 124 + 5 us, 5.4 TB/s (a large copy: 4.7); one of 263 to 526
// keys, 30 heads of 64: 9.0 us in one launch, of which the first loads from HBM and cold code are most. In fp32 at head dim 128 a
// workgroup has two waves for the LDS of a CU (128 KB): half of its SIMDs work.
#include <math.h>

#include <algorithm>
#include <climits>
#include <cmath>

#include "attn_score.h"

namespace {

struct Cache {
  const void *k, *v;
  int64_t k_sb, k_sh, k_sl, v_sb, v_sh, v_sl;  // elements
};

struct CachedArgs {
  const void* q;
  void* out;
  int64_t q_sb, q_sh, q_sl, o_sb, o_sh, o_sl;
  Cache own, prefix;
  const int32_t* lengths;
  int B, H, Hk, rep, Ln, L, Lp, window;
  int tiles, splits;                // 32-row tiles of a sequence's rows of a key head, and workgroups that share their keys
  int prefix_tiles, prefix_splits;  // of all sequences' rows of a key head, and alike for the prefix
  int own_groups;                   // B * Hk * tiles * splits workgroups, and behind them the prefix's
  int lead;                         // steps of the prefix that each sequence takes before its own; then prefix_splits is 0
  float scale_log2;
  Cap cap;
  const float* slopes;
  const void* table;
  const int32_t* buckets;
  int table_dtype, n_buckets, radius;
  float *sums, *parts;  // [workgroup][32] {offset, sum}, and [workgroup][32][kD]; null: the output is written
};

template <typename T, int kD>
struct CachedShape {
  static constexpr int kRow = kD * (int)sizeof(T);
  static constexpr int kMat = kStep * kRow;  // a step's keys or values
  // Waves of a workgroup: two stages of 2 kMat bytes each.
  static constexpr int kWaves = kRow <= 256 ? 4 : 2;
};

template <typename T>
__device__ __forceinline__ void store_four(uint8_t* row, int at, float x, float y, float z, float w) {
  if constexpr (std::is_same<T, float>::value) *reinterpret_cast<float4*>(row + 4 * at) = make_float4(x, y, z, w);
  else *reinterpret_cast<uint2*>(row + 2 * at) = make_uint2(Elem<T>::pack(x, y), Elem<T>::pack(z, w));
}

// kPieces: a piece of the row of all steps (parts is not null); else an item.
// kLead: a sequence's steps begin with those of the prefix.
template <bool kLead, bool kCap, typename T, int kD>
__global__ __launch_bounds__((64 * CachedShape<T, kD>::kWaves)) void cached_kernel(CachedArgs a) {
  constexpr int kSize = sizeof(T), kRow = CachedShape<T, kD>::kRow, kMat = CachedShape<T, kD>::kMat;
  constexpr int kWaves = CachedShape<T, kD>::kWaves;
  constexpr int kDS = kRow / 32, kDC = kD / 32, kParts = kRow / 128;
  __shared__ __attribute__((aligned(1024))) uint8_t tile0[kWaves * 2 * kMat], tile1[kWaves * 2 * kMat];
  __shared__ float joined[kWaves][2][kStep];

  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, hh = lane >> 5;
  const bool shared = !kLead && (int)blockIdx.x >= a.own_groups;
  int x = shared ? blockIdx.x - a.own_groups : blockIdx.x;
  const int splits = shared ? a.prefix_splits : a.splits, tiles = shared ? a.prefix_tiles : a.tiles;
  const int split = x % splits;
  x /= splits;
  const int tile = x % tiles;
  x /= tiles;
  const int hk = shared ? x : x % a.Hk, b0 = shared ? 0 : x / a.Hk;

  // The lane's row: of sequence b, query head h, new token i.
  const int per = a.rep * a.Ln, n_rows = shared ? a.B * per : per;
  const int row = tile * kStep + col;
  const int r = min(row, n_rows - 1);  // (rows past the last one are computed like it and not stored)
  const int b = shared ? r / per : b0, in = shared ? r - b * per : r;
  const int h = hk * a.rep + in / a.Ln, i = in % a.Ln;
  const int t = min(max(a.lengths[b], 0), a.L) - a.Ln + i;
  const int place = shared ? a.Lp + t : t;  // d = place - key
  sa_u32x4v fa[kDS];
  {
    const uint8_t* p = static_cast<const uint8_t*>(a.q) + (b * a.q_sb + h * a.q_sh + i * a.q_sl) * kSize + 16 * hh;
#pragma unroll
    for (int s = 0; s < kDS; ++s) fa[s] = *reinterpret_cast<const sa_u32x4v*>(p + 32 * s);
  }
  float slope = a.slopes ? a.slopes[h] * kLog2e : 0.f;
  auto bias_at = [&](int d) {
    const int n = min(max(a.buckets[min(max(d, -a.radius), a.radius) + a.radius], 0), a.n_buckets - 1);
    return load_as_float(a.table, a.table_dtype, (int64_t)n * a.H + h) * kLog2e;
  };
  float past = a.table ? bias_at(a.radius) : 0.f;

  // Nearest and furthest row of the tile, and whether one sees nothing.
  int near = t >= 0 ? place : INT_MAX, far = t >= 0 ? place : -1;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    near = min(near, __shfl_xor(near, o));
    far = max(far, __shfl_xor(far, o));
  }
  near = __builtin_amdgcn_readfirstlane(near);
  far = __builtin_amdgcn_readfirstlane(far);
  const bool blind = __ballot(t < 0) != 0;
  // The tile's keys: of a leading prefix those from p0 on, `lead` steps of them (keys -Lp + p0 .. -1), and then those from k0 on.
  // Both begin with the first key that a row sees: rows of the cache before a window may hold anything, and P = 0 times that
  // need not be 0.
  const int end = shared ? a.Lp : __builtin_amdgcn_readfirstlane(min(max(a.lengths[b0], 0), a.L));
  int p0 = 0, k0 = 0, lead = kLead ? a.lead : 0;
  if (a.window && near != INT_MAX) {
    const int key = near - a.window + 1;
    if (kLead && key < 0) {
      p0 = max(0, key + a.Lp);
      lead = (a.Lp - p0 + kStep - 1) / kStep;
    } else {
      lead = 0;
      k0 = max(0, min(key, end));
    }
  }
  const int n_steps = far < 0 ? 0 : lead + (end - k0 + kStep - 1) / kStep;
  const int per_split = (n_steps + splits - 1) / splits;
  const int last = min(n_steps, per_split * (split + 1));
  const int begin = split * per_split + w;  // steps begin, begin + kWaves, ..

  auto at = [&](const void* p, int64_t sb, int64_t sh) { return static_cast<const uint8_t*>(p) + (b0 * sb + hk * sh) * kSize; };
  // Copies of a step's keys and values: rows past the last cached one, and steps past the wave's last, read as zero whatever is
  // there.
  auto issue = [&](int step, lds_u8* to) __attribute__((always_inline)) {
    const bool ahead = kLead && step < lead;
    const Cache& c = shared || ahead ? a.prefix : a.own;
    const int rows = ahead ? a.Lp : end, first = ahead ? p0 + step * kStep : k0 + (step - lead) * kStep;
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const int64_t row_bytes = (m == 0 ? c.k_sl : c.v_sl) * kSize;
      const uint8_t* base = m == 0 ? at(c.k, ahead ? 0 : c.k_sb, c.k_sh) : at(c.v, ahead ? 0 : c.v_sb, c.v_sh);
#pragma unroll
      for (int r16 = 0; r16 < 2; ++r16) {
        const int row0 = first + 16 * r16;
        const int64_t left = step < last && row0 < rows ? (rows - 1 - row0) * row_bytes + 128 : 0;
        const int size = __builtin_amdgcn_readfirstlane((int)min(left, (int64_t)INT_MAX));
        const uint8_t* from = base + row0 * row_bytes;
#pragma unroll
        for (int hf = 0; hf < kParts; ++hf) {
          const __amdgpu_buffer_rsrc_t rsrc =
              __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(from + 128 * hf), (short)0, size, 0x00020000);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int lr = 8 * j + (lane >> 3);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                rsrc, (lds_u8*)(to + (w * 2 + m) * kMat + hf * kStep * 128 + 2048 * r16 + 1024 * j), 16,
                lr * (int)row_bytes + 16 * ((lane & 7) ^ swz(lr)), 0, 0, 0);
          }
        }
      }
    }
  };

  const TileReads<T, kD> reads(lane);
  sa_f32x16 acc[kDC];
#pragma unroll
  for (int dc = 0; dc < kDC; ++dc) acc[dc] = sa_f32x16{};
  float m = -INFINITY, l = 0.f;

  auto compute = [&](int step, const lds_u8* from) __attribute__((always_inline)) {
    const lds_u8* mat = from + w * 2 * kMat;
    const bool ahead = kLead && step < lead;
    const int row0 = ahead ? p0 + step * kStep - a.Lp : k0 + (step - lead) * kStep, limit = ahead ? 0 : end;
    sa_f32x16 S = {};
    sa_u32x4v x[kDS];
#pragma unroll
    for (int s = 0; s < kDS; ++s) x[s] = lds_read_b128(reads.row(mat, s));
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int s = 0; s < kDS; ++s) S = mfma_chunk<T>(x[s], fa[s], S);
    // (the first values are requested before the exponentials)
    typename TileReads<T, kD>::Columns values = reads.columns(mat + kMat, 0);
    __builtin_amdgcn_sched_barrier(0);
    float sc = a.scale_log2;
    if constexpr (kCap) {
      sa_f32x16 none;
      if (std::is_same<T, float>::value || a.cap.fine) bend_all<true, false>(a.cap.in, a.cap.log2, S, none);
      else bend_all<false, false>(a.cap.in, a.cap.log2, S, none);
      sc = 1.f;
    }
    const int base = place - row0 - 4 * hh;  // d = base - c_e
    if (a.table) {
      if (near - row0 - 31 >= a.radius) {
#pragma unroll
        for (int e = 0; e < 16; ++e) S[e] = fmaf(S[e], sc, past);
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) S[e] = fmaf(S[e], sc, bias_at(base - (8 * (e >> 2) + (e & 3))));
      }
      sc = 1.f;
    }
    // Slopes: S becomes S - slope |d| - ref, with ref the row's offset, or what the step's middle key loses where that is less. It
    // goes in before S does: of two large numbers that cancel no bits are lost.
    float ref = 0.f;
    if (a.slopes) {
      ref = fmaxf(m, -slope * fabsf((float)(place - row0 - kStep / 2)));
#pragma unroll
      for (int e = 0; e < 16; ++e)
        S[e] = fmaf(S[e], sc, fmaf(-slope, fabsf((float)(base - (8 * (e >> 2) + (e & 3)))), -ref));
      sc = 1.f;
    }
    if (blind || row0 + 31 > near || row0 + 31 >= limit || (a.window && far - row0 >= a.window)) {
      const unsigned most = a.window ? a.window : 0x80000000u;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int k = 8 * (e >> 2) + (e & 3);
        if (t < 0 || (unsigned)(base - k) >= most || row0 + 4 * hh + k >= limit) S[e] = -INFINITY;
      }
    }
    float top = S[0];
#pragma unroll
    for (int e = 1; e < 16; ++e) top = fmaxf(top, S[e]);
    top = xhalf_max(top) * sc + ref;
    if (__ballot(top > m + kAbove<T>)) {
      const float next_m = fmaxf(m, top - kBelow<T>);
      const float f = next_m == m ? 1.f : fast_exp2(m - next_m);
      m = next_m;
      l *= f;
#pragma unroll
      for (int dc = 0; dc < kDC; ++dc)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[dc][e] *= f;
    }
    const float off = m == -INFINITY ? 0.f : m - ref;
    Weights<T> P;
#pragma unroll
    for (int e = 0; e < 16; e += 2) P.set(e, fast_exp2(fmaf(S[e], sc, -off)), fast_exp2(fmaf(S[e + 1], sc, -off)));
    l = P.sum(l);
    if constexpr (std::is_same<T, float>::value) {
      reads.product(mat + kMat, P, acc);
    } else {
#pragma unroll
      for (int hf = 0; hf < kD / 64; ++hf) {
        const auto now = values;
        if (hf + 1 < kD / 64) values = reads.columns(mat + kMat, hf + 1);
        reads.product(now, hf, P, acc);
      }
    }
  };

  // Both stages' copies are in flight but for the time in which one is computed on: a stage that has been read takes the step
  // after next at once. What the row needs has landed before the first copy is on its way, and there are copies for every
  // stage, past the last step empty ones: the compiler would else wait for all copies in every step.
  lds_u8* const t0 = (lds_u8*)tile0;
  lds_u8* const t1 = (lds_u8*)tile1;
  __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
#pragma unroll
  for (int s = 0; s < kDS; ++s) asm volatile("" : "+v"(fa[s]));
  asm volatile("" : "+v"(slope), "+v"(past));
  issue(begin, t0);
  issue(begin + kWaves, t1);
  for (int s = begin; s < last; s += 2 * kWaves) {
    __builtin_amdgcn_s_waitcnt(waitcnt_vm(8 * kParts));
    compute(s, t0);
    issue(s + 2 * kWaves, t0);
    __builtin_amdgcn_s_waitcnt(waitcnt_vm(8 * kParts));
    if (s + kWaves < last) compute(s + kWaves, t1);
    issue(s + 3 * kWaves, t1);
  }
  __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));

  // ---- The waves' sums: [wave][32 rows][kD] over the stages, 16-byte chunks swizzled by the row.
  l = xhalf_sum(l);
  if (hh == 0) {
    joined[w][0][col] = m;
    joined[w][1][col] = l;
  }
  __syncthreads();  // (every wave is done with its stages, too)
  constexpr int kCh = kD / 4;
  float* mine = reinterpret_cast<float*>(tile0) + w * kStep * kD;
  static_assert(kWaves * kStep * kD * 4 <= kWaves * 2 * kMat, "the sums fit a stage");
#pragma unroll
  for (int dc = 0; dc < kDC; ++dc)
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4)
      *reinterpret_cast<float4*>(mine + col * kD + 4 * ((8 * dc + 2 * q4 + hh) ^ (col & (kCh - 1)))) =
          make_float4(acc[dc][4 * q4], acc[dc][4 * q4 + 1], acc[dc][4 * q4 + 2], acc[dc][4 * q4 + 3]);
  __syncthreads();
  const int group = blockIdx.x;
  for (int at = threadIdx.x; at < kStep * kCh; at += 64 * kWaves) {
    const int rr = at / kCh, ch = at % kCh;
    if (tile * kStep + rr >= n_rows) break;
    float top = joined[0][0][rr];
#pragma unroll
    for (int v = 1; v < kWaves; ++v) top = fmaxf(top, joined[v][0][rr]);
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
#pragma unroll
    for (int v = 0; v < kWaves; ++v) {
      const float mv = joined[v][0][rr], f = mv == top ? 1.f : fast_exp2(mv - top);
      const float4 y = *reinterpret_cast<const float4*>(reinterpret_cast<float*>(tile0) + (v * kStep + rr) * kD +
                                                        4 * (ch ^ (rr & (kCh - 1))));
      s.x = fmaf(y.x, f, s.x);
      s.y = fmaf(y.y, f, s.y);
      s.z = fmaf(y.z, f, s.z);
      s.w = fmaf(y.w, f, s.w);
      sum = fmaf(joined[v][1][rr], f, sum);
    }
    if (a.parts) {
      *reinterpret_cast<float4*>(a.parts + ((int64_t)group * kStep + rr) * kD + 4 * ch) = s;
      if (ch == 0) *reinterpret_cast<float2*>(a.sums + ((int64_t)group * kStep + rr) * 2) = make_float2(top, sum);
      continue;
    }
    const float f = sum == 0.f ? 0.f : 1.f / sum;
    const int in_ = tile * kStep + rr;  // (a row of sequence b0)
    uint8_t* p = static_cast<uint8_t*>(a.out) +
                 (b0 * a.o_sb + (hk * a.rep + in_ / a.Ln) * a.o_sh + (in_ % a.Ln) * a.o_sl) * kSize;
    store_four<T>(p, 4 * ch, s.x * f, s.y * f, s.z * f, s.w * f);
  }
}

// out = the workgroups' sums of each row, those of its own keys and then those of the prefix: a wave per row, whose groups of
// kD / 4 lanes take turns at them. A row without any is zeros.
template <typename T, int kD>
__global__ __launch_bounds__(256) void cached_merge_kernel(CachedArgs a) {
  constexpr int kCh = kD / 4, kGroups = 64 / kCh;
  const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (at >= (int64_t)a.B * a.H * a.Ln) return;  // (the whole wave)
  const int lane = threadIdx.x & 63, ch = lane % kCh, turn = lane / kCh;
  const int i = (int)(at % a.Ln), h = (int)(at / a.Ln % a.H), b = (int)(at / a.Ln / a.H);
  const int hk = h / a.rep, in = (h - hk * a.rep) * a.Ln + i, all = b * a.rep * a.Ln + in;
  // Place of the s-th sums of the row, in units of rows.
  const int n = a.splits + a.prefix_splits;
  const int64_t own = ((int64_t)(b * a.Hk + hk) * a.tiles + in / kStep) * a.splits;
  const int64_t shared = a.own_groups + ((int64_t)hk * a.prefix_tiles + all / kStep) * a.prefix_splits - a.splits;
  auto place = [&](int s) { return s < a.splits ? (own + s) * kStep + in % kStep : (shared + s) * kStep + all % kStep; };
  float top = -INFINITY;
  for (int s = lane; s < n; s += 64) top = fmaxf(top, a.sums[2 * place(s)]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  float r[5] = {};  // the chunk, and the sum
#pragma unroll 4
  for (int s = turn; s < n; s += kGroups) {
    const int64_t p = place(s);
    const float2 x = *reinterpret_cast<const float2*>(a.sums + 2 * p);
    const float f = x.x == top ? 1.f : fast_exp2(x.x - top);
    const float4 y = *reinterpret_cast<const float4*>(a.parts + p * kD + 4 * ch);
    r[0] = fmaf(y.x, f, r[0]);
    r[1] = fmaf(y.y, f, r[1]);
    r[2] = fmaf(y.z, f, r[2]);
    r[3] = fmaf(y.w, f, r[3]);
    r[4] = fmaf(x.y, f, r[4]);
  }
#pragma unroll
  for (int o = kCh; o < 64; o <<= 1)
#pragma unroll
    for (int x = 0; x < 5; ++x) r[x] += __shfl_xor(r[x], o);
  if (turn > 0) return;
  const float f = r[4] == 0.f ? 0.f : 1.f / r[4];
  store_four<T>(static_cast<uint8_t*>(a.out) + (b * a.o_sb + h * a.o_sh + i * a.o_sl) * (int64_t)sizeof(T), 4 * ch, r[0] * f,
                r[1] * f, r[2] * f, r[3] * f);
}

// ---- Host side.

constexpr int kLeastSteps = 8;   // of a workgroup, before the keys are split further
constexpr int kWholeSteps = 32;  // up to so many a workgroup takes them all: 526 keys 8.9 us in one launch, not 6.9 + 3.9 in two
// Workgroups that a call aims at, by the bytes of a row: twice as many as the 256 CUs' LDS holds at once, so that one's first
// copies and its join run beside another's steps. 32 sequences of up to 1350 own keys behind 17776 shared ones, D 64: 58 us, of
// as many as it holds 71, of four times as many 63; 4 sequences of up to 45104 keys, D 128: 117 us, of four times as many 125.
inline int target_groups(int row) { return 512 * (row <= 128 ? 2 : 1); }

struct CachedPlan {
  int tiles, splits, prefix_tiles, prefix_splits, lead;
  int64_t own_groups, groups, sums, bytes;
};

int plan_cached(const sa_attn_cached& t, const char* fn, CachedPlan& p) {
  const int64_t per = (int64_t)(t.H / t.Hk) * t.Ln;
  const int64_t tiles = (per + kStep - 1) / kStep, prefix_tiles = t.Lp ? (t.B * per + kStep - 1) / kStep : 0;
  const int64_t items = (int64_t)t.B * t.Hk * tiles, prefix_items = t.Hk * prefix_tiles;
  if (t.B * per >= 1LL << 30 || items + prefix_items >= 1LL << 20)
    return sa::fail(SA_ERR_UNSUPPORTED, "%s: too many rows", fn);
  // Splits in proportion to the keys, so that workgroups have alike many of them, about `target` in all.
  const int target = target_groups(t.D * (t.dtype == SA_DTYPE_F32 ? 4 : 2));
  const int64_t steps = (t.L + kStep - 1) / kStep, prefix_steps = t.Lp ? (t.Lp + kStep - 1) / kStep : 0;
  const int64_t all = items * steps + prefix_items * prefix_steps;
  const int64_t each = std::max<int64_t>(kLeastSteps, (all + target - 1) / target);
  p.tiles = (int)tiles;
  // A short prefix is read by each sequence for itself, ahead of its own keys, where the card holds all workgroups at once: the
  // prefix comes out of the L2 then, and there are no sums to join (4 answers of up to 77 tokens to a caption of 226: 15 us in
  // two launches, 11 in one).
  const bool whole = steps + prefix_steps <= kWholeSteps && (!t.Lp || items <= target / 2);
  p.lead = whole ? (int)prefix_steps : 0;
  p.prefix_tiles = whole ? 0 : (int)prefix_tiles;
  p.splits = whole ? 1 : (int)std::max<int64_t>(1, (steps + each - 1) / each);
  p.prefix_splits = whole || !t.Lp ? 0 : (int)std::max<int64_t>(1, (prefix_steps + each - 1) / each);
  p.own_groups = items * p.splits;
  p.groups = p.own_groups + (int64_t)t.Hk * p.prefix_tiles * p.prefix_splits;
  const bool merged = p.splits > 1 || p.prefix_splits > 0;
  p.sums = (p.groups * kStep * 8 + 255) / 256 * 256;
  p.bytes = merged ? p.sums + p.groups * kStep * t.D * 4 : 0;
  return SA_OK;
}

int check_cached(const sa_attn_cached* t, const char* fn) {
  SA_REQUIRE(t, "%s: null call", fn);
  SA_REQUIRE(t->dtype >= SA_DTYPE_BF16 && t->dtype <= SA_DTYPE_F32, "%s: dtype %d", fn, t->dtype);
  SA_REQUIRE(t->B > 0 && t->H > 0 && t->Hk > 0 && t->Ln > 0 && t->L > 0 && t->Lp >= 0,
             "%s: bad shape B=%d H=%d Hk=%d Ln=%d L=%d Lp=%d", fn, t->B, t->H, t->Hk, t->Ln, t->L, t->Lp);
  SA_REQUIRE(t->H % t->Hk == 0, "%s: %d query heads over %d key heads", fn, t->H, t->Hk);
  SA_REQUIRE(t->window >= 0, "%s: window %d", fn, t->window);
  if (t->D != 64 && t->D != 128) return sa::fail(SA_ERR_UNSUPPORTED, "%s: head_dim %d (64 or 128)", fn, t->D);
  if (t->L > 1 << 29 || t->Lp > 1 << 29) return sa::fail(SA_ERR_UNSUPPORTED, "%s: more than 2^29 keys", fn);
  SA_REQUIRE(t->sm_scale > 0.f && std::isfinite(t->sm_scale), "%s: sm_scale must be positive and finite", fn);
  SA_REQUIRE(t->cap >= 0.f && std::isfinite(t->cap), "%s: cap must be positive and finite, or 0 for none", fn);
  SA_REQUIRE(cap_in_range(t->sm_scale, t->cap), "%s: cap or sm_scale / cap out of range", fn);
  if (t->table) {
    SA_REQUIRE(t->buckets && t->n_buckets > 0, "%s: table without buckets", fn);
    SA_REQUIRE(t->table_dtype >= SA_DTYPE_BF16 && t->table_dtype <= SA_DTYPE_F32, "%s: table dtype %d", fn, t->table_dtype);
    if (t->radius < 0 || t->radius > kMostRadius)
      return sa::fail(SA_ERR_UNSUPPORTED, "%s: distances up to %d told apart (at most %d)", fn, t->radius, kMostRadius);
  }
  return SA_OK;
}

template <bool kCap, typename T, int kD>
void launch_cached(const CachedArgs& a, const CachedPlan& p, hipStream_t s) {
  const dim3 grid((unsigned)p.groups), group(64 * CachedShape<T, kD>::kWaves);
  if (p.lead) hipLaunchKernelGGL((cached_kernel<true, kCap, T, kD>), grid, group, 0, s, a);
  else hipLaunchKernelGGL((cached_kernel<false, kCap, T, kD>), grid, group, 0, s, a);
  if (!p.bytes) return;
  const int64_t rows = (int64_t)a.B * a.H * a.Ln;
  hipLaunchKernelGGL((cached_merge_kernel<T, kD>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, a);
}

template <typename T>
void launch_type(const CachedArgs& a, const CachedPlan& p, int D, bool cap, hipStream_t s) {
  if (D == 64 && cap) launch_cached<true, T, 64>(a, p, s);
  else if (D == 64) launch_cached<false, T, 64>(a, p, s);
  else if (cap) launch_cached<true, T, 128>(a, p, s);
  else launch_cached<false, T, 128>(a, p, s);
}

}  // namespace

extern "C" int sa_attn_cached_workspace(const sa_attn_cached* t, int64_t* bytes) {
  const char* fn = "sa_attn_cached_workspace";
  SA_REQUIRE(bytes, "%s: null bytes", fn);
  if (int rc = check_cached(t, fn)) return rc;
  CachedPlan p;
  if (int rc = plan_cached(*t, fn, p)) return rc;
  *bytes = p.bytes;
  return sa::ok();
}

extern "C" int sa_attn_cached_fwd(const sa_attn_cached* t, void* stream) {
  const char* fn = "sa_attn_cached_fwd";
  if (int rc = check_cached(t, fn)) return rc;
  SA_REQUIRE(t->q && t->k && t->v && t->out && t->lengths && (!t->Lp || (t->prefix_k && t->prefix_v)), "%s: null pointer", fn);
  CachedPlan p;
  if (int rc = plan_cached(*t, fn, p)) return rc;
  const int size = t->dtype == SA_DTYPE_F32 ? 4 : 2, per16 = 16 / size;
  const void* ptrs[6] = {t->q, t->out, t->k, t->v, t->prefix_k, t->prefix_v};
  for (int i = 0; i < (t->Lp ? 6 : 4); ++i) {
    if (reinterpret_cast<uintptr_t>(ptrs[i]) % 16 != 0)
      return sa::fail(SA_ERR_UNSUPPORTED, "%s: tensor base not 16-byte aligned", fn);
    for (int j = 0; j < 3; ++j)
      if (t->strides[3 * i + j] % per16 != 0)
        return sa::fail(SA_ERR_UNSUPPORTED, "%s: strides must be multiples of %d elements", fn, per16);
    // (a step's rows are reached through 32-bit offsets)
    if (t->strides[3 * i + 2] < 0 || t->strides[3 * i + 2] > 1 << 24)
      return sa::fail(SA_ERR_UNSUPPORTED, "%s: rows more than 2^24 elements apart", fn);
  }
  SA_REQUIRE(!p.bytes || (t->workspace && reinterpret_cast<uintptr_t>(t->workspace) % 256 == 0),
             "%s: workspace null or not 256-byte aligned", fn);
  SA_REQUIRE(t->workspace_bytes >= p.bytes, "%s: workspace of %lld bytes < %lld", fn, (long long)t->workspace_bytes,
             (long long)p.bytes);
  CachedArgs a{};
  const int64_t* st = t->strides;
  a.q = t->q; a.q_sb = st[0]; a.q_sh = st[1]; a.q_sl = st[2];
  a.out = t->out; a.o_sb = st[3]; a.o_sh = st[4]; a.o_sl = st[5];
  a.own = Cache{t->k, t->v, st[6], st[7], st[8], st[9], st[10], st[11]};
  a.prefix = Cache{t->prefix_k, t->prefix_v, st[12], st[13], st[14], st[15], st[16], st[17]};
  a.lengths = t->lengths;
  a.B = t->B; a.H = t->H; a.Hk = t->Hk; a.rep = t->H / t->Hk;
  a.Ln = t->Ln; a.L = t->L; a.Lp = t->Lp; a.window = t->window;
  a.tiles = p.tiles; a.splits = p.splits;
  a.prefix_tiles = p.prefix_tiles; a.prefix_splits = p.prefix_splits;
  a.own_groups = (int)p.own_groups; a.lead = p.lead;
  a.scale_log2 = t->sm_scale * kLog2e;
  a.cap = cap_of(t->sm_scale, t->cap, t->dtype);
  a.slopes = t->slopes;
  a.table = t->table; a.buckets = t->buckets;
  a.table_dtype = t->table_dtype; a.n_buckets = t->n_buckets; a.radius = t->radius;
  if (p.bytes) {
    a.sums = static_cast<float*>(t->workspace);
    a.parts = reinterpret_cast<float*>(static_cast<uint8_t*>(t->workspace) + p.sums);
  }
  hipStream_t s = sa::as_stream(stream);
  if (t->dtype == SA_DTYPE_BF16) launch_type<__bf16>(a, p, t->D, t->cap > 0, s);
  else if (t->dtype == SA_DTYPE_F16) launch_type<_Float16>(a, p, t->D, t->cap > 0, s);
  else launch_type<float>(a, p, t->D, t->cap > 0, s);
  return sa::check_launch(fn);
}
