// Rotary positions of queries and keys: pairs of a head's values turned by an angle per token.
//
//   angle[token][pair] = position[axis of pair][token] * frequency[pair]
//   (a, b) -> (a cos - b sin, b cos + a sin), and with -sin for the gradient (the transpose)
//
// The table kernel forms the angles in 64 bits, as turns, so that far positions keep their fraction, and
// takes the quarter turn off before the 32-bit sine and cosine. It is bound by arithmetic until the table
// outgrows the caches: 45 104 tokens of 64 pairs take 8.3 us (2.8 TB/s written; 10.1 with sincospif, 11.6
// with one token a thread as well), 1 350 of 32 pairs 2.4, which an empty launch takes too.
//
// The rotation is bound by memory: each value is read and written once, and a thread keeps its pairs'
// cosines and sines while it goes through the heads.
#include <math.h>

#include <algorithm>
#include <climits>
#include <cmath>

#include "sa_common.h"

namespace {

constexpr int kMaxAxes = 4;
constexpr int kMaxPairs = 128;
constexpr double kTurn = 6.283185307179586476925287;

struct TableArgs {
  const void* positions;
  int64_t stride_axis, stride_token;
  int64_t L;
  int pairs;
  int tokens, steps;  // of a workgroup: tokens at once, and how often
  int axis_end[kMaxAxes];  // pairs of the axes up to this one
  float factor[kMaxAxes];  // of the axis's cosines and sines
  double turns[kMaxPairs];  // turns per position
  float2* table;
};

// A thread keeps its pair and takes `steps` tokens, so that the axis and the frequency are found once.
template <typename P>
__global__ __launch_bounds__(256) void rotary_table_kernel(TableArgs a) {
  const int slot = threadIdx.x / (unsigned)a.pairs;
  const int pair = threadIdx.x - slot * a.pairs;
  if (slot >= a.tokens) return;
  int axis = 0;
  while (pair >= a.axis_end[axis]) ++axis;  // (axis_end of the last axis is the number of pairs)
  const double turns = a.turns[pair];
  const float m = a.factor[axis];
  const P* positions = static_cast<const P*>(a.positions) + axis * a.stride_axis;
  int64_t token = (int64_t)blockIdx.x * a.tokens * a.steps + slot;
  for (int i = 0; i < a.steps && token < a.L; ++i, token += a.tokens) {
    const double t = (double)positions[token * a.stride_token] * turns;
    const double r = t - rint(t);  // exact
    const double quarter = rint(4.0 * r);
    const float y = (float)((r - 0.25 * quarter) * kTurn);  // |y| <= pi / 4
    const float z = y * y;
    // Their power series, up to y^9 and y^10 (what is left out is below 2.5e-9 of the value).
    const float s = fmaf(y * z, fmaf(z, fmaf(z, fmaf(z, 1.f / 362880, -1.f / 5040), 1.f / 120), -1.f / 6), y);
    const float c = fmaf(z, fmaf(z, fmaf(z, fmaf(z, fmaf(z, -1.f / 3628800, 1.f / 40320), -1.f / 720), 1.f / 24), -0.5f), 1.f);
    const int q = (int)quarter & 3;  // (an infinite or NaN position gives NaN either way)
    const float sn = (q & 1) ? c : s, cs = (q & 1) ? s : c;
    a.table[token * a.pairs + pair] = make_float2((q == 1 || q == 2) ? -cs * m : cs * m, (q & 2) ? -sn * m : sn * m);
  }
}

// ---- rotation -----------------------------------------------------------------------------------

struct RotArgs {
  const void* x[2];  // q, k
  void* y[2];
  int64_t xs[2][3], ys[2][3];  // strides of b, h, l
  int heads[2];
  int B, L, D;
  const float2* table;
  int n_rows, pairs;
  const int32_t* rows;  // nullable: table row of token (b, t) at rows[b * rows_sb + t]
  int64_t rows_sb;
  int skip;             // without rows: token t has row t - skip
  float sign;           // of the sines
  int copy;             // values that do not turn are copied (0: in place, they are left)
  int units, tokens, slots;  // threads: unit + units * (token + tokens * head slot)
  int group;            // heads per workgroup (of q's and k's together)
};

// N consecutive values of a head, moved together (16 bytes at most at a time).
template <typename T, int N>
struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) Chunk {
  T v[N];
};

typedef uint32_t Words __attribute__((ext_vector_type(4)));

// A thread turns one unit of one token in every head of its group. Interleaved: V consecutive values
// (V / 2 pairs, those past the last one left alone). Halves: V values of each half (V pairs); units past
// the turned part copy 2 V values, in the same two accesses, so that the lanes of a wave stay together.
// Loads of kUnroll heads are in flight together.
//
// V values are 16 bytes, or fewer where the halves are no multiples of that (fp32 in 32 bytes, two accesses that leave
// every second 16 to each other: [1, 15 + 5, 8229, 128], 96 of 128 values, halves 42 us, in 16 bytes 35).
//
// kStream (a template argument: the choice beside the stores costs 4 %): a run of such stores fills whole lines (128
// bytes: the row, or its half), so that they need not wait in a cache for the rest and are streamed out. Other tensors
// each time, ordinary / streamed, us: bf16 interleaved [2, 30 + 30, 17776, 64] 105 / 98 (5.6 TB/s), fp16 halves [1, 16 +
// 4, 20000, 128] 48 / 41, fp32 [2, 24 + 8, 8000, 64] interleaved 50 / 47 and halves 51 / 47 (5.6 TB/s); halves of 64
// bytes, [2, 30 + 30, 17776, 64] in bf16, 107 / 109.
template <typename T, bool kHalf, int V, bool kStream>
__global__ __launch_bounds__(256) void rotary_kernel(RotArgs a) {
  constexpr int kUnroll = 4;
  constexpr int kPairs = kHalf ? V : V / 2;
  constexpr int kChunks = kHalf ? 2 : 1;
  const int unit = threadIdx.x % a.units;
  const int rest = threadIdx.x / a.units;
  const int slot = rest / a.tokens;
  const int token_groups = (a.L + a.tokens - 1) / a.tokens;
  const int b = blockIdx.x / token_groups;
  const int t = (blockIdx.x - b * token_groups) * a.tokens + (rest - slot * a.tokens);
  if (slot >= a.slots || t >= a.L) return;
  const int row = a.rows ? a.rows[b * a.rows_sb + t] : t - a.skip;
  const int turned = (a.pairs + kPairs - 1) / kPairs;  // units that turn (halves: whole ones)
  const bool turn = unit < turned && (unsigned)row < (unsigned)a.n_rows;
  if (!turn && !a.copy) return;
  float c[kPairs], s[kPairs];
  if (turn) {
    const float2* p = a.table + (int64_t)row * a.pairs + kPairs * unit;
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const bool ok = kHalf || kPairs * unit + i < a.pairs;
      const float2 x = ok ? p[i] : make_float2(1.f, 0.f);
      c[i] = x.x;
      s[i] = x.y * a.sign;
    }
  }
  const int n_heads = a.heads[0] + a.heads[1];
  const int end = min(n_heads, (int)(blockIdx.y + 1) * a.group);
  auto from = [&](int h) {
    const int w = h >= a.heads[0];
    return static_cast<const T*>(w ? a.x[1] : a.x[0]) + b * (w ? a.xs[1][0] : a.xs[0][0]) +
           (h - (w ? a.heads[0] : 0)) * (w ? a.xs[1][1] : a.xs[0][1]) + t * (w ? a.xs[1][2] : a.xs[0][2]);
  };
  auto to = [&](int h) {
    const int w = h >= a.heads[0];
    return static_cast<T*>(w ? a.y[1] : a.y[0]) + b * (w ? a.ys[1][0] : a.ys[0][0]) +
           (h - (w ? a.heads[0] : 0)) * (w ? a.ys[1][1] : a.ys[0][1]) + t * (w ? a.ys[1][2] : a.ys[0][2]);
  };
  const int at0 = kHalf && unit >= turned ? 2 * a.pairs + 2 * V * (unit - turned) : V * unit;
  const int at1 = kHalf && unit < turned ? a.pairs + V * unit : at0 + V;
  for (int h0 = blockIdx.y * a.group + slot; h0 < end; h0 += kUnroll * a.slots) {
    Chunk<T, V> x[kUnroll][kChunks];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (h0 + u * a.slots < end) {
        const T* p = from(h0 + u * a.slots);
        x[u][0] = *reinterpret_cast<const Chunk<T, V>*>(p + at0);
        if constexpr (kHalf) x[u][1] = *reinterpret_cast<const Chunk<T, V>*>(p + at1);
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (h0 + u * a.slots < end) {
        if (turn) {  // (a token without a position keeps its bits, as do values past the last pair)
#pragma unroll
          for (int i = 0; i < kPairs; ++i) {
            T& xa = kHalf ? x[u][0].v[i] : x[u][0].v[2 * i & (V - 1)];
            T& xb = kHalf ? x[u][kChunks - 1].v[i] : x[u][0].v[(2 * i + 1) & (V - 1)];
            const float va = (float)xa, vb = (float)xb;
            if (kHalf || kPairs * unit + i < a.pairs) {
              xa = (T)fmaf(va, c[i], -(vb * s[i]));
              xb = (T)fmaf(vb, c[i], va * s[i]);
            }
          }
        }
        T* p = to(h0 + u * a.slots);
        if constexpr (kStream) {
          __builtin_nontemporal_store(__builtin_bit_cast(Words, x[u][0]), reinterpret_cast<Words*>(p + at0));
          if constexpr (kHalf)
            __builtin_nontemporal_store(__builtin_bit_cast(Words, x[u][kChunks - 1]), reinterpret_cast<Words*>(p + at1));
        } else {
          *reinterpret_cast<Chunk<T, V>*>(p + at0) = x[u][0];
          if constexpr (kHalf) *reinterpret_cast<Chunk<T, V>*>(p + at1) = x[u][1];
        }
      }
    }
  }
}

// Any head dim, number of pairs, strides and alignment: a unit is one pair, then one value each.
template <typename T, bool kHalf>
__global__ __launch_bounds__(256) void rotary_any_kernel(RotArgs a) {
  const int unit = threadIdx.x % a.units;
  const int rest = threadIdx.x / a.units;
  const int slot = rest / a.tokens;
  const int token_groups = (a.L + a.tokens - 1) / a.tokens;
  const int b = blockIdx.x / token_groups;
  const int t = (blockIdx.x - b * token_groups) * a.tokens + (rest - slot * a.tokens);
  if (slot >= a.slots || t >= a.L) return;
  const int row = a.rows ? a.rows[b * a.rows_sb + t] : t - a.skip;
  const bool pair = unit < a.pairs;
  const bool turn = pair && (unsigned)row < (unsigned)a.n_rows;
  if (!turn && !a.copy) return;
  float2 cs = make_float2(1.f, 0.f);
  if (turn) cs = a.table[(int64_t)row * a.pairs + unit];
  cs.y *= a.sign;
  const int at0 = !pair ? unit + a.pairs : kHalf ? unit : 2 * unit;
  const int at1 = !pair ? at0 : kHalf ? unit + a.pairs : 2 * unit + 1;
  const int n_heads = a.heads[0] + a.heads[1];
  const int end = min(n_heads, (int)(blockIdx.y + 1) * a.group);
  for (int h = blockIdx.y * a.group + slot; h < end; h += a.slots) {
    const int w = h >= a.heads[0], hw = h - (w ? a.heads[0] : 0);
    const T* p = static_cast<const T*>(a.x[w]) + b * a.xs[w][0] + hw * a.xs[w][1] + t * a.xs[w][2];
    T* o = static_cast<T*>(a.y[w]) + b * a.ys[w][0] + hw * a.ys[w][1] + t * a.ys[w][2];
    const T va = p[at0], vb = p[at1];
    o[at0] = turn ? (T)fmaf((float)va, cs.x, -((float)vb * cs.y)) : va;
    if (pair) o[at1] = turn ? (T)fmaf((float)vb, cs.x, (float)va * cs.y) : vb;
  }
}

// Values that a thread moves together: 16 bytes, or fewer in halves that are no multiples of them (whole units have
// to fill the half and the rest of the head, and the rows have to be aligned to them); 1 for anything else.
int width_of(const RotArgs& a, bool half, int size) {
  int64_t strides = a.D;
  uint64_t ptrs = 0;
  for (int w = 0; w < (a.heads[1] ? 2 : 1); ++w) {
    for (int i = 0; i < 3; ++i) strides |= a.xs[w][i] | a.ys[w][i];
    ptrs |= reinterpret_cast<uintptr_t>(a.x[w]) | reinterpret_cast<uintptr_t>(a.y[w]);
  }
  for (int v = 16 / size; v >= (half ? 2 : 16 / size); v /= 2) {
    if (half && (a.pairs % v || (a.D - 2 * a.pairs) % (2 * v))) continue;
    if (strides % v == 0 && ptrs % std::min(16, v * size) == 0) return v;
  }
  return 1;
}

template <typename T>
int launch_rotary(RotArgs a, bool half, hipStream_t s, const char* fn) {
  constexpr int kWide = 16 / sizeof(T);
  const int v = width_of(a, half, sizeof(T));
  const bool stream = (half ? a.pairs : a.D) * sizeof(T) >= 128;
  // units per token, then as many tokens (a power of two up to the length) and head slots as fit 256 threads
  a.units = v == 1 ? a.D - a.pairs : half ? a.D / (2 * v) : a.D / v;
  const int room = 256 / a.units;
  a.tokens = 1;
  while (2 * a.tokens <= room && a.tokens < a.L) a.tokens *= 2;
  a.slots = room / a.tokens;
  const int n_heads = a.heads[0] + a.heads[1];
  const int64_t wgs = (int64_t)a.B * ((a.L + a.tokens - 1) / a.tokens);
  SA_REQUIRE(wgs < (1LL << 31), "%s: grid too large", fn);
  // A group of heads shares the table's values; groups as large as leave some 4 096 workgroups (8 192: 92 -> 90 us at
  // [2, 30, 17776, 64], but 9.3 -> 11.6 at 1 576 tokens), of at most 16 heads a slot (2 x 48 heads of 45 104 tokens: 222 us
  // in groups of 48, 206 in groups of 16).
  const int64_t want = std::max<int64_t>(1, std::min<int64_t>(n_heads, 4096 / wgs));
  a.group = std::min((int)((n_heads + want - 1) / want), 16 * a.slots);
  a.group = std::max(a.group, std::min(n_heads, a.slots));
  const dim3 grid((unsigned)wgs, (unsigned)((n_heads + a.group - 1) / a.group)), blk(256);
  if (v == 1) {
    if (half) hipLaunchKernelGGL((rotary_any_kernel<T, true>), grid, blk, 0, s, a);
    else hipLaunchKernelGGL((rotary_any_kernel<T, false>), grid, blk, 0, s, a);
  } else if (!half) {
    if (stream) hipLaunchKernelGGL((rotary_kernel<T, false, kWide, true>), grid, blk, 0, s, a);
    else hipLaunchKernelGGL((rotary_kernel<T, false, kWide, false>), grid, blk, 0, s, a);
  } else if (v == kWide) {
    if (stream) hipLaunchKernelGGL((rotary_kernel<T, true, kWide, true>), grid, blk, 0, s, a);
    else hipLaunchKernelGGL((rotary_kernel<T, true, kWide, false>), grid, blk, 0, s, a);
  } else if (v == 4) {
    if constexpr (kWide > 4) hipLaunchKernelGGL((rotary_kernel<T, true, 4, false>), grid, blk, 0, s, a);
  } else {
    hipLaunchKernelGGL((rotary_kernel<T, true, 2, false>), grid, blk, 0, s, a);
  }
  return sa::check_launch(fn);
}

}  // namespace

extern "C" int sa_rotary_table(const void* positions, int position_type, const int64_t strides[2], int64_t L, int n_axes,
                               const int32_t* axis_pairs, const double* frequencies, const double* factors,
                               float* table, void* stream) {
  const char* fn = "sa_rotary_table";
  SA_REQUIRE(positions && strides && axis_pairs && frequencies && factors && table, "%s: null pointer", fn);
  SA_REQUIRE(L > 0 && L < (1LL << 31), "%s: L=%lld", fn, (long long)L);
  SA_REQUIRE(n_axes >= 1 && n_axes <= kMaxAxes, "%s: %d axes (1 to %d)", fn, n_axes, kMaxAxes);
  SA_REQUIRE(reinterpret_cast<uintptr_t>(table) % 8 == 0, "%s: table not 8-byte aligned", fn);
  TableArgs a;
  a.positions = positions;
  a.stride_axis = strides[0];
  a.stride_token = strides[1];
  a.pairs = 0;
  for (int i = 0; i < n_axes; ++i) {
    SA_REQUIRE(axis_pairs[i] > 0 && axis_pairs[i] <= kMaxPairs - a.pairs, "%s: axes of more than %d pairs", fn, kMaxPairs);
    a.pairs += axis_pairs[i];
    a.axis_end[i] = a.pairs;
    SA_REQUIRE(std::isfinite(factors[i]), "%s: factor %d is not finite", fn, i);
    a.factor[i] = (float)factors[i];
  }
  for (int i = 0; i < a.pairs; ++i) {
    SA_REQUIRE(std::isfinite(frequencies[i]), "%s: frequency %d is not finite", fn, i);
    a.turns[i] = frequencies[i] / kTurn;
  }
  a.L = L;
  a.table = reinterpret_cast<float2*>(table);
  a.tokens = 256 / a.pairs;
  // As many steps as leave some 1 024 workgroups (45 104 tokens of 64 pairs: 12.8 us in one, 10.1 in four and more; 1 350
  // of 32: 2.4 and 3.2).
  a.steps = (int)std::min<int64_t>(8, std::max<int64_t>(1, L / ((int64_t)a.tokens * 1024)));
  const int64_t wgs = (L + (int64_t)a.tokens * a.steps - 1) / ((int64_t)a.tokens * a.steps);
  SA_REQUIRE(wgs < (1LL << 31), "%s: grid too large", fn);
  const dim3 grid((unsigned)wgs), blk(256);
  hipStream_t s = sa::as_stream(stream);
  if (position_type == SA_POSITION_I32) hipLaunchKernelGGL(rotary_table_kernel<int32_t>, grid, blk, 0, s, a);
  else if (position_type == SA_POSITION_I64) hipLaunchKernelGGL(rotary_table_kernel<int64_t>, grid, blk, 0, s, a);
  else if (position_type == SA_POSITION_F32) hipLaunchKernelGGL(rotary_table_kernel<float>, grid, blk, 0, s, a);
  else if (position_type == SA_POSITION_F64) hipLaunchKernelGGL(rotary_table_kernel<double>, grid, blk, 0, s, a);
  else return sa::fail(SA_ERR_INVALID, "%s: position type %d", fn, position_type);
  return sa::check_launch(fn);
}

extern "C" int sa_rotary_apply(int dtype, const void* q, void* q_out, const void* k, void* k_out,
                               const int64_t strides[12], int B, int H, int Hk, int L, int D, const float* table,
                               int n_rows, int pairs, const int32_t* rows, int64_t rows_batch_stride, int skip,
                               int halves, int inverse, void* stream) {
  const char* fn = "sa_rotary_apply";
  SA_REQUIRE(dtype == SA_DTYPE_BF16 || dtype == SA_DTYPE_F16 || dtype == SA_DTYPE_F32, "%s: dtype %d", fn, dtype);
  SA_REQUIRE(q && q_out && strides && table, "%s: null pointer", fn);
  SA_REQUIRE(!k == !k_out, "%s: k without its output", fn);
  SA_REQUIRE(B > 0 && H > 0 && (!k || Hk > 0) && L > 0 && D > 0, "%s: bad shape B=%d H=%d Hk=%d L=%d D=%d", fn, B, H, Hk,
             L, D);
  SA_REQUIRE(L <= INT_MAX - 255, "%s: L=%d", fn, L);  // (rounded up to a workgroup's tokens)
  SA_REQUIRE(D <= 2 * kMaxPairs, "%s: head dim %d (at most %d)", fn, D, 2 * kMaxPairs);
  SA_REQUIRE(n_rows > 0 && pairs > 0 && 2 * pairs <= D, "%s: a table of %d rows of %d pairs for head dim %d", fn, n_rows,
             pairs, D);
  SA_REQUIRE(skip >= 0 && skip <= L, "%s: skip=%d of %d tokens", fn, skip, L);
  SA_REQUIRE(rows ? skip == 0 : L - skip <= n_rows, "%s: %d tokens after %d for %d table rows", fn, L - skip, skip, n_rows);
  SA_REQUIRE(H + (int64_t)(k ? Hk : 0) < 65536, "%s: too many heads", fn);
  SA_REQUIRE(reinterpret_cast<uintptr_t>(table) % 8 == 0, "%s: table not 8-byte aligned", fn);
  RotArgs a;
  a.x[0] = q; a.y[0] = q_out;
  a.x[1] = k; a.y[1] = k_out;
  a.heads[0] = H;
  a.heads[1] = k ? Hk : 0;
  for (int w = 0; w < 2; ++w)
    for (int i = 0; i < 3; ++i) {
      a.xs[w][i] = k || w == 0 ? strides[6 * w + i] : 0;
      a.ys[w][i] = k || w == 0 ? strides[6 * w + 3 + i] : 0;
    }
  a.B = B; a.L = L; a.D = D;
  a.table = reinterpret_cast<const float2*>(table);
  a.n_rows = n_rows;
  a.pairs = pairs;
  a.rows = rows;
  a.rows_sb = rows_batch_stride;
  a.skip = skip;
  a.sign = inverse ? -1.f : 1.f;
  // Each thread reads its values before it writes them, so that out may be the input itself.
  a.copy = !(q == q_out && (!k || k == k_out));
  hipStream_t s = sa::as_stream(stream);
  if (dtype == SA_DTYPE_F32) return launch_rotary<float>(a, halves != 0, s, fn);
  if (dtype == SA_DTYPE_F16) return launch_rotary<_Float16>(a, halves != 0, s, fn);
  return launch_rotary<__bf16>(a, halves != 0, s, fn);
}
