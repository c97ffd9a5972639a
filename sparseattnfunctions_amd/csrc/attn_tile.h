// Pieces shared by the 16-bit attention kernels (attn_fwd.hip, attn_bwd.hip): operand types and
// their MFMA, LDS tile copies, operand reads and explicit waits. Tiles are rows of 128 bytes (64
// 16-bit values; a 128-dim row is two of them) in 16-byte chunks, XOR-swizzled by the row.
#pragma once

#include "sa_common.h"

namespace {

constexpr float kLog2e = 1.4426950408889634f;

typedef __attribute__((address_space(3))) uint8_t lds_u8;
typedef short sa_i16x4v __attribute__((ext_vector_type(4)));
typedef unsigned sa_u32x4v __attribute__((ext_vector_type(4)));
__device__ inline sa_bf16x8 as_bf16x8(uint4 x) { return __builtin_bit_cast(sa_bf16x8, x); }
__device__ inline sa_bf16x8 as_bf16x8(sa_u32x4v x) { return __builtin_bit_cast(sa_bf16x8, x); }

__device__ inline sa_f32x16 mfma32(sa_bf16x8 a, sa_bf16x8 b, sa_f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

__device__ inline float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

typedef __bf16 sa_bf16x2 __attribute__((ext_vector_type(2)));

// Two fp32 -> packed bf16 pair (round to nearest even, v_cvt_pk_bf16_f32).
__device__ inline uint32_t cvt_pk_bf16(float a, float b) {
  sa_bf16x2 r = {(__bf16)a, (__bf16)b};
  return __builtin_bit_cast(uint32_t, r);
}

// The three bf16 terms of x0 and x1, packed: each remainder is exact in fp32, and the last one
// has at most 8 significand bits, so hi + mid + lo = x (above bf16's subnormals).
__device__ inline void split3(float x0, float x1, uint32_t& hi, uint32_t& mid, uint32_t& lo) {
  hi = cvt_pk_bf16(x0, x1);
  const float a0 = x0 - __uint_as_float(hi << 16), a1 = x1 - __uint_as_float(hi & 0xffff0000u);
  mid = cvt_pk_bf16(a0, a1);
  lo = cvt_pk_bf16(a0 - __uint_as_float(mid << 16), a1 - __uint_as_float(mid & 0xffff0000u));
}

__device__ inline float dot2_bf16_ones(uint32_t pair, float acc) {
  const sa_bf16x2 ones = {(__bf16)1.0f, (__bf16)1.0f};
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(sa_bf16x2, pair), ones, acc, false);
}

typedef _Float16 sa_f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 sa_f16x8 __attribute__((ext_vector_type(8)));

// Operand element type of a launch: the MFMA, the rounding of P (and of the output) to the
// element type (round to nearest even), and the row-sum dot of a packed pair with ones.
template <typename T>
struct Elem;
template <>
struct Elem<__bf16> {
  typedef sa_bf16x8 v8;
  __device__ static inline v8 as8(sa_u32x4v x) { return as_bf16x8(x); }
  __device__ static inline sa_f32x16 mfma(v8 a, v8 b, sa_f32x16 c) { return mfma32(a, b, c); }
  __device__ static inline uint32_t pack(float a, float b) { return cvt_pk_bf16(a, b); }
  __device__ static inline float dot2_ones(uint32_t pair, float acc) { return dot2_bf16_ones(pair, acc); }
};
template <>
struct Elem<_Float16> {
  typedef sa_f16x8 v8;
  __device__ static inline v8 as8(sa_u32x4v x) { return __builtin_bit_cast(sa_f16x8, x); }
  __device__ static inline sa_f32x16 mfma(v8 a, v8 b, sa_f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  __device__ static inline uint32_t pack(float a, float b) {  // v_cvt_pk_f16_f32
    const sa_f16x2 r = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(uint32_t, r);
  }
  __device__ static inline float dot2_ones(uint32_t pair, float acc) {
    const sa_f16x2 ones = {(_Float16)1.0f, (_Float16)1.0f};
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(sa_f16x2, pair), ones, acc, false);
  }
};

// max / sum of x over lanes l and l ^ 32 (v_permlane32_swap: no LDS traffic).
__device__ inline float xhalf_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ inline float xhalf_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// 16-byte chunk swizzle of LDS tile row r (depends on r mod 16). Chunk c of row r is stored
// at chunk c ^ swz(r). With 64 or 32 LDS banks it makes conflict-free (a) the K operand
// reads, 16 lanes reading 16 consecutive rows at one chunk, and (b) the transposed V reads,
// 32 lanes reading 4 consecutive rows x 4 chunks.
__device__ inline int swz(int r) {
  const int j = (r >> 1) & 7;
  return (((j & 1) << 2) | (j >> 1)) ^ ((r & 1) << 1);
}

__device__ inline sa_u32x4v lds_read_b128(const lds_u8* p) {
  return *reinterpret_cast<const __attribute__((address_space(3))) sa_u32x4v*>(p);
}
// ds_read_b64_tr_b16: within each 16-lane group, lane i points at 4 consecutive bf16 (row
// i/4, columns 4(i%4)..+3 of a 4 x 16 block); lane j receives column j of that block.
__device__ inline uint2 lds_read_tr16(const lds_u8* p) {
  const sa_i16x4v v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) sa_i16x4v*)(p));
  return __builtin_bit_cast(uint2, v);
}
typedef unsigned sa_u32x2v __attribute__((ext_vector_type(2)));
// The same read issued as inline assembly: the compiler's wait analysis cannot tell these
// reads from the copies still landing in the other LDS buffers and would otherwise wait for
// all of them; the caller waits for the reads explicitly (lgkm_wait_pair).
template <int kOff>
__device__ inline sa_u32x2v lds_read_tr16_asm(uint32_t addr) {
  sa_u32x2v r;
  asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(r) : "v"(addr), "i"(kOff));
  return r;
}

// Copy one 64-row tile into LDS: instruction i, lane l -> row 8i + l/8 (tile-relative),
// 16-byte slot l of the i-th KB of `dst`. goff[p] = lane offset for rows with (row/8) odd
// (p = 1) or even (p = 0); it holds the swizzle. Offsets at or past `bytes` read as zero.
__device__ inline void dma_tile(const void* base, uint32_t bytes, uint32_t tile_off, uint32_t row_bytes,
                                const uint32_t (&goff)[2], lds_u8* dst) {
  const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0,
                                                                        (int)bytes, 0x00020000);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_u8*)(dst + 1024 * i), 16,
                                             tile_off + 8 * i * row_bytes + goff[i & 1], 0, 0, 0);
}

// dma_tile for a tile of contiguous 128-byte rows (head dim 64, row stride 64 elements): the
// same copies, with the descriptors based at the tile's rows 0 and 32, so that the lane
// offsets stay loop invariant and the instruction offset (added to both the global and the
// LDS address) steps the 8-row groups; no per-tile vector address arithmetic. Each
// descriptor's size ends at the same byte as dma_tile's (0 when row 32 lies past it): a lane
// reads offset goff + 1024 j of the descriptor at off iff off + goff + 1024 j < bytes, so rows
// past Lk read as zero as before.
__device__ inline void dma_tile_c128(const uint16_t* base, uint32_t bytes, uint32_t tile_off,
                                     const uint32_t (&goff)[2], lds_u8* dst) {
#pragma unroll
  for (int hq = 0; hq < 2; ++hq) {
    // Wave-uniform by construction; readfirstlane lets the compiler build the descriptor
    // in scalar registers.
    const uint32_t off = __builtin_amdgcn_readfirstlane(tile_off + 4096u * hq);
    const uint32_t end = __builtin_amdgcn_readfirstlane(bytes);
    const int size = __builtin_amdgcn_readfirstlane(end - min(off, end));
    const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t*>(reinterpret_cast<const uint8_t*>(base) + off), (short)0, size, 0x00020000);
    lds_u8* d = dst + 4096 * hq;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, d, 16, goff[0], 0, 0, 0);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, d, 16, goff[1], 0, 1024, 0);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, d, 16, goff[0], 0, 2048, 0);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, d, 16, goff[1], 0, 3 * 1024, 0);
  }
}

// Waits until at most n LDS reads are outstanding (n in 0..14, even), tying the wait to
// the two registers it makes valid so that nothing reads them earlier.
__device__ __forceinline__ void lgkm_wait_pair(int n, sa_u32x2v& a, sa_u32x2v& b) {
  switch (n) {
    case 14: asm volatile("s_waitcnt lgkmcnt(14)" : "+v"(a), "+v"(b)); break;
    case 12: asm volatile("s_waitcnt lgkmcnt(12)" : "+v"(a), "+v"(b)); break;
    case 10: asm volatile("s_waitcnt lgkmcnt(10)" : "+v"(a), "+v"(b)); break;
    case 8: asm volatile("s_waitcnt lgkmcnt(8)" : "+v"(a), "+v"(b)); break;
    case 6: asm volatile("s_waitcnt lgkmcnt(6)" : "+v"(a), "+v"(b)); break;
    case 4: asm volatile("s_waitcnt lgkmcnt(4)" : "+v"(a), "+v"(b)); break;
    case 2: asm volatile("s_waitcnt lgkmcnt(2)" : "+v"(a), "+v"(b)); break;
    default: asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(a), "+v"(b) : : "memory"); break;
  }
}

// s_waitcnt encodings (gfx9): vmcnt in bits 3:0 and 15:14, expcnt 6:4, lgkmcnt 11:8.
constexpr int waitcnt_vm(int n) { return (n & 15) | ((n >> 4) << 14) | 0x0F70; }
constexpr int kWaitLgkm0 = 0xC07F;
constexpr int kWaitVmLgkm0 = 0x0070;

// Workgroup barrier with no memory fence: the waits before it are explicit (a fence would
// also wait for the copies in flight). The clobber keeps the compiler from moving LDS
// accesses across it.
__device__ __forceinline__ void wg_barrier() { asm volatile("s_barrier" ::: "memory"); }

}  // namespace
