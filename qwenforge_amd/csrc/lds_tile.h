// 64-key tiles of fp16 K and V rows of 64 dims in LDS, as the streaming
// attention kernels hold them, and the reads of their matrix-core operands.
//
// LDS rows are 128 bytes, XOR-swizzled in 16-byte chunks (chunk c of row r
// lives at c ^ swz(r)).  gfx950's LDS serves 256 bytes per cycle (64 banks of 4
// bytes: a 16-byte read takes 16 lanes at a time).  With
// swz(r) = r1 | r3 << 1 | (r1 ^ r4) << 2 (ri = bit i of r) the 16 lanes of a
// K operand read (rows 8*(c/4) + 4j + c%4, one logical chunk) hit 16
// distinct 16-byte bank groups, i.e. the reads are conflict-free; a swizzle
// that breaks this doubles SQ_LDS_BANK_CONFLICT (measured).  V^T operands come
// from ds_read_b64_tr_b16: within each 16-lane group, lane i receives element
// i % 4 of the 8-byte words addressed by lanes 4t + i/4 (t = 0..3), so lanes
// that address 4 keys x 16 dims of V receive V^T[d][4 keys] directly.
#pragma once

#include "qf_common.h"

namespace qf {

constexpr int kRowBytes = 64 * 2;  // a row of 64 dims

__device__ __forceinline__ int swz(int row) {
  const int r1 = (row >> 1) & 1, r3 = (row >> 3) & 1, r4 = (row >> 4) & 1;
  return r1 | (r3 << 1) | ((r1 ^ r4) << 2);
}

typedef __attribute__((address_space(3))) void lds_void;

// 32-bit LDS address of a pointer into a __shared__ array.
__device__ __forceinline__ unsigned lds_addr(const unsigned char* p) {
  return (unsigned)(uintptr_t)(const lds_void*)p;
}

// LDS operand reads of a tile, written as inline asm.  The tiles arrive by
// LDS DMA (buffer_load ... lds), which the compiler tracks with the vector
// memory counter; it cannot tell that a read of one stage does not alias the
// DMA into another, and before every compiler-visible LDS read it would wait
// for the DMA just issued for the next tiles (vmcnt(0)), which serialises the
// prefetch.  These reads carry no such wait: the barrier of the step orders
// them after their own tile's DMA, and the caller waits for the reads
// themselves (lgkmcnt) before the first use.
template <int kOff>
__device__ __forceinline__ u32x4 lds_read_b128(unsigned addr) {
  u32x4 r;
  asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(r) : "v"(addr), "i"(kOff));
  return r;
}

// ds_read_b64_tr_b16: lane i receives the 16-bit elements that the
// transposed 8-byte reads of its lane group place there (the V^T operand).
template <int kOff>
__device__ __forceinline__ u32x2 lds_read_tr_b64(unsigned addr) {
  u32x2 r;
  asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(r) : "v"(addr), "i"(kOff));
  return r;
}

// Buffer resource over `rem` valid bytes from `base` (a tile's first row):
// the tile's address and valid byte count live in SGPRs, so a lane's load
// offset within the tile never changes, and rows past the sequence (the last
// tile's tail) read as zero (their scores are masked).  Needs row strides
// >= 64 elements so a row's 128 bytes lie below the record count.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t tile_rsrc(const unsigned char* base, int64_t rem) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(base), (short)0,
                                           (int)(rem < 0x7fffffff ? rem : 0x7fffffff), 0x00020000);
}

// v_max3_f32 on raw registers.  fmaxf would first canonicalise the MFMA
// results (v_max_f32 x, x per operand: IEEE mode quiets signalling NaNs); the
// scores here are finite or -inf, so the plain three-input max is exact.
__device__ __forceinline__ float max3_raw(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// Max of a lane's 16 scores: a depth-3 tree of seven max3.  The hazard
// recognizer does not look into inline asm, so it would insert no wait
// states between the score MFMAs and an asm read of their results: the
// s_nops, tied to all sixteen score registers (every max3 depends on them,
// and they on the MFMAs), give a matrix-core result the 16 wait states it
// may need before a VALU read, however close the scheduler puts the max.
__device__ __forceinline__ float max16(f32x4 (&sc)[4]) {
  asm volatile("s_nop 7\n\ts_nop 7" : "+v"(sc[0]), "+v"(sc[1]), "+v"(sc[2]), "+v"(sc[3]));
  const float a = max3_raw(sc[0][0], sc[0][1], sc[0][2]);
  const float b = max3_raw(sc[0][3], sc[1][0], sc[1][1]);
  const float d = max3_raw(sc[1][2], sc[1][3], sc[2][0]);
  const float e = max3_raw(sc[2][1], sc[2][2], sc[2][3]);
  const float f = max3_raw(sc[3][0], sc[3][1], sc[3][2]);
  return max3_raw(max3_raw(a, b, d), max3_raw(e, f, sc[3][3]), kNegInf);
}

// Running max is only moved when a tile's max exceeds it by more than this
// many log2 units: until then p = exp2(s - m) <= 2^8 stays exact enough in
// fp16 and the output accumulators need no rescaling (the final division by
// the running sum makes the result independent of the reference point).
constexpr float kRescaleSlack = 8.f;

}  // namespace qf
