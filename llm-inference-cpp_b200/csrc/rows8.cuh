// Keys and values held in 8 bits: what a row is, how it is made and what it stands for.
//
// A row is the D numbers of one position and kv head (a key after its rotation, a value).  It is held as D codes of 8 bits and one
// fp32 scale:
//     a = max |x|,  scale = a / MAX,  code = x / scale to the nearest (ties to even),  it stands for code * scale
// with MAX 127 (int8 codes, -127 .. 127) or 448 (e4m3 codes).  The division by the scale is a product with its reciprocal, rounded.
//   * a < 2^-100: the row counts as zeros (scale 0, codes 0): smaller scales would have no reciprocal in fp32;
//   * a row with an infinity or a NaN has the scale NaN and codes 0: it reads as NaN, as a sum over it would.
// One scale per position: a scale shared by several positions would have to grow when a later one is larger, so that codes that
// are there would be rounded again — the result would depend on how a prompt was cut into steps — and the tokens of a step would
// race for it.  It costs 4 bytes for 64 or 128 codes.
//
// Pages hold 64 positions: codes [page][kv head][64][D], scales [page][kv head][64].
#pragma once
#include <cuda_fp16.h>
#include <float.h>

#include "common.cuh"

namespace llmi {

constexpr int HELD_INT8 = 0, HELD_E4M3 = 1;
constexpr int PAGE8 = 64;
constexpr float ROW8_LEAST = 7.888609052210118e-31f;      // 2^-100

struct Paged8 {
  const int32_t* seq_pages;   // [n_seqs, pages_stride]
  int pages_stride;
  int table_pages;            // pages of a sequence that the table has room for
  int n_pages;                // pages of the pool
  int n_kv_heads;
  int head_dim;
};

// The page of position `pos`, or -1 where the table or the pool has none such (a caller's mistake: nothing is read or written there, and
// queries that see it are NaN).
__device__ __forceinline__ int page8_of(const Paged8& c, int seq, int pos) {
  const int i = pos / PAGE8;
  if (i >= c.table_pages) return -1;
  const int page = c.seq_pages[(size_t)seq * c.pages_stride + i];
  return (unsigned)page < (unsigned)c.n_pages ? page : -1;
}

// The page index of the sequence's position `pos` >= 0, no further than one behind the table's last: a sequence longer than its table
// (a caller's mistake, too) costs no time, and its first page without a place reads as NaN as an unknown one does.
__device__ __forceinline__ int page_index8(const Paged8& c, int pos) { return min(pos / PAGE8, c.table_pages); }

struct Scale8 {
  float scale, inv;
};
template <int HELD> __device__ __forceinline__ Scale8 scale8(float a, bool finite) {
  Scale8 s;
  if (!finite) {
    s.scale = __int_as_float(0x7fffffff);
    s.inv = 0.f;
  } else if (a < ROW8_LEAST) {
    s.scale = s.inv = 0.f;
  } else {
    s.scale = __fdiv_rn(a, HELD == HELD_INT8 ? 127.f : 448.f);
    s.inv = __frcp_rn(s.scale);
  }
  return s;
}
__device__ __forceinline__ bool finite8(float x) { return fabsf(x) <= FLT_MAX; }

// Two codes, the first in the low byte.  (A row that is not finite has inv 0; infinity times 0 is no number and must not become a code.)
template <int HELD> __device__ __forceinline__ uint32_t codes8(float x0, float x1, float inv, bool finite) {
  if (!finite) return 0u;
  if (HELD == HELD_INT8) {
    // (1.5 * 2^23 + x is rounded to an integer as rint does, which the low byte holds; |x| is 127 at most: a * rn(1 / rn(a / 127)))
    const float a = __fadd_rn(__fmul_rn(x0, inv), 12582912.f), b = __fadd_rn(__fmul_rn(x1, inv), 12582912.f);
    return __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x0040) & 0xffffu;
  }
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(__fmul_rn(x1, inv)), "f"(__fmul_rn(x0, inv)));
  return r;
}

// The two codes in the low half of `w` as fp16 numbers, exactly.
template <int HELD> __device__ __forceinline__ __half2 halves8(uint32_t w) {
  uint32_t r;
  if (HELD == HELD_INT8) {
    // 0x6400 | u is 1024 + u in fp16; u = code + 128
    asm("prmt.b32 %0, %1, %2, 0x4140;" : "=r"(r) : "r"(w ^ 0x80808080u), "r"(0x64646464u));
    const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));      // 1152
    return __hsub2(*reinterpret_cast<__half2*>(&r), bias);
  }
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)w));
  return *reinterpret_cast<__half2*>(&r);
}
// Four codes as fp16 numbers, exactly: bytes 0, 1 and bytes 2, 3.
template <int HELD> __device__ __forceinline__ void halves8x4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if (HELD == HELD_INT8) {
    const uint32_t u = w ^ 0x80808080u;
    asm("prmt.b32 %0, %1, %2, 0x4140;" : "=r"(lo) : "r"(u), "r"(0x64646464u));
    asm("prmt.b32 %0, %1, %2, 0x4342;" : "=r"(hi) : "r"(u), "r"(0x64646464u));
    const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
    const __half2 l = __hsub2(*reinterpret_cast<__half2*>(&lo), bias), h = __hsub2(*reinterpret_cast<__half2*>(&hi), bias);
    lo = *reinterpret_cast<const uint32_t*>(&l), hi = *reinterpret_cast<const uint32_t*>(&h);
  } else {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
  }
}

// A sum of weights relative to a maximum, relative to a new one: times 2^down, `down` the old maximum less the new one, at most 0.  In two steps: the maxima are those of score +
// log2 of a value's scale, so the factor alone may be below what fp32 has where the sum times it is not.
__device__ __forceinline__ float rescale8(float sum, float down) {
  const float h = fast_exp2(0.5f * down);
  return sum * h * h;
}
template <int HELD> __device__ __forceinline__ float code8(uint32_t byte) { return __low2float(halves8<HELD>(byte)); }

}  // namespace llmi
