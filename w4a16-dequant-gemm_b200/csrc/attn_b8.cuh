// What the two kernels of attention over a paged 8-bit cache share (attn_b8.cu, attn_b8_chunk.cu).
#pragma once

#include <cuda_bf16.h>

#include "w4b_common.cuh"
#include "w4b_kernels.h"

namespace w4b {

constexpr int AB_MAX_D = 128;
constexpr float AB_LOG2E = 1.4426950408889634f;
constexpr float AB_LN2 = 0.6931471805599453f;
// Weights are 2^(X - m) as halves. The reference point m of a row moves only when some X exceeds it by more than
// AB_SLACK (halves end at 2^16), and then to AB_BELOW under that X: the largest weight of a row is 2^9 or more, so what
// is rounded to multiples of 2^-24 (halves below 2^-14) or to zero is off by 2^-34 of it, which even a million such
// positions do not add up to an FP16 rounding. With m at the maximum itself it would be 2^-25, and a row whose first
// position outweighs each of the others by that much lost them all (price of the lower point, 9 or 5 alike: rows move
// more often; prompt chunks 209 -> 213 us, 24 drafts 17.1 -> 17.4 us, none for single tokens).
constexpr float AB_SLACK = 15.0f, AB_BELOW = 9.0f;
constexpr float AB_NONE = -1e30f;  // reference point of a row that has seen nothing

__host__ __device__ __forceinline__ size_t counter_bytes(int grid) { return 4 * (((size_t)grid + 63) / 64 * 64); }

// bytes 0, 1 (lo) and 2, 3 (hi) of w to half2 each
__device__ __forceinline__ void e4m3x4_to_h2(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n"
      ".reg .b16 a, b;\n"
      "mov.b32 {a, b}, %2;\n"
      "cvt.rn.f16x2.e4m3x2 %0, a;\n"
      "cvt.rn.f16x2.e4m3x2 %1, b;\n"
      "}\n"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// BF16 query rows become FP16 by a power of two of the row's own: with `top` the largest |q| (bits) its largest value
// lands in [2^14, 2^15), and what falls below the half range is 2^-39 of it. scale_row undoes it in the scores. The power
// ends where one of the two would not be a normal number: at 2^-113 every finite row still fits, at 2^126 rows below
// 2^-112 stay smaller, the smallest subnormal at 2^-7.
__device__ __forceinline__ void bf16_row_scale(uint32_t top, float& up, float& scale_row) {
  const int k = min(max(141 - (int)(top >> 7), -113), 126);  // 127 + 14 - the biased exponent
  up = __uint_as_float((uint32_t)(127 + k) << 23);
  scale_row = __uint_as_float((uint32_t)(127 - k) << 23);
}
__device__ __forceinline__ uint32_t bf16x2_to_h2(uint32_t w, float up) {
  return h2_as_u32(__floats2half2_rn(__uint_as_float(w << 16) * up, __uint_as_float(w & 0xFFFF0000u) * up));
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack_out(float x, float y) {
  if (BF16) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(x, y);
    return *(const uint32_t*)&b;
  }
  return h2_as_u32(__floats2half2_rn(x, y));
}
// 1 / l; a row that saw nothing gives zeros, NaN stays
__device__ __forceinline__ float row_norm(float l) { return l == 0.0f ? 0.0f : 1.0f / l; }
__device__ __forceinline__ float row_lse(float m, float l) { return l == 0.0f ? -INFINITY : (m + log2f(l)) * AB_LN2; }

// What a sequence asks for, with the device-side values held inside what the launch was sized for: positions from
// max_len on and tokens from max_q on are left out (status), but where a token stands goes by the values as they are.
struct SeqInfo {
  int len, q0, nq;
  int first;  // causal: position of token 0 (negative when there are more tokens than positions)
};
__device__ __forceinline__ SeqInfo seq_info(const AttnB8& a, int i) {
  SeqInfo s;
  const int len = max(a.seq_lens[i], 0);
  s.q0 = a.q_offsets ? a.q_offsets[i] : i;
  const int nq = a.q_offsets ? max(a.q_offsets[i + 1] - s.q0, 0) : 1;
  s.len = min(len, a.max_len);
  s.nq = min(nq, a.max_q);
  s.first = len - nq;
  if (len > a.max_len || nq > a.max_q) atomicExch(a.status, ST_ATTN_BOUNDS);
  return s;
}
// the positions token `tq` sees
__device__ __forceinline__ int positions_seen(const AttnB8& a, const SeqInfo& s, int tq) {
  return a.causal ? min(s.len, max(0, s.first + tq + 1)) : s.len;
}

// The split of T units over G CTAs: CTA c has units [T c / G, T (c + 1) / G), and unit u is CTA ((u + 1) G - 1) / T's.
// (64-bit division is some hundred instructions, so 32-bit where it suffices, and only where a row is split.)
__device__ __forceinline__ int unit_owner(long long u, long long T, long long G) {
  const unsigned long long n = (unsigned long long)(u + 1) * (unsigned long long)G - 1;
  return (n | (unsigned long long)T) < 0x100000000ULL ? (int)((unsigned)n / (unsigned)T) : (int)(n / (unsigned long long)T);
}
__device__ __forceinline__ long long range_begin(long long T, long long c, long long G) {
  const unsigned long long n = (unsigned long long)T * (unsigned long long)c;
  return n < 0x100000000ULL ? (long long)((unsigned)n / (unsigned)G) : (long long)(n / (unsigned long long)G);
}

}  // namespace w4b
