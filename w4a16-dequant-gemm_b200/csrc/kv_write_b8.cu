// The quantising write of a paged 8-bit cache: the rows of new tokens (FP16 or BF16) to E4M3 codes with one FP32 scale
// per (page, head), side by side for K and V.
//
// The tokens that a call writes into one page are one run of consecutive slots. With a = max |x| over the run's rows
// of a head and s the page's scale before the call:
//   run starts at row 0 of the page:  s' = 2^e, the smallest power of two with a <= 448 * 2^e (e in -60..60; -60 for a = 0)
//   run continues a page:             s' = s when a <= 448 * s, else 2^e as above, and the page's earlier codes are
//                                     rounded again: code' = rn(code * (s / s'))
//   new codes = rn(x / s')            (round to nearest even)
// Powers of two make x / s' exact and the second rounding exact too, except for codes that become subnormal; E4M3
// loses no precision by it, its step being relative. A row with a value that is not finite is written as zeros and
// reported through the status word, like the other quantizers do.
//
// One CTA per (run, head, side): memory-bound, every value is read once (16-byte loads, kept in registers between the
// maximum and the rounding) and every code written once. |x| of FP16 and BF16 order like their bit patterns, so the
// maximum is taken on packed 16-bit integers. A CTA looks for the runs that begin in its window of tokens.
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "w4b_common.cuh"
#include "w4b_kernels.h"

namespace w4b {
namespace {

constexpr int KW_HELD = 4;            // 8-value pieces a thread keeps in registers
constexpr int KW_MIN_EXP = -60, KW_MAX_EXP = 60;

template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
  if (BF16) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
  return __half22float2(u32_as_h2(v));
}

__device__ __forceinline__ uint32_t abs_max2(uint32_t a, uint32_t b) { return __vmaxu2(a, b & 0x7FFF7FFFu); }

// 8 values times / over the scale to 8 codes
template <bool BF16>
__device__ __forceinline__ uint2 encode8(uint4 v, float s, float inv, bool pow2) {
  const uint32_t in[4] = {v.x, v.y, v.z, v.w};
  uint32_t h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 f = unpack2<BF16>(in[i]);
    if (pow2) {
      f.x *= inv;
      f.y *= inv;
    } else {
      f.x = __fdiv_rn(f.x, s);
      f.y = __fdiv_rn(f.y, s);
    }
    h[i] = (uint32_t)__nv_cvt_float2_to_fp8x2(f, __NV_SATFINITE, __NV_E4M3);
  }
  return make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
}

// codes of a page whose scale grew: rn(code * ratio)
__device__ __forceinline__ uint32_t recode4(uint32_t w, float ratio) {
  uint32_t out = 0;
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    const float2 f = make_float2(e4m3_to_float((w >> (8 * i)) & 0xFF) * ratio,
                                 e4m3_to_float((w >> (8 * i + 8)) & 0xFF) * ratio);
    out |= (uint32_t)__nv_cvt_float2_to_fp8x2(f, __NV_SATFINITE, __NV_E4M3) << (8 * i);
  }
  return out;
}

template <bool BF16, int D>
__global__ void kv_write_b8_kernel(const KvWriteB8 a) {
  constexpr int LPR = D / 8;  // lanes per row
  __shared__ uint32_t wmax[16];
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5, nthreads = blockDim.x;
  const int h = (int)blockIdx.y;
  const bool v_side = blockIdx.z != 0;
  const uint16_t* x = (const uint16_t*)(v_side ? a.v_new : a.k_new) + (size_t)h * D;
  const long long xs = v_side ? a.v_stride : a.k_stride;
  const long long rows = (long long)a.npages * a.page;
  uint8_t* codes = (v_side ? a.q_v : a.q_k) + (size_t)h * rows * D;
  float* scales = (v_side ? a.s_v : a.s_k) + (size_t)h * a.npages;
  const uint32_t inf_bits = BF16 ? 0x7F80u : 0x7C00u;

  // tokens that head a run, 32 at a time
  const int t_begin = (int)blockIdx.x * a.window, t_end = min(t_begin + a.window, a.T);
  for (int t0 = t_begin; t0 < t_end; t0 += 32) {
    uint32_t heads = 0;
    {
      const int t = t0 + lane;
      bool head = false, wrong = false;
      if (t < t_end) {
        const int slot = a.slots[t], before = t > 0 ? a.slots[t - 1] : -1;
        if (slot >= rows) {
          wrong = true;
        } else if (slot >= 0 && (slot % a.page == 0 || before != slot - 1)) {
          // a second run in the page of the token before: its scale would be a race
          wrong = before >= 0 && before / a.page == slot / a.page;
          head = !wrong;
        }
      }
      if (wrong && wid == 0) atomicExch(a.status, ST_KV_WRITE_SLOT);
      heads = __ballot_sync(0xffffffffu, head);
    }
    while (heads != 0) {
      const int t = t0 + __ffs(heads) - 1;
      heads &= heads - 1;
      const int slot = a.slots[t];
      const int p = slot / a.page, row0 = slot - p * a.page;
      // the run: tokens t .. t + n - 1 in slots slot, slot + 1, ... of the page
      int n = 1;
      const int most = min(a.page - row0, a.T - t);
      while (n < most) {  // every warp by itself
        const int j = n + lane;
        const uint32_t on = __ballot_sync(0xffffffffu, j < most && a.slots[t + j] == slot + j);
        n += on == 0xffffffffu ? 32 : __ffs(~on) - 1;
        if (on != 0xffffffffu) break;
      }
      const int pieces = n * LPR;
      uint4 held[KW_HELD];
      uint32_t top = 0;
      bool finite = true;
      // rows with a value that is not finite count as zeros
      auto row_of = [&](int i) -> uint4 {
        const uint16_t* src = x + (long long)(t + i / LPR) * xs + (i % LPR) * 8;
        return i < pieces ? *(const uint4*)src : make_uint4(0, 0, 0, 0);
      };
      auto row_max = [&](uint4& v) {
        uint32_t m = abs_max2(abs_max2(abs_max2(abs_max2(0u, v.x), v.y), v.z), v.w);
        m = max(m & 0xFFFFu, m >> 16);
#pragma unroll
        for (int d = LPR / 2; d > 0; d >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
        if (m >= inf_bits) {
          finite = false;
          v = make_uint4(0, 0, 0, 0);
          m = 0;
        }
        return m;
      };
#pragma unroll
      for (int k = 0; k < KW_HELD; ++k) {
        held[k] = make_uint4(0, 0, 0, 0);
        if (k * nthreads < pieces) held[k] = row_of(k * nthreads + tid);
      }
      const float old = scales[p];
#pragma unroll
      for (int k = 0; k < KW_HELD; ++k)
        if (k * nthreads < pieces) top = max(top, row_max(held[k]));
      for (int k = KW_HELD; k * nthreads < pieces; ++k) {
        uint4 v = row_of(k * nthreads + tid);
        top = max(top, row_max(v));
      }
      top = __reduce_max_sync(0xffffffffu, top);
      if (lane == 0) wmax[wid] = top;
      __syncthreads();
      for (int w = 0; w < nthreads / 32; ++w) top = max(top, wmax[w]);
      __syncthreads();  // wmax is free for the next run; scales[p] has been read by all
      const float amax = BF16 ? __uint_as_float(top << 16) : __half2float(__ushort_as_half((unsigned short)top));

      float s = old;
      bool moved = false;
      if (row0 == 0 || !(amax <= 448.0f * old)) {
        int e = KW_MIN_EXP;
        if (amax > 0.0f) {
          int b;
          const float m = frexpf(amax, &b);
          e = b - 9 + (m > 0.875f ? 1 : 0);  // 448 = 0.875 * 2^9
          if (e > KW_MAX_EXP && tid == 0) atomicExch(a.status, ST_QUANT_INVALID);
          e = min(max(e, KW_MIN_EXP), KW_MAX_EXP);
        }
        s = __uint_as_float((uint32_t)(e + 127) << 23);
        moved = row0 > 0;
      }
      if (tid == 0 && s != old) scales[p] = s;
      if (!finite && (lane % LPR) == 0) atomicExch(a.status, ST_QUANT_INVALID);
      uint8_t* page_codes = codes + (size_t)p * a.page * D;
      if (moved) {
        const float ratio = old / s;
        uint32_t* w = (uint32_t*)page_codes;
        for (int i = tid; i < row0 * (D / 4); i += nthreads) w[i] = recode4(w[i], ratio);
      }
      const bool pow2 = (__float_as_uint(s) & 0x007FFFFFu) == 0;
      const float inv = 1.0f / s;
      uint2* dst = (uint2*)(page_codes + (size_t)row0 * D);
#pragma unroll
      for (int k = 0; k < KW_HELD; ++k) {
        const int i = k * nthreads + tid;
        if (i < pieces) dst[i] = encode8<BF16>(held[k], s, inv, pow2);
      }
      for (int k = KW_HELD; k * nthreads < pieces; ++k) {
        const int i = k * nthreads + tid;
        uint4 v = row_of(i);
        row_max(v);
        if (i < pieces) dst[i] = encode8<BF16>(v, s, inv, pow2);
      }
    }
  }
}

}  // namespace

cudaError_t kv_write_b8_launch(const KvWriteB8& args, int H, int D, int bf16, int sm_count, cudaStream_t stream) {
  KvWriteB8 a = args;
  // threads: a full page's pieces, KW_HELD per thread
  int threads = a.page * (D / 8) / KW_HELD;
  threads = threads < 64 ? 64 : (threads > 512 ? 512 : (threads + 31) / 32 * 32);
  // window: single-token runs (a decode step) want a CTA each; prompt steps want about a page per CTA, or most of the
  // grid would only find that its token heads no run. About two waves of CTAs decide between the two.
  const long long items = (long long)a.T * H * 2, grid = 2LL * sm_count * (2048 / threads);
  long long w = items / grid;
  a.window = (int)(w < 1 ? 1 : (w > a.page ? a.page : w));
  const dim3 g((unsigned)((a.T + a.window - 1) / a.window), (unsigned)H, 2);
  if (D == 128) {
    if (bf16) kv_write_b8_kernel<true, 128><<<g, threads, 0, stream>>>(a);
    else kv_write_b8_kernel<false, 128><<<g, threads, 0, stream>>>(a);
  } else {
    if (bf16) kv_write_b8_kernel<true, 64><<<g, threads, 0, stream>>>(a);
    else kv_write_b8_kernel<false, 64><<<g, threads, 0, stream>>>(a);
  }
  return cudaGetLastError();
}

}  // namespace w4b
