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
// Memory-bound: every value is read once (16-byte loads, kept in registers between the maximum and the rounding) and
// every code written once. |x| of FP16 and BF16 order like their bit patterns, so the maximum is taken on packed 16-bit
// integers. A CTA looks for the runs that begin in its window of tokens and takes some of the 2 H (side, head) items of
// each: finding a run is two dependent reads of the slot map, which a long step's CTAs share between several items.
// Measured: 64 single tokens, 8 heads of 128, FP16: 3.3 us; 17,417 tokens, 8 heads of 128 out of rows of 12 KB, BF16:
// 26.0 us = 4.1 TB/s, 0.63 of the measured copy rate (39.6 us with a CTA for every run and item). What is left there
// are the waits for each item's loads and the instructions around each run (issue 0.59, DRAM 0.37 of their peaks); loads
// one item ahead in registers cost more of them than they hid, copies into shared memory were not tried.
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "w4b_common.cuh"
#include "w4b_kernels.h"

namespace w4b {
namespace {

constexpr int KW_HELD = 8;            // 8-value pieces a thread keeps in registers (4: 34.8 us where 8 take 26.0)
constexpr int KW_BLOCKS = 2;          // CTAs of 512 threads per SM: 64 registers a thread
constexpr int KW_MIN_EXP = -60, KW_MAX_EXP = 60;

template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
  if (BF16) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
  return __half22float2(u32_as_h2(v));
}

// 8 values over the scale to 8 codes; a scale that is a power of two (every one this kernel makes) is a multiplication
template <bool BF16>
__device__ __forceinline__ uint2 encode8(uint4 v, float inv) {
  const uint32_t in[4] = {v.x, v.y, v.z, v.w};
  uint32_t h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack2<BF16>(in[i]);
    h[i] = (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(f.x * inv, f.y * inv), __NV_SATFINITE, __NV_E4M3);
  }
  return make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
}
template <bool BF16>
__device__ __noinline__ uint2 encode8_div(uint4 v, float s) {
  const uint32_t in[4] = {v.x, v.y, v.z, v.w};
  uint32_t h[4];
#pragma unroll 1
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack2<BF16>(in[i]);
    h[i] = (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(f.x, s), __fdiv_rn(f.y, s)), __NV_SATFINITE, __NV_E4M3);
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

// Whether one of the `reach` tokens before token t has a slot in the page that begins at row `base`. (Out of line: only
// tokens behind skipped ones ask, and its instructions in the kernel's way cost a decode step 0.4 us of 3.3.)
__device__ __noinline__ bool page_before(const int* slots, int t, int reach, unsigned base, unsigned page) {
  bool found = false;
#pragma unroll 4
  for (int j = 1; j <= reach; ++j) found = found || (unsigned)slots[t - j] - base < page;
  return found;
}

template <bool BF16, int D>
__global__ void __launch_bounds__(512, KW_BLOCKS) kv_write_b8_kernel(const KvWriteB8 a) {
  constexpr int LPR = D / 8;  // lanes per row
  __shared__ uint32_t wmax[2][16];
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5, nthreads = blockDim.x;
  const long long rows = (long long)a.npages * a.page;
  const uint32_t inf_bits = BF16 ? 0x7F80u : 0x7C00u;

  // this CTA's tokens and items (sides and heads; the CTAs of neighbouring items are launched together, since they
  // read the same tokens' rows)
  const int groups = (2 * a.H + a.items - 1) / a.items, win = (int)(blockIdx.x / groups);
  const int item0 = (int)(blockIdx.x - (unsigned)win * groups) * a.items, item1 = min(item0 + a.items, 2 * a.H);
  const int t_begin = win * a.window, t_end = (int)min((long long)t_begin + a.window, (long long)a.T);

  struct Task {
    int t, n;     // tokens t .. t + n - 1: a run
    int p, row0;  // its page, the row it starts at
    int item;     // < H: keys of head `item`; else values of head item - H
  };
  int t0 = t_begin - 32;
  uint32_t heads = 0;  // tokens t0 + bit that head a run
  auto advance = [&](Task& k) {  // the next item of the run, or the first of the next run; the same in every thread
    if (k.n > 0 && ++k.item < item1) return true;
    while (heads == 0) {
      t0 += 32;
      if (t0 >= t_end) return false;
      const int t = t0 + lane;
      bool head = false, wrong = false;
      if (t < t_end) {
        const int slot = a.slots[t], before = t > 0 ? a.slots[t - 1] : -1;
        if (slot >= rows) {
          wrong = true;
        } else if (slot >= 0 && (slot % a.page == 0 || before != slot - 1)) {
          // a second run in the page of the token before: its scale would be a race
          wrong = before >= 0 && before / a.page == slot / a.page;
          if ((before < 0 || before >= rows) && t > 1)  // behind tokens that are not written: as many as a page has rows
            wrong = page_before(a.slots, t, min(a.page - 1, t), (unsigned)(slot - slot % a.page), (unsigned)a.page);
          head = !wrong;
        }
      }
      if (wrong && wid == 0) atomicExch(a.status, ST_KV_WRITE_SLOT);
      heads = __ballot_sync(0xffffffffu, head);
    }
    k.t = t0 + __ffs(heads) - 1;
    heads &= heads - 1;
    const int slot = a.slots[k.t];
    k.p = slot / a.page;
    k.row0 = slot - k.p * a.page;
    k.item = item0;
    k.n = 1;
    const int most = min(a.page - k.row0, a.T - k.t);
    while (k.n < most) {
      const int j = k.n + lane;
      const uint32_t on = __ballot_sync(0xffffffffu, j < most && a.slots[k.t + j] == slot + j);
      k.n += on == 0xffffffffu ? 32 : __ffs(~on) - 1;
      if (on != 0xffffffffu) break;
    }
    return true;
  };
  Task k = {0, 0, 0, 0, 0};
  for (int turn = 0; advance(k); turn ^= 1) {
    const bool v_side = k.item >= a.H;
    const int h = v_side ? k.item - a.H : k.item, pieces = k.n * LPR;
    // this thread's pieces: i * nthreads + tid, row (i * nthreads + tid) / LPR of the run
    const long long stride = v_side ? a.v_stride : a.k_stride;
    const uint16_t* x = (const uint16_t*)(v_side ? a.v_new : a.k_new) + (size_t)h * D + (long long)(k.t + tid / LPR) * stride +
                        (tid % LPR) * 8;
    const long long pass = (long long)(nthreads / LPR) * stride;
    float* scale = (v_side ? a.s_v : a.s_k) + (size_t)h * a.npages + k.p;
    uint4 held[KW_HELD];
#pragma unroll
    for (int i = 0; i < KW_HELD; ++i)
      held[i] = i * nthreads + tid < pieces ? *(const uint4*)(x + i * pass) : make_uint4(0, 0, 0, 0);
    const float old = *scale;
    uint32_t top = 0;
    bool finite = true;
    auto row_max = [&](uint4& v) {  // a row with a value that is not finite counts as zeros
      uint32_t m = __vmaxu2(__vmaxu2(v.x & 0x7FFF7FFFu, v.y & 0x7FFF7FFFu), __vmaxu2(v.z & 0x7FFF7FFFu, v.w & 0x7FFF7FFFu));
      const bool bad = (m & 0xFFFFu) >= inf_bits || (m >> 16) >= inf_bits;
      if (__any_sync(0xffffffffu, bad)) {
        bool row = bad;
#pragma unroll
        for (int d = LPR / 2; d > 0; d >>= 1) row = __shfl_xor_sync(0xffffffffu, (int)row, d) || row;
        if (row) {
          finite = false;
          v = make_uint4(0, 0, 0, 0);
          m = 0;
        }
      }
      return m;
    };
#pragma unroll
    for (int i = 0; i < KW_HELD; ++i)
      if (i * nthreads < pieces) top = __vmaxu2(top, row_max(held[i]));
#pragma unroll 1
    for (int i = KW_HELD; i * nthreads < pieces; ++i) {  // pages larger than the registers: read twice
      uint4 v = i * nthreads + tid < pieces ? *(const uint4*)(x + i * pass) : make_uint4(0, 0, 0, 0);
      top = __vmaxu2(top, row_max(v));
    }
    top = __reduce_max_sync(0xffffffffu, max(top & 0xFFFFu, top >> 16));
    if (lane == 0) wmax[turn][wid] = top;
    __syncthreads();  // (and the scale has been read by all)
    for (int w = 0; w < nthreads / 32; ++w) top = max(top, wmax[turn][w]);
    const float amax = BF16 ? __uint_as_float(top << 16) : __half2float(__ushort_as_half((unsigned short)top));

    float s = old;
    bool moved = false;
    if (k.row0 == 0 || !(amax <= 448.0f * old)) {
      int e = KW_MIN_EXP;
      if (amax > 0.0f) {
        int b;
        const float m = frexpf(amax, &b);
        e = b - 9 + (m > 0.875f ? 1 : 0);  // 448 = 0.875 * 2^9
        if (e > KW_MAX_EXP && tid == 0) atomicExch(a.status, ST_QUANT_INVALID);
        e = min(max(e, KW_MIN_EXP), KW_MAX_EXP);
      }
      s = __uint_as_float((uint32_t)(e + 127) << 23);
      moved = k.row0 > 0;
    }
    if (tid == 0 && s != old) *scale = s;
    if (!finite && (lane % LPR) == 0) atomicExch(a.status, ST_QUANT_INVALID);
    uint8_t* page_codes = (v_side ? a.q_v : a.q_k) + ((size_t)h * rows + (size_t)k.p * a.page) * D;
    if (moved) {
      const float ratio = old / s;
      uint32_t* w = (uint32_t*)page_codes;
#pragma unroll 1
      for (int i = tid; i < k.row0 * (D / 4); i += nthreads) w[i] = recode4(w[i], ratio);
    }
    uint2* dst = (uint2*)(page_codes + (size_t)k.row0 * D) + tid;
    if ((__float_as_uint(s) & 0x007FFFFFu) == 0) {
      const float inv = 1.0f / s;
#pragma unroll
      for (int i = 0; i < KW_HELD; ++i)
        if (i * nthreads + tid < pieces) dst[i * nthreads] = encode8<BF16>(held[i], inv);
#pragma unroll 1
      for (int i = KW_HELD; i * nthreads < pieces; ++i) {
        uint4 v = i * nthreads + tid < pieces ? *(const uint4*)(x + i * pass) : make_uint4(0, 0, 0, 0);
        row_max(v);
        if (i * nthreads + tid < pieces) dst[i * nthreads] = encode8<BF16>(v, inv);
      }
    } else {
#pragma unroll 1
      for (int i = 0; i * nthreads < pieces; ++i) {
        uint4 v = i * nthreads + tid < pieces ? *(const uint4*)(x + i * pass) : make_uint4(0, 0, 0, 0);
        row_max(v);
        if (i * nthreads + tid < pieces) dst[i * nthreads] = encode8_div<BF16>(v, s);
      }
    }
  }
}

}  // namespace

cudaError_t kv_write_b8_launch(const KvWriteB8& args, int D, int bf16, int sm_count, cudaStream_t stream) {
  KvWriteB8 a = args;
  // threads: a full page's pieces, KW_HELD per thread
  int threads = a.page * (D / 8) / KW_HELD;
  threads = threads < 32 ? 32 : (threads > 512 ? 512 : (threads + 31) / 32 * 32);
  // One wave of CTAs: single-token runs (a decode step) get a CTA for each item; longer steps first wider windows, up
  // to a page (a narrower one would mostly find that its token heads no run), then several items per CTA.
  const long long wave = (long long)sm_count * (KW_BLOCKS * 512 / threads), all = 2LL * a.H * a.T;
  const long long w = (all + wave - 1) / wave;
  a.window = (int)(w > a.page ? a.page : w);
  const long long windows = (a.T + (long long)a.window - 1) / a.window;
  long long groups = wave / windows;
  groups = groups < 1 ? 1 : (groups > 2 * a.H ? 2 * a.H : groups);
  a.items = (int)((2 * a.H + groups - 1) / groups);
  const long long grid = windows * ((2 * a.H + a.items - 1) / a.items);
  const dim3 g((unsigned)grid);
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
