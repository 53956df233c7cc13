// Attention over a paged 8-bit cache for sequences with many query rows per key/value head (prompt chunks, encoder
// states): the same operator as attn_b8.cu, bound by the tensor pipe instead of HBM, on tcgen05.
//
// One CTA works on 128 query rows (token-major: row = token * group + head of the group) of one sequence and
// key/value head, and walks the positions in tiles of 64:
//   S = Q K^T        tcgen05.mma M = 128, N = 64; A = Q from tensor memory, B = the K tile in shared memory
//   w = 2^(S * s_k * scale * log2 e + log2 s_v - m)      (why V's scale goes into the weights: attn_b8.cu)
//   O += w V         M = 128, N = D, K = 64; A = w from tensor memory (over S), B = the V tile
// Both A operands come from tensor memory because that form issues a 128 x 128 x 16 product every 74 cycles against
// 103 with A in shared memory (64 ideal; measured alone), and because it leaves shared memory to the conversion.
//   warps 0-3  one thread per query row (its TMEM lane): no reduction across threads anywhere. The reference point m
//              moves only when a score exceeds it by 2^8 (see attn_b8.cu); then O is rescaled in place.
//   warps 4-7  E4M3 -> FP16 (exact): 16-byte loads of the next tile in flight while the current one is written to
//              swizzled operand tiles. K is K-major; V is stored the same way (row = position) and read MN-major.
//   One elected thread of warp 0 issues the MMAs, when the four warps' weights are in place: it has nothing else to do
//   until the next scores are there, and with eight warps a thread may use 128 registers. (elect.sync, not "lane == 0":
//   with a plain thread test an instruction took 92 cycles to issue whatever its size.)
// Two CTAs per SM (TMEM: S 64 + O 128 + Q 64 = 256 columns each): one's softmax overlaps the other's products.
//
// Split: units of one tile over all (sequence, head, row tile) in order, cut into equal ranges, as in attn_b8.cu; the
// causal limit of every row tile is in the count.
#include <cuda_bf16.h>
#include <float.h>

#include "attn_b8.cuh"

namespace w4b {
namespace {

constexpr int AC_ROWS = 128;
constexpr int AC_TILE = 64;   // positions per tile
constexpr int AC_THREADS = 256;
constexpr int AC_WARPS = AC_THREADS / 32;
constexpr int AC_CTAS_PER_SM = 2;
constexpr int AC_MIN_UNITS = 4;  // tiles per CTA below which no further split pays

__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
  return p != 0;
}

// 128-byte swizzle, 8-row groups of 1024 bytes. K-major: lbo unused (1). MN-major: lbo = bytes to the next 64 columns.
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr, uint32_t lbo16) {
  uint64_t d = 0;
  d |= (uint64_t)((addr >> 4) & 0x3FFFu);
  d |= (uint64_t)lbo16 << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

__device__ __forceinline__ void mma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t db, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
      "}\n" ::"r"(tmem_d),
      "r"(tmem_a), "l"(db), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tc_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

#define W4B_R8(v, o) "r"(v[o]), "r"(v[o + 1]), "r"(v[o + 2]), "r"(v[o + 3]), "r"(v[o + 4]), "r"(v[o + 5]), "r"(v[o + 6]), "r"(v[o + 7])
#define W4B_W8(v, o) "=r"(v[o]), "=r"(v[o + 1]), "=r"(v[o + 2]), "=r"(v[o + 3]), "=r"(v[o + 4]), "=r"(v[o + 5]), "=r"(v[o + 6]), "=r"(v[o + 7])
// 32 columns of this thread's lane; the caller waits (tmem_wait_ld / _st)
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,"
      "%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : W4B_W8(v, 0), W4B_W8(v, 8), W4B_W8(v, 16), W4B_W8(v, 24)
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
      "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::W4B_R8(v, 0),
      W4B_R8(v, 8), W4B_R8(v, 16), W4B_R8(v, 24), "r"(addr)
      : "memory");
}
#undef W4B_R8
#undef W4B_W8
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Positions the rows of a row tile see, and its tiles.
struct RowTile {
  int rows;      // query rows in use
  int end;       // positions any row sees
  int all_see;   // positions every row sees
  int units;     // tiles (at least one: a row tile that sees nothing still writes its zeros)
};
__device__ __forceinline__ RowTile row_tile(const AttnB8& a, const SeqInfo& s, int qt) {
  RowTile t;
  const int first = qt * AC_ROWS;
  t.rows = min(AC_ROWS, s.nq * a.group - first);
  const int before = s.len - s.nq;
  t.end = a.causal ? min(s.len, max(0, before + (first + t.rows - 1) / a.group + 1)) : s.len;
  t.all_see = a.causal ? max(0, before + first / a.group + 1) : s.len;
  t.units = max(1, (t.end + AC_TILE - 1) / AC_TILE);
  return t;
}
__device__ __forceinline__ int row_tiles(const AttnB8& a, const SeqInfo& s) {
  const int rows = s.nq * a.group;
  return rows >= a.chunk_rows ? (rows + AC_ROWS - 1) / AC_ROWS : 0;
}
// Units of one head of a sequence, by a warp (the same value in every lane).
__device__ __forceinline__ long long head_units(const AttnB8& a, const SeqInfo& s, int lane) {
  const int n = row_tiles(a, s);
  long long sum = 0;
  for (int qt = lane; qt < n; qt += 32) sum += row_tile(a, s, qt).units;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  return sum;
}

template <int D>
struct ChunkSmem {
  static constexpr int TILE_BYTES = AC_TILE * D * 2;  // an FP16 operand tile: D / 64 blocks of 64 rows x 128 bytes
  static constexpr int STAGES = 2;
  static constexpr int META = 4 * 4 * 16;              // four tiles of four blocks of 16 positions
  static constexpr int K_OFF = 0, V_OFF = STAGES * TILE_BYTES, META_OFF = 2 * STAGES * TILE_BYTES;
  static constexpr int BAR_OFF = META_OFF + META;
  static constexpr int BYTES = BAR_OFF + 128 + 1024;   // + alignment
};

// where a CTA's range of units starts
struct RangeStart {
  long long u_begin, u_end, total, ctas;
  int seq, head, qt, r0;
};

template <int D, bool BF16>
__global__ void __launch_bounds__(AC_THREADS, AC_CTAS_PER_SM) attn_b8_chunk_kernel(const AttnB8 a) {
  using L = ChunkSmem<D>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ long long wsum[AC_WARPS];
  __shared__ RangeStart start;
  __shared__ uint32_t tmem_slot;
  __shared__ int is_last;
  const int tid = threadIdx.x, lane = tid & 31, wid = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const uint32_t sm = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smp = smem_raw + (sm - smem_u32(smem_raw));

  // ---- this CTA's range of units: warps take consecutive runs of sequences -------------------------------------
  {
    const int per = (a.nseq + AC_WARPS - 1) / AC_WARPS;
    const int i0 = min(wid * per, a.nseq), i1 = min(i0 + per, a.nseq);
    long long mine = 0;
    for (int i = i0; i < i1; ++i) mine += a.H * head_units(a, seq_info(a, i), lane);
    if (lane == 0) wsum[wid] = mine;
    __syncthreads();
    long long before = 0, T = 0;
    for (int w = 0; w < AC_WARPS; ++w) {
      if (w < wid) before += wsum[w];
      T += wsum[w];
    }
    const long long most = (T + AC_MIN_UNITS - 1) / AC_MIN_UNITS;
    const long long G = most < (long long)gridDim.x ? most : (long long)gridDim.x;
    const long long cta = blockIdx.x;
    if (cta >= G) return;
    const long long ub = T * cta / G, ue = T * (cta + 1) / G;
    if (ub >= before && ub < before + mine) {
      long long off = ub - before, hu = 0;
      int i = i0;
      SeqInfo s;
      for (;; ++i) {
        s = seq_info(a, i);
        hu = head_units(a, s, lane);
        if (off < hu * a.H) break;
        off -= hu * a.H;
      }
      const int head = (int)(off / hu);
      off -= (long long)head * hu;
      int qt = 0;
      for (;; qt += 32) {  // 32 row tiles at a time
        const int n = row_tiles(a, s);
        long long v = qt + lane < n ? row_tile(a, s, qt + lane).units : 0, x = v;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const long long o = __shfl_up_sync(0xffffffffu, x, d);
          if (lane >= d) x += o;
        }
        const uint32_t in = __ballot_sync(0xffffffffu, off < x);
        if (in != 0) {
          const int k = __ffs(in) - 1;
          off -= __shfl_sync(0xffffffffu, x - v, k);
          qt += k;
          break;
        }
        off -= __shfl_sync(0xffffffffu, x, 31);
      }
      if (lane == 0) start = RangeStart{ub, ue, T, G, i, head, qt, (int)off};
    }
  }

  // ---- barriers, tensor memory ---------------------------------------------------------------------------------
  const uint32_t bars = sm + L::BAR_OFF;
  auto k_full = [&](int s) { return bars + 8u * s; };
  auto k_free = [&](int s) { return bars + 16u + 8u * s; };
  auto v_full = [&](int s) { return bars + 32u + 8u * s; };
  auto v_free = [&](int s) { return bars + 48u + 8u * s; };
  const uint32_t s_full = bars + 64u, o_done = bars + 72u;
  if (tid == 0) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(k_full(s), 4);
      mbar_init(k_free(s), 1);
      mbar_init(v_full(s), 4);
      mbar_init(v_free(s), 1);
    }
    mbar_init(s_full, 2);   // the MMAs' completion and the issuing thread itself (for the tile's factors)
    mbar_init(o_done, 1);
    mbar_init_fence();
  }
  constexpr uint32_t COLS = 256;
  if (wid == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_before_sync();
  __syncthreads();
  tc_after_sync();
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0);
  const uint32_t t_s = tmem, t_q = tmem + 64, t_o = tmem + 128;  // S (and the weights over it), Q, O

  long long u = start.u_begin;
  const long long u_end = start.u_end, T = start.total, G = start.ctas;
  int seq = start.seq, head = start.head, qt = start.qt, r0 = start.r0;
  SeqInfo s = seq_info(a, seq);
  int it = 0;        // tiles so far: stage and phase of every ring
  // A wait that gave up: from there on this thread only walks through, so that every barrier of the four softmax
  // warps is met by all of them.
  bool ok = true;

  while (u < u_end) {
    while (row_tiles(a, s) == 0) s = seq_info(a, ++seq);  // sequences of the other kernel
    const RowTile t = row_tile(a, s, qt);
    const int r1 = (int)min((long long)t.units, r0 + (u_end - u));
    const int n_tiles = r1 - r0;

    if (wid >= 4) {
      // ------------------------------ conversion ------------------------------
      constexpr int PIECES = D / 16, PASSES = AC_TILE * PIECES / 128;
      const int ct = tid - 128;
      const int* bt = a.bt + (long long)seq * a.bt_stride;
      const size_t slab = (size_t)head * a.npages;
      uint4 kr[PASSES], vr[PASSES];
      float sk = 0.0f, sv = -1.0f;  // of block ct of the tile (threads 0-3)
      auto load = [&](int r) {
        const int p0 = r * AC_TILE;
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
          const int e = i * 128 + ct, row = e / PIECES, pos = p0 + row;
          kr[i] = vr[i] = make_uint4(0, 0, 0, 0);
          if (pos < s.len) {
            const int pi = a.page_div.div(pos), pg = bt[pi];
            if ((unsigned)pg < (unsigned)a.npages) {
              const size_t at = ((slab + pg) * a.page + (pos - pi * a.page)) * D + (e - row * PIECES) * 16;
              kr[i] = __ldg((const uint4*)(a.q_k + at));
              vr[i] = __ldg((const uint4*)(a.q_v + at));
            }
          }
        }
        if (ct < 4) {
          const int pos = p0 + 16 * ct;
          sk = 0.0f;
          sv = -1.0f;
          if (pos < s.len) {
            const int pg = bt[a.page_div.div(pos)];
            if ((unsigned)pg < (unsigned)a.npages) {
              sk = a.s_k[slab + pg];
              sv = a.s_v[slab + pg];
            } else {
              atomicExch(a.status, ST_KV_PAGE);
            }
          }
        }
      };
      auto store = [&](const uint4& raw, uint32_t tile, int i) {
        const int e = i * 128 + ct, row = e / PIECES, piece = e - row * PIECES;
        uint4 h0, h1;
        e4m3x4_to_h2(raw.x, h0.x, h0.y);
        e4m3x4_to_h2(raw.y, h0.z, h0.w);
        e4m3x4_to_h2(raw.z, h1.x, h1.y);
        e4m3x4_to_h2(raw.w, h1.z, h1.w);
        const int blk = piece >> 2, c = (piece & 3) * 2;
        const uint32_t base = tile + blk * (AC_TILE * 128) + row * 128;
        // the two blocks' lanes take the halves in opposite order: all eight 16-byte slots at once
        const uint32_t a0 = base + ((c ^ (row & 7)) << 4), a1 = base + (((c + 1) ^ (row & 7)) << 4);
        sts128(blk ? a1 : a0, blk ? h1 : h0);
        sts128(blk ? a0 : a1, blk ? h0 : h1);
      };
      load(r0);
      for (int j = 0; j < n_tiles && ok; ++j) {
        const int st = (it + j) & 1;
        const uint32_t ph = (uint32_t)((it + j) >> 1) & 1u;
        ok = __all_sync(0xffffffffu, mbar_wait(k_free(st), ph ^ 1u, a.status, ST_FLASH_TIMEOUT));
        if (!ok) break;
#pragma unroll
        for (int i = 0; i < PASSES; ++i) store(kr[i], sm + L::K_OFF + st * L::TILE_BYTES, i);
        if (ct < 4) {
          // a block without positions (behind the end, or of no page) weighs nothing: exponent -inf
          const bool on = sv >= 0.0f;
          const float v = fmaxf(sv, 1e-30f);
          *(float4*)(smp + L::META_OFF + (((it + j) & 3) * 4 + ct) * 16) =
              make_float4(on ? sk * (a.scale * AB_LOG2E) : 0.0f, on ? lg2(v) : -INFINITY, on ? 1.0f / v : 0.0f, 0.0f);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(k_full(st));
        ok = __all_sync(0xffffffffu, mbar_wait(v_free(st), ph ^ 1u, a.status, ST_FLASH_TIMEOUT));
        if (!ok) break;
#pragma unroll
        for (int i = 0; i < PASSES; ++i) store(vr[i], sm + L::V_OFF + st * L::TILE_BYTES, i);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(v_full(st));
        if (j + 1 < n_tiles) load(r0 + j + 1);
      }
    } else {
      // ------------------------------ softmax: one thread per query row ------------------------------
      const uint32_t lane_off = (uint32_t)(wid * 32) << 16;
      const int row = qt * AC_ROWS + tid;
      const bool on = tid < t.rows;
      const int tq = on ? row / a.group : 0, hq = head * a.group + (on ? row - tq * a.group : 0);
      const int lim = !on ? 0 : (a.causal ? s.len - s.nq + tq + 1 : s.len);
      // D = F32, A = B = F16; S: B (K) K-major; O: B (V) MN-major. By the elected thread of warp 0.
      constexpr uint32_t id_s = (1u << 4) | ((uint32_t)(AC_TILE >> 3) << 17) | ((uint32_t)(AC_ROWS >> 4) << 24);
      constexpr uint32_t id_o = (1u << 4) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(AC_ROWS >> 4) << 24);
      auto scores = [&](int j) {
        const int st = (it + j) & 1;
        if (!mbar_wait(k_full(st), (uint32_t)((it + j) >> 1) & 1u, a.status, ST_FLASH_TIMEOUT)) return;
        tc_after_sync();
        const uint64_t db = operand_desc(sm + L::K_OFF + st * L::TILE_BYTES, 1);
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          mma_ts(t_s, t_q + 8 * k, db + (uint64_t)((k >> 2) * (AC_TILE * 128 / 16) + (k & 3) * 2), id_s, k > 0);
        mma_commit(k_free(st));
        mma_commit(s_full);
        mbar_arrive(s_full);
      };
      auto values = [&](int j) {
        const int st = (it + j) & 1;
        if (!mbar_wait(v_full(st), (uint32_t)((it + j) >> 1) & 1u, a.status, ST_FLASH_TIMEOUT)) return;
        tc_after_sync();
        const uint64_t db = operand_desc(sm + L::V_OFF + st * L::TILE_BYTES, AC_TILE * 128 / 16);
#pragma unroll
        for (int k = 0; k < AC_TILE / 16; ++k)  // 16 positions: 16 rows of 128 bytes
          mma_ts(t_o, t_s + 8 * k, db + (uint64_t)(k * (16 * 128 / 16)), id_o, j > 0 || k > 0);
        mma_commit(v_free(st));
        mma_commit(o_done);
      };
      // all four warps' stores to tensor memory are done
      auto meet = [&]() {
        tmem_wait_st();
        tc_before_sync();
        asm volatile("bar.sync 1, 128;" ::: "memory");
        tc_after_sync();
      };
      // Q to tensor memory as FP16 (BF16: by a power of two of the row's own, see attn_b8.cu)
      float scale_row = 1.0f;
      {
        const uint4* q = (const uint4*)((const uint16_t*)a.q + (long long)(s.q0 + tq) * a.q_stride + (size_t)hq * D);
        float up = 1.0f;
        if (BF16) {
          uint32_t top = 0;
          for (int i = 0; i < D / 8; ++i) {
            const uint4 v = on ? q[i] : make_uint4(0, 0, 0, 0);
            top = __vmaxu2(top, __vmaxu2(__vmaxu2(v.x & 0x7FFF7FFFu, v.y & 0x7FFF7FFFu),
                                         __vmaxu2(v.z & 0x7FFF7FFFu, v.w & 0x7FFF7FFFu)));
          }
          bf16_row_scale(max(top & 0xFFFFu, top >> 16), up, scale_row);
        }
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
          uint32_t h[32];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const uint4 v = on ? q[8 * c + i] : make_uint4(0, 0, 0, 0);
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) h[4 * i + k] = BF16 ? bf16x2_to_h2(w[k], up) : w[k];
          }
          tmem_st32(t_q + 32 * c + lane_off, h);
        }
        meet();
        if (wid == 0 && ok && elect_one()) scores(0);
        __syncwarp();
      }
      float m = AB_NONE, l = 0.0f;
      for (int j = 0; j < n_tiles; ++j) {
        ok = ok && mbar_wait(s_full, (uint32_t)(it + j) & 1u, a.status, ST_FLASH_TIMEOUT);
        ok = __all_sync(0xffffffffu, ok);
        tc_after_sync();
        float x[AC_TILE];
        tmem_ld32(t_s + lane_off, (uint32_t*)x);
        tmem_ld32(t_s + 32 + lane_off, (uint32_t*)x + 32);
        tmem_wait_ld();
        const float4* meta = (const float4*)(smp + L::META_OFF) + ((it + j) & 3) * 4;
        float inv[4];
        const int p0 = (r0 + j) * AC_TILE;
        float top = -INFINITY;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const float4 f = meta[b];
          const float fk = f.x * scale_row;
          inv[b] = f.z;
#pragma unroll
          for (int i = 0; i < 16; ++i) x[16 * b + i] = fmaf(x[16 * b + i], fk, f.y);
        }
        if (p0 + AC_TILE > t.all_see) {
#pragma unroll
          for (int i = 0; i < AC_TILE; ++i)
            if (p0 + i >= lim) x[i] = -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < AC_TILE; ++i) top = fmaxf(top, x[i]);
        if (__any_sync(0xffffffffu, top > m + AB_SLACK)) {
          const float mn = top > m + AB_SLACK ? top : m, f = ex2(m - mn);
          m = mn;
          l *= f;
          if (j > 0) {
            ok = ok && mbar_wait(o_done, (uint32_t)(it + j - 1) & 1u, a.status, ST_FLASH_TIMEOUT);
            ok = __all_sync(0xffffffffu, ok);
            tc_after_sync();
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              uint32_t o[32];
              tmem_ld32(t_o + 32 * c + lane_off, o);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
              tmem_st32(t_o + 32 * c + lane_off, o);
            }
            tmem_wait_st();
          }
        }
        uint32_t w[32];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          float sum = 0.0f;
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            const float w0 = ex2(x[16 * b + i] - m), w1 = ex2(x[16 * b + i + 1] - m);
            sum += w0 + w1;
            w[8 * b + i / 2] = h2_as_u32(__floats2half2_rn(w0, w1));
          }
          l = fmaf(sum, inv[b], l);
        }
        tmem_st32(t_s + lane_off, w);
        meet();
        if (wid == 0 && ok && elect_one()) {
          values(j);
          if (j + 1 < n_tiles) scores(j + 1);
        }
        __syncwarp();
      }
      // ---- the row's result, or its part of it ----
      ok = ok && mbar_wait(o_done, (uint32_t)(it + n_tiles - 1) & 1u, a.status, ST_FLASH_TIMEOUT);
      ok = __all_sync(0xffffffffu, ok);
      {
        tc_after_sync();
        const long long cta = blockIdx.x;
        const long long row_begin = u - r0, row_end = row_begin + t.units;
        const int first_cta = (int)(((row_begin + 1) * G - 1) / T), last_cta = (int)((row_end * G - 1) / T);
        const bool whole = first_cta == last_cta;
        uint16_t* out = (uint16_t*)a.out + (long long)(s.q0 + tq) * a.out_stride + (size_t)hq * D;
        auto finish = [&](float ms, float ls) {
          if (a.lse) a.lse[(long long)(s.q0 + tq) * (a.H * a.group) + hq] = row_lse(ms, ls);
        };
        auto store32 = [&](int c, const float* v, float scale) {
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            uint32_t h[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) h[k] = pack_out<BF16>(v[i + 2 * k] * scale, v[i + 2 * k + 1] * scale);
            *(uint4*)(out + 32 * c + i) = make_uint4(h[0], h[1], h[2], h[3]);
          }
        };
        int* counters = (int*)a.chunk_ws;
        float* parts = (float*)((uint8_t*)a.chunk_ws + counter_bytes((int)gridDim.x));
        constexpr size_t PART = (size_t)AC_ROWS * (D + 2);
        auto slot = [&](int k) { return parts + (size_t)(k == first_cta ? 2 * k + 1 : 2 * k) * PART; };
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          float o[32];
          tmem_ld32(t_o + 32 * c + lane_off, (uint32_t*)o);
          tmem_wait_ld();
          if (whole) {
            if (on) store32(c, o, row_norm(l));
          } else {
            // [D / 4][row][4]: consecutive rows next to each other
            float* p = slot((int)cta) + 2 * AC_ROWS + (size_t)(8 * c) * AC_ROWS * 4 + tid * 4;
#pragma unroll
            for (int i = 0; i < 8; ++i)
              *(float4*)(p + (size_t)i * AC_ROWS * 4) = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
          }
        }
        tc_before_sync();
        if (whole) {
          if (on) finish(m, l);
        } else {
          *(float2*)(slot((int)cta) + 2 * tid) = make_float2(m, l);
          __threadfence();
          asm volatile("bar.sync 1, 128;" ::: "memory");
          if (tid == 0) {
            const int want = last_cta - first_cta + 1;
            is_last = atomicAdd(counters + first_cta, 1) + 1 == want;
            if (is_last) counters[first_cta] = 0;  // as the next launch expects it
          }
          asm volatile("bar.sync 1, 128;" ::: "memory");
          if (is_last && on) {
            __threadfence();
            float ms = AB_NONE, ls = 0.0f;
            for (int k = first_cta; k <= last_cta; ++k) ms = fmaxf(ms, __ldcg(slot(k) + 2 * tid));
            for (int k = first_cta; k <= last_cta; ++k) {
              const float2 ml = __ldcg((const float2*)(slot(k) + 2 * tid));
              ls = fmaf(ml.y, ex2(ml.x - ms), ls);
            }
            const float norm = row_norm(ls);
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              float v[32];
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = 0.0f;
#pragma unroll 1
              for (int k = first_cta; k <= last_cta; ++k) {
                const float* p = slot(k) + 2 * AC_ROWS + (size_t)(8 * c) * AC_ROWS * 4 + tid * 4;
                const float f = ex2(__ldcg(slot(k) + 2 * tid) - ms);
                float4 o[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) o[i] = __ldcg((const float4*)(p + (size_t)i * AC_ROWS * 4));
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                  v[4 * i] = fmaf(o[i].x, f, v[4 * i]);
                  v[4 * i + 1] = fmaf(o[i].y, f, v[4 * i + 1]);
                  v[4 * i + 2] = fmaf(o[i].z, f, v[4 * i + 2]);
                  v[4 * i + 3] = fmaf(o[i].w, f, v[4 * i + 3]);
                }
              }
              store32(c, v, norm);
            }
            finish(ms, ls);
          }
        }
      }
    }
    // next row tile
    u += n_tiles;
    it += n_tiles;
    r0 = 0;
    if (++qt == row_tiles(a, s)) {
      qt = 0;
      if (++head == a.H) {
        head = 0;
        if (u < u_end) s = seq_info(a, ++seq);
      }
    }
  }
  tc_before_sync();
  __syncthreads();
  if (wid == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(COLS));
}

template <int D, bool BF16>
cudaError_t launch(const AttnB8& a, int sm_count, cudaStream_t stream) {
  auto* k = attn_b8_chunk_kernel<D, BF16>;
  const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, ChunkSmem<D>::BYTES);
  if (e != cudaSuccess) return e;
  k<<<AC_CTAS_PER_SM * sm_count, AC_THREADS, ChunkSmem<D>::BYTES, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace

size_t attn_b8_chunk_ws_bytes(int sm_count) {
  const int grid = AC_CTAS_PER_SM * sm_count;
  return counter_bytes(grid) + (size_t)2 * grid * AC_ROWS * (AB_MAX_D + 2) * sizeof(float);
}

cudaError_t attn_b8_chunk_launch(const AttnB8& a, int D, int bf16, int sm_count, cudaStream_t stream) {
  if (D == 128) return bf16 ? launch<128, true>(a, sm_count, stream) : launch<128, false>(a, sm_count, stream);
  return bf16 ? launch<64, true>(a, sm_count, stream) : launch<64, false>(a, sm_count, stream);
}

}  // namespace w4b
