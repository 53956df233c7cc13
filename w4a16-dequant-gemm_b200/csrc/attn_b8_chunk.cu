// Attention over a paged 8-bit cache for sequences with many query rows per key/value head (prompt chunks, encoder
// states): the same operator as attn_b8.cu, bound by the tensor pipe instead of HBM, on tcgen05.
//
// One CTA per SM works on a group of up to 256 query rows (token-major: row = token * group + head of the group) of one
// sequence and key/value head, and walks the positions in tiles of 64. Two warpgroups hold 128 rows each:
//   S = Q K^T        tcgen05.mma M = 128, N = 64; B = the K tile in shared memory
//   w = 2^(S * s_k * scale * log2 e + log2 s_v - m)      (why V's scale goes into the weights: attn_b8.cu)
//   O += w V         M = 128, N = D, K = 64; A = w from tensor memory, B = the V tile
// A group of at most 128 rows is given to both warpgroups, which take the tiles in turn and join their results in
// shared memory.
//   warps 0-7   one thread per query row (its TMEM lane): no reduction across threads anywhere. The reference point m
//               moves only when a score exceeds it by 2^15 (see attn_b8.cu); then O is rescaled in place.
//   warps 8-11  E4M3 -> FP16 (exact), once for both warpgroups: 16-byte loads two tiles ahead in registers, written to
//               swizzled operand tiles. K is K-major; V is stored the same way (row = position) and read MN-major.
//   warp 12     one elected thread issues all MMAs: the scores of a warpgroup's next tile as soon as it has read the
//               present ones, so that they run under its exponentials, then the weights' product. (With each warpgroup
//               issuing its own it waits them out: 280 us instead of 224 for the case below. elect.sync, not
//               "lane == 0": with a plain thread test an instruction took 92 cycles to issue whatever its size.)
// Tensor memory: S 2 x 64, w 2 x 32, O 2 x 128 columns and the first 64 dims of Q, 2 x 32; with D = 128 the other half
// of Q is in shared memory. An A operand in tensor memory is worth having: 42 cycles for 128 x 64 x 16 against 72 with
// A in shared memory (32 ideal; measured alone).
// Registers: 512 threads of 128 at launch, split 160 / 160 / 112 / 80 between the warpgroups.
//
// Split: units of one tile (two, for a group that both warpgroups share) over all (sequence, head, row group) in
// order, cut into equal ranges, as in attn_b8.cu; the causal limit of every group is in the count.
//
// Measured: 2 x 1k tokens on 4 to 6k positions, 32 query heads on 8 of 128, BF16: 210-214 us = 0.87-0.88 PFLOP/s, 0.53
// of the measured matrix rate. A tile takes about 2200 cycles where its products take 1500 and its exponentials 1024:
// what bounds it is the chain of one warpgroup - scores from tensor memory, maximum, exponentials, weights back - of
// which only two run side by side. Tried without gain: a quarter to a half of the exponentials as polynomials on the
// FMA pipe (215-228 against 218), holding the warpgroups half a tile apart (228), codes brought into L2 four tiles
// ahead (212 against 207; all with the reference point at the maximum, attn_b8.cuh). A group costs about 8 us besides its tiles when it is split between CTAs.
#include <cuda_bf16.h>
#include <float.h>

#include "attn_b8.cuh"

namespace w4b {
namespace {

constexpr int AC_ROWS = 128;          // query rows per warpgroup
constexpr int AC_GROUP = 2 * AC_ROWS;  // per CTA
constexpr int AC_TILE = 64;            // positions per tile
constexpr int AC_THREADS = 512;
constexpr int AC_WARPS = AC_THREADS / 32;
constexpr int AC_LIST = 32;            // sequences of a CTA's range that are looked up beforehand
constexpr int AC_MIN_UNITS = 4;        // units per CTA below which no further split pays
constexpr int AC_ROW_COST = 6;         // units a group counts for besides its tiles: its start, join and store take that long

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
__device__ __forceinline__ void mma_ss(uint32_t tmem_d, uint64_t da, uint64_t db, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
      "}\n" ::"r"(tmem_d),
      "l"(da), "l"(db), "r"(idesc), "r"((uint32_t)accumulate)
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

// two FP32 values in one register pair: one instruction for both
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pair(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ f32x2 pair(float a) { return pair(a, a); }
__device__ __forceinline__ float lo(f32x2 v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float hi(f32x2 v) { return __uint_as_float((uint32_t)(v >> 32)); }
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// A group of query rows, the positions it sees, and its units.
struct RowGroup {
  int rows;    // query rows in use
  int tiles;   // position tiles any row sees
  int units;   // AC_ROW_COST of no tiles, then at least one: a group that sees nothing still writes its zeros
  bool split;  // both warpgroups share the rows
};
__device__ __forceinline__ RowGroup row_group(const AttnB8& a, const SeqInfo& s, int gi) {
  RowGroup t;
  const int first = gi * AC_GROUP;
  t.rows = min(AC_GROUP, s.nq * a.group - first);
  t.split = t.rows <= AC_ROWS;
  const int end = positions_seen(a, s, (first + t.rows - 1) / a.group);
  t.tiles = max(1, (end + AC_TILE - 1) / AC_TILE);
  t.units = (t.split ? (t.tiles + 1) / 2 : t.tiles) + AC_ROW_COST;
  return t;
}
__device__ __forceinline__ int row_groups(const AttnB8& a, const SeqInfo& s) {
  const int rows = s.nq * a.group;
  return rows >= a.chunk_rows ? (rows + AC_GROUP - 1) / AC_GROUP : 0;
}
__device__ __forceinline__ long long warp_scan(long long v, int lane) {  // inclusive
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long o = __shfl_up_sync(0xffffffffu, v, d);
    if (lane >= d) v += o;
  }
  return v;
}
// Units of sequences i0 + lane (lane < n <= 32), all heads: a sequence of many groups by the whole warp, 32 at a time.
__device__ __forceinline__ long long warp_units(const AttnB8& a, int i0, int n, int lane) {
  SeqInfo s = {0, 0, 0, 0};
  if (lane < n) s = seq_info(a, i0 + lane);
  const int groups = row_groups(a, s);
  long long mine = 0;  // (a prompt of a million tokens over millions of positions has more units than 32 bits hold)
  if (groups <= 8)
    for (int gi = 0; gi < groups; ++gi) mine += row_group(a, s, gi).units;
  for (uint32_t big = __ballot_sync(0xffffffffu, groups > 8); big != 0; big &= big - 1) {
    const int k = __ffs(big) - 1, all = __shfl_sync(0xffffffffu, groups, k);
    const SeqInfo t = {__shfl_sync(0xffffffffu, s.len, k), 0, __shfl_sync(0xffffffffu, s.nq, k),
                       __shfl_sync(0xffffffffu, s.first, k)};
    long long sum = 0;
    for (int gi = lane; gi < all; gi += 32) sum += row_group(a, t, gi).units;
    sum = __shfl_sync(0xffffffffu, warp_scan(sum, lane), 31);
    if (lane == k) mine = sum;
  }
  return a.H * mine;
}

template <int D>
struct ChunkSmem {
  static constexpr int TILE_BYTES = AC_TILE * D * 2;  // an FP16 operand tile: D / 64 blocks of 64 rows x 128 bytes
  static constexpr int STAGES = 4;
  static constexpr int METAS = 2 * STAGES;             // a tile's factors outlive its stage: they are read after the scores
  static constexpr int META = METAS * 4 * 16;          // per tile: four blocks of 16 positions
  static constexpr int JOIN = AC_ROWS * (D + 2) * 4;   // the second warpgroup's result of a shared group
  // dims 64 .. 127 of both warpgroups' query rows (D = 128) share their place with the join buffer
  static constexpr int K_OFF = 0, V_OFF = STAGES * TILE_BYTES, Q_OFF = 2 * STAGES * TILE_BYTES, JOIN_OFF = Q_OFF;
  static constexpr int META_OFF = JOIN_OFF + JOIN, BAR_OFF = META_OFF + META;
  static constexpr int BYTES = BAR_OFF + 256 + 1024;   // + alignment
};

// 16 bytes, or zeros
__device__ __forceinline__ uint4 load_if(const uint8_t* p, bool on) {
  uint4 v;
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.u32 p, %5, 0;\n"
      "mov.b32 %0, 0;\nmov.b32 %1, 0;\nmov.b32 %2, 0;\nmov.b32 %3, 0;\n"
      "@p ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];\n"
      "}\n"
      : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w)
      : "l"(p), "r"((uint32_t)on));
  return v;
}

// where a CTA's range of units starts
struct RangeStart {
  long long u_begin, u_end, total, ctas;
  int head, gi, r0;
  int count;               // sequences with work in the range (the first AC_LIST of them are listed)
  int seq[AC_LIST];
  SeqInfo s[AC_LIST];
};

// A role's walk over its CTA's row groups.
struct Walk {
  int left;  // units still to do
  int idx;   // the sequence's place in the list
  int seq, head, gi, r0;
  int it;    // tiles so far: stage and phase of the rings
  SeqInfo s;
  RowGroup t;
  int n_units, tile0, n_tiles;  // of the present group
  __device__ __forceinline__ explicit Walk(const RangeStart& b)
      : left((int)(b.u_end - b.u_begin)), idx(0), seq(b.seq[0]), head(b.head), gi(b.gi), r0(b.r0), it(0), s(b.s[0]) {}
  __device__ __forceinline__ void next_sequence(const AttnB8& a, const RangeStart& b) {
    if (++idx < b.count) {
      seq = b.seq[idx];
      s = b.s[idx];
    } else {  // behind the list: one after the other, past those of the other kernel
      do s = seq_info(a, ++seq);
      while (row_groups(a, s) == 0);
    }
  }
  __device__ __forceinline__ bool more(const AttnB8& a, const RangeStart& b) {
    while (left > 0) {
      t = row_group(a, s, gi);
      n_units = min(t.units - r0, left);
      const int u0 = max(0, r0 - AC_ROW_COST), u1 = r0 + n_units - AC_ROW_COST;  // units that stand for tiles
      if (u1 > 0) {
        tile0 = t.split ? 2 * u0 : u0;
        n_tiles = min(t.split ? 2 * (u1 - u0) : u1 - u0, t.tiles - tile0);
        return true;
      }
      n_tiles = 0;
      next(a, b);
    }
    return false;
  }
  __device__ __forceinline__ void next(const AttnB8& a, const RangeStart& b) {
    left -= n_units;
    it += n_tiles;
    r0 = 0;
    if (++gi == row_groups(a, s)) {
      gi = 0;
      if (++head == a.H) {
        head = 0;
        if (left > 0) next_sequence(a, b);
      }
    }
  }
};

template <int D, bool BF16>
__global__ void __launch_bounds__(AC_THREADS, 1) attn_b8_chunk_kernel(const AttnB8 a) {
  using L = ChunkSmem<D>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ long long wsum[AC_WARPS];
  __shared__ RangeStart start;
  __shared__ uint32_t tmem_slot;
  __shared__ int is_last[2];
  const int tid = threadIdx.x, lane = tid & 31, wid = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const uint32_t sm = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smp = smem_raw + (sm - smem_u32(smem_raw));

  pdl_launch_dependents();  // the kernel for the short sequences may fill what this one leaves
  // ---- barriers and tensor memory by the last warp, beside the range by the others ------------------------------
  const uint32_t bars = sm + L::BAR_OFF;
  auto k_full = [&](int s) { return bars + 8u * s; };
  auto k_free = [&](int s) { return bars + 32u + 8u * s; };
  auto v_full = [&](int s) { return bars + 64u + 8u * s; };
  auto v_free = [&](int s) { return bars + 96u + 8u * s; };
  auto s_full = [&](int w) { return bars + 128u + 8u * w; };   // scores are there
  auto s_free = [&](int w) { return bars + 144u + 8u * w; };   // scores have been read
  auto w_full = [&](int w) { return bars + 160u + 8u * w; };   // weights are there
  auto o_done = [&](int w) { return bars + 176u + 8u * w; };   // their product is done: O may be read, w overwritten
  auto q_full = [&](int w) { return bars + 192u + 8u * w; };   // query rows are there
  constexpr uint32_t COLS = 512;
  if (wid == AC_WARPS - 1) {
    if (lane == 0) {
      for (int s = 0; s < L::STAGES; ++s) {
        mbar_init(k_full(s), 4);  // the conversion warps
        mbar_init(k_free(s), 1);
        mbar_init(v_full(s), 4);
        mbar_init(v_free(s), 1);
      }
      for (int w = 0; w < 2; ++w) {
        mbar_init(s_full(w), 2);  // the MMAs' completion and the issuing thread itself (for the tile's factors)
        mbar_init(s_free(w), 4);
        mbar_init(w_full(w), 4);
        mbar_init(o_done(w), 1);
        mbar_init(q_full(w), 4);
      }
      mbar_init_fence();
    }
    __syncwarp();
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // This CTA's range of units: the other warps take consecutive runs of sequences.
  constexpr int PLANNERS = AC_WARPS - 1;
  const int per = (a.nseq + PLANNERS - 1) / PLANNERS;
  const int i0 = min(wid * per, a.nseq), i1 = wid < PLANNERS ? min(i0 + per, a.nseq) : i0;
  long long mine = 0;
  for (int i = i0; i < i1; i += 32) mine += warp_units(a, i, min(32, i1 - i), lane);
  mine = __shfl_sync(0xffffffffu, warp_scan(mine, lane), 31);
  if (lane == 0) wsum[wid] = mine;
  tc_before_sync();
  __syncthreads();
  tc_after_sync();
  const long long upto = warp_scan(lane < AC_WARPS ? wsum[lane] : 0, lane);  // over the warps
  const long long T = __shfl_sync(0xffffffffu, upto, 31), before = __shfl_sync(0xffffffffu, upto, wid) - mine;
  const long long most = (T + AC_MIN_UNITS - 1) / AC_MIN_UNITS;
  const long long G = most < (long long)gridDim.x ? most : (long long)gridDim.x;
  const bool idle = (long long)blockIdx.x >= G;
  if (!idle) {
    const long long ub = range_begin(T, blockIdx.x, G), ue = range_begin(T, blockIdx.x + 1, G);
    if (ub >= before && ub < before + mine) {
      // the sequence that unit ub is in, and those after it up to unit ue
      long long base = before;
      int count = 0;
      for (int i = i0; i < a.nseq && base < ue; i += 32) {
        const int n = min(32, a.nseq - i);
        const long long v = warp_units(a, i, n, lane), end = base + warp_scan(v, lane);
        const bool in = v > 0 && end > ub && end - v < ue;
        const uint32_t all = __ballot_sync(0xffffffffu, in);
        const int at = count + __popc(all & ((1u << lane) - 1));
        if (in && at < AC_LIST) {
          start.seq[at] = i + lane;
          start.s[at] = seq_info(a, i + lane);
        }
        if (count == 0 && all != 0) {
          const int k = __ffs(all) - 1;
          const long long first = __shfl_sync(0xffffffffu, end - v, k), units = __shfl_sync(0xffffffffu, v, k);
          const SeqInfo s = seq_info(a, i + k);
          long long off = ub - first;
          const long long hu = (unsigned long long)units < 0x100000000ULL ? (unsigned)units / (unsigned)a.H : units / a.H;
          const int head = (off | hu) < 0x7FFFFFFF ? (int)off / (int)hu : (int)(off / hu);
          off -= (long long)head * hu;
          int gi = 0;
          for (;; gi += 32) {  // 32 groups at a time
            const long long u = gi + lane < row_groups(a, s) ? row_group(a, s, gi + lane).units : 0, x = warp_scan(u, lane);
            const uint32_t here = __ballot_sync(0xffffffffu, off < x);
            if (here != 0) {
              const int b = __ffs(here) - 1;
              off -= __shfl_sync(0xffffffffu, x - u, b);
              gi += b;
              break;
            }
            off -= __shfl_sync(0xffffffffu, x, 31);
          }
          if (lane == 0) {
            start.head = head;
            start.gi = gi;
            start.r0 = (int)off;
          }
        }
        count += __popc(all);
        base = __shfl_sync(0xffffffffu, end, 31);
      }
      if (lane == 0) {
        start.u_begin = ub;
        start.u_end = ue;
        start.total = T;
        start.ctas = G;
        start.count = min(count, AC_LIST);
      }
    }
  } else if (tid == 0) {
    start.u_begin = start.u_end = 0;  // nothing to do: every role's walk is empty
  }
  __syncthreads();
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0);

  // A wait that gave up: from there on this thread only walks through, so that every barrier of the warpgroups is met
  // by all of them.
  bool ok = true;
  // Registers: 128 threads x (160 + 160 + 112 + 80) = the 512 x 128 of the launch.
  if (wid >= 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    // ------------------------------ MMA issue ------------------------------
    if (wid == 12 && elect_one()) {
      int mine = 0, other = 0, segments = 0;  // tiles of the warpgroups, row groups so far: phases
      for (Walk k(start); k.more(a, start); k.next(a, start)) {
        const RowGroup& t = k.t;
        const int n_tiles = k.n_tiles, it = k.it;
        // D = F32, A = B = F16; S: B (K) K-major; O: B (V) MN-major
        constexpr uint32_t id_s = (1u << 4) | ((uint32_t)(AC_TILE >> 3) << 17) | ((uint32_t)(AC_ROWS >> 4) << 24);
        constexpr uint32_t id_o = (1u << 4) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(AC_ROWS >> 4) << 24);
        const int n[2] = {t.split ? (n_tiles + 1) / 2 : n_tiles, t.split ? n_tiles / 2 : n_tiles};
        auto wait = [&](uint32_t bar, int phase) {
          ok = ok && mbar_wait(bar, (uint32_t)phase & 1u, a.status, ST_FLASH_TIMEOUT);
        };
        auto scores = [&](int w, int i) {  // of the warpgroup's tile i
          const int j = it + (t.split ? 2 * i + w : i), st = j % L::STAGES, c = (w ? other : mine) + i;
          if (t.split || w == 0) wait(k_full(st), j / L::STAGES);
          if (c > 0) wait(s_free(w), c - 1);
          if (!ok) return;
          tc_after_sync();
          const uint32_t t_s = tmem + 64 * w, t_q = tmem + 192 + 32 * w;
          const uint64_t db = operand_desc(sm + L::K_OFF + st * L::TILE_BYTES, 1);
          const uint64_t da = operand_desc(sm + L::Q_OFF + w * (AC_ROWS * 128), 1);
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint64_t b = db + (uint64_t)((k >> 2) * (AC_TILE * 128 / 16) + (k & 3) * 2);
            if (k < 4) mma_ts(t_s, t_q + 8 * k, b, id_s, k > 0);
            else mma_ss(t_s, da + (uint64_t)((k & 3) * 2), b, id_s, true);
          }
          if (t.split || w == 1) mma_commit(k_free(st));
          mma_commit(s_full(w));
          mbar_arrive(s_full(w));
        };
        auto values = [&](int w, int i) {
          const int j = it + (t.split ? 2 * i + w : i), st = j % L::STAGES, c = (w ? other : mine) + i;
          if (t.split || w == 0) wait(v_full(st), j / L::STAGES);
          wait(w_full(w), c);
          if (!ok) return;
          tc_after_sync();
          const uint32_t t_w = tmem + 128 + 32 * w, t_o = tmem + 256 + 128 * w;
          const uint64_t db = operand_desc(sm + L::V_OFF + st * L::TILE_BYTES, AC_TILE * 128 / 16);
#pragma unroll
          for (int k = 0; k < AC_TILE / 16; ++k)  // 16 positions: 16 rows of 128 bytes
            mma_ts(t_o, t_w + 8 * k, db + (uint64_t)(k * (16 * 128 / 16)), id_o, i > 0 || k > 0);
          if (t.split || w == 1) mma_commit(v_free(st));
          mma_commit(o_done(w));
        };
        wait(q_full(0), segments);
        wait(q_full(1), segments);
        scores(0, 0);
        if (n[1] > 0) scores(1, 0);
#pragma unroll 1
        for (int i = 0; i < n[0]; ++i) {
          if (i + 1 < n[0]) scores(0, i + 1);
          if (i + 1 < n[1]) scores(1, i + 1);
          values(0, i);
          if (i < n[1]) values(1, i);
        }
        mine += n[0];
        other += n[1];
        ++segments;
      }
    }
    __syncwarp();
  } else if (wid >= 8) {
    // ------------------------------ conversion ------------------------------
    asm volatile("setmaxnreg.dec.sync.aligned.u32 112;");
    for (Walk k(start); k.more(a, start); k.next(a, start)) {
      const SeqInfo& s = k.s;
      const int n_tiles = k.n_tiles, tile0 = k.tile0, it = k.it;
      // A pass covers 128 pieces of 16 bytes: 16 rows (D = 128) or 32 (D = 64). Eight consecutive lanes take four
      // pieces of the same 64 columns in two neighbouring rows: their FP16 halves meet all eight 16-byte slots.
      constexpr int PASSES = D / 32, ROWS = 64 / PASSES;
      const int ct = tid - 256, quad = lane >> 3;
      const int row0 = (D == 128 ? 4 * (wid - 8) + 2 * (quad >> 1) : 8 * (wid - 8) + 2 * quad) + ((lane >> 2) & 1);
      const int blk = D == 128 ? quad & 1 : 0, piece = 4 * blk + (lane & 3);
      const uint32_t dst = blk * (AC_TILE * 128) + row0 * 128;  // (ROWS is a multiple of 8: the swizzle is every pass's)
      const uint32_t dst0 = dst + (((2 * (lane & 3)) ^ (row0 & 7)) << 4), dst1 = dst + (((2 * (lane & 3) + 1) ^ (row0 & 7)) << 4);
      const int* bt = a.bt + (long long)k.seq * a.bt_stride;
      const size_t slab = (size_t)k.head * a.npages, base = slab * a.page * D + piece * 16;
      const uint8_t *kb = a.q_k + base, *vb = a.q_v + base;
      // Two tiles' codes in registers: while one is converted the other is on its way.
      struct Raw {
        uint4 k[PASSES], v[PASSES];
        float sk, sv;  // of block ct of the tile (threads 0-3)
      } raw[2];
      // Lane b < 4 of every warp looks up the row of block b of a tile, one tile ahead of the loads that need it.
      // (Looked up where it is used, four dependent loads in a row made this the slowest role: 1600 cycles a tile.)
      int pg = -1, in_page = 0;
      const bool scales = ct < 4;
      auto pages = [&](int r) {
        const int pos = r * AC_TILE + 16 * (lane & 3), pi = a.page_div.div(pos);
        pg = pos < s.len && lane < 4 ? __ldg(bt + pi) : -1;
        in_page = pos - pi * a.page;
      };
      auto load = [&](Raw& w, int r) {
        const bool there = (unsigned)pg < (unsigned)a.npages;
        const int row = there ? pg * a.page + in_page : -1;
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
          const int b = D == 128 ? i : 2 * i + (row0 >> 4);  // block of this pass's row
          const int first = __shfl_sync(0xffffffffu, row, b);
          const int in = row0 & 15;
          const bool on = first >= 0 && r * AC_TILE + 16 * b + in < s.len;
          const size_t at = (size_t)(on ? first + in : 0) * D;
          w.k[i] = load_if(kb + at, on);
          w.v[i] = load_if(vb + at, on);
        }
        if (scales) {
          w.sk = there ? __ldg(a.s_k + slab + pg) : 0.0f;
          w.sv = there ? __ldg(a.s_v + slab + pg) : -1.0f;
          if (!there && r * AC_TILE + 16 * ct < s.len) atomicExch(a.status, ST_KV_PAGE);
        }
      };
      auto store = [&](const uint4& raw, uint32_t tile, int i) {
        uint4 h0, h1;
        e4m3x4_to_h2(raw.x, h0.x, h0.y);
        e4m3x4_to_h2(raw.y, h0.z, h0.w);
        e4m3x4_to_h2(raw.z, h1.x, h1.y);
        e4m3x4_to_h2(raw.w, h1.z, h1.w);
        sts128(tile + i * (ROWS * 128) + dst0, h0);
        sts128(tile + i * (ROWS * 128) + dst1, h1);
      };
      auto convert = [&](const Raw& w, int j) {
        const int st = (it + j) % L::STAGES;
        const uint32_t ph = (uint32_t)((it + j) / L::STAGES) & 1u;
        ok = ok && mbar_wait(k_free(st), ph ^ 1u, a.status, ST_FLASH_TIMEOUT);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) return;
#pragma unroll
        for (int i = 0; i < PASSES; ++i) store(w.k[i], sm + L::K_OFF + st * L::TILE_BYTES, i);
        if (ct < 4) {
          // a block without positions (behind the end, or of no page) weighs nothing: exponent -inf
          const bool on = w.sv >= 0.0f;
          const float v = fmaxf(w.sv, 1e-30f);
          *(float4*)(smp + L::META_OFF + ((it + j) % L::METAS * 4 + ct) * 16) =
              make_float4(on ? w.sk : 0.0f, on ? lg2(v) : -INFINITY, on ? 1.0f / v : 0.0f, 0.0f);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(k_full(st));
        ok = __all_sync(0xffffffffu, mbar_wait(v_free(st), ph ^ 1u, a.status, ST_FLASH_TIMEOUT));
        if (!ok) return;
#pragma unroll
        for (int i = 0; i < PASSES; ++i) store(w.v[i], sm + L::V_OFF + st * L::TILE_BYTES, i);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(v_full(st));
      };
      pages(tile0);
      load(raw[0], tile0);
      pages(tile0 + 1);
      for (int j = 0; j < n_tiles && ok; j += 2) {
        if (j + 1 < n_tiles) {
          load(raw[1], tile0 + j + 1);
          pages(tile0 + j + 2);
        }
        convert(raw[0], j);
        if (j + 2 < n_tiles) {
          load(raw[0], tile0 + j + 2);
          pages(tile0 + j + 3);
        }
        if (j + 1 < n_tiles) convert(raw[1], j + 1);
      }
    }
  } else {
    // ------------------------------ softmax: one thread per query row ------------------------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 160;");
    int mine = 0;  // tiles of this warpgroup so far: phase of its barriers
    for (Walk k(start); k.more(a, start); k.next(a, start)) {
      const SeqInfo& s = k.s;
      const RowGroup& t = k.t;
      const int n_tiles = k.n_tiles, tile0 = k.tile0, it = k.it;
      const int head = k.head;
      const int w = wid >> 2, rt = tid & (AC_ROWS - 1);  // warpgroup, row of its tile
      const uint32_t lane_off = (uint32_t)((wid & 3) * 32) << 16;
      const uint32_t t_s = tmem + 64 * w, t_w = tmem + 128 + 32 * w, t_q = tmem + 192 + 32 * w, t_o = tmem + 256 + 128 * w;
      const int row_in = rt + (t.split ? 0 : AC_ROWS * w), row = k.gi * AC_GROUP + row_in;
      const bool on = row_in < t.rows;
      const int tq = on ? row / a.group : 0, hq = head * a.group + (on ? row - tq * a.group : 0);
      const int lim = on ? positions_seen(a, s, tq) : 0;
      const int all_see = positions_seen(a, s, (row - rt) / a.group);  // positions all rows of the warpgroup see
      const int j_first = t.split ? w : 0, j_step = t.split ? 2 : 1;
      // this warp's accesses to tensor memory are done: tell the issuing thread
      auto signal = [&](uint32_t bar) {
        tc_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar);
      };
      // Q: each warp reads its 32 rows along the rows (one thread a row would touch 32 lines at every load: 6000
      // cycles) into swizzled 128-byte rows of shared memory; then each thread makes its own row FP16 (BF16: by a
      // power of two of the row's own, see attn_b8.cu), the first 64 dims to tensor memory, the others in place.
      float scale_row = 1.0f;
      {
        constexpr int LPR = D / 8, RPL = 32 / LPR;  // lanes per row, rows per load
        const uint32_t q_hi = sm + L::Q_OFF + w * (AC_ROWS * 128), q_lo = q_hi + (D == 128 ? 2 * AC_ROWS * 128 : 0);
        const int piece = lane % LPR;
        uint4 v[32 / RPL];
#pragma unroll
        for (int i = 0; i < 32 / RPL; ++i) {
          const int r_in = (wid & 3) * 32 + i * RPL + lane / LPR + (t.split ? 0 : AC_ROWS * w);
          const int r = k.gi * AC_GROUP + r_in, tok = r / a.group, hh = k.head * a.group + (r - tok * a.group);
          v[i] = r_in < t.rows ? __ldg((const uint4*)((const uint16_t*)a.q + (long long)(s.q0 + tok) * a.q_stride + (size_t)hh * D) + piece)
                               : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 32 / RPL; ++i) {
          const int r = (wid & 3) * 32 + i * RPL + lane / LPR;
          sts128((piece >= 8 ? q_hi : q_lo) + r * 128 + (((piece & 7) ^ (r & 7)) << 4), v[i]);
        }
        __syncwarp();
        auto at = [&](int p) { return (p >= 8 ? q_hi : q_lo) + rt * 128 + (((p & 7) ^ (rt & 7)) << 4); };
        float up = 1.0f;
        if (BF16) {
          uint32_t top = 0;
#pragma unroll
          for (int p = 0; p < LPR; ++p) {
            const uint4 x = lds128(at(p));
            top = __vmaxu2(top, __vmaxu2(__vmaxu2(x.x & 0x7FFF7FFFu, x.y & 0x7FFF7FFFu),
                                         __vmaxu2(x.z & 0x7FFF7FFFu, x.w & 0x7FFF7FFFu)));
          }
          bf16_row_scale(max(top & 0xFFFFu, top >> 16), up, scale_row);
#pragma unroll
          for (int p = 8; p < LPR; ++p) {
            const uint4 x = lds128(at(p));
            sts128(at(p), make_uint4(bf16x2_to_h2(x.x, up), bf16x2_to_h2(x.y, up), bf16x2_to_h2(x.z, up), bf16x2_to_h2(x.w, up)));
          }
        }
        uint32_t h[32];
#pragma unroll
        for (int p = 0; p < 8; ++p) {
          const uint4 x = lds128(at(p));
          h[4 * p] = BF16 ? bf16x2_to_h2(x.x, up) : x.x;
          h[4 * p + 1] = BF16 ? bf16x2_to_h2(x.y, up) : x.y;
          h[4 * p + 2] = BF16 ? bf16x2_to_h2(x.z, up) : x.z;
          h[4 * p + 3] = BF16 ? bf16x2_to_h2(x.w, up) : x.w;
        }
        scale_row *= a.scale * AB_LOG2E;  // (in this order: a large row may come with a small scale, and the other way round)
        tmem_st32(t_q + lane_off, h);
        if (D == 128) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        tmem_wait_st();
        signal(q_full(w));
      }
      // While a row has seen nothing (`bare`) its reference point is 0; the first tile with a score sets it.
      float m = 0.0f, l = 0.0f;
      bool bare = true;
      // A barrier that is through costs some 150 cycles to ask all the same; so it is asked while the exponentials
      // run, and waited for only if it was not through then. (Nothing the warp does depends on `ok` but its waits.)
      auto await = [&](uint32_t bar, int phase, bool through) {
        if (!through) ok = ok && mbar_wait(bar, (uint32_t)phase & 1u, a.status, ST_FLASH_TIMEOUT);
        __syncwarp();
        tc_after_sync();
      };
      bool s_there = false;
      for (int j = j_first; j < n_tiles; j += j_step, ++mine) {
        await(s_full(w), mine, s_there);
        union {
          uint32_t u[AC_TILE];
          float f[AC_TILE];
          f32x2 p[AC_TILE / 2];
        } x;
        const float4* meta = (const float4*)(smp + L::META_OFF) + ((it + j) % L::METAS) * 4;
        const int p0 = (tile0 + j) * AC_TILE;
        float inv[4], top = -INFINITY;
        // exponents X - m; the second half's load runs under the first half's arithmetic
        tmem_ld32(t_s + lane_off, x.u);
        tmem_wait_ld();
        tmem_ld32(t_s + 32 + lane_off, x.u + 32);
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          if (b == 2) {
            tmem_wait_ld();
            signal(s_free(w));
          }
          const float4 f = meta[b];
          const f32x2 fk = pair(f.x * scale_row), fc = pair(f.y - m);
          inv[b] = f.z;
#pragma unroll
          for (int i = 0; i < 8; ++i) x.p[8 * b + i] = fma2(x.p[8 * b + i], fk, fc);
        }
        if (p0 + AC_TILE > all_see) {
#pragma unroll
          for (int i = 0; i < AC_TILE; ++i)
            if (p0 + i >= lim) x.f[i] = -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < AC_TILE; i += 2) top = max3(top, x.f[i], x.f[i + 1]);
        const bool move = bare ? top > -INFINITY : top > AB_SLACK;
        if (__any_sync(0xffffffffu, move)) {
          const float by = move ? top - AB_BELOW : 0.0f, f = bare ? 0.0f : ex2(-by);  // (nothing to scale while bare)
          m += by;
          l *= f;
          bare = bare && !move;
          const f32x2 neg = pair(-by);
#pragma unroll
          for (int i = 0; i < AC_TILE / 2; ++i) x.p[i] = add2(x.p[i], neg);
          if (j > j_first) {
            await(o_done(w), mine - 1, false);
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
        // O and the place of the weights are free again; the next scores are there
        // (unconditionally: a branch on the answer would wait for it here)
        const bool o_test = mbar_test(o_done(w), (uint32_t)(mine - 1) & 1u), s_test = mbar_test(s_full(w), (uint32_t)(mine + 1) & 1u);
        uint32_t wt[32];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          f32x2 sum = pair(0.0f);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const f32x2 e = pair(ex2(x.f[16 * b + 2 * i]), ex2(x.f[16 * b + 2 * i + 1]));
            sum = add2(sum, e);
            wt[8 * b + i] = h2_as_u32(__floats2half2_rn(lo(e), hi(e)));
          }
          l = fmaf(lo(sum) + hi(sum), inv[b], l);
        }
        await(o_done(w), mine - 1, o_test || j == j_first);
        s_there = s_test;
        tmem_st32(t_w + lane_off, wt);
        tmem_wait_st();
        signal(w_full(w));
      }
      if (bare) m = AB_NONE;
      // the join buffer lies over Q: both warpgroups have seen their last scores
      if (t.split) asm volatile("bar.sync 3, 256;" ::: "memory");
      // ---- the row's result, or its part of it ----
      const bool some = j_first < n_tiles;  // (the second warpgroup of a shared group of one tile has none)
      if (some) await(o_done(w), mine - 1, false);
      float* join = (float*)(smp + L::JOIN_OFF);  // [row][2], then [D / 4][row][4]
      if (t.split && w == 1) {
        *(float2*)(join + 2 * rt) = make_float2(m, l);
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          float o[32];
          if (some) {
            tmem_ld32(t_o + 32 * c + lane_off, (uint32_t*)o);
            tmem_wait_ld();
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = 0.0f;
          }
          float* p = join + 2 * AC_ROWS + (8 * c * AC_ROWS + rt) * 4;
#pragma unroll
          for (int i = 0; i < 8; ++i)
            *(float4*)(p + i * AC_ROWS * 4) = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
        }
        tc_before_sync();
        asm volatile("bar.sync 3, 256;" ::: "memory");
      } else {
        float f0 = 1.0f, f1 = 0.0f;  // factors of this warpgroup's and the other's part
        if (t.split) {
          asm volatile("bar.sync 3, 256;" ::: "memory");
          const float2 other = *(const float2*)(join + 2 * rt);
          const float ms = fmaxf(m, other.x);
          f0 = ex2(m - ms);
          f1 = ex2(other.x - ms);
          m = ms;
          l = l * f0 + other.y * f1;
        }
        const long long G = start.ctas, T = start.total;
        const int cta = (int)blockIdx.x;
        const bool whole = k.r0 <= AC_ROW_COST && k.r0 + k.n_units == t.units;
        const long long row_begin = start.u_end - k.left - k.r0;
        const int first_cta = whole ? cta : unit_owner(row_begin + AC_ROW_COST, T, G);
        const int last_cta = whole ? cta : unit_owner(row_begin + t.units - 1, T, G);
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
        int* counter = (int*)a.chunk_ws + 2 * first_cta + w;
        const int want = last_cta - first_cta + 1;
        constexpr size_t PART = (size_t)AC_ROWS * (D + 2);  // floats per warpgroup
        float* parts = (float*)((uint8_t*)a.chunk_ws + counter_bytes(2 * (int)gridDim.x)) + w * PART;
        auto slot = [&](int k) { return parts + (size_t)(k == first_cta ? 2 * k + 1 : 2 * k) * (2 * PART); };
        // this CTA's 32 columns of chunk c
        auto own = [&](int c, float* o) {
          tmem_ld32(t_o + 32 * c + lane_off, (uint32_t*)o);
          tmem_wait_ld();
          if (t.split) {
            const float* p = join + 2 * AC_ROWS + (8 * c * AC_ROWS + rt) * 4;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float4 v = *(const float4*)(p + i * AC_ROWS * 4);
              o[4 * i] = fmaf(o[4 * i], f0, v.x * f1);
              o[4 * i + 1] = fmaf(o[4 * i + 1], f0, v.y * f1);
              o[4 * i + 2] = fmaf(o[4 * i + 2], f0, v.z * f1);
              o[4 * i + 3] = fmaf(o[4 * i + 3], f0, v.w * f1);
            }
          }
        };
        if (whole) {
          const float norm = row_norm(l);
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            float o[32];
            own(c, o);
            if (on) store32(c, o, norm);
          }
          if (on) finish(m, l);
        } else {
          // The CTA that comes last joins all parts, in CTA order, its own from tensor memory. One that finds itself
          // last already need not write its part.
          auto ask = [&](bool add) {
            asm volatile("bar.sync %0, 128;" ::"r"(1 + w) : "memory");
            if (rt == 0) {
              int before;
              if (add) {
                // release (after the barrier: the whole warpgroup's writes) and acquire
                asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(before) : "l"(counter) : "memory");
              } else {
                asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(before) : "l"(counter) : "memory");
              }
              is_last[w] = before == want - 1;
              if (before == want - 1) *counter = 0;  // as the next launch expects it
            }
            asm volatile("bar.sync %0, 128;" ::"r"(1 + w) : "memory");
            return is_last[w] != 0;
          };
          bool last = ask(false);
          if (!last) {
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              float o[32];
              own(c, o);
              // [D / 4][row][4]: consecutive rows next to each other
              float* p = slot(cta) + 2 * AC_ROWS + (size_t)(8 * c * AC_ROWS + rt) * 4;
#pragma unroll
              for (int i = 0; i < 8; ++i)
                *(float4*)(p + (size_t)i * AC_ROWS * 4) = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
            }
            *(float2*)(slot(cta) + 2 * rt) = make_float2(m, l);
            last = ask(true);
          }
          if (last) {
            auto ml = [&](int k) { return k == cta ? make_float2(m, l) : __ldcg((const float2*)(slot(k) + 2 * rt)); };
            float ms = AB_NONE, ls = 0.0f;
            for (int k0 = first_cta; k0 <= last_cta; k0 += 4) {
              float2 v[4];
#pragma unroll
              for (int b = 0; b < 4; ++b) v[b] = ml(min(k0 + b, last_cta));
              float mn = ms;
#pragma unroll
              for (int b = 0; b < 4; ++b) mn = fmaxf(mn, v[b].x);
              ls *= ex2(ms - mn);
              ms = mn;
#pragma unroll
              for (int b = 0; b < 4; ++b)
                if (k0 + b <= last_cta) ls = fmaf(v[b].y, ex2(v[b].x - ms), ls);
            }
            const float norm = row_norm(ls);
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              float v[32];
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = 0.0f;
#pragma unroll 1
              for (int k = first_cta; k <= last_cta; ++k) {
                const float f = ex2(ml(k).x - ms);
                float o[32];
                if (k == cta) {
                  own(c, o);
                } else {
                  const float* p = slot(k) + 2 * AC_ROWS + (size_t)(8 * c * AC_ROWS + rt) * 4;
#pragma unroll
                  for (int i = 0; i < 8; ++i) *(float4*)(o + 4 * i) = __ldcg((const float4*)(p + (size_t)i * AC_ROWS * 4));
                }
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] = fmaf(o[i], f, v[i]);
              }
              if (on) store32(c, v, norm);
            }
            if (on) finish(ms, ls);
          }
        }
        tc_before_sync();
      }
      if (t.split) asm volatile("bar.sync 3, 256;" ::: "memory");  // the join buffer is free again
    }
  }
  tc_before_sync();
  __syncthreads();
  if (wid == AC_WARPS - 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(COLS));
}

template <int D, bool BF16>
cudaError_t launch(const AttnB8& a, int sm_count, cudaStream_t stream) {
  const cudaError_t e = opt_in_smem<attn_b8_chunk_kernel<D, BF16>>(ChunkSmem<D>::BYTES);
  if (e != cudaSuccess) return e;
  attn_b8_chunk_kernel<D, BF16><<<sm_count, AC_THREADS, ChunkSmem<D>::BYTES, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace

size_t attn_b8_chunk_ws_bytes(int sm_count) {
  return counter_bytes(2 * sm_count) + (size_t)2 * sm_count * AC_GROUP * (AB_MAX_D + 2) * sizeof(float);
}

cudaError_t attn_b8_chunk_launch(const AttnB8& a, int D, int bf16, int sm_count, cudaStream_t stream) {
  if (D == 128) return bf16 ? launch<128, true>(a, sm_count, stream) : launch<128, false>(a, sm_count, stream);
  return bf16 ? launch<64, true>(a, sm_count, stream) : launch<64, false>(a, sm_count, stream);
}

}  // namespace w4b
