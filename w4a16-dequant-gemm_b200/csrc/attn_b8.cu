// Attention over a paged 8-bit cache (E4M3 codes, one FP32 scale per page and key/value head), for a few query tokens
// per sequence: decode steps, drafted tokens, and the same without the causal mask over an encoder's states.
//
// Mathematics, per sequence and key/value head. The R = tokens * group query rows that share the head are columns of
//   X[pos][n] = (K q)[pos][n] * (s_k * scale * log2 e) + log2(s_v)         x = log2 of the weight of the CODE row of V
//   w = 2^(X - m),  O^T[d][n] += sum_pos Vcode[pos][d] * w[pos][n],  l[n] += w / s_v
// with m a reference point near the running maximum of X: taking log2(s_v) into the exponent puts V's scale into the
// weights for free, whatever its size, and w / s_v is the plain softmax weight. out = O / l, lse = ln 2 (m + log2 l).
// m moves only when some X exceeds it by more than 15 (a warp vote), so the usual block needs no reduction across
// lanes: weights up to 2^15 are halves like others, and sums are FP32.
//
// Both products run on mma.sync.m16n8k16 with the CACHE as the 16-row operand and the query rows as the 8 columns
// (a decode step has 1 to 16 rows: as the 128-row operand of the larger tensor instructions they would leave most of
// it empty, and at HBM speed this form needs a sixth of the mma.sync rate):
//   K: ldmatrix hands lane (g, c) bytes 4c..4c+3 of a 16-byte piece of positions g and g + 8; two conversions
//      E4M3x2 -> half2 make them the operand's registers (the k order is permuted, q is loaded in the same order);
//   V: ldmatrix.trans hands over dims 2g, 2g+1 of positions 2c, 2c+1; one byte permute pairs the positions, two
//      conversions make the transposed operand (row g = dim 2g, row g + 8 = dim 2g + 1).
// E4M3 -> FP16 is exact. The weights go from accumulator to operand layout by movmatrix.
//
// Bound by HBM: the cache is read once per column tile, so once for up to 16 query rows a head and twice for 17 to 32.
// Each warp keeps its own ring of 16-position blocks (K and V, 4 KB at D = 128) filled by cp.async two blocks ahead
// (D = 64: five), without any barrier between warps.
//
// Split: all work - 64-position units of all (sequence, head, column tile) rows in order - is cut into equal ranges,
// one per CTA, whatever the lengths; the lengths are on the device, so every CTA sums them itself. A row that spans
// CTAs is joined by whichever of them arrives last, in CTA order (bit-identical from run to run).
//
// Measured (device time in a graph): 4 sequences x 131,072 positions, 32 query heads on 8 of 128: 191 us = 5.6 TB/s,
// 0.86 of the measured copy rate; 64 sequences of 100 to 8192 positions, 64 heads on 8 of 128: 56 us = 4.5 TB/s (0.68;
// 5 us of it are launch, the sums over the lengths and the first loads, 70 us without AB_ROW_COST: CTAs with many
// short rows came late); one sequence of 778: 8.5 us. (The 16-column form at D = 128 spills 76 bytes: four CTAs an SM
// leave 128 registers.)
#include "attn_b8.cuh"

namespace w4b {
namespace {

constexpr int AB_WARPS = 4;
constexpr int AB_THREADS = 32 * AB_WARPS;
constexpr int AB_CTAS_PER_SM = 4;
constexpr int AB_UNIT = 64;      // positions per work unit: one block of 16 per warp
constexpr int AB_ROW_COST = 2;   // units a row counts for besides its positions: its start, join and store take that long
constexpr int AB_JOIN = 16;      // parts of a row up to which one CTA joins them all
constexpr int AB_MAX_COLS = 16;  // query rows per column tile

__device__ __forceinline__ void cp_async16_zfill(uint32_t dst, const void* src, bool on) {
  const int n = on ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t r[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t r[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
template <int NC>
__device__ __forceinline__ long long seq_units(const AttnB8& a, const SeqInfo& s, int& tiles, int& units) {
  const int rows = s.nq * a.group;
  tiles = rows < a.chunk_rows ? (rows + NC - 1) / NC : 0;  // the others are the chunk kernel's
  units = max(1, (s.len + AB_UNIT - 1) / AB_UNIT) + AB_ROW_COST;
  return (long long)a.H * tiles * units;
}

template <typename T>
__device__ __forceinline__ T block_exclusive(T v, T* sums, T& total) {  // AB_THREADS threads
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  T x = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const T o = __shfl_up_sync(0xffffffffu, x, d);
    if (lane >= d) x += o;
  }
  if (lane == 31) sums[wid] = x;
  __syncthreads();
  T before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < AB_WARPS; ++w) {
    if (w < wid) before += sums[w];
    total += sums[w];
  }
  __syncthreads();
  return before + x - v;
}

template <int D, int NT, bool BF16>
struct AttnB8Kernel {
  static constexpr int NC = 8 * NT;
  static constexpr int KSTEPS = D / 16;             // MMAs per 16 positions and column octet, each product
  static constexpr int PIECES = D / 16;             // 16-byte pieces per row
  static constexpr int SIDE = 16 * D;               // bytes of K (or V) in a block
  static constexpr int STAGE = 2 * SIDE + 16;       // + s_k, s_v
  static constexpr int STAGES = 384 / D;            // 16 warps x 3 x 4 KB (6 x 2 KB): all the shared memory there is
  static constexpr int RING = STAGES * STAGE;       // per warp
  static constexpr int OPITCH = D + 8;              // floats per column of the merge buffer
  static constexpr int MERGE = AB_WARPS * NC * (OPITCH + 2) * 4;
  static constexpr int SMEM = (AB_WARPS * RING > MERGE ? AB_WARPS * RING : MERGE);
  static constexpr size_t PART = (size_t)NC * (D + 2);  // floats of a partial result

  // 16-byte piece j of row r of a block, swizzled so that eight rows of one piece meet all banks
  static __device__ __forceinline__ uint32_t piece(int r, int j) {
    if (D == 128) return (uint32_t)(r * 128 + ((j ^ (r & 7)) << 4));
    return (uint32_t)(r * 64 + ((j ^ ((r >> 1) & 3)) << 4));
  }
};

template <int D, int NT, bool BF16>
__global__ void __launch_bounds__(AB_THREADS, AB_CTAS_PER_SM) attn_b8_kernel(const AttnB8 a) {
  using C = AttnB8Kernel<D, NT, BF16>;
  constexpr int NC = C::NC;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ long long sums[AB_WARPS];
  __shared__ long long found_off;
  __shared__ int found_seq, is_last;
  __shared__ SeqInfo found_info;
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5, g = lane >> 2, c = lane & 3;

  // ---- this CTA's range of units -----------------------------------------------------------------------------
  const int per = (a.nseq + AB_THREADS - 1) / AB_THREADS;
  const int i_begin = min(tid * per, a.nseq), i_end = min(i_begin + per, a.nseq);
  long long mine = 0;
  int tiles, units;
#pragma unroll 4
  for (int i = i_begin; i < i_end; ++i) mine += seq_units<NC>(a, seq_info(a, i), tiles, units);
  long long T;
  const long long before = block_exclusive(mine, sums, T);
  const long long G = T < (long long)gridDim.x ? T : (long long)gridDim.x;
  const long long cta = blockIdx.x;
  if (cta >= G) {
    if (cta == 0 && a.after_chunk) pdl_wait();
    return;
  }
  const long long u_begin = range_begin(T, cta, G), u_end = range_begin(T, cta + 1, G);
  if (u_begin >= before && u_begin < before + mine) {
    long long off = u_begin - before;
    int i = i_begin;
    SeqInfo s;
    for (;; ++i) {
      s = seq_info(a, i);
      const long long n = seq_units<NC>(a, s, tiles, units);
      if (off < n) break;
      off -= n;
    }
    found_seq = i;
    found_off = off;
    found_info = s;
  }
  __syncthreads();
  int seq = found_seq;
  long long off = found_off;  // units into the sequence
  long long u = u_begin;

  int* counters = (int*)a.ws;
  float* parts = (float*)((uint8_t*)a.ws + counter_bytes(3 * (int)gridDim.x));
  const uint32_t ring = smem_u32(smem) + wid * C::RING;

  SeqInfo s = found_info;
  while (u < u_end) {
    const long long seq_n = seq_units<NC>(a, s, tiles, units);
    if (off >= seq_n) {
      s = seq_info(a, ++seq);
      off = 0;
      continue;
    }
    // row = (head, column tile) of the sequence; units [r0, r1) of it are this CTA's
    const int row = off < 0x7FFFFFFF ? (int)off / units : (int)(off / units), at = (int)(off - (long long)row * units);
    const int step = (int)min((long long)(units - at), u_end - u);
    // (the first AB_ROW_COST units of a row stand for no positions)
    const int r0 = max(0, at - AB_ROW_COST), r1 = at + step - AB_ROW_COST;
    if (r1 <= 0) {
      u += step;
      off += step;
      continue;
    }
    const int head = row / tiles, tile = row - head * tiles;
    const int rows = min(NC, s.nq * a.group - tile * NC);   // query rows in this tile
    const int tq0 = tile * NC / a.group;                      // first and last query token of the tile
    const int tq1 = (tile * NC + rows - 1) / a.group;
    const int end = positions_seen(a, s, tq1), all_see = positions_seen(a, s, tq0);  // seen by any row, by every row
    const int p_begin = r0 * AB_UNIT, p_end = min(r1 * AB_UNIT, end);
    const int nblocks = p_end > p_begin ? (p_end - p_begin + 15) / 16 : 0;
    const int mine_n = nblocks > wid ? (nblocks - wid + AB_WARPS - 1) / AB_WARPS : 0;

    // ---- the ring ------------------------------------------------------------------------------------------------
    const int* bt = a.bt + (long long)seq * a.bt_stride;
    const size_t slab = (size_t)head * a.npages;
    auto position = [&](int j) { return p_begin + (wid + j * AB_WARPS) * 16; };
    // the page of block j (-1 behind the end), and the row of the page it starts at
    struct Place {
      int pg, in;
    };
    auto page_of = [&](int j) {
      const int p0 = position(j), pi = a.page_div.div(p0);
      return Place{j < mine_n ? bt[pi] : -1, p0 - pi * a.page};
    };
    // where this lane's 16 bytes of a copy go: rows lane / PIECES, then on from there
    const uint32_t lane0 = C::piece(lane / C::PIECES, lane % C::PIECES);
    const uint32_t lane1 = D == 128 ? C::piece(lane / C::PIECES + 4, lane % C::PIECES) - 512 : lane0;
    auto issue = [&](int j, Place at) {
      const uint32_t st = ring + (j % C::STAGES) * C::STAGE;
      if (j < mine_n) {
        const int pg = at.pg;
        const bool good = (unsigned)pg < (unsigned)a.npages;
        const size_t r = (slab + (good ? pg : 0)) * a.page + at.in;
        const uint8_t* ks = a.q_k + r * D + lane * 16;
        const uint8_t* vs = a.q_v + r * D + lane * 16;
        if (good && position(j) + 16 <= s.len) {
#pragma unroll
          for (int i = 0; i < C::SIDE / 512; ++i) {
            const uint32_t to = st + ((i & 1) ? lane1 : lane0) + i * 512;
            cp_async16(to, ks + i * 512);
            cp_async16(to + C::SIDE, vs + i * 512);
          }
        } else {
#pragma unroll
          for (int i = 0; i < C::SIDE / 512; ++i) {
            const uint32_t to = st + ((i & 1) ? lane1 : lane0) + i * 512;
            const bool on = good && position(j) + (i * 32 + lane) / C::PIECES < s.len;
            cp_async16_zfill(to, ks + (on ? i * 512 : 0), on);
            cp_async16_zfill(to + C::SIDE, vs + (on ? i * 512 : 0), on);
          }
        }
        if (lane < 2) {
          const float* sc = (lane == 0 ? a.s_k : a.s_v) + slab + (good ? pg : 0);
          if (good) {
            cp_async<4>(st + 2 * C::SIDE + 4 * lane, sc);
          } else {
            asm volatile("st.shared.f32 [%0], %1;" ::"r"(st + 2 * C::SIDE + 4 * lane), "f"(-1.0f) : "memory");
            if (lane == 0) atomicExch(a.status, ST_KV_PAGE);
          }
        }
      }
      cp_async_commit();
    };
    // ---- query rows as operand registers: lane (g, c) holds row g, dims 16 i + 4 c .. + 3 ----------------------
    // (read between the first look-up of a page and the copies that wait for it)
    uint32_t qf[NT][C::KSTEPS][2];
    float fs[NT][2];     // per column (2c, 2c + 1): score factor without s_k
    int lim[NT][2];      // per column: positions it sees
    Place pg_next = page_of(0);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int n = t * 8 + g, r = tile * NC + n;
      const bool on = n < rows;
      const int tq = on ? r / a.group : 0, hh = on ? r - tq * a.group : 0;
      const uint16_t* qrow =
          (const uint16_t*)a.q + (long long)(s.q0 + tq) * a.q_stride + (size_t)(head * a.group + hh) * D + 4 * c;
#pragma unroll
      for (int i = 0; i < C::KSTEPS; ++i) {
        const uint2 v = on ? *(const uint2*)(qrow + 16 * i) : make_uint2(0, 0);
        qf[t][i][0] = v.x;
        qf[t][i][1] = v.y;
      }
    }
#pragma unroll
    for (int j = 0; j < C::STAGES - 1; ++j) {
      const Place pg = pg_next;
      pg_next = page_of(j + 1);
      issue(j, pg);
    }

#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float scale_row = 1.0f;
      if (BF16) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < C::KSTEPS; ++i)
          top = __vmaxu2(top, __vmaxu2(qf[t][i][0] & 0x7FFF7FFFu, qf[t][i][1] & 0x7FFF7FFFu));
        top = max(top & 0xFFFFu, top >> 16);
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        float up;
        bf16_row_scale(top, up, scale_row);
#pragma unroll
        for (int i = 0; i < C::KSTEPS; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) qf[t][i][j] = bf16x2_to_h2(qf[t][i][j], up);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int col = 2 * c + j;
        fs[t][j] = __shfl_sync(0xffffffffu, scale_row, col * 4) * (a.scale * AB_LOG2E);
        const int rr = tile * NC + t * 8 + col;
        lim[t][j] = t * 8 + col < rows ? positions_seen(a, s, rr / a.group) : 0;
      }
    }

    float acc[C::KSTEPS][NT][4];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int i = 0; i < C::KSTEPS; ++i)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][t][j] = 0.0f;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        m[t][j] = AB_NONE;
        l[t][j] = 0.0f;
      }

    for (int j = 0; j < mine_n; ++j) {
      cp_async_wait<C::STAGES - 2>();
      __syncwarp();
      {
        const Place pg = pg_next;
        pg_next = page_of(j + C::STAGES);
        issue(j + C::STAGES - 1, pg);
      }
      const uint32_t st = ring + (j % C::STAGES) * C::STAGE;
      const int p0 = position(j);
      const float sk = __uint_as_float(lds32(st + 2 * C::SIDE)), sv = __uint_as_float(lds32(st + 2 * C::SIDE + 4));
      // scores
      float x[NT][4];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[t][i] = 0.0f;
#pragma unroll
      for (int i = 0; i < C::KSTEPS; i += 2) {
        uint32_t r[4];
        // matrices: positions 0-7 and 8-15 of piece i, then of piece i + 1
        ldsm4(r, st + C::piece((lane & 7) + (lane & 8), i + (lane >> 4)));
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          uint32_t f[4];
          e4m3x4_to_h2(r[2 * k], f[0], f[2]);
          e4m3x4_to_h2(r[2 * k + 1], f[1], f[3]);
#pragma unroll
          for (int t = 0; t < NT; ++t) mma_16816(x[t], f, qf[t][i + k][0], qf[t][i + k][1]);
        }
      }
      // weights
      const bool bad = sv < 0.0f;
      const float svc = fmaxf(sv, 1e-30f), lv = lg2(svc), inv_sv = __frcp_rn(svc);
      const bool partial = bad || p0 + 16 > all_see;
      float y[NT][4], most = -INFINITY;  // X - m
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const float f0 = fs[t][0] * sk, f1 = fs[t][1] * sk;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[t][i] = fmaf(x[t][i], i & 1 ? f1 : f0, lv);
        if (partial) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (bad || p0 + g + (i >> 1) * 8 >= lim[t][i & 1]) x[t][i] = -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          y[t][i] = x[t][i] - m[t][i & 1];
          most = fmaxf(most, y[t][i]);
        }
      }
      if (__any_sync(0xffffffffu, most > AB_SLACK)) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float top = fmaxf(x[t][i], x[t][i + 2]);
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
            // (only the columns that need it: a column's bits do not depend on the others')
            const float mn = top > m[t][i] + AB_SLACK ? top - AB_BELOW : m[t][i], f = ex2(m[t][i] - mn);
            m[t][i] = mn;
            l[t][i] *= f;
#pragma unroll
            for (int k = 0; k < C::KSTEPS; ++k) {
              acc[k][t][i] *= f;
              acc[k][t][i + 2] *= f;
            }
            y[t][i] = x[t][i] - mn;
            y[t][i + 2] = x[t][i + 2] - mn;
          }
      }
      uint32_t pf[NT][2];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          w[i] = ex2(y[t][i]);
          l[t][i & 1] = fmaf(w[i], inv_sv, l[t][i & 1]);
        }
        // rounded to halves, the type V's codes convert to exactly and both operands of the product share: off by at most
        // 2^-11 of a weight, independently for each position, beside an output rounded by as much (FP16) or 2^-8 (BF16).
        // The denominator sums them unrounded, so lse is as exact as the scores.
        pf[t][0] = movmatrix_trans(h2_as_u32(__floats2half2_rn(w[0], w[1])));
        pf[t][1] = movmatrix_trans(h2_as_u32(__floats2half2_rn(w[2], w[3])));
      }
      // values
#pragma unroll
      for (int i = 0; i < C::KSTEPS; i += 2) {
        uint32_t r[4];
        ldsm4_trans(r, st + C::SIDE + C::piece((lane & 7) + (lane & 8), i + (lane >> 4)));
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          uint32_t f[4];
          e4m3x4_to_h2(__byte_perm(r[2 * k], 0, 0x3120), f[0], f[1]);
          e4m3x4_to_h2(__byte_perm(r[2 * k + 1], 0, 0x3120), f[2], f[3]);
#pragma unroll
          for (int t = 0; t < NT; ++t) mma_16816(acc[i + k][t], f, pf[t][0], pf[t][1]);
        }
      }
      __syncwarp();
    }

    // ---- join the warps ------------------------------------------------------------------------------------------
    cp_async_wait<0>();
    __syncthreads();  // the ring becomes the merge buffer
    float* om = (float*)smem;                           // [warp][NC][OPITCH]
    float* ml = om + AB_WARPS * NC * C::OPITCH;           // [warp][NC][2]
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float sum = l[t][j];
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        const int n = t * 8 + 2 * c + j;
        if (g == 0) {
          ml[(wid * NC + n) * 2] = m[t][j];
          ml[(wid * NC + n) * 2 + 1] = sum;
        }
#pragma unroll
        for (int i = 0; i < C::KSTEPS; ++i)
          *(float2*)(om + (wid * NC + n) * C::OPITCH + 16 * i + 2 * g) = make_float2(acc[i][t][j], acc[i][t][j + 2]);
      }
    __syncthreads();

    // where the row begins and ends among the CTAs
    const bool whole = r0 == 0 && r1 == units - AB_ROW_COST;
    const int first_cta = whole ? (int)cta : unit_owner(u - at + AB_ROW_COST, T, G);
    const int last_cta = whole ? (int)cta : unit_owner(u - at + units - 1, T, G);
    constexpr int LANES = D / 8;  // threads per column
    auto store_row = [&](int n, int d, const float v[8], float ms, float ls) {
      // d: first of eight dims; v unnormalised
      const int r = tile * NC + n, tq = r / a.group, hq = head * a.group + (r - tq * a.group);
      const float inv = row_norm(ls);
      uint32_t h[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) h[i] = pack_out<BF16>(v[2 * i] * inv, v[2 * i + 1] * inv);
      *(uint4*)((uint16_t*)a.out + (long long)(s.q0 + tq) * a.out_stride + (size_t)hq * D + d) =
          make_uint4(h[0], h[1], h[2], h[3]);
      if (a.lse && d == 0)
        a.lse[(long long)(s.q0 + tq) * (a.H * a.group) + hq] = row_lse(ms, ls);
    };
    float* part = parts + (size_t)(2 * cta + (r0 == 0 ? 1 : 0)) * C::PART;
    for (int e = tid; e < NC * LANES; e += AB_THREADS) {
      const int n = e / LANES, d = (e - n * LANES) * 8;
      if (n >= rows) continue;
      float ms = AB_NONE, ls = 0.0f, v[8];
#pragma unroll
      for (int w = 0; w < AB_WARPS; ++w) ms = fmaxf(ms, ml[(w * NC + n) * 2]);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.0f;
#pragma unroll
      for (int w = 0; w < AB_WARPS; ++w) {
        const float f = ex2(ml[(w * NC + n) * 2] - ms);
        ls = fmaf(ml[(w * NC + n) * 2 + 1], f, ls);
        const float4* o = (const float4*)(om + (w * NC + n) * C::OPITCH + d);
        const float4 o0 = o[0], o1 = o[1];
        v[0] = fmaf(o0.x, f, v[0]);
        v[1] = fmaf(o0.y, f, v[1]);
        v[2] = fmaf(o0.z, f, v[2]);
        v[3] = fmaf(o0.w, f, v[3]);
        v[4] = fmaf(o1.x, f, v[4]);
        v[5] = fmaf(o1.y, f, v[5]);
        v[6] = fmaf(o1.z, f, v[6]);
        v[7] = fmaf(o1.w, f, v[7]);
      }
      if (whole) {
        store_row(n, d, v, ms, ls);
      } else {
        float4* dst = (float4*)(part + 2 * NC + n * D + d);
        dst[0] = make_float4(v[0], v[1], v[2], v[3]);
        dst[1] = make_float4(v[4], v[5], v[6], v[7]);
        if (d == 0) *(float2*)(part + 2 * n) = make_float2(ms, ls);
      }
    }
    if (!whole) {
      auto slot = [&](int k) { return parts + (size_t)(k == first_cta ? 2 * k + 1 : 2 * k) * C::PART; };
      // whether this CTA is the last of `want` at a counter (left at zero, as the next launch expects it)
      auto arrive = [&](int* counter, int want) {
        __syncthreads();
        if (tid == 0) {
          __threadfence();  // (after the barrier: covers the whole CTA's writes, and below its reads)
          const int got = atomicAdd(counter, 1) + 1;
          __threadfence();
          is_last = got == want;
          if (got == want) *counter = 0;
        }
        __syncthreads();
        return is_last != 0;
      };
      // A row of many parts is joined in two steps: groups of about the square root of their number, then the groups
      // (one sequence of 121k positions, 8 heads, 74 parts a row: 77 us in one step, 61 us in two). The code is there
      // once for both: a CTA comes here cold, and every instruction is fetched for the one row.
      const int count = last_cta - first_cta + 1;
      int width = count;
      if (count > AB_JOIN) {
        width = AB_JOIN / 2;
        while (width * width < count) ++width;
      }
      const int gi = ((int)cta - first_cta) / width;
      int k0 = first_cta + gi * width, cnt = min(width, last_cta + 1 - k0), stride = 1;
      // (a CTA leads at most one group of a row that it begins and one of a row that it continues)
      int* counter = counters + (width == count ? 0 : gi == 0 ? 1 : 2) * (int)gridDim.x + k0;
      while (arrive(counter, cnt)) {
        const bool final = width == count || stride > 1;
        for (int e = tid; e < NC * LANES; e += AB_THREADS) {
          const int n = e / LANES, d = (e - n * LANES) * 8;
          if (n >= rows) continue;
          // the parts of CTAs k0, k0 + stride, ..., in this order, four on their way at once
          float ms = AB_NONE, ls = 0.0f, v[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = 0.0f;
          for (int q = 0; q < cnt; q += 4) {
            float2 st[4];
            float4 o[4][2];
#pragma unroll
            for (int b = 0; b < 4; ++b) {
              const float* src = slot(k0 + min(q + b, cnt - 1) * stride);
              st[b] = __ldcg((const float2*)(src + 2 * n));
              o[b][0] = __ldcg((const float4*)(src + 2 * NC + n * D + d));
              o[b][1] = __ldcg((const float4*)(src + 2 * NC + n * D + d) + 1);
            }
            float mn = ms;
#pragma unroll
            for (int b = 0; b < 4; ++b) mn = fmaxf(mn, st[b].x);  // (a repeated last one changes nothing)
            const float f0 = ex2(ms - mn);
            ms = mn;
            ls *= f0;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] *= f0;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
              const float f = q + b < cnt ? ex2(st[b].x - ms) : 0.0f;
              ls = fmaf(st[b].y, f, ls);
              v[0] = fmaf(o[b][0].x, f, v[0]);
              v[1] = fmaf(o[b][0].y, f, v[1]);
              v[2] = fmaf(o[b][0].z, f, v[2]);
              v[3] = fmaf(o[b][0].w, f, v[3]);
              v[4] = fmaf(o[b][1].x, f, v[4]);
              v[5] = fmaf(o[b][1].y, f, v[5]);
              v[6] = fmaf(o[b][1].z, f, v[6]);
              v[7] = fmaf(o[b][1].w, f, v[7]);
            }
          }
          if (final) {
            store_row(n, d, v, ms, ls);
          } else {
            // over the leader's own part, which this thread has read here before; its (m, l) after all have read them
            float4* dst = (float4*)(slot(k0) + 2 * NC + n * D + d);
            dst[0] = make_float4(v[0], v[1], v[2], v[3]);
            dst[1] = make_float4(v[4], v[5], v[6], v[7]);
            if (d == 0) *(float2*)((float*)smem + 2 * n) = make_float2(ms, ls);
          }
        }
        if (final) break;
        __syncthreads();
        if (tid < rows) *(float2*)(slot(k0) + 2 * tid) = *(const float2*)((float*)smem + 2 * tid);
        k0 = first_cta;
        cnt = (count + width - 1) / width;
        stride = width;
        counter = counters + first_cta;
      }
    }
    __syncthreads();  // the merge buffer becomes the ring again
    u += step;
    off += step;
  }
  // The chunk kernel before this one ran beside it; the stream's next kernel has to find both done.
  if (cta == 0 && a.after_chunk) pdl_wait();
}

int attn_b8_grid(int sm_count) { return AB_CTAS_PER_SM * sm_count; }

template <int D, int NT, bool BF16>
cudaError_t launch(const AttnB8& a, int sm_count, cudaStream_t stream) {
  using C = AttnB8Kernel<D, NT, BF16>;
  const cudaError_t e = opt_in_smem<attn_b8_kernel<D, NT, BF16>>(C::SMEM);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)attn_b8_grid(sm_count));
  cfg.blockDim = dim3(AB_THREADS);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = a.after_chunk ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, attn_b8_kernel<D, NT, BF16>, a);
}

}  // namespace

size_t attn_b8_ws_bytes(int sm_count) {
  const int grid = attn_b8_grid(sm_count);
  return counter_bytes(3 * grid) + (size_t)2 * grid * AB_MAX_COLS * (AB_MAX_D + 2) * sizeof(float);
}

cudaError_t attn_b8_launch(const AttnB8& args, int D, int bf16, int sm_count, cudaStream_t stream, int* launches) {
  AttnB8 a = args;
  const long long rows = (long long)a.max_q * a.group;
  const bool wide = rows > 8;
  *launches = 1;
  if (rows >= a.chunk_rows) {
    const cudaError_t e = attn_b8_chunk_launch(a, D, bf16, sm_count, stream);
    // The counts are on the device, max_q only bounds them: unless a single token already reaches the threshold, a
    // sequence may be the kernel's below, also when there is only one. (That costs one long sequence 2 us. The chunk
    // kernel taking a sequence alone whatever its count would cost a short one under a large max_q, 32 heads on 8 of
    // 128: 1 token on 777 / 131,072 positions 23 / 178 us instead of 14 / 79.)
    if (e != cudaSuccess || a.group >= a.chunk_rows) return e;
    *launches = 2;
    a.after_chunk = 1;
  }
#define W4B_GO(DD)                                                                                      \
  (bf16 ? (wide ? launch<DD, 2, true>(a, sm_count, stream) : launch<DD, 1, true>(a, sm_count, stream)) \
        : (wide ? launch<DD, 2, false>(a, sm_count, stream) : launch<DD, 1, false>(a, sm_count, stream)))
  return D == 128 ? W4B_GO(128) : W4B_GO(64);
#undef W4B_GO
}

}  // namespace w4b
