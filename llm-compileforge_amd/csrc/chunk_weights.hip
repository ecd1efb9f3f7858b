// Accounts of prompt chunks (gfx950): for each cached token t, the weight that
// a chunk's rows put on it,
//   w[n, hw, t] = (t of the chunk ? 0 : decay * w[n, hw, t])
//                 + sum over rows i and heads h of exp(s[i, h, t] - m[i, h]) / l[i, h],
// row i at position c + i seeing tokens up to its own.  The sum runs over
// rows, across the softmax's own direction, so every row's l is needed before
// any token's sum; the scores of a prompt (4 bytes a row, head and token) are
// far more than K, so they are computed twice:
//   rows kernel    m and l of every (row, head): Q of 256 columns (query rows
//                  x heads of one KV head) in registers, K tiles streamed
//                  through LDS, an online softmax per lane;
//   tokens kernel  K of 256 tokens in registers, Q streamed through LDS with
//                  each column's (m, 1 / l), the sums per lane.
//   short kernel   both at once, for tables of a workgroup's tokens: the scores of
//                  64 columns in registers, their maxima and sums joined in LDS.
// All form S^T = K Q^T (v_mfma_f32_16x16x32; a lane's outputs are four tokens
// of one column), so m, l, and 1 / l are lane-local and the tokens' sums meet
// across the 16 lanes of a column group once a run.  The work of a head is a
// line of steps, 64 tokens for a block of 256 columns (rows kernel) or 64
// columns for a block of 256 tokens (tokens kernel), block after block; every
// resident workgroup takes an equal stretch of it, which is a run or two: it
// leaves (m, l) or sums of each run in the workspace, joined in a fixed order,
// so there are no atomics.  (Units of a fixed length, dealt out in turn, left
// the busiest workgroup a third more steps than the mean.)  Per visible pair the
// kernels issue a fused multiply-add, an exponential (almost three times the
// time of one), an addition and half a maximum next to 2 * D operations of the
// matrix pipe, which the vector pipe hardly overlaps: 64 by 64 pairs at head_dim
// 64 take a SIMD 1,480 cycles with nothing else to do, and some 2,800 here, the
// staging, masks and the end, when the older waves of a SIMD are done, included.
// Two prompts of 1,500 to 4,000 rows, 32 heads of 64: rows 90 us, tokens 85
// (3.6e10 operations of the matrix pipe each); 64 observers behind 4,000 to
// 12,000 tokens, 4 sequences, 32 heads of 128, e4m3: 35 and 42 us.
#include <algorithm>
#include <type_traits>

#include "cf_device.hpp"
#include "cf_host.hpp"
#include "chunk_weights.hpp"
#include "mfma_tile.hpp"

namespace cf {

namespace {

constexpr int kCols = 256;   // columns of a row block, tokens of a token block
constexpr int kStage = 64;   // tokens or columns of a step
constexpr int kSegment = 8192;  // tokens whose block offsets the rows kernel holds
constexpr int kColumns = 960;   // columns whose (m, 1 / l) the tokens kernel holds

// A chunk, as the kernels see it.  All wave-uniform.
struct Chunk {
  int n;
  int start;  // first q row
  int row0;   // first observed q row
  int rows;   // observed rows
  int c0;     // position of the first observed row (negative: rows before the sequence's start)
  int cap;    // tokens that exist: min(len, Mb * 16)
  int fresh;  // tokens from here on came with the chunk
};

// q rows start .. end of chunk n (the chunks taken in order and made disjoint).
__device__ __forceinline__ Chunk chunk_of(const ChunkWeightsParams& p, int n, int start, int end, int len) {
  Chunk c;
  c.n = n;
  c.start = start;
  const int rows = end - start;
  c.rows = p.observe > 0 ? min(rows, p.observe) : rows;
  c.row0 = end - c.rows;
  c.c0 = len - c.rows;
  c.cap = min(len, p.Mb * 16);
  c.fresh = len - rows;
  return c;
}

__device__ __forceinline__ int len_of(const ChunkWeightsParams& p, int n) {
  return max(p.seq_lens[(int64_t)n * p.sl_s], 0);
}

__device__ __forceinline__ int start_of(const ChunkWeightsParams& p, int n) {
  return min(max(p.q_start[(int64_t)n * p.qs_s], 0), p.Tq);
}

// Tokens visible to rows below `end` of the chunk.
__device__ __forceinline__ int visible(const Chunk& c, int end) { return min(max(c.c0 + min(end, c.rows), 0), c.cap); }

__device__ __forceinline__ int cdiv(int a, int b) { return (a + b - 1) / b; }

// The line of steps of one KV head: for each chunk its blocks, for each block its
// steps.  A workgroup lists the chunks of a window with the steps before them
// once, so that a step is found in LDS.
constexpr int kWindow = 256;

struct Window {
  int start[kWindow], end[kWindow];  // q rows
  int len[kWindow];                  // tokens of the sequence
  int before[kWindow + 1];           // steps of the chunks before
};

// Blocks of R rows, steps of 64 tokens that some of the rows see.
struct RowBlocks {
  int R;
  __device__ __forceinline__ int blocks(const Chunk& c) const { return cdiv(c.rows, R); }
  __device__ __forceinline__ int steps(const Chunk& c, int b) const {
    return (visible(c, (b + 1) * R) + kStage - 1) / kStage;
  }
};

// Blocks of TOKENS tokens, steps of 64 columns from the first that sees the
// block's first token on.
template <int TOKENS>
struct TokenBlocks {
  int G;
  __device__ __forceinline__ int blocks(const Chunk& c) const { return (visible(c, c.rows) + TOKENS - 1) / TOKENS; }
  __device__ __forceinline__ int first(const Chunk& c, int b) const { return max(b * TOKENS - c.c0, 0) * G / kStage; }
  __device__ __forceinline__ int steps(const Chunk& c, int b) const {
    return (c.rows * G + kStage - 1) / kStage - first(c, b);
  }
};

// Lists chunks w0 .. w0 + kWindow - 1; `ends`: where the chunks before them end,
// and then these.  Ends with a barrier.
template <class Blocks>
__device__ void list_chunks(const ChunkWeightsParams& p, Window* w, int w0, const Blocks& blocks, int* ends) {
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int n_here = min(p.N - w0, kWindow);
  int carry = *ends;
  for (int base = 0; base < n_here; base += 64) {  // (every wave alike; wave 0 writes)
    const int i = base + lane;
    // a chunk starts where the ones before it end, if q_start has it earlier
    const int start = max(wave_incl_max(i < n_here ? start_of(p, w0 + i) : 0, lane), carry);
    const int end = i < n_here ? max(start_of(p, w0 + i + 1), start) : start;
    if (wave == 0 && i < n_here) {
      w->start[i] = start;
      w->end[i] = end;
      w->len[i] = len_of(p, w0 + i);
    }
    carry = wave_last(start);
  }
  *ends = carry;
  __syncthreads();
  for (int i = wave; i < n_here; i += 4) {
    const Chunk c = chunk_of(p, w0 + i, w->start[i], w->end[i], w->len[i]);
    const int nb = blocks.blocks(c);
    int n = 0;
    for (int b = lane; b < nb; b += 64) n += blocks.steps(c, b);
    n = wave_last(wave_incl_scan(n, lane));
    if (lane == 0) w->before[i + 1] = n;
  }
  __syncthreads();
  if (wave == 0) {
    int total = 0;
    for (int base = 0; base < n_here; base += 64) {
      const int i = base + lane;
      const int incl = wave_incl_scan(i < n_here ? w->before[i + 1] : 0, lane) + total;
      if (i < n_here) w->before[i + 1] = incl;
      total = wave_last(incl);
    }
    if (lane == 0) w->before[0] = 0;
  }
  __syncthreads();
}

// Steps at .. at + n - 1 of a block, that one workgroup does.
struct Run {
  Chunk c;
  int block, at, n;
  int piece, pieces;  // the run's number among the block's, and how many they are
  bool last;
};

// The runs of a workgroup, one after the other.
template <class Blocks>
struct Runs {
  const ChunkWeightsParams& p;
  Window* win;
  Blocks blocks;
  int least;  // steps that a workgroup takes at least
  int lane;
  int x = 0, end = 0, share = 1;  // the stretch's steps left, and its length
  int w0 = -kWindow, ends = 0;

  __device__ __forceinline__ Runs(const ChunkWeightsParams& params, Window* w, Blocks b, int least_steps)
      : p(params), win(w), blocks(b), least(least_steps), lane(threadIdx.x & 63) {}

  // The next one, false after the last.  Called by all threads, with a barrier
  // between a run's use and the next call.
  __device__ __forceinline__ bool next(Run* run) {
    while (x >= end) {  // on to the next window
      w0 += kWindow;
      if (w0 >= p.N) return false;
      __syncthreads();
      list_chunks(p, win, w0, blocks, &ends);
      const int total = uniform(win->before[min(p.N - w0, kWindow)]);
      share = max(cdiv(total, (int)(gridDim.x / p.Hkv)), least);
      x = min((int)(blockIdx.x / p.Hkv) * share, total);
      end = min(x + share, total);
    }
    int v = x, i = 0;
    for (int base = 0; base + w0 < p.N && base < kWindow; base += 64) {  // the last chunk with before[i] <= v
      const uint64_t hit = __ballot(w0 + base + lane < p.N && win->before[base + lane] <= v);
      if (hit == 0) break;
      i = base + 63 - __builtin_clzll(hit);
    }
    v -= uniform(win->before[i]);
    run->c = chunk_of(p, w0 + i, uniform(win->start[i]), uniform(win->end[i]), uniform(win->len[i]));
    const int nb = blocks.blocks(run->c);
    int steps = 0;
    for (int base = 0; base < nb; base += 64) {
      const int b = base + lane, n = b < nb ? blocks.steps(run->c, b) : 0;
      const int incl = wave_incl_scan(n, lane);
      const uint64_t hit = __ballot(incl > v);
      if (hit != 0) {
        const int at = __builtin_ctzll(hit);
        run->block = base + at;
        steps = uniform(__shfl(n, at, 64));
        v -= uniform(__shfl(incl - n, at, 64));
        break;
      }
      v -= wave_last(incl);
    }
    run->at = v;
    run->n = min(end - x, steps - v);
    run->last = v + run->n == steps;
    const int first = (x - v) / share;  // the workgroup that has the block's first step
    run->piece = x / share - first;
    run->pieces = (x - v + steps - 1) / share - first + 1;
    x += run->n;
    return true;
  }
};

// Where a chunk's observed row r lies in ws_ml, and its first piece in ws_p: by
// the chunk where a window of observers makes that shorter, else by the row (a
// chunk has at most two pieces more than its rows fill).
__device__ __forceinline__ int64_t stat_row(const ChunkWeightsParams& p, const Chunk& c, int r) {
  return p.compact ? (int64_t)c.n * p.observe + r : (int64_t)c.row0 + r;
}
__device__ __forceinline__ int64_t piece0(const ChunkWeightsParams& p, const Chunk& c) {
  return p.compact ? (int64_t)c.n * (cdiv(p.observe, p.piece_rows) + 1) : (int64_t)(c.start / p.piece_rows) + 2 * c.n;
}

// Waves of a SIMD that the registers are cut for: at head_dim 128 the operands
// held (64 registers) leave room for two.
template <int D>
constexpr int waves_per_simd() {
  return D == 64 ? 3 : 2;
}

// Columns to query rows: j / G for j below 1,024 and G up to 64, where
// j * (G * ceil(2^16 / G) - 2^16) < 2^16 makes the rounded-up reciprocal exact.
struct Columns {
  uint32_t recip;
  int G;
  __device__ __forceinline__ explicit Columns(int group) : recip((65536u + (uint32_t)group - 1u) / (uint32_t)group), G(group) {}
  __device__ __forceinline__ int row(int j) const { return (int)(((uint32_t)j * recip) >> 16); }
};

template <int D>
constexpr int row_bytes() {
  return D * 2 + 16;  // a staged row: 16 bytes more than whole bank rounds, so 16 rows lie in different banks
}

__device__ __forceinline__ int block_of(const ChunkWeightsParams& p, int n, int j) {
  if (j >= p.Mb) return -1;
  const int id = p.tables[(int64_t)n * p.t_sb + (int64_t)j * p.t_sm];
  return id >= 0 && id < p.NB ? id : -1;
}

// 8 channels of a K row at element offset `at`, as stored, and as 16 bytes of
// operand (converted exactly).
template <int KT>
using Stored = typename std::conditional<KT == kE4M3, uint2, uint4>::type;

template <int KT>
__device__ __forceinline__ Stored<KT> k_piece(const ChunkWeightsParams& p, int64_t at) {
  if constexpr (KT == kE4M3) return *(const uint2*)((const uint8_t*)p.k + at);
  else return *(const uint4*)((const uint16_t*)p.k + at);
}

template <int QT, int KT>
__device__ __forceinline__ uint4 operand(const Stored<KT>& v) {
  if constexpr (KT != kE4M3) return v;
  else if constexpr (QT == kF16) return __builtin_bit_cast(uint4, e4m3x8_to_f16(v.x, v.y));
  else return __builtin_bit_cast(uint4, e4m3x8_to_bf16(v.x, v.y));
}

// Rows of q from a block's or step's first on, for the heads of one KV head: offsets fit 32
// bits (the launcher's bound on the strides).
struct QRows {
  const uint16_t* base;
  int row, head;    // strides
  uint32_t flip;    // changes the sign of every element
  __device__ __forceinline__ QRows(const ChunkWeightsParams& p, int row0, int h, uint32_t sign)
      : base((const uint16_t*)p.q + (int64_t)row0 * p.q_sr + (int64_t)(h * p.G) * p.q_sh), row((int)p.q_sr),
        head((int)p.q_sh), flip(sign) {}
  __device__ __forceinline__ uint4 piece(int r, int g, int d) const {
    uint4 v = *(const uint4*)(base + (uint32_t)(r * row + g * head + d));
    v.x ^= flip;
    v.y ^= flip;
    v.z ^= flip;
    v.w ^= flip;
    return v;
  }
};

// Scores in log2 units are scale_of() times the products of K and Q, which
// carry the scale's sign: the factor is never negative.
struct Factor {
  float qk;
  uint32_t flip;
};
__device__ __forceinline__ Factor factor_of(const ChunkWeightsParams& p, int h) {
  const float ks = p.k_scale ? p.k_scale[h * p.ks_s] : 1.0f;
  const float f = p.scale * ks * kLog2e;
  return Factor{fabsf(f), f < 0.0f ? 0x80008000u : 0u};
}

// ---- rows: m and l of every (row, head) over a piece of its tokens --------------

template <int QT, int KT, int D>
__global__ __launch_bounds__(256, waves_per_simd<D>()) void chunk_rows_kernel(ChunkWeightsParams p) {
  constexpr int NC = D / 32, RB = row_bytes<D>(), PPR = D / 8;  // MFMAs a tile, 16-byte pieces a row
  constexpr int LOADS = kStage * PPR / 256;
  __shared__ __align__(16) uint8_t stage[2][kStage * RB];
  __shared__ int64_t where[kSegment / 16];  // offsets of the segment's blocks (-1: none)
  __shared__ Window win;
  const int tid = threadIdx.x, lane = tid & 63, li = lane & 15, lq = lane >> 4, wave = uniform(tid >> 6);
  const int R = kCols / p.G;
  const Columns col(p.G);
  // where a lane's pieces of a stage lie in their blocks
  int64_t in_block[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const int e = i * 256 + tid;
    in_block[i] = (e / PPR & 15) * p.k_s[1] + e % PPR * 8;
  }
  const int h = (int)(blockIdx.x % (unsigned)p.Hkv);
  Runs<RowBlocks> runs(p, &win, RowBlocks{R}, p.row_steps);
  Run un;
  while (runs.next(&un)) {
    const Chunk& c = un.c;
    const int r0 = un.block * R, nr = min(R, c.rows - r0), ncol = nr * p.G;
    const int t_begin = un.at * kStage, t_end = min(t_begin + un.n * kStage, visible(c, r0 + nr));
    const Factor f = factor_of(p, h);
    const QRows rows(p, c.row0 + r0, h, f.flip);
    // this wave's 64 columns: four tiles of 16
    QOp<QT> q[4][NC];
    int pos[4];  // last token that the lane's column of tile ct sees
#pragma unroll
    for (int ct = 0; ct < 4; ++ct) {
      const int j = wave * 64 + ct * 16 + li, r = col.row(j), g = j - r * p.G;
      pos[ct] = j < ncol ? c.c0 + r0 + r : -1;
#pragma unroll
      for (int x = 0; x < NC; ++x)
        q[ct][x] = as_qop<QT>(j < ncol ? rows.piece(r, g, 32 * x + 8 * lq) : make_uint4(0, 0, 0, 0));
    }
    // positions of the wave's first and last column
    const int w_lo = c.c0 + r0 + col.row(wave * 64), w_hi = c.c0 + r0 + col.row(min(wave * 64 + 63, ncol - 1));
    const bool busy = wave * 64 < ncol;
    float m[4], l[4];
#pragma unroll
    for (int ct = 0; ct < 4; ++ct) m[ct] = -INFINITY, l[ct] = 0.0f;

    for (int seg = t_begin; seg < t_end; seg += kSegment) {
      const int seg_end = min(seg + kSegment, t_end);
      for (int i = tid; seg + i * 16 < seg_end; i += 256) {
        const int blk = block_of(p, c.n, (seg >> 4) + i);
        where[i] = blk < 0 ? -1 : (int64_t)blk * p.k_s[0] + (int64_t)h * p.k_s[2];
      }
      // A step's loads go out at the start of the one before it, from offsets
      // looked up in the one before that.
      Stored<KT> reg[LOADS];
      int64_t at[LOADS];
      uint32_t absent = 0, next_absent = 0;  // blocks of a step that are none of the cache's
      auto locate = [&](int t0) {  // tokens t0 .. + 63 (those past the end: the last one's block, masked)
        const int last = (seg_end - 1 - seg) >> 4, i0 = (t0 - seg) >> 4;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) at[i] = where[min(i0 + (i * 256 + tid) / PPR / 16, last)];
        const bool none = t0 + li * 16 >= seg_end || where[min(i0 + li, last)] < 0;
        next_absent = (uint32_t)__ballot(none) & 15u;
      };
      auto fetch = [&] {
#pragma unroll
        for (int i = 0; i < LOADS; ++i)
          reg[i] = k_piece<KT>(p, (at[i] < 0 ? (int64_t)h * p.k_s[2] : at[i]) + in_block[i]);
      };
      auto store = [&](int buf) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
          const int e = i * 256 + tid;
          *(uint4*)(stage[buf] + e / PPR * RB + e % PPR * 16) = operand<QT, KT>(reg[i]);
        }
      };
      __syncthreads();
      locate(seg);
      fetch();
      absent = next_absent;
      if (seg + kStage < seg_end) locate(seg + kStage);
      store(0);
      __syncthreads();
      for (int t0 = seg, buf = 0; t0 < seg_end; t0 += kStage, buf ^= 1) {
        const bool more = t0 + kStage < seg_end;
        const uint32_t here = absent;
        if (more) {
          fetch();
          absent = next_absent;
          if (t0 + 2 * kStage < seg_end) locate(t0 + 2 * kStage);
        }
        if (busy && t0 <= w_hi) {
          const bool whole = t0 + kStage - 1 <= w_lo && t0 + kStage <= t_end && here == 0;
          // (two bodies: the masks' selects would double the vector work of a tile
          // that needs none)
          auto tiles = [&](auto masked) {
            constexpr bool kMasked = decltype(masked)::value;
#pragma unroll
            for (int ct = 0; ct < 4; ++ct) {
              f32x4_t s[4];
#pragma unroll
              for (int tt = 0; tt < 4; ++tt) {
                s[tt] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int x = 0; x < NC; ++x)
                  s[tt] = mfma16(as_qop<QT>(*(const uint4*)(stage[buf] + (tt * 16 + li) * RB + x * 64 + lq * 16)),
                                 q[ct][x], s[tt]);
              }
              if constexpr (kMasked) {
#pragma unroll
                for (int tt = 0; tt < 4; ++tt) {
                  const int last = (here >> tt & 1) == 0 ? min(pos[ct], t_end - 1) : -1;
#pragma unroll
                  for (int v = 0; v < 4; ++v)
                    if (t0 + tt * 16 + 4 * lq + v > last) s[tt][v] = -INFINITY;
                }
              }
              float mx = s[0][0];
#pragma unroll
              for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i >> 2][i & 3]);
              mx = kMasked && mx == -INFINITY ? mx : mx * f.qk;
              // the reference moves only when a score exceeds it by more than 8
              // (log2 units): sums of e <= 256 are as exact in float32
              if (mx > m[ct] + 8.0f) {
                l[ct] *= __builtin_amdgcn_exp2f(m[ct] - mx);
                m[ct] = mx;
              }
              const float ref = m[ct] == -INFINITY ? 0.0f : m[ct];
              float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const float sv = s[i >> 2][i & 3];
                const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(sv, f.qk, -ref));
                sum[i & 3] += !kMasked || sv != -INFINITY ? e : 0.0f;
              }
              l[ct] += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            }
          };
          if (whole) tiles(std::false_type{});
          else tiles(std::true_type{});
        }
        if (more) store(buf ^ 1);
        __syncthreads();
      }
    }
    // the four lanes of a column
#pragma unroll
    for (int ct = 0; ct < 4; ++ct) {
      float M = fmaxf(m[ct], __shfl_xor(m[ct], 16, 64));
      M = fmaxf(M, __shfl_xor(M, 32, 64));
      // (no finite score: l is 0, or NaN where a score was)
      float L = l[ct] * (m[ct] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m[ct] - M));
      L += __shfl_xor(L, 16, 64);
      L += __shfl_xor(L, 32, 64);
      const int j = wave * 64 + ct * 16 + li, r = col.row(j), g = j - r * p.G;
      if (lq == 0 && j < ncol)
        p.ws_ml[(un.piece * p.stat_rows + stat_row(p, c, r0 + r)) * p.Hq + h * p.G + g] = make_float2(M, L);
    }
    if (un.last && h == 0 && tid < nr) p.ws_np[stat_row(p, c, r0 + tid)] = un.pieces;
  }
}

// (-reference, 1 / sum) of a row and head from its runs, kBatch of them in flight
// at a time.
__device__ __forceinline__ float2 joined(const ChunkWeightsParams& p, int64_t row, int head) {
  const float2* ml = p.ws_ml + row * p.Hq + head;
  const int64_t step = p.stat_rows * p.Hq;
  // (a row without tokens has no runs, and what is read for it goes nowhere)
  const int np = min(max(p.ws_np[row], 0), p.ml_pieces);
  float M = -INFINITY, L = 0.0f;
  constexpr int kBatch = 8;
  for (int i0 = 0; i0 < np; i0 += kBatch) {
    float2 x[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) x[k] = ml[min(i0 + k, np - 1) * step];
    float mn = M;
#pragma unroll
    for (int k = 0; k < kBatch; ++k) mn = fmaxf(mn, x[k].x);
    L *= M == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(M - mn);
#pragma unroll
    for (int k = 0; k < kBatch; ++k)
      if (i0 + k < np) L += x[k].y * (x[k].x == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(x[k].x - mn));
    M = mn;
  }
  return make_float2(M == -INFINITY ? 0.0f : -M, L == 0.0f ? 0.0f : 1.0f / L);
}

// In the place of the first run's, for calls whose tokens kernel would join a
// row many times; one (row, head) a thread.  (Rows that no chunk has hold
// anything, and nobody reads what comes of it.)
__global__ __launch_bounds__(256) void chunk_stats_kernel(ChunkWeightsParams p) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, row = i / p.Hq;
  if (row < p.stat_rows) p.ws_ml[i] = joined(p, row, (int)(i - row * p.Hq));
}

// A wave's sums of tokens tw .. + 63 over the run's columns: the 16 columns of a
// lane group, then the run's place.
__device__ __forceinline__ void leave_sums(const ChunkWeightsParams& p, const Chunk& c, const Run& un, int h, int tw,
                                           float acc[4][4]) {
  const int lane = threadIdx.x & 63, li = lane & 15, lq = lane >> 4;
#pragma unroll
  for (int tt = 0; tt < 4; ++tt)
#pragma unroll
    for (int v = 0; v < 4; ++v)
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) acc[tt][v] += __shfl_xor(acc[tt][v], o, 64);
  if (li == 0) {
    float* out = p.ws_p + ((piece0(p, c) + un.piece) * p.Hkv + h) * (int64_t)p.Mb * 16;
#pragma unroll
    for (int tt = 0; tt < 4; ++tt) {
      const int t = tw + tt * 16 + 4 * lq;
      if (t < p.Mb * 16) *(float4*)(out + t) = make_float4(acc[tt][0], acc[tt][1], acc[tt][2], acc[tt][3]);
    }
  }
  // (a short sequence's one block of 512 tokens is two of the join's)
  const int blocks = cdiv(p.Mb * 16, kCols), own = blockDim.x == 256 ? 1 : blocks;
  if (un.last && h == 0 && (int)threadIdx.x < own) p.ws_tp[c.n * blocks + un.block + threadIdx.x] = un.pieces;
}

// ---- tokens: sums over a run of columns ----------------------------------------

template <int QT, int KT, int D>
__global__ __launch_bounds__(256, waves_per_simd<D>()) void chunk_tokens_kernel(ChunkWeightsParams p) {
  constexpr int NC = D / 32, RB = row_bytes<D>(), PPR = D / 8;
  constexpr int LOADS = kStage * PPR / 256;
  __shared__ __align__(16) uint8_t stage[2][kStage * RB];
  __shared__ float2 fin[kColumns];  // (-m, 1 / l) of the segment's columns
  __shared__ Window win;
  const int tid = threadIdx.x, lane = tid & 63, li = lane & 15, lq = lane >> 4, wave = uniform(tid >> 6);
  const Columns colm(p.G);
  const int h = (int)(blockIdx.x % (unsigned)p.Hkv);
  const TokenBlocks<kCols> blocks{p.G};
  Runs<TokenBlocks<kCols>> runs(p, &win, blocks, p.col_steps);
  Run un;
  while (runs.next(&un)) {
    const Chunk& c = un.c;
    const int ncol = c.rows * p.G, vis = visible(c, c.rows);
    const int t0 = un.block * kCols, tw = t0 + wave * 64;  // the block's and the wave's first token
    const int j_begin = (blocks.first(c, un.block) + un.at) * kStage, j_end = j_begin + un.n * kStage;
    const Factor f = factor_of(p, h);

    // this wave's 64 tokens: four blocks of 16
    QOp<QT> k[4][NC];
    int live[4];  // tokens of the block that exist
#pragma unroll
    for (int tt = 0; tt < 4; ++tt) {
      const int t = tw + tt * 16;
      const int blk = t < vis ? block_of(p, c.n, t >> 4) : -1;
      live[tt] = blk < 0 ? 0 : min(vis - t, 16);
#pragma unroll
      for (int x = 0; x < NC; ++x)
        k[tt][x] = as_qop<QT>(operand<QT, KT>(k_piece<KT>(p, (int64_t)(blk < 0 ? 0 : blk) * p.k_s[0] +
                                                                 (int64_t)h * p.k_s[2] + li * p.k_s[1] + 32 * x + 8 * lq)));
    }
    const bool all_live = live[0] + live[1] + live[2] + live[3] == 64;
    float acc[4][4];
#pragma unroll
    for (int tt = 0; tt < 4; ++tt)
#pragma unroll
      for (int v = 0; v < 4; ++v) acc[tt][v] = 0.0f;

    uint4 reg[LOADS];  // a step's first column: head `head` of row `row`
    auto fetch = [&](int j0, int row, int head) {  // columns j0 .. + 63 (zeros past the last)
      const QRows rows(p, c.row0 + row, h, f.flip);
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int e = i * 256 + tid, j = head + e / PPR, r = colm.row(j), g = j - r * p.G;
        reg[i] = j0 + e / PPR < ncol ? rows.piece(r, g, e % PPR * 8) : make_uint4(0, 0, 0, 0);
      }
    };
    auto store = [&](int buf) {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int e = i * 256 + tid;
        *(uint4*)(stage[buf] + e / PPR * RB + e % PPR * 16) = reg[i];
      }
    };
    int row = j_begin / p.G, head = j_begin - row * p.G;
    for (int seg = j_begin; seg < j_end; seg += kColumns) {
      const int seg_end = min(seg + kColumns, j_end);
      fetch(seg, row, head);
      for (int i = tid; i < seg_end - seg; i += 256) {
        const int r = colm.row(head + i), g = head + i - r * p.G;
        const int64_t at = stat_row(p, c, row + r);
        fin[i] = seg + i >= ncol ? make_float2(0.0f, 0.0f)
                                 : (p.joined ? p.ws_ml[at * p.Hq + h * p.G + g] : joined(p, at, h * p.G + g));
      }
      store(0);
      __syncthreads();
      for (int j0 = seg, buf = 0; j0 < seg_end; j0 += kStage, buf ^= 1) {
        const bool more = j0 + kStage < seg_end;
        const int on = colm.row(head + kStage), next_row = row + on, next_head = head + kStage - on * p.G;
        if (more) fetch(j0 + kStage, next_row, next_head);
        // the last of these columns sees the wave's first token, and the first its last
        const int pos = c.c0 + row;
        if (tw < vis && pos + colm.row(head + min(kStage - 1, ncol - 1 - j0)) >= tw) {
          // (columns past the last are zeros, which make NaN of an infinity of K)
          const bool whole = all_live && pos >= tw + 63 && j0 + kStage <= ncol;
          auto tiles = [&](auto masked) {
            constexpr bool kMasked = decltype(masked)::value;
#pragma unroll
            for (int ct = 0; ct < 4; ++ct) {
              const float2 col = fin[j0 - seg + ct * 16 + li];
              QOp<QT> q[NC];
#pragma unroll
              for (int x = 0; x < NC; ++x)
                q[x] = as_qop<QT>(*(const uint4*)(stage[buf] + (ct * 16 + li) * RB + x * 64 + lq * 16));
              const int j = ct * 16 + li, last = !kMasked ? 0 : (j0 + j < ncol ? pos + colm.row(head + j) : -1);
              f32x4_t s[4];
#pragma unroll
              for (int tt = 0; tt < 4; ++tt) {
                s[tt] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int x = 0; x < NC; ++x) s[tt] = mfma16(k[tt][x], q[x], s[tt]);
              }
#pragma unroll
              for (int tt = 0; tt < 4; ++tt) {
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                  const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[tt][v], f.qk, col.x));
                  const float sum = __builtin_fmaf(e, col.y, acc[tt][v]);
                  if constexpr (kMasked) {
                    // the block's tokens that exist, up to the column's own position
                    const int end = min(live[tt], last + 1 - (tw + tt * 16));
                    acc[tt][v] = 4 * lq + v < end ? sum : acc[tt][v];
                  } else {
                    acc[tt][v] = sum;
                  }
                }
              }
            }
          };
          if (whole) tiles(std::false_type{});
          else tiles(std::true_type{});
        }
        if (more) store(buf ^ 1);
        __syncthreads();
        row = next_row;
        head = next_head;
      }
    }
    leave_sums(p, c, un, h, tw, acc);
  }
}

// ---- short sequences: rows and tokens at once -----------------------------------

// Tables of at most 256 or 512 tokens: a workgroup of four or eight waves that
// holds them all (64 a wave) has a
// column's whole row of scores, so one pass does: the scores of 64 columns stay in
// registers, the waves' maxima and sums of a column meet in LDS, and the weights
// are added up as in the tokens kernel.
// It forms masked scores, too, so eight waves are for few rows: of 500 rows and
// tokens and 32 heads of 64, one chunk takes 20.5 us against 29.4, eight (6.6e7
// row, head and token triples) 65.9 and 67.7, 32 209 and 159; of 12 heads eight
// 36.5 and 53.1, 32 (9.8e7) 106 both.  Of 253 rows and tokens 64 chunks take 114 and
// 123, one 15 and 24.
constexpr double kShortMost = 1e8;
constexpr int kShortWaves = 2;  // of a SIMD: the scores held leave room for no more

template <int QT, int KT, int D, int WAVES>
__global__ __launch_bounds__(WAVES * 64, kShortWaves) void chunk_short_kernel(ChunkWeightsParams p) {
  constexpr int NC = D / 32, RB = row_bytes<D>(), PPR = D / 8;
  constexpr int THREADS = WAVES * 64, LOADS = kStage * PPR / THREADS;
  __shared__ __align__(16) uint8_t stage[2][kStage * RB];
  __shared__ float wave_m[WAVES][kStage], wave_l[WAVES][kStage];
  __shared__ Window win;
  const int tid = threadIdx.x, lane = tid & 63, li = lane & 15, lq = lane >> 4, wave = uniform(tid >> 6);
  const Columns colm(p.G);
  const int h = (int)(blockIdx.x % (unsigned)p.Hkv);
  const TokenBlocks<WAVES * 64> blocks{p.G};
  Runs<TokenBlocks<WAVES * 64>> runs(p, &win, blocks, p.col_steps);
  Run un;
  while (runs.next(&un)) {
    const Chunk& c = un.c;
    const int ncol = c.rows * p.G, vis = visible(c, c.rows), tw = wave * 64;
    const int j_begin = (blocks.first(c, un.block) + un.at) * kStage, j_end = j_begin + un.n * kStage;
    const Factor f = factor_of(p, h);
    QOp<QT> k[4][NC];
    int live[4];  // tokens of the block that exist
#pragma unroll
    for (int tt = 0; tt < 4; ++tt) {
      const int t = tw + tt * 16;
      const int blk = t < vis ? block_of(p, c.n, t >> 4) : -1;
      live[tt] = blk < 0 ? 0 : min(vis - t, 16);
#pragma unroll
      for (int x = 0; x < NC; ++x)
        k[tt][x] = as_qop<QT>(operand<QT, KT>(k_piece<KT>(p, (int64_t)(blk < 0 ? 0 : blk) * p.k_s[0] +
                                                                 (int64_t)h * p.k_s[2] + li * p.k_s[1] + 32 * x + 8 * lq)));
    }
    float acc[4][4];
#pragma unroll
    for (int tt = 0; tt < 4; ++tt)
#pragma unroll
      for (int v = 0; v < 4; ++v) acc[tt][v] = 0.0f;

    uint4 reg[LOADS];
    auto fetch = [&](int j0, int row, int head) {  // columns j0 .. + 63, the first head `head` of row `row`
      const QRows rows(p, c.row0 + row, h, f.flip);
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int e = i * THREADS + tid, j = head + e / PPR, r = colm.row(j), g = j - r * p.G;
        reg[i] = j0 + e / PPR < ncol ? rows.piece(r, g, e % PPR * 8) : make_uint4(0, 0, 0, 0);
      }
    };
    auto store = [&](int buf) {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int e = i * THREADS + tid;
        *(uint4*)(stage[buf] + e / PPR * RB + e % PPR * 16) = reg[i];
      }
    };
    int row = j_begin / p.G, head = j_begin - row * p.G;
    fetch(j_begin, row, head);
    store(0);
    __syncthreads();
    for (int j0 = j_begin, buf = 0; j0 < j_end; j0 += kStage, buf ^= 1) {
      const bool more = j0 + kStage < j_end;
      const int on = colm.row(head + kStage), next_row = row + on, next_head = head + kStage - on * p.G;
      if (more) fetch(j0 + kStage, next_row, next_head);
      f32x4_t s[4][4];
#pragma unroll
      for (int ct = 0; ct < 4; ++ct) {
        const int j = ct * 16 + li;
        // the lane's column sees this many of the wave's tokens
        const int seen = (j0 + j < ncol ? c.c0 + row + colm.row(head + j) + 1 : 0) - tw;
        QOp<QT> q[NC];
#pragma unroll
        for (int x = 0; x < NC; ++x)
          q[x] = as_qop<QT>(*(const uint4*)(stage[buf] + j * RB + x * 64 + lq * 16));
#pragma unroll
        for (int tt = 0; tt < 4; ++tt) {
          s[ct][tt] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int x = 0; x < NC; ++x) s[ct][tt] = mfma16(k[tt][x], q[x], s[ct][tt]);
        }
        float mx = -INFINITY;
#pragma unroll
        for (int tt = 0; tt < 4; ++tt) {
          const int end = min(live[tt], seen - tt * 16);
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            if (4 * lq + v >= end) s[ct][tt][v] = -INFINITY;
            mx = fmaxf(mx, s[ct][tt][v]);
          }
        }
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        if (lq == 0) wave_m[wave][j] = mx;
      }
      __syncthreads();
#pragma unroll
      for (int ct = 0; ct < 4; ++ct) {
        const int j = ct * 16 + li;
        float mx = wave_m[0][j];
#pragma unroll
        for (int i = 1; i < WAVES; ++i) mx = fmaxf(mx, wave_m[i][j]);
        const float ref = mx == -INFINITY ? 0.0f : mx * f.qk;
        float sum = 0.0f;
#pragma unroll
        for (int tt = 0; tt < 4; ++tt)
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const float sv = s[ct][tt][v], e = __builtin_amdgcn_exp2f(__builtin_fmaf(sv, f.qk, -ref));
            s[ct][tt][v] = sv != -INFINITY ? e : -1.0f;  // (-1: masked)
            sum += sv != -INFINITY ? e : 0.0f;
          }
        sum += __shfl_xor(sum, 16, 64);
        sum += __shfl_xor(sum, 32, 64);
        if (lq == 0) wave_l[wave][j] = sum;
      }
      __syncthreads();
#pragma unroll
      for (int ct = 0; ct < 4; ++ct) {
        const int j = ct * 16 + li;
        float L = wave_l[0][j];
#pragma unroll
        for (int i = 1; i < WAVES; ++i) L += wave_l[i][j];
        const float inv = L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll
        for (int tt = 0; tt < 4; ++tt)
#pragma unroll
          for (int v = 0; v < 4; ++v) {  // (a NaN reaches the row's own tokens only)
            const float e = s[ct][tt][v];
            acc[tt][v] = e != -1.0f ? __builtin_fmaf(e, inv, acc[tt][v]) : acc[tt][v];
          }
      }
      if (more) store(buf ^ 1);
      __syncthreads();
      row = next_row;
      head = next_head;
    }
    leave_sums(p, c, un, h, tw, acc);
  }
}

// ---- join --------------------------------------------------------------------

// SPLIT: 64 tokens a workgroup, each wave summing every fourth piece, and the
// four meet in LDS; else a token a thread.
template <bool SPLIT>
__global__ __launch_bounds__(256) void chunk_join_kernel(ChunkWeightsParams p) {
  constexpr int kTokens = SPLIT ? 64 : 256;
  __shared__ float sums[4][64];
  const int lane = threadIdx.x & 63, wave = SPLIT ? uniform(threadIdx.x >> 6) : 0;
  const int per = p.Mb * 16, groups = cdiv(per, kTokens);
  const int nh = blockIdx.x / groups, n = nh / p.Hw, hw = nh - n * p.Hw;
  const int t = (blockIdx.x - nh * groups) * kTokens + (SPLIT ? lane : (int)threadIdx.x);
  int start = 0;  // the end of the chunks before, and this one's own start
  for (int i = lane; i <= n; i += 64) start = max(start, start_of(p, i));
  start = wave_last(wave_incl_max(start, 0));
  const Chunk c = chunk_of(p, n, start, max(start_of(p, n + 1), start), len_of(p, n));
  if (c.rows == 0) return;
  const int heads = p.Hkv / p.Hw;
  // the pieces of the token's block and their heads: one head's sums are Hkv
  // rows apart, those of all heads follow each other
  const int seen = t < visible(c, c.rows) ? p.ws_tp[n * cdiv(per, kCols) + t / kCols] : 0, count = seen * heads;
  const int64_t step = (int64_t)per * (p.Hw == 1 ? 1 : p.Hkv);
  const float* part = p.ws_p + (piece0(p, c) * p.Hkv + hw * heads) * (int64_t)per + t;
  float sum = 0.0f;
#pragma unroll 8
  for (int i = wave; i < count; i += SPLIT ? 4 : 1) sum += part[i * step];
  if constexpr (SPLIT) {
    sums[wave][lane] = sum;
    __syncthreads();
    if (wave != 0) return;
    sum = (sums[0][lane] + sums[1][lane]) + (sums[2][lane] + sums[3][lane]);
  }
  if (t >= c.cap) return;
  float* w = p.weights + (int64_t)n * p.w_sb + (int64_t)hw * p.w_sh + t;
  *w = t >= c.fresh || p.decay == 0.0f ? sum : __builtin_fmaf(*w, p.decay, sum);
}

// ---- launch ------------------------------------------------------------------

// How a call is cut, from its sizes alone: the workspace query and the launch
// agree on it.
struct Cut {
  bool compact;         // rows stored by the chunk (a window of observers)
  int64_t stat_rows;    // rows of ws_ml
  int64_t ml_pieces;    // runs of a row's tokens, at most
  int64_t pieces;       // of ws_p
  int row_steps, col_steps, piece_rows;
};

// The least that a workgroup takes bounds the runs of a block, and with them the
// workspace: a row's tokens are at most 33 runs; a token's columns runs of 64
// columns at least, or of more (up to 4,096) where the sums would exceed 32 MB.
Cut cut_of(int64_t Tq, int64_t N, int64_t Hkv, int64_t G, int64_t cap, int64_t observe) {
  Cut c;
  c.compact = observe > 0 && N * observe < Tq;
  c.stat_rows = c.compact ? N * observe : Tq;
  const int64_t steps = std::max<int64_t>(ceil_div(cap, kStage), 1);
  c.row_steps = (int)ceil_div(steps, 32);
  c.ml_pieces = (steps - 1) / c.row_steps + 2;
  for (c.col_steps = 1;; c.col_steps *= 2) {
    c.piece_rows = (int)(c.col_steps * kStage / G);  // (G <= 64)
    c.pieces = c.compact ? N * (ceil_div(observe, c.piece_rows) + 1) : Tq / c.piece_rows + 2 * N;
    if (c.col_steps == 64 || c.pieces * Hkv * cap * 4 <= 32 << 20) break;
  }
  return c;
}

uint64_t pad(uint64_t x) { return (x + 255) & ~(uint64_t)255; }

// (row, head, token) triples from which a kernel of its own joins the rows'
// runs: 256 observers of 32 heads over 12,000 tokens (9.8e7) take 41.1 us in the
// tokens kernel and 4.0 before it, 48.0 where it joins them itself; 35 rows of
// 64 heads over 4,200 (9.4e6) 13.6 in all.
constexpr double kJoinFirst = 3.2e7;

struct Layout {
  Cut cut;
  uint64_t p, np, tp, bytes;  // byte offsets behind ws_ml
};

Layout layout_of(int64_t Tq, int64_t N, int64_t Hq, int64_t Hkv, int64_t cap, int64_t observe) {
  Layout w;
  w.cut = cut_of(Tq, N, Hkv, Hq / Hkv, cap, observe);
  w.p = pad((uint64_t)w.cut.ml_pieces * w.cut.stat_rows * Hq * 8);
  w.np = w.p + pad((uint64_t)w.cut.pieces * Hkv * cap * 4);
  w.tp = w.np + pad((uint64_t)w.cut.stat_rows * 4);
  w.bytes = w.tp + pad((uint64_t)N * ceil_div(cap, kCols) * 4);
  return w;
}

template <int QT, int KT, int D>
int32_t launch_d(const ChunkWeightsParams& p, hipStream_t stream) {
  const int64_t cap = (int64_t)p.Mb * 16;
  // as many workgroups as are resident, the same number for every head
  const int resident = waves_per_simd<D>() * device_cu_count();
  const dim3 grid((unsigned)(std::max(resident / p.Hkv, 1) * p.Hkv));
  const auto few = [&](int waves) {
    return dim3((unsigned)(std::max(kShortWaves * 4 / waves * device_cu_count() / p.Hkv, 1) * p.Hkv));
  };
  if (cap <= kCols) {
    ProfileScope prof("cf_chunk_short", stream);
    CF_LAUNCH((chunk_short_kernel<QT, KT, D, 4>), few(4), dim3(256), 0, stream, p);
    CF_HIP_CHECK(hipGetLastError());
  } else if (cap <= 2 * kCols && (double)p.stat_rows * p.Hq * cap <= kShortMost) {
    ProfileScope prof("cf_chunk_short", stream);
    CF_LAUNCH((chunk_short_kernel<QT, KT, D, 8>), few(8), dim3(512), 0, stream, p);
    CF_HIP_CHECK(hipGetLastError());
  } else {
    {
      ProfileScope prof("cf_chunk_rows", stream);
      CF_LAUNCH((chunk_rows_kernel<QT, KT, D>), grid, dim3(256), 0, stream, p);
      CF_HIP_CHECK(hipGetLastError());
    }
    if (p.joined) {
      ProfileScope prof("cf_chunk_stats", stream);
      CF_LAUNCH(chunk_stats_kernel, dim3((unsigned)ceil_div(p.stat_rows * p.Hq, 256)), dim3(256), 0, stream, p);
      CF_HIP_CHECK(hipGetLastError());
    }
    {
      ProfileScope prof("cf_chunk_tokens", stream);
      CF_LAUNCH((chunk_tokens_kernel<QT, KT, D>), grid, dim3(256), 0, stream, p);
      CF_HIP_CHECK(hipGetLastError());
    }
  }
  ProfileScope prof("cf_chunk_join", stream);
  // Many pieces a token: more loads in flight.  Two prompts of 4,000 rows 4.0 us
  // against 4.6, 469 rows of 64 heads into one account 4.0 and 7.6; 64 observers
  // of four sequences, whose pieces are few, 8.2 and 4.4.
  if (ceil_div(p.compact ? p.observe : ceil_div(p.Tq, p.N), p.piece_rows) * (p.Hkv / p.Hw) >= 8)
    CF_LAUNCH((chunk_join_kernel<true>), dim3((unsigned)(ceil_div(cap, 64) * p.N * p.Hw)), dim3(256), 0, stream, p);
  else
    CF_LAUNCH((chunk_join_kernel<false>), dim3((unsigned)(ceil_div(cap, 256) * p.N * p.Hw)), dim3(256), 0, stream, p);
  CF_HIP_CHECK(hipGetLastError());
  return CF_OK;
}

template <int QT, int KT>
int32_t launch_t(const ChunkWeightsParams& p, hipStream_t stream) {
  return p.D == 128 ? launch_d<QT, KT, 128>(p, stream) : launch_d<QT, KT, 64>(p, stream);
}

}  // namespace

bool chunk_weights_supported(const ChunkWeightsParams& p, int q_dt, int k_dt) {
  if (!(q_dt == kBF16 && (k_dt == kBF16 || k_dt == kE4M3)) && !(q_dt == kF16 && (k_dt == kF16 || k_dt == kE4M3)))
    return false;
  if (p.D != 64 && p.D != 128) return false;
  if (p.G > 64 || p.NB < 1) return false;
  // a step's offsets into q: up to 256 rows and 64 heads
  if (p.q_sr >= 1 << 20 || p.q_sh >= 1 << 20) return false;
  const int kb = k_dt == kE4M3 ? 1 : 2;
  if (p.k_s[3] != 1 || ((uintptr_t)p.k & 15) != 0 || ((uintptr_t)p.q & 15) != 0) return false;
  for (int i = 0; i < 3; ++i)
    if ((p.k_s[i] * kb) % 16 != 0) return false;
  return (p.q_sr * 2) % 16 == 0 && (p.q_sh * 2) % 16 == 0;
}

uint64_t chunk_weights_workspace_bytes(int64_t num_q_tokens, int64_t num_chunks, int64_t num_q_heads,
                                       int64_t num_kv_heads, int64_t max_blocks, int64_t observe) {
  return layout_of(num_q_tokens, num_chunks, num_q_heads, num_kv_heads, max_blocks * 16, observe).bytes;
}

void chunk_weights_bind_workspace(ChunkWeightsParams& p, void* workspace) {
  const Layout w = layout_of(p.Tq, p.N, p.Hq, p.Hkv, (int64_t)p.Mb * 16, p.observe);
  p.compact = w.cut.compact;
  p.stat_rows = w.cut.stat_rows;
  p.ml_pieces = (int)w.cut.ml_pieces;
  p.row_steps = w.cut.row_steps;
  p.col_steps = w.cut.col_steps;
  p.piece_rows = w.cut.piece_rows;
  p.joined = (double)p.stat_rows * p.Hq * p.Mb * 16 >= kJoinFirst;
  p.ws_ml = (float2*)workspace;
  p.ws_p = (float*)((char*)workspace + w.p);
  p.ws_np = (int*)((char*)workspace + w.np);
  p.ws_tp = (int*)((char*)workspace + w.tp);
}

int32_t launch_chunk_weights(const ChunkWeightsParams& p, int q_dt, int k_dt, hipStream_t stream) {
  if (q_dt == kF16) return k_dt == kE4M3 ? launch_t<kF16, kE4M3>(p, stream) : launch_t<kF16, kF16>(p, stream);
  return k_dt == kE4M3 ? launch_t<kBF16, kE4M3>(p, stream) : launch_t<kBF16, kBF16>(p, stream);
}

}  // namespace cf
