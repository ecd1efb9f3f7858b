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
// Both form S^T = K Q^T (v_mfma_f32_16x16x32; a lane's outputs are four tokens
// of one column), so m, l, and 1 / l are lane-local and the tokens' sums meet
// across the 16 lanes of a column group once a unit.  Work is cut into units
// of 256 columns x TP tokens (rows kernel) and CB columns x 256 tokens (tokens
// kernel), dealt out evenly to the resident workgroups; a unit leaves (m, l) or
// sums of its piece in the workspace, joined in a fixed order, so there are no
// atomics.  Per visible pair the kernels
// issue a fused multiply-add, an exponential (four times the time of one) and
// an addition next to 2 * D operations of the matrix pipe: the exponentials
// bound them at head_dim 64, both about equally at 128.
#include <algorithm>
#include <type_traits>

#include "cf_device.hpp"
#include "cf_host.hpp"
#include "chunk_weights.hpp"
#include "mfma_tile.hpp"

namespace cf {

namespace {

constexpr int kCols = 256;   // columns of a rows-kernel unit, tokens of a tokens-kernel unit
constexpr int kStage = 64;   // tokens or columns staged at a time
constexpr int kMaxCB = 1024;
constexpr int kMaxTP = 16384;

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

// Units of a launch: (chunk, block of R rows, block of TB tokens that some of
// the rows see, KV head), the head innermost.  A workgroup lists the chunks of a
// window with their units before them once, so that a unit is found in LDS.
constexpr int kWindow = 256;

struct Window {
  int start[kWindow], end[kWindow];  // q rows
  int len[kWindow];                  // tokens of the sequence
  int before[kWindow + 1];           // (row block, token block) pairs of the chunks before
};

__device__ __forceinline__ int token_blocks(const Chunk& c, int rb, int R, int TB) {
  return cdiv(visible(c, (rb + 1) * R), TB);
}

// Lists chunks w0 .. w0 + kWindow - 1; `ends`: where the chunks before them end,
// and then these.  Ends with a barrier.
__device__ void list_chunks(const ChunkWeightsParams& p, Window* w, int w0, int R, int TB, int* ends) {
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
    const int nb = cdiv(c.rows, R);
    int n = 0;
    for (int rb = lane; rb < nb; rb += 64) n += token_blocks(c, rb, R, TB);
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

struct Unit {
  Chunk c;
  int h, rb, tb;
};

// Unit u of the window at w0 (0 <= u < units of the window).
__device__ __forceinline__ Unit unit_of(const ChunkWeightsParams& p, const Window* w, int w0, int64_t u, int R, int TB,
                                        int lane) {
  Unit out;
  out.h = (int)(u % p.Hkv);
  int v = (int)(u / p.Hkv), i = 0;
  for (int base = 0; base + w0 < p.N && base < kWindow; base += 64) {  // the last chunk with before[i] <= v
    const uint64_t hit = __ballot(w0 + base + lane < p.N && w->before[base + lane] <= v);
    if (hit == 0) break;
    i = base + 63 - __builtin_clzll(hit);
  }
  v -= uniform(w->before[i]);
  out.c = chunk_of(p, w0 + i, uniform(w->start[i]), uniform(w->end[i]), uniform(w->len[i]));
  const int nb = cdiv(out.c.rows, R);
  for (int base = 0; base < nb; base += 64) {
    const int rb = base + lane, n = rb < nb ? token_blocks(out.c, rb, R, TB) : 0;
    const int incl = wave_incl_scan(n, lane);
    const uint64_t hit = __ballot(incl > v);
    if (hit != 0) {
      const int at = __builtin_ctzll(hit);
      out.rb = base + at;
      out.tb = v - uniform(__shfl(incl - n, at, 64));
      return out;
    }
    v -= wave_last(incl);
  }
  out.rb = out.tb = 0;  // (not reached: v is below the chunk's units)
  return out;
}

// Where a chunk's observed row r lies in ws_ml, and its first row piece in ws_p:
// by the chunk where a window of observers makes that shorter, else by the row
// (chunks before it use at most one piece more than their rows fill).
__device__ __forceinline__ int64_t stat_row(const ChunkWeightsParams& p, const Chunk& c, int r) {
  return p.compact ? (int64_t)c.n * p.observe + r : (int64_t)c.row0 + r;
}
__device__ __forceinline__ int64_t piece0(const ChunkWeightsParams& p, const Chunk& c, int R) {
  return p.compact ? (int64_t)c.n * cdiv(p.observe, R) : (int64_t)(c.start / R) + c.n;
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

// 16 bytes of operand (8 channels) of a K row at element offset `at`: as stored,
// or converted (exactly).
template <int QT, int KT>
__device__ __forceinline__ uint4 k_piece(const ChunkWeightsParams& p, int64_t at) {
  if constexpr (KT == kE4M3) {
    const uint2 v = *(const uint2*)((const uint8_t*)p.k + at);
    if constexpr (QT == kF16) return __builtin_bit_cast(uint4, e4m3x8_to_f16(v.x, v.y));
    else return __builtin_bit_cast(uint4, e4m3x8_to_bf16(v.x, v.y));
  } else {
    return *(const uint4*)((const uint16_t*)p.k + at);
  }
}

// Rows of q from a unit's first on, for the heads of one KV head: offsets fit 32
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
  __shared__ int64_t where[kMaxTP / 16];  // offsets of the unit's blocks (-1: none)
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
  int ends = 0, w0 = 0;
  list_chunks(p, &win, 0, R, p.TP, &ends);
  int64_t u = blockIdx.x, units = (int64_t)win.before[min(p.N, kWindow)] * p.Hkv;
  for (;; u += gridDim.x) {
    while (u >= units) {  // on to the next window
      u -= units;
      w0 += kWindow;
      if (w0 >= p.N) return;
      __syncthreads();
      list_chunks(p, &win, w0, R, p.TP, &ends);
      units = (int64_t)win.before[min(p.N - w0, kWindow)] * p.Hkv;
    }
    const Unit un = unit_of(p, &win, w0, u, R, p.TP, lane);
    const Chunk& c = un.c;
    const int r0 = un.rb * R, nr = min(R, c.rows - r0), ncol = nr * p.G;
    const int t_begin = un.tb * p.TP, t_end = min(t_begin + p.TP, visible(c, r0 + nr));
    const Factor f = factor_of(p, un.h);
    for (int i = tid; t_begin + i * 16 < t_end; i += 256) {
      const int blk = block_of(p, c.n, (t_begin >> 4) + i);
      where[i] = blk < 0 ? -1 : (int64_t)blk * p.k_s[0] + (int64_t)un.h * p.k_s[2];
    }
    const QRows rows(p, c.row0 + r0, un.h, f.flip);
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

    uint4 reg[LOADS];
    auto fetch = [&](int t0) {  // tokens t0 .. + 63 (those past the end: the last one's block, masked)
      const int last = (t_end - 1 - t_begin) >> 4, i0 = (t0 - t_begin) >> 4;
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int64_t at = where[min(i0 + (i * 256 + tid) / PPR / 16, last)];
        reg[i] = k_piece<QT, KT>(p, (at < 0 ? (int64_t)un.h * p.k_s[2] : at) + in_block[i]);
      }
    };
    auto store = [&](int buf) {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int e = i * 256 + tid;
        *(uint4*)(stage[buf] + e / PPR * RB + e % PPR * 16) = reg[i];
      }
    };
    __syncthreads();
    fetch(t_begin);
    store(0);
    __syncthreads();
    for (int t0 = t_begin, buf = 0; t0 < t_end; t0 += kStage, buf ^= 1) {
      const bool more = t0 + kStage < t_end;
      if (more) fetch(t0 + kStage);
      if (busy && t0 <= w_hi) {
        const int i0 = (t0 - t_begin) >> 4;
        bool whole = t0 + kStage - 1 <= w_lo && t0 + kStage <= t_end;
        int valid[kStage / 16];  // whether a block is one of the cache
#pragma unroll
        for (int tt = 0; tt < kStage / 16; ++tt) {
          valid[tt] = uniform((int)(t0 + tt * 16 < t_end ? where[i0 + tt] >> 32 : -1)) >= 0;
          whole = whole && valid[tt];
        }
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
                const int last = valid[tt] ? min(pos[ct], t_end - 1) : -1;
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
        p.ws_ml[(un.tb * p.stat_rows + stat_row(p, c, r0 + r)) * p.Hq + un.h * p.G + g] = make_float2(M, L);
    }
    __syncthreads();  // the stage is filled anew
  }
}

// ---- tokens: sums over the rows of a piece -----------------------------------

template <int QT, int KT, int D>
__global__ __launch_bounds__(256, waves_per_simd<D>()) void chunk_tokens_kernel(ChunkWeightsParams p) {
  constexpr int NC = D / 32, RB = row_bytes<D>(), PPR = D / 8;
  constexpr int LOADS = kStage * PPR / 256;
  __shared__ __align__(16) uint8_t stage[2][kStage * RB];
  __shared__ float2 fin[kMaxCB];  // (-m, 1 / l) of the unit's columns
  __shared__ Window win;
  const int tid = threadIdx.x, lane = tid & 63, li = lane & 15, lq = lane >> 4, wave = uniform(tid >> 6);
  const int R = p.CB / p.G, RA = kCols / p.G;
  const Columns colm(p.G);
  int ends = 0, w0 = 0;
  list_chunks(p, &win, 0, R, kCols, &ends);
  int64_t u = blockIdx.x, units = (int64_t)win.before[min(p.N, kWindow)] * p.Hkv;
  for (;; u += gridDim.x) {
    while (u >= units) {  // on to the next window
      u -= units;
      w0 += kWindow;
      if (w0 >= p.N) return;
      __syncthreads();
      list_chunks(p, &win, w0, R, kCols, &ends);
      units = (int64_t)win.before[min(p.N - w0, kWindow)] * p.Hkv;
    }
    const Unit un = unit_of(p, &win, w0, u, R, kCols, lane);
    const Chunk& c = un.c;
    const int r0 = un.rb * R, nr = min(R, c.rows - r0), ncol = nr * p.G;
    const int vis = visible(c, r0 + nr);
    const int t0 = un.tb * kCols, tw = t0 + wave * 64;  // the unit's and the wave's first token
    const Factor f = factor_of(p, un.h);
    // columns before the first row that sees the unit's tokens are left out
    const int j_begin = max(t0 - c.c0 - r0, 0) * p.G & ~(kStage - 1);

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
        k[tt][x] = as_qop<QT>(k_piece<QT, KT>(p, (int64_t)(blk < 0 ? 0 : blk) * p.k_s[0] + (int64_t)un.h * p.k_s[2] +
                                                      li * p.k_s[1] + 32 * x + 8 * lq));
    }
    const bool all_live = live[0] + live[1] + live[2] + live[3] == 64;
    float acc[4][4];
#pragma unroll
    for (int tt = 0; tt < 4; ++tt)
#pragma unroll
      for (int v = 0; v < 4; ++v) acc[tt][v] = 0.0f;

    const QRows rows(p, c.row0 + r0, un.h, f.flip);
    uint4 reg[LOADS];
    auto fetch = [&](int j0) {  // columns j0 .. + 63 (zeros past the last)
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int e = i * 256 + tid, j = j0 + e / PPR, r = colm.row(j), g = j - r * p.G;
        reg[i] = j < ncol ? rows.piece(r, g, e % PPR * 8) : make_uint4(0, 0, 0, 0);
      }
    };
    auto store = [&](int buf) {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int e = i * 256 + tid;
        *(uint4*)(stage[buf] + e / PPR * RB + e % PPR * 16) = reg[i];
      }
    };
    fetch(j_begin);
    // the rows' references and sums, from their pieces: kBatch of them in
    // flight at a time
    for (int j = j_begin + tid; j < cdiv(ncol, kStage) * kStage; j += 256) {
      float2 v = make_float2(0.0f, 0.0f);
      if (j < ncol) {
        const int r = colm.row(j), g = j - r * p.G, row = r0 + r;
        const float2* ml = p.ws_ml + stat_row(p, c, row) * p.Hq + un.h * p.G + g;
        const int64_t step = p.stat_rows * p.Hq;
        const int np = cdiv(visible(c, (row / RA + 1) * RA), p.TP);  // pieces that the rows kernel wrote
        float M = -INFINITY, L = 0.0f;
        constexpr int kBatch = 8;
        for (int i0 = 0; i0 < np; i0 += kBatch) {
          float2 x[kBatch];
#pragma unroll
          for (int i = 0; i < kBatch; ++i) x[i] = ml[min(i0 + i, np - 1) * step];
          float mn = M;
#pragma unroll
          for (int i = 0; i < kBatch; ++i) mn = fmaxf(mn, x[i].x);
          L *= M == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(M - mn);
#pragma unroll
          for (int i = 0; i < kBatch; ++i)
            if (i0 + i < np) L += x[i].y * (x[i].x == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(x[i].x - mn));
          M = mn;
        }
        v = make_float2(M == -INFINITY ? 0.0f : -M, L == 0.0f ? 0.0f : 1.0f / L);
      }
      fin[j] = v;
    }

    store(0);
    __syncthreads();
    for (int j0 = j_begin, buf = 0; j0 < ncol; j0 += kStage, buf ^= 1) {
      const bool more = j0 + kStage < ncol;
      if (more) fetch(j0 + kStage);
      // the last of these columns sees the wave's first token, and the first its last
      if (tw < vis && c.c0 + r0 + colm.row(min(j0 + kStage - 1, ncol - 1)) >= tw) {
        const bool whole = all_live && c.c0 + r0 + colm.row(j0) >= tw + 63;
        auto tiles = [&](auto masked) {
          constexpr bool kMasked = decltype(masked)::value;
#pragma unroll
          for (int ct = 0; ct < 4; ++ct) {
            const float2 col = fin[j0 + ct * 16 + li];
            QOp<QT> q[NC];
#pragma unroll
            for (int x = 0; x < NC; ++x)
              q[x] = as_qop<QT>(*(const uint4*)(stage[buf] + (ct * 16 + li) * RB + x * 64 + lq * 16));
            const int j = j0 + ct * 16 + li, last = !kMasked ? 0 : (j < ncol ? c.c0 + r0 + colm.row(j) : -1);
#pragma unroll
            for (int tt = 0; tt < 4; ++tt) {
              f32x4_t s = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
              for (int x = 0; x < NC; ++x) s = mfma16(k[tt][x], q[x], s);
#pragma unroll
              for (int v = 0; v < 4; ++v) {
                const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[v], f.qk, col.x));
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
    }
    // the 16 columns of a lane group
#pragma unroll
    for (int tt = 0; tt < 4; ++tt)
#pragma unroll
      for (int v = 0; v < 4; ++v)
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) acc[tt][v] += __shfl_xor(acc[tt][v], o, 64);
    if (li == 0) {
      float* out = p.ws_p + ((piece0(p, c, R) + un.rb) * p.Hkv + un.h) * (int64_t)p.Mb * 16;
#pragma unroll
      for (int tt = 0; tt < 4; ++tt) {
        const int t = tw + tt * 16 + 4 * lq;
        if (t < p.Mb * 16) *(float4*)(out + t) = make_float4(acc[tt][0], acc[tt][1], acc[tt][2], acc[tt][3]);
      }
    }
    __syncthreads();  // fin and the stage are filled anew
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
  const int R = p.CB / p.G, nb = cdiv(c.rows, R), heads = p.Hkv / p.Hw;
  // the row blocks from the first that sees token t on, and their heads: one
  // head's sums are Hkv rows apart, those of all heads follow each other
  const int first = max(t - c.c0, 0) / R, count = t < c.cap ? (nb - first) * heads : 0;
  const int64_t step = (int64_t)per * (p.Hw == 1 ? 1 : p.Hkv);
  const float* part = p.ws_p + ((piece0(p, c, R) + first) * p.Hkv + hw * heads) * (int64_t)per + t;
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
  int64_t row_pieces;   // of ws_p
  int TP, CB;
};

// Long units reuse what they hold in registers more often, short ones even out
// what the workgroups get: the longest that give each at least kUnitsEach, of
// about half of the (row, token) blocks (causal).
constexpr double kUnitsEach = 2.5;

Cut cut_of(int64_t Tq, int64_t N, int64_t Hkv, int64_t G, int64_t D, int64_t cap, int64_t observe) {
  Cut c;
  c.compact = observe > 0 && N * observe < Tq;
  c.stat_rows = c.compact ? N * observe : Tq;
  const double want = kUnitsEach * (D == 64 ? 3 : 2) * device_cu_count();
  const double seen = observe > 0 ? 1.0 : 0.5;
  auto pieces = [&](int64_t cols) { return c.compact ? N * ceil_div(observe, cols / G) : Tq / (cols / G) + N; };
  c.TP = 1024;
  while (c.TP > 128 && (double)pieces(kCols) * Hkv * ceil_div(cap, c.TP) * seen < want) c.TP /= 2;
  // (at most 64 pieces of a long row's tokens, as long as kMaxTP holds them)
  c.TP = (int)std::min<int64_t>(kMaxTP, std::max<int64_t>(c.TP, ceil_div(ceil_div(cap, 64), kStage) * kStage));
  c.CB = kMaxCB;
  while (c.CB > kCols && (double)pieces(c.CB) * Hkv * ceil_div(cap, kCols) * seen < want) c.CB /= 2;
  c.row_pieces = pieces(c.CB);
  return c;
}

uint64_t pad(uint64_t x) { return (x + 255) & ~(uint64_t)255; }

template <int QT, int KT, int D>
int32_t launch_d(const ChunkWeightsParams& p, hipStream_t stream) {
  const int64_t cap = (int64_t)p.Mb * 16;
  // as many workgroups as are resident: each takes every grid-th unit
  const dim3 grid((unsigned)(waves_per_simd<D>() * device_cu_count()));
  {
    ProfileScope prof("cf_chunk_rows", stream);
    CF_LAUNCH((chunk_rows_kernel<QT, KT, D>), grid, dim3(256), 0, stream, p);
    CF_HIP_CHECK(hipGetLastError());
  }
  {
    ProfileScope prof("cf_chunk_tokens", stream);
    CF_LAUNCH((chunk_tokens_kernel<QT, KT, D>), grid, dim3(256), 0, stream, p);
    CF_HIP_CHECK(hipGetLastError());
  }
  ProfileScope prof("cf_chunk_join", stream);
  // (many pieces a token: more loads in flight)
  if (ceil_div(p.Tq, p.N * (p.CB / p.G)) * (p.Hkv / p.Hw) >= 8)
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
  // a unit's offsets into q: 1,024 rows and 64 heads
  if (p.q_sr >= 1 << 20 || p.q_sh >= 1 << 20) return false;
  const int kb = k_dt == kE4M3 ? 1 : 2;
  if (p.k_s[3] != 1 || ((uintptr_t)p.k & 15) != 0 || ((uintptr_t)p.q & 15) != 0) return false;
  for (int i = 0; i < 3; ++i)
    if ((p.k_s[i] * kb) % 16 != 0) return false;
  return (p.q_sr * 2) % 16 == 0 && (p.q_sh * 2) % 16 == 0;
}

uint64_t chunk_weights_workspace_bytes(int64_t num_q_tokens, int64_t num_chunks, int64_t num_q_heads,
                                       int64_t num_kv_heads, int64_t head_dim, int64_t max_blocks, int64_t observe) {
  const int64_t cap = max_blocks * 16;
  const Cut c = cut_of(num_q_tokens, num_chunks, num_kv_heads, num_q_heads / num_kv_heads, head_dim, cap, observe);
  return pad((uint64_t)ceil_div(cap, c.TP) * c.stat_rows * num_q_heads * 8) +
         pad((uint64_t)c.row_pieces * num_kv_heads * cap * 4);
}

void chunk_weights_bind_workspace(ChunkWeightsParams& p, void* workspace) {
  const int64_t cap = (int64_t)p.Mb * 16;
  const Cut c = cut_of(p.Tq, p.N, p.Hkv, p.G, p.D, cap, p.observe);
  p.compact = c.compact;
  p.stat_rows = c.stat_rows;
  p.TP = c.TP;
  p.CB = c.CB;
  p.ws_ml = (float2*)workspace;
  p.ws_p = (float*)((char*)workspace + pad((uint64_t)ceil_div(cap, c.TP) * c.stat_rows * p.Hq * 8));
}

int32_t launch_chunk_weights(const ChunkWeightsParams& p, int q_dt, int k_dt, hipStream_t stream) {
  if (q_dt == kF16) return k_dt == kE4M3 ? launch_t<kF16, kE4M3>(p, stream) : launch_t<kF16, kF16>(p, stream);
  return k_dt == kE4M3 ? launch_t<kBF16, kE4M3>(p, stream) : launch_t<kBF16, kBF16>(p, stream);
}

}  // namespace cf
