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
// kernel); a unit leaves (m, l) or sums of its piece in the workspace, joined
// in a fixed order, so there are no atomics.  Per visible pair the kernels
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
__device__ __forceinline__ Chunk chunk_of(const ChunkWeightsParams& p, int n, int start, int end) {
  Chunk c;
  c.n = n;
  c.start = start;
  const int len = max(p.seq_lens[(int64_t)n * p.sl_s], 0);
  const int rows = end - start;
  c.rows = p.observe > 0 ? min(rows, p.observe) : rows;
  c.row0 = end - c.rows;
  c.c0 = len - c.rows;
  c.cap = min(len, p.Mb * 16);
  c.fresh = len - rows;
  return c;
}

__device__ __forceinline__ int start_of(const ChunkWeightsParams& p, int n) {
  return min(max(p.q_start[(int64_t)n * p.qs_s], 0), p.Tq);
}

// Tokens visible to rows below `end` of the chunk.
__device__ __forceinline__ int visible(const Chunk& c, int end) { return min(max(c.c0 + min(end, c.rows), 0), c.cap); }

__device__ __forceinline__ int cdiv(int a, int b) { return (a + b - 1) / b; }

// Units of a chunk and head: blocks of R rows times blocks of TB tokens.  A
// causal chunk's first rows see few tokens and its last ones many, so row
// block k shares a line of `width` units with block nb - 1 - k: the lines of a
// chunk are then about equally long, and few of their units are empty.
struct Grid {
  int nb, width, units;
};

__device__ __forceinline__ Grid grid_of(const Chunk& c, int R, int TB) {
  Grid g;
  g.nb = cdiv(c.rows, R);
  if (g.nb <= 1) {
    g.width = cdiv(visible(c, c.rows), TB);
  } else {
    const int64_t both = 2 * (int64_t)max(c.c0, 0) + (int64_t)(g.nb + 1) * R;
    const int64_t most = 2 * (int64_t)cdiv(c.cap, TB);
    g.width = (int)min((both + TB - 1) / TB + 1, most);
  }
  g.units = ((g.nb + 1) / 2) * g.width;
  return g;
}

// Unit u of a launch: its chunk, head, row block and token block.  False past
// the last unit; empty (tb < 0) where a line ends early.
struct Unit {
  Chunk c;
  int h, rb, tb;
};

__device__ bool unit_of(const ChunkWeightsParams& p, int64_t u, int R, int TB, int lane, Unit* out) {
  const int h = (int)(u % p.Hkv);
  int64_t v = u / p.Hkv;
  int before = 0;  // where the chunks before the lanes' end
  for (int base = 0; base < p.N; base += 64) {
    const int n = base + lane;
    // a chunk starts where the ones before it end, if q_start has it earlier
    const int start = max(wave_incl_max(n < p.N ? start_of(p, n) : 0, lane), before);
    const int end = n < p.N ? max(start_of(p, n + 1), start) : start;
    int units = 0;
    if (n < p.N) units = grid_of(chunk_of(p, n, start, end), R, TB).units;
    const int incl = wave_incl_scan(units, lane);
    const uint64_t hit = __ballot(incl > v);
    if (hit == 0) {
      v -= wave_last(incl);
      before = wave_last(start);
      continue;
    }
    const int at = __ffsll((long long)hit) - 1;
    v -= uniform(__shfl(incl - units, at, 64));
    out->c = chunk_of(p, base + at, uniform(__shfl(start, at, 64)), uniform(__shfl(end, at, 64)));
    const Grid g = grid_of(out->c, R, TB);
    const int k = (int)v / g.width, t = (int)v - k * g.width;
    const int first = cdiv(visible(out->c, (k + 1) * R), TB);
    const int mate = g.nb - 1 - k;
    out->h = h;
    out->rb = t < first ? k : mate;
    out->tb = t < first ? t : t - first;
    if (t >= first && (mate == k || out->tb >= cdiv(visible(out->c, (mate + 1) * R), TB))) out->tb = -1;
    return true;
  }
  return false;
}

template <int D>
constexpr int row_bytes() {
  return D * 2 + 16;  // a staged row: 16 bytes more than whole bank rounds, so 16 rows lie in different banks
}

__device__ __forceinline__ int block_of(const ChunkWeightsParams& p, int n, int j) {
  if (j >= p.Mb) return -1;
  const int id = p.tables[(int64_t)n * p.t_sb + (int64_t)j * p.t_sm];
  return id >= 0 && id < p.NB ? id : -1;
}

// 16 bytes of operand (8 channels) of a K row: as stored, or converted (exactly).
template <int QT, int KT>
__device__ __forceinline__ uint4 k_piece(const ChunkWeightsParams& p, int blk, int off, int h, int d) {
  const int64_t at = (int64_t)blk * p.k_s[0] + (int64_t)off * p.k_s[1] + (int64_t)h * p.k_s[2] + d;
  if constexpr (KT == kE4M3) {
    const uint2 v = *(const uint2*)((const uint8_t*)p.k + at);
    if constexpr (QT == kF16) return __builtin_bit_cast(uint4, e4m3x8_to_f16(v.x, v.y));
    else return __builtin_bit_cast(uint4, e4m3x8_to_bf16(v.x, v.y));
  } else {
    return *(const uint4*)((const uint16_t*)p.k + at);
  }
}

// 16 bytes of a q row; `flip` changes the sign of every element.
__device__ __forceinline__ uint4 q_piece(const ChunkWeightsParams& p, int row, int hq, int d, uint32_t flip) {
  uint4 v = *(const uint4*)((const uint16_t*)p.q + (int64_t)row * p.q_sr + (int64_t)hq * p.q_sh + d);
  v.x ^= flip;
  v.y ^= flip;
  v.z ^= flip;
  v.w ^= flip;
  return v;
}

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
__global__ __launch_bounds__(256) void chunk_rows_kernel(ChunkWeightsParams p, int64_t max_units) {
  constexpr int NC = D / 32, RB = row_bytes<D>(), PPR = D / 8;  // MFMAs a tile, 16-byte pieces a row
  constexpr int LOADS = kStage * PPR / 256;
  __shared__ __align__(16) uint8_t stage[2][kStage * RB];
  __shared__ int ids[2][kStage / 16];
  const int tid = threadIdx.x, lane = tid & 63, li = lane & 15, lq = lane >> 4, wave = uniform(tid >> 6);
  const int R = kCols / p.G;
  for (int64_t u = blockIdx.x; u < max_units; u += gridDim.x) {
    Unit un;
    if (!unit_of(p, u, R, p.TP, lane, &un)) return;
    if (un.tb < 0) continue;
    const Chunk& c = un.c;
    const int r0 = un.rb * R, nr = min(R, c.rows - r0), ncol = nr * p.G;
    const int t_begin = un.tb * p.TP, t_end = min(t_begin + p.TP, visible(c, r0 + nr));
    const Factor f = factor_of(p, un.h);
    // this wave's 64 columns: four tiles of 16
    QOp<QT> q[4][NC];
    int pos[4];  // last token that the lane's column of tile ct sees
#pragma unroll
    for (int ct = 0; ct < 4; ++ct) {
      const int j = wave * 64 + ct * 16 + li, r = j / p.G, g = j - r * p.G;
      pos[ct] = j < ncol ? c.c0 + r0 + r : -1;
#pragma unroll
      for (int x = 0; x < NC; ++x)
        q[ct][x] = as_qop<QT>(j < ncol ? q_piece(p, c.row0 + r0 + r, un.h * p.G + g, 32 * x + 8 * lq, f.flip)
                                       : make_uint4(0, 0, 0, 0));
    }
    // positions of the wave's first and last column
    const int w_lo = c.c0 + r0 + wave * 64 / p.G, w_hi = c.c0 + r0 + min(wave * 64 + 63, ncol - 1) / p.G;
    const bool busy = wave * 64 < ncol;
    float m[4], l[4];
#pragma unroll
    for (int ct = 0; ct < 4; ++ct) m[ct] = -INFINITY, l[ct] = 0.0f;

    uint4 reg[LOADS];
    auto fetch = [&](int t0) {  // tokens t0 .. + 63 (those past the end: the last one's block, masked)
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int e = i * 256 + tid, t = t0 + e / PPR;
        const int blk = block_of(p, c.n, min(t, t_end - 1) >> 4);
        reg[i] = k_piece<QT, KT>(p, blk < 0 ? 0 : blk, t & 15, un.h, e % PPR * 8);
      }
    };
    auto store = [&](int t0, int buf) {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int e = i * 256 + tid;
        *(uint4*)(stage[buf] + e / PPR * RB + e % PPR * 16) = reg[i];
      }
      if (tid < kStage / 16) ids[buf][tid] = t0 + tid * 16 < t_end ? block_of(p, c.n, (t0 >> 4) + tid) : -1;
    };
    fetch(t_begin);
    store(t_begin, 0);
    __syncthreads();
    for (int t0 = t_begin, buf = 0; t0 < t_end; t0 += kStage, buf ^= 1) {
      const bool more = t0 + kStage < t_end;
      if (more) fetch(t0 + kStage);
      if (busy && t0 <= w_hi) {
        bool whole = t0 + kStage - 1 <= w_lo && t0 + kStage <= t_end;
#pragma unroll
        for (int tt = 0; tt < kStage / 16; ++tt) whole = whole && uniform(ids[buf][tt]) >= 0;
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
                const int last = ids[buf][tt] < 0 ? -1 : min(pos[ct], t_end - 1);
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
      if (more) store(t0 + kStage, buf ^ 1);
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
      const int j = wave * 64 + ct * 16 + li, r = j / p.G, g = j - r * p.G;
      if (lq == 0 && j < ncol)
        p.ws_ml[((int64_t)un.tb * p.Tq + c.row0 + r0 + r) * p.Hq + un.h * p.G + g] = make_float2(M, L);
    }
    __syncthreads();  // the stage is filled anew
  }
}

// ---- tokens: sums over the rows of a piece -----------------------------------

// Index of a chunk's first row piece of R rows in ws_p: chunks before it use at
// most one piece more than their rows fill.
__device__ __forceinline__ int64_t piece0(const Chunk& c, int R) { return (int64_t)(c.start / R) + c.n; }

template <int QT, int KT, int D>
__global__ __launch_bounds__(256) void chunk_tokens_kernel(ChunkWeightsParams p, int64_t max_units) {
  constexpr int NC = D / 32, RB = row_bytes<D>(), PPR = D / 8;
  constexpr int LOADS = kStage * PPR / 256;
  __shared__ __align__(16) uint8_t stage[2][kStage * RB];
  __shared__ float2 fin[kMaxCB];  // (-m, 1 / l) of the unit's columns
  const int tid = threadIdx.x, lane = tid & 63, li = lane & 15, lq = lane >> 4, wave = uniform(tid >> 6);
  const int R = p.CB / p.G, RA = kCols / p.G;
  for (int64_t u = blockIdx.x; u < max_units; u += gridDim.x) {
    Unit un;
    if (!unit_of(p, u, R, kCols, lane, &un)) return;
    if (un.tb < 0) continue;
    const Chunk& c = un.c;
    const int r0 = un.rb * R, nr = min(R, c.rows - r0), ncol = nr * p.G;
    const int vis = visible(c, r0 + nr);
    const int t0 = un.tb * kCols, tw = t0 + wave * 64;  // the unit's and the wave's first token
    const Factor f = factor_of(p, un.h);
    // columns before the first row that sees the unit's tokens are left out
    const int j_begin = max(t0 - c.c0 - r0, 0) * p.G & ~(kStage - 1);

    // the rows' references and sums, from their pieces
    for (int j = j_begin + tid; j < cdiv(ncol, kStage) * kStage; j += 256) {
      float2 v = make_float2(0.0f, 0.0f);
      if (j < ncol) {
        const int r = j / p.G, g = j - r * p.G, row = r0 + r;
        const float2* ml = p.ws_ml + (int64_t)(c.row0 + row) * p.Hq + un.h * p.G + g;
        const int64_t step = (int64_t)p.Tq * p.Hq;
        const int np = cdiv(visible(c, (row / RA + 1) * RA), p.TP);  // pieces that the rows kernel wrote
        float M = -INFINITY, L = 0.0f;
        for (int i = 0; i < np; ++i) {
          const float2 x = ml[i * step];
          const float mn = fmaxf(M, x.x);
          L = L * (M == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(M - mn)) +
              x.y * (x.x == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(x.x - mn));
          M = mn;
        }
        v = make_float2(M == -INFINITY ? 0.0f : -M, L == 0.0f ? 0.0f : 1.0f / L);
      }
      fin[j] = v;
    }

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
        k[tt][x] = as_qop<QT>(k_piece<QT, KT>(p, blk < 0 ? 0 : blk, li, un.h, 32 * x + 8 * lq));
    }
    const bool all_live = live[0] + live[1] + live[2] + live[3] == 64;
    float acc[4][4];
#pragma unroll
    for (int tt = 0; tt < 4; ++tt)
#pragma unroll
      for (int v = 0; v < 4; ++v) acc[tt][v] = 0.0f;

    uint4 reg[LOADS];
    auto fetch = [&](int j0) {  // columns j0 .. + 63 (zeros past the last)
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int e = i * 256 + tid, j = j0 + e / PPR, r = j / p.G, g = j - r * p.G;
        reg[i] = j < ncol ? q_piece(p, c.row0 + r0 + r, un.h * p.G + g, e % PPR * 8, f.flip) : make_uint4(0, 0, 0, 0);
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
    store(0);
    __syncthreads();
    for (int j0 = j_begin, buf = 0; j0 < ncol; j0 += kStage, buf ^= 1) {
      const bool more = j0 + kStage < ncol;
      if (more) fetch(j0 + kStage);
      // the last of these columns sees the wave's first token, and the first its last
      if (tw < vis && c.c0 + r0 + min(j0 + kStage - 1, ncol - 1) / p.G >= tw) {
        const bool whole = all_live && c.c0 + r0 + j0 / p.G >= tw + 63;
        auto tiles = [&](auto masked) {
          constexpr bool kMasked = decltype(masked)::value;
#pragma unroll
          for (int ct = 0; ct < 4; ++ct) {
            const float2 col = fin[j0 + ct * 16 + li];
            QOp<QT> q[NC];
#pragma unroll
            for (int x = 0; x < NC; ++x)
              q[x] = as_qop<QT>(*(const uint4*)(stage[buf] + (ct * 16 + li) * RB + x * 64 + lq * 16));
            const int j = j0 + ct * 16 + li, last = !kMasked ? 0 : (j < ncol ? c.c0 + r0 + j / p.G : -1);
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
      float* out = p.ws_p + ((piece0(c, R) + un.rb) * p.Hkv + un.h) * (int64_t)p.Mb * 16;
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

__global__ __launch_bounds__(256) void chunk_join_kernel(ChunkWeightsParams p) {
  const int per = p.Mb * 16, chunks = cdiv(per, 256);
  const int nh = blockIdx.x / chunks, n = nh / p.Hw, hw = nh - n * p.Hw;
  const int t = (blockIdx.x - nh * chunks) * 256 + threadIdx.x;
  int start = 0;  // the end of the chunks before, and this one's own start
  for (int i = (int)(threadIdx.x & 63); i <= n; i += 64) start = max(start, start_of(p, i));
  start = wave_last(wave_incl_max(start, 0));
  const Chunk c = chunk_of(p, n, start, max(start_of(p, n + 1), start));
  if (c.rows == 0 || t >= c.cap) return;
  const int R = p.CB / p.G, nb = cdiv(c.rows, R), heads = p.Hkv / p.Hw;
  // the first row block that sees token t
  const int first = max(t - c.c0, 0) / R;
  float sum = 0.0f;
  for (int rb = first; rb < nb; ++rb)
    for (int h = hw * heads; h < (hw + 1) * heads; ++h)
      sum += p.ws_p[((piece0(c, R) + rb) * p.Hkv + h) * (int64_t)per + t];
  float* w = p.weights + (int64_t)n * p.w_sb + (int64_t)hw * p.w_sh + t;
  *w = t >= c.fresh || p.decay == 0.0f ? sum : __builtin_fmaf(*w, p.decay, sum);
}

// ---- launch ------------------------------------------------------------------

int64_t row_pieces(int64_t Tq, int64_t N, int64_t G, int64_t CB) { return Tq / (CB / G) + N; }

// Columns of a tokens-kernel unit and tokens of a rows-kernel unit: long ones
// reuse what they hold in registers more often, short ones spread a small call
// over the GPU.
int col_block(int64_t Tq, int64_t N, int64_t Hkv, int64_t G, int64_t cap) {
  return row_pieces(Tq, N, G, kMaxCB) * Hkv * ceil_div(cap, kCols) / 2 >= 2 * (int64_t)device_cu_count() ? kMaxCB : kCols;
}
int token_piece(int64_t Tq, int64_t N, int64_t Hkv, int64_t G, int64_t cap) {
  const int64_t few = row_pieces(Tq, N, G, kCols) * Hkv * ceil_div(cap, 1024) / 2 < 2 * (int64_t)device_cu_count();
  const int64_t most = ceil_div(cap, 16);  // at most 16 pieces of a long row
  return (int)std::max<int64_t>(few ? 256 : 1024, ceil_div(most, kStage) * kStage);
}

uint64_t pad(uint64_t x) { return (x + 255) & ~(uint64_t)255; }

template <int QT, int KT, int D>
int32_t launch_d(const ChunkWeightsParams& p, hipStream_t stream) {
  const int64_t cap = (int64_t)p.Mb * 16;
  // upper bounds of the units (a chunk's lines hold at most both of their blocks')
  const int64_t ua = (row_pieces(p.Tq, p.N, p.G, kCols) + p.N) * p.Hkv * (ceil_div(cap, p.TP) + 1);
  const int64_t ub = (row_pieces(p.Tq, p.N, p.G, p.CB) + p.N) * p.Hkv * (ceil_div(cap, kCols) + 1);
  const int64_t most = 3 * (int64_t)device_cu_count();
  {
    ProfileScope prof("cf_chunk_rows", stream);
    CF_LAUNCH((chunk_rows_kernel<QT, KT, D>), dim3((unsigned)std::min(ua, most)), dim3(256), 0, stream, p, ua);
    CF_HIP_CHECK(hipGetLastError());
  }
  {
    ProfileScope prof("cf_chunk_tokens", stream);
    CF_LAUNCH((chunk_tokens_kernel<QT, KT, D>), dim3((unsigned)std::min(ub, most)), dim3(256), 0, stream, p, ub);
    CF_HIP_CHECK(hipGetLastError());
  }
  ProfileScope prof("cf_chunk_join", stream);
  CF_LAUNCH(chunk_join_kernel, dim3((unsigned)(ceil_div(cap, 256) * p.N * p.Hw)), dim3(256), 0, stream, p);
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
  const int kb = k_dt == kE4M3 ? 1 : 2;
  if (p.k_s[3] != 1 || ((uintptr_t)p.k & 15) != 0 || ((uintptr_t)p.q & 15) != 0) return false;
  for (int i = 0; i < 3; ++i)
    if ((p.k_s[i] * kb) % 16 != 0) return false;
  return (p.q_sr * 2) % 16 == 0 && (p.q_sh * 2) % 16 == 0;
}

uint64_t chunk_weights_workspace_bytes(int64_t num_q_tokens, int64_t num_chunks, int64_t num_q_heads,
                                       int64_t num_kv_heads, int64_t max_blocks) {
  const int64_t cap = max_blocks * 16, G = num_q_heads / num_kv_heads;
  const int64_t tp = token_piece(num_q_tokens, num_chunks, num_kv_heads, G, cap);
  const int64_t cb = col_block(num_q_tokens, num_chunks, num_kv_heads, G, cap);
  return pad((uint64_t)ceil_div(cap, tp) * num_q_tokens * num_q_heads * 8) +
         pad((uint64_t)row_pieces(num_q_tokens, num_chunks, G, cb) * num_kv_heads * cap * 4);
}

void chunk_weights_bind_workspace(ChunkWeightsParams& p, void* workspace) {
  const int64_t cap = (int64_t)p.Mb * 16;
  p.TP = token_piece(p.Tq, p.N, p.Hkv, p.G, cap);
  p.CB = col_block(p.Tq, p.N, p.Hkv, p.G, cap);
  p.ws_ml = (float2*)workspace;
  p.ws_p = (float*)((char*)workspace + pad((uint64_t)ceil_div(cap, p.TP) * p.Tq * p.Hq * 8));
}

int32_t launch_chunk_weights(const ChunkWeightsParams& p, int q_dt, int k_dt, hipStream_t stream) {
  if (q_dt == kF16) return k_dt == kE4M3 ? launch_t<kF16, kE4M3>(p, stream) : launch_t<kF16, kF16>(p, stream);
  return k_dt == kE4M3 ? launch_t<kBF16, kE4M3>(p, stream) : launch_t<kBF16, kBF16>(p, stream);
}

}  // namespace cf
