// New K and V rows into paged caches in 8 bits with a scale for each block and
// head (block_scale.hpp).
//
// Sequence n's rows take the last positions of its seq_lens[n].  For every block
// they touch, and every head: with m the largest magnitude of its new rows, and
// s0 its scale if it held rows before (it does where its first new row is not at
// offset 0; otherwise it starts anew, whatever was there),
//   s1 = max(s0, least scale for m);   new codes = code(x / s1);
//   the rows before the first new one, if s1 is not s0: code(old code * s0 / s1).
// So a block's codes always hold under its one scale, no row is ever out of range,
// and a block whose scale stands is not read.
//
// One wave takes one (block, head) of keys or of values, so nothing is shared
// between waves: no atomics, one launch, and results that do not depend on the
// order of anything.
#include "block_scale.hpp"
#include "cf_host.hpp"
#include "kv_blocks.hpp"

namespace cf {

namespace {

constexpr int kTaskWaves = 4;  // (block, head, keys or values) tasks of a workgroup

// Sequences own units of at least the blocks that their rows can touch: L rows
// touch at most L / bs + 2, so sequence n's first unit is start[n] / bs + 2 n.
// BS: the block size (0: the parameters').
template <int BS>
__device__ __forceinline__ int block_size(const KvBlocksParams& p) {
  return BS > 0 ? BS : p.bs;
}
__device__ __forceinline__ int row_start(const KvBlocksParams& p, int n) {
  return min(max(p.start[n * p.st_s], 0), (int)p.T);
}
template <int BS>
__device__ __forceinline__ int64_t first_unit(const KvBlocksParams& p, int n) {
  return (unsigned)row_start(p, n) / (unsigned)block_size<BS>(p) + 2 * (int64_t)n;
}

// What a unit writes: rows [row, row + rows) go to offsets off ... of block id.
struct Place {
  int64_t id;  // may lie outside of the cache: nothing is written then
  int row, off, rows;
};

// The sequence of unit u is the last whose first unit is at most u: 64 probes at a
// time, and the last of these rounds brings the sequence's rows and length along,
// so that up to 64 sequences take two dependent loads up to the block.
template <int BS>
__device__ __forceinline__ bool place_of(const KvBlocksParams& p, int64_t u, int lane, Place* at) {
  const int bs = block_size<BS>(p);
  int n = (int)u, a = n, b = n + 1, j = 0, len;
  if (p.start != nullptr) {
    int lo = 0, count = p.N;
    while (count > 64) {
      const int step = (count + 63) >> 6, off = lane * step;
      const unsigned long long below = __ballot(off < count && first_unit<BS>(p, lo + off) <= u);
      if (below == 0) return false;
      const int idx = uniform(63 - __clzll((long long)below));
      lo += idx * step;
      count = min(step, count - idx * step);
    }
    const int i = lo + min(lane, count - 1);
    const int ia = row_start(p, i), ib = row_start(p, i + 1), il = p.lens[i * p.l_s];
    const int64_t first = (unsigned)ia / (unsigned)bs + 2 * (int64_t)i;
    const unsigned long long below = __ballot(lane < count && first <= u);
    if (below == 0) return false;
    const int idx = uniform(63 - __clzll((long long)below));
    n = lo + idx;
    a = __builtin_amdgcn_readlane(ia, idx);
    b = __builtin_amdgcn_readlane(ib, idx);
    len = __builtin_amdgcn_readlane(il, idx);
    j = (int)(u - ((unsigned)a / (unsigned)bs + 2 * (int64_t)n));
  } else {
    len = p.lens[n * p.l_s];
  }
  if (b <= a || len <= 0) return false;
  const int64_t before = (int64_t)len - (b - a);  // position of row a
  const int first = before > 0 ? (int)before : 0;
  const int64_t jb = (unsigned)first / (unsigned)bs + j;
  const int64_t lo = max(jb * bs, (int64_t)first), hi = min((jb + 1) * bs, (int64_t)len);
  if (lo >= hi || jb >= p.Mb) return false;
  at->id = p.tables[n * p.t_sn + jb * p.t_sm];
  at->row = a + (int)(lo - before);
  at->off = (int)(lo - jb * bs);
  at->rows = (int)(hi - lo);
  return true;
}

__device__ __forceinline__ bool in_cache(const KvBlocksParams& p, const Place& at) { return at.id >= 0 && at.id < p.NB; }

// Any layout and block size, a lane a channel.
template <int XT, int CT>
__device__ void write_any(const KvBlocksParams& p, const Place& at, int kv, int h, int lane) {
  using X = Elem<XT>;
  using C = Elem<CT>;
  const typename X::T* x = (const typename X::T*)p.x[kv] + at.row * p.x_s[kv][0] + h * p.x_s[kv][1];
  uint8_t* c = (uint8_t*)p.cache[kv] + at.id * p.c_s[kv][0] + h * p.c_s[kv][2];
  float* scale = p.scale[kv] + at.id * p.s_s[kv][0] + h * p.s_s[kv][1];
  const int64_t xt = p.x_s[kv][0], xd = p.x_s[kv][2], ct = p.c_s[kv][1], cd = p.c_s[kv][3];
  const float old = at.off > 0 ? read_scale(*scale) : 0.0f;
  uint32_t m = 0;
  for (int r = 0; r < at.rows; ++r)
    for (int d = lane; d < p.D; d += 64) m = max(m, f2u(X::load(x + r * xt + d * xd)) & 0x7FFFFFFFu);
  const float s = widened(old, least_scale<CT>(wave_umax(m)));
  if (at.off > 0 && !(s == old)) {
    for (int r = 0; r < at.off; ++r)
      for (int d = lane; d < p.D; d += 64) {
        uint8_t* to = c + r * ct + d * cd;
        *to = block_code<CT>(C::load((const typename C::T*)to) * old, s);
      }
  }
  for (int r = 0; r < at.rows; ++r)
    for (int d = lane; d < p.D; d += 64)
      c[(at.off + r) * ct + d * cd] = block_code<CT>(X::load(x + r * xt + d * xd), s);
  if (lane == 0) *scale = s;
}

template <int XT, int CT>
__global__ __launch_bounds__(64 * kTaskWaves) void kv_blocks_kernel(KvBlocksParams p) {
  const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6);
  const int task = (int)blockIdx.y * kTaskWaves + wave;
  if (task >= 2 * p.H) return;
  Place at;
  if (!place_of<0>(p, blockIdx.x, lane, &at) || !in_cache(p, at)) return;
  write_any<XT, CT>(p, at, task & 1, task >> 1, lane);
}

// Blocks of 16 tokens of 64 or 128 channels whose rows (or channels) are whole
// pieces: a task's new rows are read once, into registers, by wide loads that are
// all in flight together, and its codes are stored in pieces of 8 or 16 bytes.
// Rows outside of the new ones are read as the nearest new one, which leaves the
// maximum as it is, so nothing but the stores of a block written in part is
// predicated.
//   rows: a lane has 8 channels of every (512 / D)-th token.
//   channels (V of the native layouts, tokens side by side): a lane has 2 channels
//   of all 16 tokens, at D = 64 of 8.
// Four prompts of 700-2,000 tokens (8 heads of 128, bf16 to e4m3; 25 MB read and
// written) take 9.5 us, a chunk step of 1,085 rows (f16 to int8, 6.7 MB) 6.1, 32
// single rows 4.6; every lane a byte at a time 27.8, 16.6 and 4.5.  The bytes alone
// would take 5.2 at a large copy's 4.8 TB/s: what is left is one launch's start and
// end and a wave's chain of dependent loads (lengths, table, rows) at the latency of
// HBM; 2 to 16 waves a workgroup and units or heads first in the grid measured alike.
constexpr int kTok = 16;

// Two new values in their type, and what of them orders as their magnitudes do.
template <int XT>
struct Pair {
  uint32_t u;
  __device__ __forceinline__ uint32_t mag() const { return u & 0x7FFF7FFFu; }
  __device__ __forceinline__ float2 values() const {
    if constexpr (XT == kBF16) return make_float2(u2f(u << 16), u2f(u & 0xFFFF0000u));
    else return make_float2((float)__builtin_bit_cast(_Float16, (uint16_t)u), (float)__builtin_bit_cast(_Float16, (uint16_t)(u >> 16)));
  }
};
template <>
struct Pair<kF32> {
  float2 f;
  __device__ __forceinline__ uint32_t mag() const { return max(f2u(f.x) & 0x7FFFFFFFu, f2u(f.y) & 0x7FFFFFFFu); }
  __device__ __forceinline__ float2 values() const { return f; }
};
template <int XT>
__device__ __forceinline__ uint32_t mag_max(uint32_t a, uint32_t b) {
  if constexpr (XT == kF32) {
    return max(a, b);
  } else {
    using H2 = uint16_t __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(H2, a), __builtin_bit_cast(H2, b)));
  }
}
// float32 bits of the largest magnitude of a wave (a NaN's above infinity's).
template <int XT>
__device__ __forceinline__ uint32_t wave_mag(uint32_t m) {
  if constexpr (XT == kF32) return wave_umax(m);
  const uint32_t h = wave_umax(max(m & 0xFFFFu, m >> 16));
  return XT == kBF16 ? h << 16 : f2u((float)__builtin_bit_cast(_Float16, (uint16_t)h));
}

// Quotients by one scale s < 2^126 without the division's instructions.  With r
// the rounded 1 / s, two steps q += r * (x - q * s) by fused products give the
// rounded quotient: after one q is within one step of it, and from such a q the
// next one rounds as the exact quotient does (Markstein, 1990).  The remainder is
// exact where the quotient is of at least 2^-60, as s >= 2^-40; below, every code
// is 0.  By a power of two the product alone is exact.
template <int CT>
struct BlockQuant {
  float s, r;
  bool two;  // s is a power of two
  __device__ __forceinline__ explicit BlockQuant(float scale) : s(scale), r(1.0f / scale), two((f2u(scale) & 0x7FFFFFu) == 0u) {}
  __device__ __forceinline__ float quotient(float x) const {
    float q = x * r;
    if (CT == kE4M3 && two) return q;
    q = __builtin_fmaf(__builtin_fmaf(-q, s, x), r, q);
    return __builtin_fmaf(__builtin_fmaf(-q, s, x), r, q);
  }
  // Four codes, the first in byte 0.  |x / s| is at most 448 (int8: 127, the
  // quotient's own rounding aside).
  __device__ __forceinline__ uint32_t codes(float a, float b, float c, float d) const {
    a = quotient(a), b = quotient(b), c = quotient(c), d = quotient(d);
    if constexpr (CT == kI8) {
      // the sum rounds to a whole number, ties to even, in the low bits
      constexpr float kWhole = 12582912.0f;  // 1.5 * 2^23
      const uint32_t ab = __builtin_amdgcn_perm(f2u(b + kWhole), f2u(a + kWhole), 0x0C0C0400u);
      return ab | __builtin_amdgcn_perm(f2u(d + kWhole), f2u(c + kWhole), 0x04000C0Cu);
    } else {
      int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
      return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
    }
  }
  // Four codes of scale `old` as codes of s (a NaN code stays as it is).
  __device__ __forceinline__ uint32_t recode(uint32_t w, float old) const {
    float f[4];
    if constexpr (CT == kI8) {
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = (float)max((int)(int8_t)(w >> (8 * i)), -127) * old;
      return codes(f[0], f[1], f[2], f[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint8_t c = (uint8_t)(w >> (8 * i));
        f[i] = Elem<CT>::load(&c) * old;
      }
      const uint32_t nan = ((((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) >> 7) * 0xFFu;
      return (codes(f[0], f[1], f[2], f[3]) & ~nan) | (w & nan);
    }
  }
};

template <int XT, int CT, int D, bool CHANNELS>
__device__ __forceinline__ bool write_wide(const KvBlocksParams& p, const Place& at, int kv, int h, int lane) {
  using T = typename Elem<XT>::T;
  using P = Pair<XT>;
  constexpr int LANES = CHANNELS ? D / 2 : D / 8;  // lanes of a token
  constexpr int STEP = 64 / LANES;                 // tokens of a pass (channels: halves of the tile)
  constexpr int N = kTok / STEP;                   // passes
  constexpr int W = CHANNELS ? 1 : 4;              // pairs of a pass
  const int d0 = (lane % LANES) * 2 * W, part = lane / LANES;
  auto token = [&](int i) { return CHANNELS ? part * N + i : i * STEP + part; };
  const T* x = (const T*)p.x[kv] + at.row * p.x_s[kv][0] + h * p.x_s[kv][1] + d0;
  // (an id outside of the cache is known only behind the rows' loads, which wait
  // for nothing but their place)
  const int64_t id = in_cache(p, at) ? at.id : 0;
  uint8_t* c = (uint8_t*)p.cache[kv] + id * p.c_s[kv][0] + h * p.c_s[kv][2];
  float* scale = p.scale[kv] + id * p.s_s[kv][0] + h * p.s_s[kv][1];
  const int64_t xt = p.x_s[kv][0];
  const int end = at.off + at.rows;
  P v[N][W];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int r = min(max(token(i) - at.off, 0), at.rows - 1);
    __builtin_memcpy(v[i], __builtin_assume_aligned(x + r * xt, sizeof(v[i]) < 16 ? sizeof(v[i]) : 16), sizeof(v[i]));
  }
  const float old = at.off > 0 ? read_scale(*scale) : 0.0f;
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int k = 0; k < W; ++k) m = mag_max<XT>(m, v[i][k].mag());
  const float s = widened(old, least_scale<CT>(wave_mag<XT>(m)));
  if (!in_cache(p, at)) return true;
  if (!(s < 0x1p126f)) return false;
  const BlockQuant<CT> q(s);
  const bool moved = at.off > 0 && s != old;
  if (lane == 0) *scale = s;
  if constexpr (CHANNELS) {
    const int64_t cd = p.c_s[kv][3];
    c += d0 * cd + part * N;
    uint32_t w[2][N / 4];
#pragma unroll
    for (int g = 0; g < N / 4; ++g) {
      float2 f[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = v[4 * g + i][0].values();
      w[0][g] = q.codes(f[0].x, f[1].x, f[2].x, f[3].x);
      w[1][g] = q.codes(f[0].y, f[1].y, f[2].y, f[3].y);
    }
    if (at.rows < kTok && !moved) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (token(i) >= at.off && token(i) < end)
#pragma unroll
          for (int k = 0; k < 2; ++k) c[k * cd + i] = (uint8_t)(w[k][i / 4] >> (8 * (i & 3)));
      return true;
    }
    if (moved) {
      uint32_t was[2][N / 4];
#pragma unroll
      for (int k = 0; k < 2; ++k) __builtin_memcpy(was[k], __builtin_assume_aligned(c + k * cd, N), N);
#pragma unroll
      for (int g = 0; g < N / 4; ++g) {
        uint32_t before = 0, after = 0;  // bytes of tokens ahead of and behind the new ones
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          before |= token(4 * g + i) < at.off ? 0xFFu << (8 * i) : 0u;
          after |= token(4 * g + i) >= end ? 0xFFu << (8 * i) : 0u;
        }
#pragma unroll
        for (int k = 0; k < 2; ++k)
          w[k][g] = (w[k][g] & ~(before | after)) | (was[k][g] & after) | (q.recode(was[k][g], old) & before);
      }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) __builtin_memcpy(__builtin_assume_aligned(c + k * cd, N), w[k], N);
  } else {
    const int64_t ct = p.c_s[kv][1];
    c += d0;
    if (moved) {
      uint2 was[N];
#pragma unroll
      for (int i = 0; i < N; ++i) was[i] = *(const uint2*)(c + min(token(i), at.off - 1) * ct);
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (token(i) < at.off)
          *(uint2*)(c + token(i) * ct) = make_uint2(q.recode(was[i].x, old), q.recode(was[i].y, old));
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float2 f[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) f[k] = v[i][k].values();
      const uint2 w = make_uint2(q.codes(f[0].x, f[0].y, f[1].x, f[1].y), q.codes(f[2].x, f[2].y, f[3].x, f[3].y));
      if (token(i) >= at.off && token(i) < end) *(uint2*)(c + token(i) * ct) = w;
    }
  }
  return true;
}

template <int XT, int CT, int D>
__global__ __launch_bounds__(64 * kTaskWaves) void kv_blocks_wide_kernel(KvBlocksParams p, int channels) {
  const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6);
  const int task = (int)blockIdx.y * kTaskWaves + wave;
  if (task >= 2 * p.H) return;
  const int kv = task & 1, h = task >> 1;
  Place at;
  if (!place_of<kTok>(p, blockIdx.x, lane, &at)) return;
  const bool done = (channels >> kv) & 1 ? write_wide<XT, CT, D, true>(p, at, kv, h, lane)
                                         : write_wide<XT, CT, D, false>(p, at, kv, h, lane);
  if (!done) write_any<XT, CT>(p, at, kv, h, lane);
}

// Whether the wide kernel takes the tensors; *channels: whose channels (bit 0: keys,
// bit 1: values) rather than rows hold whole pieces.
bool takes_wide(const KvBlocksParams& p, int x_size, int* channels) {
  if (p.bs != kTok || (p.D != 64 && p.D != 128)) return false;
  *channels = 0;
  for (int i = 0; i < 2; ++i) {
    const int64_t* x = p.x_s[i];
    const int64_t* c = p.c_s[i];
    if (x[2] != 1 || ((uintptr_t)p.x[i] | (uintptr_t)((x[0] | x[1]) * x_size)) % 16 != 0) return false;
    const uintptr_t far = (uintptr_t)p.cache[i] | (uintptr_t)(c[0] | c[2]);
    if (c[3] == 1 && (far | (uintptr_t)c[1]) % 8 == 0) continue;
    if (c[1] != 1 || (far | (uintptr_t)c[3]) % 16 != 0) return false;
    *channels |= 1 << i;
  }
  return true;
}

template <int XT, int CT>
int32_t launch_c(const KvBlocksParams& p, hipStream_t stream) {
  const dim3 grid((unsigned)p.units, (unsigned)ceil_div(2 * p.H, kTaskWaves)), block(64 * kTaskWaves);
  ProfileScope prof("cf_kv_write_blocks", stream);
  int channels;
  if (!takes_wide(p, XT == kF32 ? 4 : 2, &channels)) CF_LAUNCH((kv_blocks_kernel<XT, CT>), grid, block, 0, stream, p);
  else if (p.D == 64) CF_LAUNCH((kv_blocks_wide_kernel<XT, CT, 64>), grid, block, 0, stream, p, channels);
  else CF_LAUNCH((kv_blocks_wide_kernel<XT, CT, 128>), grid, block, 0, stream, p, channels);
  CF_HIP_CHECK(hipGetLastError());
  return CF_OK;
}

template <int XT>
int32_t launch_x(const KvBlocksParams& p, int cache_dt, hipStream_t stream) {
  return cache_dt == kI8 ? launch_c<XT, kI8>(p, stream) : launch_c<XT, kE4M3>(p, stream);
}

}  // namespace

int32_t launch_kv_blocks(KvBlocksParams p, int x_dt, int cache_dt, hipStream_t stream) {
  switch (x_dt) {
    case kF32: return launch_x<kF32>(p, cache_dt, stream);
    case kF16: return launch_x<kF16>(p, cache_dt, stream);
    default: return launch_x<kBF16>(p, cache_dt, stream);
  }
}

}  // namespace cf
