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
__device__ __forceinline__ int64_t row_start(const KvBlocksParams& p, int64_t n) {
  const int64_t a = p.start[n * p.st_s];
  return a < 0 ? 0 : (a > p.T ? p.T : a);
}
__device__ __forceinline__ int64_t first_unit(const KvBlocksParams& p, int64_t n) {
  return row_start(p, n) / p.bs + 2 * n;
}

// The last sequence whose first unit is at most u (64 probes at a time); -1: none.
__device__ int sequence_of(const KvBlocksParams& p, int64_t u, int lane) {
  int lo = 0, len = p.N;
  for (;;) {
    const int step = (len + 63) >> 6, off = lane * step;
    const unsigned long long at = __ballot(off < len && first_unit(p, lo + off) <= u);
    if (at == 0) return -1;
    const int idx = uniform(63 - __clzll((long long)at));
    lo += idx * step;
    if (step == 1) return lo;
    len = min(step, len - idx * step);
  }
}

// What a unit writes: rows [row, row + rows) go to offsets off ... of block id.
struct Place {
  int64_t id, row;
  int off, rows;
};

__device__ __forceinline__ bool place_of(const KvBlocksParams& p, int64_t u, int lane, Place* at) {
  int64_t n = u, a = u, b = u + 1, j = 0;
  if (p.start != nullptr) {
    n = sequence_of(p, u, lane);
    if (n < 0) return false;
    a = row_start(p, n);
    b = row_start(p, n + 1);
    j = u - first_unit(p, n);
  }
  const int64_t len = p.lens[n * p.l_s], before = len - (b - a);  // position of row a
  const int64_t first = before > 0 ? before : 0;
  const int64_t jb = first / p.bs + j;
  const int64_t lo = jb * p.bs > first ? jb * p.bs : first;
  const int64_t hi = (jb + 1) * p.bs < len ? (jb + 1) * p.bs : len;
  if (lo >= hi || b <= a || jb >= p.Mb) return false;
  at->id = p.tables[n * p.t_sn + jb * p.t_sm];
  if (at->id < 0 || at->id >= p.NB) return false;
  at->row = a + (lo - before);
  at->off = (int)(lo - jb * p.bs);
  at->rows = (int)(hi - lo);
  return true;
}

// Any layout, a lane a channel.
template <int XT, int CT>
__global__ __launch_bounds__(64 * kTaskWaves) void kv_blocks_kernel(KvBlocksParams p) {
  const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6);
  const int task = (int)blockIdx.y * kTaskWaves + wave;
  if (task >= 2 * p.H) return;
  const int kv = task & 1, h = task >> 1;
  Place at;
  if (!place_of(p, blockIdx.x, lane, &at)) return;
  using X = Elem<XT>;
  using C = Elem<CT>;
  const typename X::T* x = (const typename X::T*)p.x[kv] + at.row * p.x_s[kv][0] + h * p.x_s[kv][1];
  uint8_t* c = (uint8_t*)p.cache[kv] + at.id * p.c_s[kv][0] + h * p.c_s[kv][2];
  float* scale = p.scale[kv] + at.id * p.s_s[kv][0] + h * p.s_s[kv][1];
  const int64_t xt = p.x_s[kv][0], xd = p.x_s[kv][2], ct = p.c_s[kv][1], cd = p.c_s[kv][3];
  const float old = at.off > 0 ? *scale : 0.0f;
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

template <int XT>
int32_t launch_x(const KvBlocksParams& p, int cache_dt, hipStream_t stream) {
  const dim3 grid((unsigned)p.units, (unsigned)ceil_div(2 * p.H, kTaskWaves));
  ProfileScope prof("cf_kv_write_blocks", stream);
  if (cache_dt == kI8) CF_LAUNCH((kv_blocks_kernel<XT, kI8>), grid, dim3(64 * kTaskWaves), 0, stream, p);
  else CF_LAUNCH((kv_blocks_kernel<XT, kE4M3>), grid, dim3(64 * kTaskWaves), 0, stream, p);
  CF_HIP_CHECK(hipGetLastError());
  return CF_OK;
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
