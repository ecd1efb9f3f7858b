// Rotary positions on query and key rows, keys and values into the paged cache.
//
// Channel pair j of a row at position p (of the pair's axis) turns by the
// angle p * inv_freq[j]:
//   (x1, x2) -> (x1 cos - x2 sin, x2 cos + x1 sin),
// the pair's channels being (j, j + pairs) or (2 j, 2 j + 1); channels from
// 2 * pairs on pass.  Images and video give a token several positions (time,
// height, width), and a pair follows one of these axes: the first section[0]
// pairs axis 0, the next section[1] axis 1, ... or, cycled, pair j axis
// a = j % axes while j < axes * section[a], else axis 0.
//
// A rotated row is rounded once, to its output's type: e4m3fn cache codes are
// those of the float32 row divided by the head's scale, not of a row rounded
// to bf16 before.
//
// Angles are whole turns and a rest: p * inv_freq / (2 pi) is formed in 64
// bits (a position of 1e6 has an angle known to 0.06 rad only in 32), and its
// distance to the nearest whole number goes to sincospi.  A token's cosines
// and sines are computed once for eight heads and kept in LDS.
//
// A workgroup takes one token or a group of 16 and some heads of the queries,
// the keys or the values; a thread takes eight pairs (two 16-byte pieces of a
// 16-bit row).  Bound by bytes for prompts (about 4,900 rows of 32 + 8 + 8 heads
// of 128, bf16 to e4m3 with channel-major values: 110 MB in 26.3 us, 4.2 TB/s,
// with two sets of inputs in turn, of which the last-level cache still holds some,
// and 30.7 us, 3.6 TB/s, with three; launch-stamped events), by the launch for a
// decode step (32 rows: 4.2 us).
#include <algorithm>

#include "cf_device.hpp"
#include "cf_host.hpp"
#include "rotary.hpp"

namespace cf {

namespace {

constexpr int kHeads = 8;     // heads of a workgroup, for single tokens
constexpr int kMostHeads = 16;  // ... and for groups of tokens, kLeast to kMostHeads
constexpr int kLeast = 4;
constexpr int kWorkgroups = 1024;
constexpr int kTileD = 128;   // longest value row the transposing stage holds
constexpr int kPiece = 8;     // channels of a piece

template <int DT>
constexpr int esize() {
  return (int)sizeof(typename Elem<DT>::T);
}

// kPiece consecutive elements as f32, by accesses of 8 or 16 bytes.
template <int DT>
__device__ __forceinline__ void load8(const void* base, int64_t off, float* f) {
  using T = typename Elem<DT>::T;
  union {
    uint4 q[DT == kF32 ? 2 : 1];
    T e[kPiece];
  } u;
  const uint4* src = (const uint4*)((const T*)base + off);
#pragma unroll
  for (int i = 0; i < (DT == kF32 ? 2 : 1); ++i) u.q[i] = src[i];
#pragma unroll
  for (int i = 0; i < kPiece; ++i) f[i] = Elem<DT>::load(&u.e[i]);
}

template <int DT>
__device__ __forceinline__ typename Elem<DT>::T encode(float f, const Fp8Quant& qz) {
  typename Elem<DT>::T v;
  if constexpr (DT == kE4M3) v = qz(f);
  else Elem<DT>::store(&v, f);
  return v;
}

// kPiece elements as stored.
template <int DT>
union Encoded {
  uint32_t w[kPiece * esize<DT>() / 4];
  typename Elem<DT>::T e[kPiece];
  __device__ __forceinline__ Encoded(const float* f, const Fp8Quant& qz) {
    if constexpr (DT == kE4M3) {
      const uint2 v = qz.pack8(f);
      w[0] = v.x;
      w[1] = v.y;
    } else {
#pragma unroll
      for (int i = 0; i < kPiece; ++i) e[i] = encode<DT>(f[i], qz);
    }
  }
};

// Elements of a staged value row: one bank past a whole number of them.
template <int DT>
constexpr int turned_row() {
  return kTileD + 4 / esize<DT>();
}

template <int DT>
__device__ __forceinline__ void store8(void* base, int64_t off, const float* f, const Fp8Quant& qz) {
  const Encoded<DT> u(f, qz);
  typename Elem<DT>::T* dst = (typename Elem<DT>::T*)base + off;
  if constexpr (DT == kE4M3) {
    *(uint2*)dst = make_uint2(u.w[0], u.w[1]);
  } else {
#pragma unroll
    for (int i = 0; i < esize<DT>() / 2; ++i)
      ((uint4*)dst)[i] = make_uint4(u.w[4 * i], u.w[4 * i + 1], u.w[4 * i + 2], u.w[4 * i + 3]);
  }
}

__device__ __forceinline__ int axis_of(const RotaryParams& p, int j) {
  if (p.axes == 1) return 0;
  if (p.cycled) {
    const int a = j % p.axes;
    return j < p.axes * p.section[a] ? a : 0;
  }
  int a = 0, end = p.section[0];
  while (a + 1 < p.axes && j >= end) end += p.section[++a];
  return a;
}

__device__ __forceinline__ float2 cos_sin(const RotaryParams& p, int64_t t, int j) {
  const int64_t at = axis_of(p, j) * p.p_sa + t * p.p_st;
  const int64_t pos = p.pos64 ? ((const int64_t*)p.positions)[at] : (int64_t)((const int32_t*)p.positions)[at];
  double turns = (double)pos * (double)p.inv_freq[j * p.f_s] * 0.15915494309189533577;
  turns -= __builtin_rint(turns);
  float s, c;
  sincospif(2.0f * (float)turns, &s, &c);
  return make_float2(c * p.rotary_scale, s * p.rotary_scale);
}

// Element offset of token t's row in a cache, without its head and channel;
// -1 where its slot lies outside the cache.
__device__ __forceinline__ int64_t slot_offset(const RotaryParams& p, int64_t t, const int64_t* s) {
  const int64_t sl =
      p.slot64 ? ((const int64_t*)p.slots)[t * p.slot_s] : (int64_t)((const int32_t*)p.slots)[t * p.slot_s];
  if (sl < 0 || sl >= p.NB * p.bs) return -1;
  const int64_t blk = (sl >> 32) == 0 ? (int64_t)((uint32_t)sl / (uint32_t)p.bs) : sl / p.bs;
  return blk * s[0] + (sl - blk * p.bs) * s[1];
}

// Rows of nh heads of the queries (WHAT 0) or keys (1): rotated
// pieces, then the pieces that pass.
template <int XT, int OT, int TT, int THREADS, int WHAT>
__device__ __forceinline__ void rotate_rows(const RotaryParams& p, int64_t t0, int nt, int h0, int nh,
                                            const float2* cs, const int64_t* dst) {
  const int64_t* xs = p.x_s[WHAT];
  const int64_t os_h = WHAT == 0 ? p.o_s[1] : p.c_s[0][2], os_d = WHAT == 0 ? p.o_s[2] : p.c_s[0][3];
  void* out = WHAT == 0 ? p.out : p.cache[0];
  using X = typename Elem<XT>::T;
  using O = typename Elem<OT>::T;
  const bool vec = p.vec[WHAT];
  const int step = vec ? kPiece : 1;
  const int rot = p.pairs / step, items = rot + (p.D - 2 * p.pairs) / step;
  for (int u = threadIdx.x; u < nt * nh * items; u += THREADS) {
    const int th = u / items, c = u - th * items, t = th / nh, h = h0 + th - t * nh;
    if (dst[t] < 0) continue;
    const int64_t src = (t0 + t) * xs[0] + h * xs[1];
    const int64_t to = dst[t] + h * os_h;
    const Fp8Quant qz(OT == kE4M3 ? p.scale[0][h * p.sc_s[0]] : 1.0f);
    if (vec) {
      if (c >= rot) {
        float f[kPiece];
        const int d = 2 * p.pairs + (c - rot) * kPiece;
        load8<XT>(p.x[WHAT], src + d, f);
        store8<OT>(out, to + d, f, qz);
        continue;
      }
      float a[kPiece], b[kPiece], ra[kPiece], rb[kPiece];
      const int j0 = c * kPiece;
      const int da = p.adjacent ? 2 * j0 : j0, db = p.adjacent ? da + kPiece : j0 + p.pairs;
      load8<XT>(p.x[WHAT], src + da, a);
      load8<XT>(p.x[WHAT], src + db, b);
      const float2* w = cs + t * p.pairs + j0;
      if (p.adjacent) {  // a, b: pairs j0 .. + 3 and j0 + 4 .. + 7, each as x1, x2, x1, x2, ...
#pragma unroll
        for (int i = 0; i < kPiece / 2; ++i) {
          const float2 wa = w[i], wb = w[i + kPiece / 2];
          ra[2 * i] = a[2 * i] * wa.x - a[2 * i + 1] * wa.y;
          ra[2 * i + 1] = a[2 * i + 1] * wa.x + a[2 * i] * wa.y;
          rb[2 * i] = b[2 * i] * wb.x - b[2 * i + 1] * wb.y;
          rb[2 * i + 1] = b[2 * i + 1] * wb.x + b[2 * i] * wb.y;
        }
      } else {
#pragma unroll
        for (int i = 0; i < kPiece; ++i) {
          const float2 wi = w[i];
          ra[i] = a[i] * wi.x - b[i] * wi.y;
          rb[i] = b[i] * wi.x + a[i] * wi.y;
        }
      }
      store8<OT>(out, to + da, ra, qz);
      store8<OT>(out, to + db, rb, qz);
    } else {
      const X* x = (const X*)p.x[WHAT] + src;
      O* o = (O*)out + to;
      if (c >= rot) {
        const int d = 2 * p.pairs + c - rot;
        o[d * os_d] = encode<OT>(Elem<XT>::load(x + d * xs[2]), qz);
        continue;
      }
      const int d1 = p.adjacent ? 2 * c : c, d2 = p.adjacent ? d1 + 1 : c + p.pairs;
      const float a = Elem<XT>::load(x + d1 * xs[2]), b = Elem<XT>::load(x + d2 * xs[2]);
      const float2 w = cs[t * p.pairs + c];
      o[d1 * os_d] = encode<OT>(a * w.x - b * w.y, qz);
      o[d2 * os_d] = encode<OT>(b * w.x + a * w.y, qz);
    }
  }
}

// Value rows by pieces, or one channel a thread.
template <int XT, int CT, int THREADS>
__device__ __forceinline__ void copy_values(const RotaryParams& p, int64_t t0, int nt, int h0, int nh,
                                            const int64_t* dst) {
  const int64_t *xs = p.x_s[2], *s = p.c_s[1];
  const bool vec = p.vec[2];
  const int items = vec ? p.D / kPiece : p.D;
  for (int u = threadIdx.x; u < nt * nh * items; u += THREADS) {
    const int th = u / items, c = u - th * items, t = th / nh, h = h0 + th - t * nh;
    if (dst[t] < 0) continue;
    const Fp8Quant qz(CT == kE4M3 ? p.scale[1][h * p.sc_s[1]] : 1.0f);
    const int64_t src = (t0 + t) * xs[0] + h * xs[1], to = dst[t] + h * s[2];
    if (vec) {
      float f[kPiece];
      load8<XT>(p.x[2], src + c * kPiece, f);
      store8<CT>(p.cache[1], to + c * kPiece, f, qz);
    } else {
      const float f = Elem<XT>::load((const typename Elem<XT>::T*)p.x[2] + src + c * xs[2]);
      ((typename Elem<CT>::T*)p.cache[1])[to + c * s[3]] = encode<CT>(f, qz);
    }
  }
}

// Value rows into a channel-major tile (tokens of a channel side by side):
// the heads' 16 rows are turned over in LDS, so that both reads and writes are
// whole runs; four tokens of a channel go out in one store where their slots
// follow each other.
template <int XT, int CT, int THREADS>
__device__ __forceinline__ void turn_values(const RotaryParams& p, int64_t t0, int nt, int h0, int nh,
                                            const int64_t* dst, uint8_t* stage_all) {
  using C = typename Elem<CT>::T;
  constexpr int kRow = turned_row<CT>();
  C* stage = (C*)stage_all;
  const int64_t *xs = p.x_s[2], *s = p.c_s[1];
  const int per = p.D / kPiece;
  for (int u = threadIdx.x; u < nh * 16 * per; u += THREADS) {
    const int th = u / per, c = (u - th * per) * kPiece, t = th & 15, h = h0 + (th >> 4);
    if (t >= nt) continue;
    const Fp8Quant qz(CT == kE4M3 ? p.scale[1][h * p.sc_s[1]] : 1.0f);
    float f[kPiece];
    load8<XT>(p.x[2], (t0 + t) * xs[0] + h * xs[1] + c, f);
    const Encoded<CT> v(f, qz);
    uint32_t* row = (uint32_t*)(stage + th * kRow + c);  // (a row is a whole number of words)
#pragma unroll
    for (int i = 0; i < kPiece * esize<CT>() / 4; ++i) row[i] = v.w[i];
  }
  __syncthreads();
  for (int u = threadIdx.x; u < nh * p.D * 4; u += THREADS) {
    const int hc = u >> 2, hh = hc / p.D, c = hc - hh * p.D, t = (u & 3) * 4;
    const C* from = stage + (hh * 16 + t) * kRow + c;
    const int64_t at = dst[t];
    C* to = (C*)p.cache[1] + (h0 + hh) * s[2] + c * s[3];
    union {
      uint32_t w[esize<CT>()];
      C e[4];
    } q;
#pragma unroll
    for (int i = 0; i < 4; ++i) q.e[i] = from[i * kRow];
    const bool run = t + 3 < nt && at >= 0 && dst[t + 1] == at + 1 && dst[t + 2] == at + 2 && dst[t + 3] == at + 3 &&
                     ((uintptr_t)(to + at) & (4 * sizeof(C) - 1)) == 0;
    if (run) {
      if constexpr (sizeof(C) == 1) *(uint32_t*)(to + at) = q.w[0];
      else if constexpr (sizeof(C) == 2) *(uint2*)(to + at) = make_uint2(q.w[0], q.w[1]);
      else *(uint4*)(to + at) = make_uint4(q.w[0], q.w[1], q.w[2], q.w[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (t + i < nt && dst[t + i] >= 0) to[dst[t + i]] = q.e[i];
    }
  }
}

// TT tokens a workgroup.  Dynamic LDS: (cos, sin) [TT][pairs], or the stage
// of turned values.
template <int XT, int CT, int TT, int THREADS>
__global__ __launch_bounds__(THREADS) void rotary_kernel(RotaryParams p, int parts, int q_parts, int k_parts, int most,
                                                         int v_most) {
  extern __shared__ __align__(16) uint8_t lds[];
  __shared__ int64_t dst[TT];
  const int64_t group = blockIdx.x / parts;
  int part = (int)(blockIdx.x - group * parts);
  const int64_t t0 = group * TT;
  const int nt = (int)(p.T - t0 < TT ? p.T - t0 : TT);
  const int what = part < q_parts ? 0 : (part < q_parts + k_parts ? 1 : 2);
  part -= what == 0 ? 0 : (what == 1 ? q_parts : q_parts + k_parts);
  const int heads = what == 0 ? p.Hq : p.Hkv, each = what == 2 ? v_most : most;
  const int h0 = part * each, nh = min(each, heads - h0);
  if (threadIdx.x < nt) {
    const int64_t t = t0 + threadIdx.x;
    dst[threadIdx.x] = what == 0 ? t * p.o_s[0] : slot_offset(p, t, p.c_s[what - 1]);
  }
  float2* cs = (float2*)lds;
  if (what != 2)
    for (int u = threadIdx.x; u < nt * p.pairs; u += THREADS) {
      const int t = u / p.pairs;
      cs[u] = cos_sin(p, t0 + t, u - t * p.pairs);
    }
  __syncthreads();
  if (what == 0) {
    rotate_rows<XT, XT, TT, THREADS, 0>(p, t0, nt, h0, nh, cs, dst);
  } else if (what == 1) {
    rotate_rows<XT, CT, TT, THREADS, 1>(p, t0, nt, h0, nh, cs, dst);
  } else {
    if constexpr (TT == 16) {
      if (p.v_tile) {
        turn_values<XT, CT, THREADS>(p, t0, nt, h0, nh, dst, lds);
        return;
      }
    }
    copy_values<XT, CT, THREADS>(p, t0, nt, h0, nh, dst);
  }
}

template <int XT, int CT, int TT, int THREADS>
int32_t launch_tt(const RotaryParams& p, hipStream_t stream) {
  // Heads of a workgroup: many share a token's cosines and sines, few make
  // enough workgroups for the card.  Rows as above: 16 heads 26.9 us, 8 30.2,
  // 32 42; 1,237 rows of 12 heads in f32: 4 heads 7.0 us, 16 8.1.  Values that
  // are turned over have no cosines to share: of 4,900 rows 4 heads at a time
  // take 27.2 us, 2 30.8; of 2,048 17.1 and 14.6; single ones are scattered by
  // channel, a head a wave (64 rows: 4.8 us, by eight heads 10).
  int most = TT == 1 ? kHeads : kMostHeads, v_most = most, q_parts, k_parts, parts;
  int64_t groups;
  for (;; most /= 2) {
    v_most = p.vec[2] ? most : (TT == 1 ? 1 : std::max(most / 4, 2));
    q_parts = (p.Hq + most - 1) / most;
    k_parts = (p.Hkv + most - 1) / most;
    parts = q_parts + k_parts + (p.Hkv + v_most - 1) / v_most;
    groups = ceil_div(p.T, TT) * parts;
    if (TT == 1 || most == kLeast || groups >= kWorkgroups) break;
  }
  if (groups >= (int64_t)INT32_MAX) {
    set_error("rotary: too many rows");
    return CF_ERR_UNSUPPORTED;
  }
  size_t lds = (size_t)TT * p.pairs * sizeof(float2);
  if (TT == 16 && p.v_tile)
    lds = std::max(lds, (size_t)v_most * 16 * turned_row<CT>() * esize<CT>());
  ProfileScope prof("cf_rotary", stream);
  CF_LAUNCH((rotary_kernel<XT, CT, TT, THREADS>), dim3((unsigned)groups), dim3(THREADS), lds, stream, p, parts, q_parts,
            k_parts, most, v_most);
  CF_HIP_CHECK(hipGetLastError());
  return CF_OK;
}

template <int XT, int CT>
int32_t launch_t(const RotaryParams& p, hipStream_t stream) {
  // groups against single tokens, e4m3 caches of 8 heads of 128: 256 rows 6.9
  // and 6.0 us, 512 rows 7.5 and 8.6, 2,048 rows 14.8 and 21.4
  if (p.T >= 512 && p.pairs <= 256) return launch_tt<XT, CT, 16, 256>(p, stream);
  return launch_tt<XT, CT, 1, 64>(p, stream);
}

template <int XT>
int32_t launch_x(const RotaryParams& p, int cache_dt, hipStream_t stream) {
  switch (cache_dt) {
    case kF32: return launch_t<XT, kF32>(p, stream);
    case kF16: return launch_t<XT, kF16>(p, stream);
    case kBF16: return launch_t<XT, kBF16>(p, stream);
    default: return launch_t<XT, kE4M3>(p, stream);
  }
}

bool pieces(const void* base, const int64_t* stride, int n, int bytes) {
  if (((uintptr_t)base & 15) != 0 || stride[n - 1] != 1) return false;
  for (int i = 0; i < n - 1; ++i)
    if ((stride[i] * bytes) % 16 != 0) return false;
  return true;
}

}  // namespace

int32_t launch_rotary(RotaryParams p, int x_dt, int cache_dt, hipStream_t stream) {
  const int xb = dtype_bytes(x_dt), cb = dtype_bytes(cache_dt);
  const bool rows8 = p.pairs % kPiece == 0 && (p.D - 2 * p.pairs) % kPiece == 0;
  p.vec[0] = rows8 && pieces(p.x[0], p.x_s[0], 3, xb) && pieces(p.out, p.o_s, 3, xb);
  const bool kv = p.Hkv > 0;
  p.vec[1] = kv && rows8 && pieces(p.x[1], p.x_s[1], 3, xb) && pieces(p.cache[0], p.c_s[0], 4, cb);
  const bool v8 = kv && p.D % kPiece == 0 && pieces(p.x[2], p.x_s[2], 3, xb);
  p.vec[2] = v8 && pieces(p.cache[1], p.c_s[1], 4, cb);
  p.v_tile = v8 && !p.vec[2] && p.c_s[1][1] == 1 && p.D <= kTileD;
  if (p.T == 0 || p.D == 0) return CF_OK;
  switch (x_dt) {
    case kF32: return launch_x<kF32>(p, cache_dt, stream);
    case kF16: return launch_x<kF16>(p, cache_dt, stream);
    default: return launch_x<kBF16>(p, cache_dt, stream);
  }
}

}  // namespace cf
