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
// A workgroup takes a group of tokens and up to kHeads heads of the queries,
// the keys or the values; a thread takes eight pairs (two 16-byte pieces of a
// 16-bit row).  Bound by bytes for prompts, by the launch for a decode step.
#include <algorithm>

#include "cf_device.hpp"
#include "cf_host.hpp"
#include "rotary.hpp"

namespace cf {

namespace {

constexpr int kHeads = 8;     // heads of a workgroup
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

template <int DT>
__device__ __forceinline__ void store8(void* base, int64_t off, const float* f, const Fp8Quant& qz) {
  using T = typename Elem<DT>::T;
  constexpr int B = kPiece * esize<DT>();
  union {
    uint2 d[B / 8];
    T e[kPiece];
  } u;
#pragma unroll
  for (int i = 0; i < kPiece; ++i) u.e[i] = encode<DT>(f[i], qz);
  T* dst = (T*)base + off;
  if constexpr (B == 8) {
    *(uint2*)dst = u.d[0];
  } else {
#pragma unroll
    for (int i = 0; i < B / 16; ++i)
      ((uint4*)dst)[i] = make_uint4(u.d[2 * i].x, u.d[2 * i].y, u.d[2 * i + 1].x, u.d[2 * i + 1].y);
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

// Rows of up to kHeads heads of the queries (WHAT 0) or keys (1): rotated
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
// a wave turns one head's 16 rows over in LDS, so that both its reads and its
// writes are whole runs; four tokens of a channel go out in one store where
// their slots follow each other.
template <int XT, int CT>
__device__ __forceinline__ void turn_values(const RotaryParams& p, int64_t t0, int nt, int h0, int nh,
                                            const int64_t* dst, uint8_t* stage_all) {
  using C = typename Elem<CT>::T;
  constexpr int kRow = kTileD + 4 / esize<CT>();  // one bank past a whole number of them
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  C* stage = (C*)stage_all + wave * 16 * kRow;
  const int64_t *xs = p.x_s[2], *s = p.c_s[1];
  const int per = p.D / kPiece;
  for (int hh = wave; hh < nh; hh += 4) {
    const int h = h0 + hh;
    const Fp8Quant qz(CT == kE4M3 ? p.scale[1][h * p.sc_s[1]] : 1.0f);
    for (int u = lane; u < nt * per; u += 64) {
      const int t = u / per, c = (u - t * per) * kPiece;
      float f[kPiece];
      load8<XT>(p.x[2], (t0 + t) * xs[0] + h * xs[1] + c, f);
#pragma unroll
      for (int i = 0; i < kPiece; ++i) stage[t * kRow + c + i] = encode<CT>(f[i], qz);
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    for (int u = lane; u < p.D * 4; u += 64) {
      const int c = u >> 2, t = (u & 3) * 4;
      const int64_t at = dst[t];
      C* to = (C*)p.cache[1] + h * s[2] + c * s[3];
      union {
        uint32_t w[esize<CT>()];
        C e[4];
      } q;
#pragma unroll
      for (int i = 0; i < 4; ++i) q.e[i] = stage[(t + i) * kRow + c];
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
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
}

// TT tokens a workgroup.  Dynamic LDS: (cos, sin) [TT][pairs], or the stage
// of turned values.
template <int XT, int CT, int TT, int THREADS>
__global__ __launch_bounds__(THREADS) void rotary_kernel(RotaryParams p, int parts, int q_parts, int kv_parts) {
  extern __shared__ __align__(16) uint8_t lds[];
  __shared__ int64_t dst[TT];
  const int64_t group = blockIdx.x / parts;
  int part = (int)(blockIdx.x - group * parts);
  const int64_t t0 = group * TT;
  const int nt = (int)(p.T - t0 < TT ? p.T - t0 : TT);
  const int what = part < q_parts ? 0 : (part < q_parts + kv_parts ? 1 : 2);
  part -= what == 0 ? 0 : (what == 1 ? q_parts : q_parts + kv_parts);
  const int heads = what == 0 ? p.Hq : p.Hkv, h0 = part * kHeads, nh = min(kHeads, heads - h0);
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
        turn_values<XT, CT>(p, t0, nt, h0, nh, dst, lds);
        return;
      }
    }
    copy_values<XT, CT, THREADS>(p, t0, nt, h0, nh, dst);
  }
}

template <int XT, int CT, int TT, int THREADS>
int32_t launch_tt(const RotaryParams& p, hipStream_t stream) {
  const int q_parts = (p.Hq + kHeads - 1) / kHeads, kv_parts = (p.Hkv + kHeads - 1) / kHeads;
  const int parts = q_parts + 2 * kv_parts;
  const int64_t groups = ceil_div(p.T, TT) * parts;
  if (groups >= (int64_t)INT32_MAX) {
    set_error("rotary: too many rows");
    return CF_ERR_UNSUPPORTED;
  }
  size_t lds = (size_t)TT * p.pairs * sizeof(float2);
  if (TT == 16 && p.v_tile)
    lds = std::max(lds, (size_t)4 * 16 * (kTileD + 4 / esize<CT>()) * esize<CT>());
  ProfileScope prof("cf_rotary", stream);
  CF_LAUNCH((rotary_kernel<XT, CT, TT, THREADS>), dim3((unsigned)groups), dim3(THREADS), lds, stream, p, parts, q_parts,
            kv_parts);
  CF_HIP_CHECK(hipGetLastError());
  return CF_OK;
}

template <int XT, int CT>
int32_t launch_t(const RotaryParams& p, hipStream_t stream) {
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
