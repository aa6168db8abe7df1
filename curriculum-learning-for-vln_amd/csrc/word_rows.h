// Rows of word logits [N, V] for constrain.hip, top_logits.hip and distill.hip: 16-byte accesses at any row alignment, and the
// running (maximum, sum) pair of a softmax.
#pragma once
#include <float.h>

#include "vln_internal.h"

namespace vln {

// what one launch takes: fewer than 2^32 threads along x, 65535 workgroups along y
inline bool grid_fits(int64_t x, int threads, int64_t y) { return x * threads < (int64_t)1 << 32 && y <= 65535; }

// One row seen as  head | nv vectors of 16 bytes | tail : rows of an odd vocabulary start at any element, so the first `head` (< VEC)
// elements in front of a 16-byte boundary and the last `tail` (< VEC) are taken singly.  Vector i covers columns head + i * VEC ...
template <typename E> struct RowGeo {
  static constexpr int VEC = Elt<E>::kVec;
  int head, nv, tail;
  __device__ __forceinline__ RowGeo(const E* p, int V) {
    const int mis = (int)((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(E));
    head = mis ? min(VEC - mis, V) : 0;
    nv = (V - head) / VEC;
    tail = V - head - nv * VEC;
  }
  __device__ __forceinline__ int tail0() const { return head + nv * VEC; }
};

template <typename E> __device__ __forceinline__ void unpack16(const uint4& r, float* o);
template <> __device__ __forceinline__ void unpack16<float>(const uint4& r, float* o) {
  o[0] = __uint_as_float(r.x); o[1] = __uint_as_float(r.y); o[2] = __uint_as_float(r.z); o[3] = __uint_as_float(r.w);
}
template <> __device__ __forceinline__ void unpack16<bf16_raw>(const uint4& r, float* o) {
  o[0] = __uint_as_float(r.x << 16); o[1] = __uint_as_float(r.x & 0xffff0000u);
  o[2] = __uint_as_float(r.y << 16); o[3] = __uint_as_float(r.y & 0xffff0000u);
  o[4] = __uint_as_float(r.z << 16); o[5] = __uint_as_float(r.z & 0xffff0000u);
  o[6] = __uint_as_float(r.w << 16); o[7] = __uint_as_float(r.w & 0xffff0000u);
}
template <typename E> __device__ __forceinline__ uint4 pack16(const float* o);
template <> __device__ __forceinline__ uint4 pack16<float>(const float* o) {
  return make_uint4(__float_as_uint(o[0]), __float_as_uint(o[1]), __float_as_uint(o[2]), __float_as_uint(o[3]));
}
template <> __device__ __forceinline__ uint4 pack16<bf16_raw>(const float* o) {
  auto two = [](float a, float b) { return (uint32_t)f32_to_bf16_bits(a) | ((uint32_t)f32_to_bf16_bits(b) << 16); };
  return make_uint4(two(o[0], o[1]), two(o[2], o[3]), two(o[4], o[5]), two(o[6], o[7]));
}
template <typename E> __device__ __forceinline__ uint4 ld_vec(const E* p) { return *reinterpret_cast<const uint4*>(p); }
template <typename E> __device__ __forceinline__ void st_vec(E* p, const uint4& v) { *reinterpret_cast<uint4*>(p) = v; }

template <typename E> __device__ __forceinline__ void st_vec_nt(E* p, const uint4& v) {
  __builtin_nontemporal_store(__builtin_bit_cast(u32x4_t, v), reinterpret_cast<u32x4_t*>(p));
}

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }   // v_exp_f32: 1 ulp, results below 2^-126 are 0
constexpr float kLog2e = 1.4426950408889634f;

// Reductions over the wave by data-parallel moves -- row shifts of 1, 2, 4, 8 (a scan of every row of 16), then two broadcasts of row ends;
// lane 63 holds the result -- a few cycles a step, where a shuffle through LDS takes a hundred.  The same bits in every lane.
#define VLN_DPP(v, old, ctrl, rows) __builtin_amdgcn_update_dpp((old), (v), (ctrl), (rows), 0xf, false)
__device__ __forceinline__ unsigned wave_umax(unsigned x) {
  auto step = [](unsigned a, int o) { return (unsigned)o > a ? (unsigned)o : a; };
  x = step(x, VLN_DPP((int)x, 0, 0x111, 0xf)); x = step(x, VLN_DPP((int)x, 0, 0x112, 0xf)); x = step(x, VLN_DPP((int)x, 0, 0x114, 0xf));
  x = step(x, VLN_DPP((int)x, 0, 0x118, 0xf)); x = step(x, VLN_DPP((int)x, 0, 0x142, 0xa)); x = step(x, VLN_DPP((int)x, 0, 0x143, 0xc));
  return (unsigned)__builtin_amdgcn_readlane((int)x, 63);
}
__device__ __forceinline__ unsigned wave_umin(unsigned v) { return ~wave_umax(~v); }
__device__ __forceinline__ float wave_fmax(float x) {
  auto step = [](float a, int o) { return fmaxf(a, __int_as_float(o)); };
  const int low = __float_as_int(-INFINITY);
  x = step(x, VLN_DPP(__float_as_int(x), low, 0x111, 0xf)); x = step(x, VLN_DPP(__float_as_int(x), low, 0x112, 0xf));
  x = step(x, VLN_DPP(__float_as_int(x), low, 0x114, 0xf)); x = step(x, VLN_DPP(__float_as_int(x), low, 0x118, 0xf));
  x = step(x, VLN_DPP(__float_as_int(x), low, 0x142, 0xa)); x = step(x, VLN_DPP(__float_as_int(x), low, 0x143, 0xc));
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}
__device__ __forceinline__ float wave_fsum(float x) {
  auto step = [](float a, int o) { return a + __int_as_float(o); };
  x = step(x, VLN_DPP(__float_as_int(x), 0, 0x111, 0xf)); x = step(x, VLN_DPP(__float_as_int(x), 0, 0x112, 0xf));
  x = step(x, VLN_DPP(__float_as_int(x), 0, 0x114, 0xf)); x = step(x, VLN_DPP(__float_as_int(x), 0, 0x118, 0xf));
  x = step(x, VLN_DPP(__float_as_int(x), 0, 0x142, 0xa)); x = step(x, VLN_DPP(__float_as_int(x), 0, 0x143, 0xc));
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}
// inclusive sum over the lanes up to this one, and the total
__device__ __forceinline__ int wave_scan(int x, int& total) {
  x += VLN_DPP(x, 0, 0x111, 0xf); x += VLN_DPP(x, 0, 0x112, 0xf); x += VLN_DPP(x, 0, 0x114, 0xf); x += VLN_DPP(x, 0, 0x118, 0xf);
  x += VLN_DPP(x, 0, 0x142, 0xa); x += VLN_DPP(x, 0, 0x143, 0xc);
  total = __builtin_amdgcn_readlane(x, 63);
  return x;
}
__device__ __forceinline__ int wave_isum(int x) { int t; wave_scan(x, t); return t; }
#undef VLN_DPP

// sum_i exp((x_i - m) / T) with m = max x_i, in fp32.  m starts at the lowest FINITE value, not at -inf: x - m is then never
// inf - inf, a row of -inf keeps sum 0 (log: -inf), and a row masked with the type's lowest value is still a distribution.
// (x - m) is formed before the scaling: its rounding is relative to the distance, not to the logits' magnitude.
struct OnlineSum {
  float m = -FLT_MAX, s = 0.f;
  __device__ __forceinline__ void raise(float mx, float c) {
    if (mx > m) { s *= exp2_hw((m - mx) * c); m = mx; }
  }
  template <int N> __device__ __forceinline__ void add(const float (&x)[N], float c) {
    float mx = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) mx = fmaxf(mx, x[i]);
    add_max(x, mx, c);
  }
  template <int N> __device__ __forceinline__ void add_max(const float (&x)[N], float mx, float c) {
    raise(mx, c);
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) t += exp2_hw((x[i] - m) * c);
    s += t;
  }
  __device__ __forceinline__ void add1(float x, float c) { raise(x, c); s += exp2_hw((x - m) * c); }
  __device__ __forceinline__ void merge(float mo, float so, float c) {
    const float M = fmaxf(m, mo);
    s = s * exp2_hw((m - M) * c) + so * exp2_hw((mo - M) * c);
    m = M;
  }
  __device__ __forceinline__ void wave(float c) {      // the wave's total, the same bits in every lane
    const float M = wave_fmax(m);
    s = wave_fsum(s * exp2_hw((m - M) * c));
    m = M;
  }
};

// what the wave's lanes wrote to LDS, visible to all of them (one wave's accesses are carried out in order; a workgroup barrier is not needed)
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

__device__ __forceinline__ int lanes_below(unsigned long long mask) {
  return __builtin_amdgcn_mbcnt_hi((unsigned)(mask >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)mask, 0u));
}

}  // namespace vln
