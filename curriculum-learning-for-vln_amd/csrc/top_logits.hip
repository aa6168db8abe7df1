// The k largest logits of every row, sorted, and the log-mass of all others (vln_top_logits): a teacher's targets for vln_distill_*,
// and with k = 1 the greedy word.  include/vln_hip.h states the contract.
//
// Bound: bytes for many rows (the row is read once), the length of one workgroup's chain for few.  A workgroup of W waves takes a row, or
// one of S segments of it, as NVR vectors of 16 bytes per thread:
//   1. as they arrive, the maximum and the sum of exp((z - maximum) / T) of every UNIT of 8 elements -- the exponentials, most of the
//      arithmetic, run under the loads -- and the largest element of every thread (G groups per thread, so that there are >= 4 k groups): at
//      least k elements reach the k-th largest of these group maxima, and hardly more than k do -- a bound that costs a bisection over
//      64 W G numbers;
//   2. units below the bound are joined: one exponential each.  The few that are not are read again, a lane each: elements above the bound
//      are candidates (an LDS list), the rest goes into the running (maximum, sum) -- the others' mass is a sum of positive terms, never a
//      difference;
//   3. a candidate's place is the number of larger ones; places from k on belong to the others.
// Short rows stay in registers and are swept there once the bound is known: k is no small part of their units.
// Elements are ordered by (order-preserving bits of the value, lower index first): all distinct, so ties fall to the lowest index and the
// order in which candidates were collected does not show.  Where more reach the bound than a list holds, or the bound is -inf (rows with
// fewer words allowed than asked for), the elements above the bound and, in index order, as many equal to it as are missing are taken
// (their places from a scan of the counts); only if those above are too many as well is the border itself searched by bisection.
// Segments leave their candidates, and one workgroup per row selects among them.
//
// Measured, us: 4096 rows x 32000 bf16 58 with k 16, 60 with k 64 (4.4 TB/s; loads and bound alone 51, a copy's rate), 100 with k 256;
// 8192 x 4000 bf16, k 16: 22; 5120 x 992 fp32, k 16: 11; 64 x 992, k 1: 4.5, of which a launch is most; 4 x 131072 fp32, k 128: 16.5 (two
// launches).  With rows held in registers until the bound is known 4096 x 32000, k 64, takes 85: every element's exponential, 25 us of
// instructions, then comes after the loads.  Tried: the next row's loads issued from that sweep, 115 (spilled registers); a wave per row that
// streams with a running bound, 120 - 145.
#include "word_rows.h"
#include "../../include/vln_hip.h"

namespace vln {

typedef unsigned long long u64;

// value <-> order-preserving bits; every NaN is the largest, -0 equals +0.  0 is no element's.
__device__ __forceinline__ unsigned order_bits(float x) {
  const unsigned b = __float_as_uint(x + 0.f);
  return x != x ? 0xffffffffu : b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float order_value(unsigned o) {
  if (o == 0xffffffffu) return __builtin_nanf("");
  return __uint_as_float((o & 0x80000000u) ? (o ^ 0x80000000u) : ~o);
}

struct TopArgs {
  const void* logits; int64_t ld;
  int N, V, k, S, ks, vps;         // S segments per row of vps vectors, ks candidates of a segment
  float c, invT;                   // log2(e) / T, 1 / T
  void* values; long long* ids; float* rest;
  u64* keys; float2* sums;         // S > 1: [N, S, ks] (order bits << 32 | ~index; 0: none) and [N, S]
};

__device__ __forceinline__ float nan_max(float a, float b) { return __builtin_elementwise_maximum(a, b); }   // NaN wins (v_maximum3_f32)

// Largest element of a vector, an UNDERESTIMATE where it holds NaN or infinities (enough for a bound that k elements must reach).  bf16: of
// the pair in a register, the upper element is taken with the lower one as extra mantissa bits -- the order of the upper ones is kept, and
// cutting the bits off afterwards gives the exact largest -- so only the lower elements are unpacked.
template <typename E> struct VecMax;
template <> struct VecMax<float> {
  float m = -INFINITY;
  __device__ __forceinline__ void add(const uint4& r) {
    m = fmaxf(m, fmaxf(fmaxf(__uint_as_float(r.x), __uint_as_float(r.y)), fmaxf(__uint_as_float(r.z), __uint_as_float(r.w))));
  }
  __device__ __forceinline__ float get() const { return m; }
};
template <> struct VecMax<bf16_raw> {
  float lo = -INFINITY, hi = -INFINITY;
  __device__ __forceinline__ void add(const uint4& r) {
    hi = fmaxf(hi, fmaxf(fmaxf(__uint_as_float(r.x), __uint_as_float(r.y)), fmaxf(__uint_as_float(r.z), __uint_as_float(r.w))));
    lo = fmaxf(lo, fmaxf(fmaxf(__uint_as_float(r.x << 16), __uint_as_float(r.y << 16)), fmaxf(__uint_as_float(r.z << 16), __uint_as_float(r.w << 16))));
  }
  __device__ __forceinline__ float get() const { return fmaxf(lo, __uint_as_float(__float_as_uint(hi) & 0xffff0000u)); }
};
// The largest t in [lo, hi] that at least `want` of the wave's values reach -- lo must be reached by that many; ends early at a t that
// exactly `want` reach (`exact`).  count(t): how many values are >= t.
template <typename F> __device__ __forceinline__ unsigned bisect(unsigned lo, unsigned hi, int want, bool& exact, F&& count) {
  int n = count(hi);
  exact = n == want;
  if (n >= want) return hi;
  while (hi - lo > 1) {                  // count(lo) >= want > count(hi)
    const unsigned mid = lo + ((hi - lo) >> 1);
    n = count(mid);
    if (n >= want) { lo = mid; if (n == want) { exact = true; return lo; } }
    else hi = mid;
  }
  return lo;
}
// Some t in [lo, hi] that at least `want` and, if few steps find it, at most `most` values reach: a bound need not be exact.
template <typename F> __device__ __forceinline__ unsigned bisect_near(unsigned lo, unsigned hi, int want, int most, int steps, F&& count) {
  if (count(hi) >= want) return hi;
  while (hi - lo > 1 && steps-- > 0) {
    const unsigned mid = lo + ((hi - lo) >> 1);
    const int n = count(mid);
    if (n >= want) { lo = mid; if (n <= most) break; }
    else hi = mid;
  }
  return lo;
}
// Calls emit(place, key) for the nc keys of an LDS list, place = the number of larger ones.  Threads that are left over share the
// comparisons of a key: T / C threads each look at a part of the list (C: the power of two from 64 that holds nc).  Ends with the places
// emitted by the threads below nc; every thread of the workgroup calls it.
template <int T, typename F> __device__ __forceinline__ void place_by_rank(const u64* cand, int* place, int nc, int tid, F&& emit) {
  int C = 64;
  while (C < nc && C < T) C *= 2;
  const int P = T / C, part = tid / C, step = ((nc + P - 1) / P + 1) & ~1;      // an even share each
  const int j0 = min(nc, part * step), j1 = min(nc, j0 + step);
  if (P > 1) {
    if (tid < C) place[tid] = 0;
    __syncthreads();
  }
  for (int c = tid & (C - 1); c < nc; c += C) {
    const u64 mine = cand[c];
    const ulonglong2* l = reinterpret_cast<const ulonglong2*>(cand + j0);
    int r = 0;
#pragma unroll 8
    for (int j = 0; j < (j1 - j0) / 2; ++j) { const ulonglong2 q = l[j]; r += (q.x > mine ? 1 : 0) + (q.y > mine ? 1 : 0); }
    if ((j1 - j0) & 1) r += cand[j1 - 1] > mine ? 1 : 0;
    if (P > 1) atomicAdd(&place[c], r);
    else emit(r, mine);
  }
  if (P > 1) {
    __syncthreads();
    if (tid < nc) emit(place[tid], cand[tid]);
  }
}

template <typename E> __device__ __forceinline__ void emit_row(const TopArgs& a, long n, int rank, unsigned order, unsigned idx) {
  Elt<E>::st(static_cast<E*>(a.values) + n * a.k + rank, order_value(order));
  a.ids[n * a.k + rank] = (long long)idx;
}
__device__ __forceinline__ float log_mass(float m, float s, float invT) {
  return s == 0.f ? -INFINITY : (m == INFINITY ? INFINITY : m * invT + logf(s));
}

// (waves per SIMD that the registers are limited to)
template <typename E, int W, int NVR, int G> __global__ __launch_bounds__(64 * W, NVR == 16 ? 5 : W == 1 && NVR == 4 ? 7 : 8) void top_row_kernel(TopArgs a) {
  constexpr int VEC = RowGeo<E>::VEC, T = 64 * W, CAP = VLN_TOP_LOGITS_MAX, GU = NVR / G;      // CAP: candidates of a wave
  __shared__ alignas(16) u64 cand[W * CAP];                   // (first: {value bits, column}, a list per wave)
  constexpr bool STREAM = NVR > 4;
  __shared__ unsigned short dirty[STREAM ? W * CAP : 1];      // units to be looked at again, a list per wave
  __shared__ int place[T];
  __shared__ unsigned gmax[T * G];
  __shared__ int counts[W], redo, part[2][W], gt_n[W], eq_n[NVR * W];
  __shared__ unsigned bound;
  __shared__ float2 sums[W];
  const long n = blockIdx.x;
  const int s = blockIdx.y, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const E* p = static_cast<const E*>(a.logits) + n * a.ld;
  const RowGeo<E> g(p, a.V);
  const int v0 = min(g.nv, s * a.vps), v1 = min(g.nv, v0 + a.vps);
  constexpr unsigned none = sizeof(E) == 2 ? 0xff80ff80u : 0xff800000u;      // -inf elements
  auto ask = [&](int u) {
    uint4 r = make_uint4(none, none, none, none);
    if (v0 + u * T + tid < v1) r = ld_vec<E>(p + g.head + (int64_t)(v0 + u * T + tid) * VEC);
    return r;
  };
  constexpr int UV = 8 / VEC, NU = NVR / UV;   // units of 8 elements: vectors of one, units of a thread
  constexpr int HELD = NVR > 8 ? 8 : NVR;      // vectors in registers at once
  uint4 raw[HELD];
#pragma unroll
  for (int u = 0; u < HELD; ++u) raw[u] = ask(u);
  // the single elements in front of the first and behind the last vector: threads of the first segment
  int scol = -1;
  if (s == 0) scol = tid < g.head ? tid : (tid >= VEC && tid - VEC < g.tail ? g.tail0() + tid - VEC : -1);
  const float sx = scol >= 0 ? Elt<E>::ld(p + scol) : -INFINITY;
  if (tid == 0) redo = 0;
  float tmax = sx;
  float um[STREAM ? NU : 1], us[STREAM ? NU : 1];
  if constexpr (STREAM) {                      // maximum and sum of every unit, as it arrives
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      float x[8];
#pragma unroll
      for (int h = 0; h < UV; ++h) {
        unpack16<E>(raw[(u * UV + h) % HELD], x + h * VEC);
        if (u * UV + h + HELD < NVR) raw[(u * UV + h) % HELD] = ask(u * UV + h + HELD);
      }
      float m = -FLT_MAX, t = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) m = fmaxf(m, x[i]);
#pragma unroll
      for (int i = 0; i < 8; ++i) t += exp2_hw((x[i] - m) * a.c);
      um[u] = m; us[u] = t;
    }
  }
#pragma unroll
  for (int q = 0; q < G; ++q) {
    float t = -INFINITY;
    if constexpr (STREAM) {
#pragma unroll
      for (int u = q * (NU / G); u < (q + 1) * (NU / G); ++u) t = fmaxf(t, us[u] == 0.f ? -INFINITY : um[u]);
    } else {
      VecMax<E> m;
#pragma unroll
      for (int u = q * GU; u < (q + 1) * GU; ++u) m.add(raw[u]);
      t = m.get();
    }
    bool has = v0 + q * GU * T + tid < v1;
    if (q == 0 && scol >= 0) { t = fmaxf(t, sx); has = true; }
    tmax = fmaxf(tmax, t);
    gmax[q * T + tid] = has ? order_bits(t) : 0u;
  }
  __syncthreads();
  if (w == 0) {
    unsigned gm[W * G], least = 0xffffffffu, most = 0u;
    int groups = 0;
#pragma unroll
    for (int i = 0; i < W * G; ++i) {
      gm[i] = gmax[i * 64 + lane];
      groups += __popcll(__ballot(gm[i] != 0u));
      most = max(most, gm[i]);
      least = min(least, gm[i] - 1u);          // (0 - 1: an empty group)
    }
    unsigned th = 0u;                          // fewer groups than k: no bound
    if (groups >= a.k)
      th = bisect_near(wave_umin(least) + 1u, wave_umax(most), a.k, a.k + a.k / 8 + 2, 12, [&](unsigned b) {
        int c = 0;
#pragma unroll
        for (int i = 0; i < W * G; ++i) c += gm[i] >= b ? 1 : 0;
        return wave_isum(c);
      });
    if (lane == 0) bound = th;
  }
  __syncthreads();
  unsigned border = bound;                     // candidates reach it: !(x <= tval), tval just below (below +0 comes -0, which compares equal)
  const float tval = border == 0u ? 0.f : order_value(border == 0x80000000u ? border - 2 : border - 1);
  constexpr unsigned kNegInf = 0x007fffffu;    // order bits of -inf
  int len = 0;                                 // this wave's list
  uint2* list = reinterpret_cast<uint2*>(cand) + w * CAP;
  // The others' sum (rows in registers).  Every element that is no candidate is at most ref = min(the thread's largest, the bound), so the exponentials are
  // taken relative to ref, one fused multiply-add each (the rounding of ref * c is taken out again at the end).  Where that is no good
  // reference -- not finite, or everything below it underflows -- the sweep is repeated with a running maximum (`slow`).
  OnlineSum others;
  float ref = fminf(tmax, tval);
  bool slow = __ballot(!(fabsf(ref) < 1e30f) && ref != -INFINITY) != 0, redone = false;
  if (!(fabsf(ref) < 1e30f)) ref = 0.f;
  const float nm = -ref * a.c, cut_off = fmaf(ref, a.c, nm);
  bool full = border == kNegInf || border == 0u;      // (0: fewer groups than k)
  if constexpr (STREAM) {
   if (!full) {
    // Units that hold a candidate, or whose sum is none (infinities, NaN), are looked at again, a lane each; the others' sums are joined.
    int n_dirty = 0;
    float top = -FLT_MAX;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const bool d = us[u] != 0.f && !(um[u] <= tval && us[u] <= 8.f);
      const u64 mask = __ballot(d);
      if (mask) {
        const int at = n_dirty + lanes_below(mask);
        if (d && at < CAP) dirty[w * CAP + at] = (unsigned short)(u * T + tid);
        n_dirty += __popcll(mask);
      }
      if (d) { um[u] = -FLT_MAX; us[u] = 0.f; }
      top = fmaxf(top, um[u]);
    }
    others.m = top;
#pragma unroll
    for (int u = 0; u < NU; ++u) others.s += us[u] * exp2_hw((um[u] - top) * a.c);
    wave_sync();
    for (int j = lane; j - lane < min(n_dirty, CAP); j += 64) {
      int at = -1;
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = -INFINITY;
      if (j < n_dirty) {
        at = dirty[w * CAP + j];
#pragma unroll
        for (int h = 0; h < UV; ++h) {
          const int i = v0 + (at / T * UV + h) * T + at % T;
          if (i < v1) unpack16<E>(ld_vec<E>(p + g.head + (int64_t)i * VEC), x + h * VEC);
        }
      }
      int mine = 0, total;
#pragma unroll
      for (int i = 0; i < 8; ++i) mine += !(x[i] <= tval) ? 1 : 0;
      int to = len - mine + wave_scan(mine, total);
      len += total;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (!(x[i] <= tval)) {
          if (to < CAP) list[to] = make_uint2(__float_as_uint(x[i]), g.head + (v0 + (at / T * UV + i / VEC) * T + at % T) * VEC + i % VEC);
          ++to;
          x[i] = -INFINITY;
        }
      }
      others.add(x, a.c);
    }
    if (n_dirty > CAP) len = CAP + 1;          // (the rare forms)
    if (s == 0) {
      const bool in = scol >= 0 && !(sx <= tval);
      int total;
      const int at = len - 1 + wave_scan(in ? 1 : 0, total);
      len += total;
      if (in) { if (at < CAP) list[at] = make_uint2(__float_as_uint(sx), scol); }
      else if (scol >= 0) others.add1(sx, a.c);
    }
    if (lane == 0) counts[w] = len;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < W; ++i) full = full || counts[i] > CAP;
   }
  } else while (!full) {
    len = 0;
    float sum = 0.f;
#pragma unroll
    for (int u = 0; u < NVR; u += UV) {
      int i = v0 + u * T + tid;
      if (v0 + u * T >= v1) continue;           // uniform
      // (unpacked, and columns formed, where they are needed: prepared ahead for all vectors they would take three times the registers)
#pragma unroll
      for (int h = 0; h < UV; ++h) asm volatile("" : "+v"(raw[u + h].x), "+v"(raw[u + h].y), "+v"(raw[u + h].z), "+v"(raw[u + h].w), "+v"(i));
      float x[8];
#pragma unroll
      for (int h = 0; h < UV; ++h) unpack16<E>(raw[u + h], x + h * VEC);
      float mx = x[0];
#pragma unroll
      for (int j = 1; j < 8; ++j) mx = nan_max(mx, x[j]);
      if (__ballot(!(mx <= tval))) {
        auto column = [&](int j) { return g.head + (i + j / VEC * T) * VEC + j % VEC; };
        // most units of a wave have a candidate in some lane: one scan places them all
        int mine = 0, total;
        bool in[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) { in[j] = !(x[j] <= tval); mine += in[j] ? 1 : 0; }
        int at = len - mine + wave_scan(mine, total);
        len += total;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (in[j]) {
            if (at < CAP) list[at] = make_uint2(__float_as_uint(x[j]), column(j));
            ++at;
            x[j] = -INFINITY;
          }
        }
      }
      if (!slow) {
#pragma unroll
        for (int j = 0; j < 8; ++j) sum += exp2_hw(fmaf(x[j], a.c, nm));
      } else {
        others.add(x, a.c);
      }
    }
    if (!slow) {
      if (sum != 0.f) { others.m = ref; others.s = sum * exp2_hw(-cut_off); }
      if (sum < 1e-30f && tmax != -INFINITY) {  // candidates and masked words only, or an underflow?
        for (int u = v0 + tid; u < v1; u += T) {
          float x[VEC];
          unpack16<E>(ld_vec<E>(p + g.head + (int64_t)u * VEC), x);
          for (int j = 0; j < VEC; ++j) if (x[j] <= tval && x[j] != -INFINITY) redo = 1;
        }
      }
    }
    if (s == 0) {
      const bool in = scol >= 0 && !(sx <= tval);
      int total;
      const int at = len - 1 + wave_scan(in ? 1 : 0, total);
      len += total;
      if (in) { if (at < CAP) list[at] = make_uint2(__float_as_uint(sx), scol); }
      else if (scol >= 0) others.add1(sx, a.c);
    }
    if (lane == 0) counts[w] = len;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < W; ++i) full = full || counts[i] > CAP;
    const bool again = redo != 0 && !redone;   // (the same in every wave; `slow` may differ)
    if (full || !again) break;
    slow = redone = true;
    others = OnlineSum();
    __syncthreads();
  }
  if (full) {
    // The rare forms, in loops over the vectors in memory (the caches hold them).  Nothing but -inf: the first k columns.  Otherwise the
    // elements above the border and, in index order, the first `need` equal to it.
    others = OnlineSum();
    __syncthreads();
    if (tid == 0) redo = 0;
    __syncthreads();
    auto each = [&](int u, auto&& f) {       // f(element, column) of this thread's vector u
      const int i = v0 + u * T + tid;
      if (i >= v1) return;
      float x[VEC];
      unpack16<E>(ld_vec<E>(p + g.head + (int64_t)i * VEC), x);
#pragma unroll
      for (int j = 0; j < VEC; ++j) f(x[j], g.head + i * VEC + j);
    };
    bool other = sx != -INFINITY;
#pragma unroll 4
    for (int u = 0; u < NVR; ++u) each(u, [&](float x, int) { other = other || x != -INFINITY; });
    if (__ballot(other) && lane == 0) redo = 1;
    __syncthreads();
    if (!redo) {
      const int c0 = s == 0 ? 0 : g.head + v0 * VEC, n_col = (v1 - v0) * VEC + (s == 0 ? g.head + g.tail : 0);
      len = w == 0 ? min(a.k, n_col) : 0;
      for (int c = lane; c < len; c += 64) {
        const int body = g.head + (v1 - v0) * VEC;
        list[c] = make_uint2(0xff800000u, s == 0 && c >= body ? g.tail0() + c - body : c0 + c);
      }
    } else {
      int turn = 0;
      auto block_count = [&](unsigned t) {     // elements of the segment with order bits >= t
        int c = scol >= 0 && order_bits(sx) >= t ? 1 : 0;
#pragma unroll 2
        for (int u = 0; u < NVR; ++u) each(u, [&](float x, int) { c += order_bits(x) >= t ? 1 : 0; });
        c = wave_isum(c);
        if (lane == 0) part[turn][w] = c;
        __syncthreads();
        c = 0;
        for (int i = 0; i < W; ++i) c += part[turn][i];
        turn ^= 1;
        return c;
      };
      int above;
      for (int go = 0; go < 2; ++go) {
        // above the border, per wave, and equal to it, per vector and wave: index order is head, vectors by (u, wave, lane), tail
        int gt = scol >= 0 && order_bits(sx) > border ? 1 : 0;
#pragma unroll 2
        for (int u = 0; u < NVR; ++u) {
          int eq = 0;
          each(u, [&](float x, int) { const unsigned o = order_bits(x); gt += o > border ? 1 : 0; eq += o == border ? 1 : 0; });
          eq = wave_isum(eq);
          if (lane == 0) eq_n[u * W + w] = eq;
        }
        gt = wave_isum(gt);
        if (lane == 0) gt_n[w] = gt;
        __syncthreads();
        above = 0;
        bool many = false;
        for (int i = 0; i < W; ++i) { above += gt_n[i]; many = many || gt_n[i] > CAP; }
        if (!many || above < a.k) break;       // (fewer than k above: k in all, which a list holds)
        bool exact;                            // too many above it as well: the k-th largest value itself (fewer than k above)
        border = bisect(border + 1u, 0xffffffffu, a.k, exact, block_count);
        __syncthreads();
      }
      const int need = max(0, a.k - above);
      int eq_head = 0;
      if (s == 0) for (int c = 0; c < g.head; ++c) eq_head += order_bits(Elt<E>::ld(p + c)) == border ? 1 : 0;
      int eq_before = eq_head;
      len = 0;
      for (int u = 0; u < NVR; ++u) {
        int eq = 0, all;
        each(u, [&](float x, int) { eq += order_bits(x) == border ? 1 : 0; });
        int before = eq_before - eq + wave_scan(eq, all);
        for (int q = 0; q < W; ++q) { const int c = eq_n[u * W + q]; eq_before += c; if (q < w) before += c; }
        int mine = 0, rank = before;
        auto in = [&](float x) { const unsigned o = order_bits(x); return o > border || (o == border && rank++ < need); };
        each(u, [&](float x, int) { mine += in(x) ? 1 : 0; });
        int at = len - mine + wave_scan(mine, all);
        len += all;
        rank = before;
        each(u, [&](float x, int col) {
          if (in(x)) list[at++] = make_uint2(__float_as_uint(x), col);
          else others.add1(x, a.c);
        });
      }
      if (s == 0) {
        const unsigned o = order_bits(sx);
        const bool tail = scol >= g.head;
        int all;
        const int before = wave_scan(scol >= 0 && o == border ? 1 : 0, all) - 1 - (tail ? eq_head : 0) + (tail ? eq_before : 0);
        const bool in = scol >= 0 && (o > border || (o == border && before < need));
        const int at = len - 1 + wave_scan(in ? 1 : 0, all);
        len += all;
        if (in) list[at] = make_uint2(__float_as_uint(sx), scol);
        else if (scol >= 0) others.add1(sx, a.c);
      }
    }
    if (lane == 0) counts[w] = len;
    __syncthreads();
  }
  // the waves' lists as one list of keys, in a fixed order
  int nc = 0, before = 0;
#pragma unroll
  for (int i = 0; i < W; ++i) { if (i == w) before = nc; nc += counts[i]; }
  uint2 e[CAP / 64];
#pragma unroll
  for (int i = 0; i < CAP / 64; ++i) if (i * 64 + lane < counts[w]) e[i] = reinterpret_cast<const uint2*>(cand)[w * CAP + i * 64 + lane];
  u64* seg = a.S > 1 ? a.keys + (n * a.S + s) * a.ks : nullptr;
  u64* to = seg && nc <= a.ks ? seg + before : cand + before;      // a segment's candidates need no order
  __syncthreads();
#pragma unroll
  for (int i = 0; i < CAP / 64; ++i)
    if (i * 64 + lane < counts[w]) to[i * 64 + lane] = ((u64)order_bits(__uint_as_float(e[i].x)) << 32) | ~e[i].y;
  if (seg) for (int c = min(nc, a.ks) + tid; c < a.ks; c += T) seg[c] = 0ull;
  if (!seg || nc > a.ks) {
    __syncthreads();
    place_by_rank<T>(cand, place, nc, tid, [&](int at, u64 v) {
      if (at >= (seg ? a.ks : a.k)) others.add1(order_value((unsigned)(v >> 32)), a.c);
      else if (seg) seg[at] = v;
      else emit_row<E>(a, n, at, (unsigned)(v >> 32), ~(unsigned)v);
    });
  }
  others.wave(a.c);
  if (lane == 0) sums[w] = make_float2(others.m, others.s);
  __syncthreads();
  if (tid == 0) {
    OnlineSum o;
    for (int i = 0; i < W; ++i) o.merge(sums[i].x, sums[i].y, a.c);
    if (seg) a.sums[n * a.S + s] = make_float2(o.m, o.s);
    else a.rest[n] = log_mass(o.m, o.s, a.invT);
  }
}

// One workgroup selects the k best of up to `per` segments' candidates, all of them in registers.  The bound again comes from the threads'
// largest, searched by one wave; what reaches it is placed by rank.  Only if that is more than a list holds do all waves search on among the
// candidates themselves (a barrier per step), and only where that many are equal among the indices too.  A row with more segments is merged
// in levels: blockIdx.y is the group, its result one segment of the next level (last level: the row's result).
constexpr int kMergeThreads = 512, kMergeRegs = 16, kMergeMax = kMergeThreads * kMergeRegs, kMergeList = 512;

template <typename E> __global__ __launch_bounds__(kMergeThreads) void top_merge_kernel(TopArgs a, int per, u64* keys_out, float2* sums_out) {
  constexpr int W = kMergeThreads / 64;
  __shared__ alignas(16) u64 cand[kMergeList];
  __shared__ int place[kMergeThreads];
  __shared__ int part[2][W];
  __shared__ unsigned tops[kMergeThreads], ends[2];
  __shared__ float2 sums[W];
  const long n = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, s0 = blockIdx.y * per, segs = min(per, a.S - s0), total = segs * a.ks;
  const u64* keys = a.keys + (n * a.S + s0) * a.ks;
  OnlineSum others;
  for (int i = tid; i < segs; i += kMergeThreads) {
    const float2 o = a.sums[n * a.S + s0 + i];
    others.merge(o.x, o.y, a.c);
  }
  unsigned hi[kMergeRegs], lo[kMergeRegs], most = 0u;
  const int regs = (total + kMergeThreads - 1) / kMergeThreads;
#pragma unroll
  for (int i = 0; i < kMergeRegs; ++i) {
    const int at = i * kMergeThreads + tid;
    const u64 v = i < regs && at < total ? keys[at] : 0ull;
    hi[i] = (unsigned)(v >> 32); lo[i] = (unsigned)v;
    most = max(most, hi[i]);
  }
  tops[tid] = most;
  __syncthreads();
  if (w == 0) {
    unsigned gm[W], least = 0xffffffffu;
    int groups = 0;
    most = 0u;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      gm[i] = tops[i * 64 + lane];
      groups += __popcll(__ballot(gm[i] != 0u));
      most = max(most, gm[i]);
      least = min(least, gm[i] - 1u);          // (0 - 1: a thread without any)
    }
    most = wave_umax(most);
    unsigned th = 1u;
    if (groups >= a.k)
      th = bisect_near(wave_umin(least) + 1u, most, a.k, a.k + a.k / 8 + 2, 16, [&](unsigned b) {
        int c = 0;
#pragma unroll
        for (int i = 0; i < W; ++i) c += gm[i] >= b ? 1 : 0;
        return wave_isum(c);
      });
    if (lane == 0) { ends[0] = th; ends[1] = most; }
  }
  __syncthreads();
  most = ends[1];
  int turn = 0, before;                       // before: what the waves in front of this one counted
  auto block_count = [&](auto&& has) {
    int c = 0;
#pragma unroll
    for (int i = 0; i < kMergeRegs; ++i) if (i < regs) c += has(hi[i], lo[i]) ? 1 : 0;
    c = wave_isum(c);
    if (lane == 0) part[turn][w] = c;
    __syncthreads();
    c = before = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) { if (i == w) before = c; c += part[turn][i]; }
    turn ^= 1;
    return c;
  };
  unsigned th = ends[0], tl = 0u;
  int nc = block_count([&](unsigned h, unsigned) { return h >= th; });
  if (nc > kMergeList) {
    th = bisect_near(th, most, a.k, kMergeList, 32, [&](unsigned t) { return block_count([&](unsigned h, unsigned) { return h >= t; }); });
    nc = block_count([&](unsigned h, unsigned) { return h >= th; });
    if (nc > kMergeList) {
      const int need = a.k - block_count([&](unsigned h, unsigned) { return h > th; });
      bool e;
      tl = bisect(0u, 0xffffffffu, need, e, [&](unsigned t) { return block_count([&](unsigned h, unsigned l) { return h == th && l >= t; }); });
      nc = block_count([&](unsigned h, unsigned l) { return h > th || (h == th && l >= tl); });
    }
  }
  int mine = 0, all;
#pragma unroll
  for (int i = 0; i < kMergeRegs; ++i) if (i < regs) mine += hi[i] > th || (hi[i] == th && lo[i] >= tl) ? 1 : 0;
  int at = before - mine + wave_scan(mine, all);
#pragma unroll
  for (int i = 0; i < kMergeRegs; ++i) {
    if (i >= regs) continue;
    if (hi[i] > th || (hi[i] == th && lo[i] >= tl)) cand[at++] = ((u64)hi[i] << 32) | lo[i];
    else if (hi[i]) others.add1(order_value(hi[i]), a.c);
  }
  __syncthreads();
  const long slot = n * gridDim.y + blockIdx.y;
  if (keys_out) for (int c = min(nc, a.k) + tid; c < a.ks; c += kMergeThreads) keys_out[slot * a.ks + c] = 0ull;
  place_by_rank<kMergeThreads>(cand, place, nc, tid, [&](int at, u64 v) {
    if (at >= a.k) others.add1(order_value((unsigned)(v >> 32)), a.c);
    else if (keys_out) keys_out[slot * a.ks + at] = v;
    else emit_row<E>(a, n, at, (unsigned)(v >> 32), ~(unsigned)v);
  });
  others.wave(a.c);
  if (lane == 0) sums[w] = make_float2(others.m, others.s);
  __syncthreads();
  if (tid == 0) {
    OnlineSum o;
    for (int i = 0; i < W; ++i) o.merge(sums[i].x, sums[i].y, a.c);
    if (keys_out) sums_out[slot] = make_float2(o.m, o.s);
    else a.rest[n] = log_mass(o.m, o.s, a.invT);
  }
}

struct TopPlan {
  int W, NVR, G, S, vps, ks, per;       // waves, vectors per thread, groups per thread; segments, vectors and candidates of one, segments of one merge
  int levels; int count[8];     // segments left after each merge level
};
// One wave holds a row of up to 256 vectors (k <= 64) in its registers: no barrier to wait for (5120 x 992 fp32, k 8: 10.6 us; four waves: 22.5;
// k 1 | 64: 8.4 | 17, as units: 9.1 | 21).  One wave that keeps units takes up to 512 (8192 x 4000 bf16, k 16: 22 us; two waves 25 - 31, four
// 40), two waves up to 1024 (k <= 128; 8192 x 8000 bf16, k 32: 35; four: 43), four waves the rest: rows of up to 64 KB whole, with the fewest
// vectors per thread that hold them -- with few rows too, where segments would occupy more of the chip but their merge is a second launch
// (64 x 32000 bf16, k 1, whole | in segments of 16 KB: 8 | 11; 300 x 16000, k 32: 10 | 18).  Longer rows are cut: into 64 KB where that gives
// every CU two workgroups (512 x 131072 bf16, k 32: 38.6; 32 KB: 39.3; 16 KB: 53), into 32 KB where it does not (64 x 50000, k 32: 13.6; 64 KB:
// 14.8; 16 KB: 14.4.  1 x 131072, k 1: 10.5; 12.2; 10.5).
// Units only pay where there are many more of them than k: rows with fewer than 4 k stay in registers, 16 KB a workgroup (2000 x 992 fp32, k
// 128: 18 us; as units: 49).
// Groups per thread: one maximum of a thread's vectors is cheaper than four (8192 x 4000, k 16, two waves: 25 us; 30), but k has to stay well below
// the number of maxima, or too much reaches the bound (4096 x 32000, k 256, in registers: 1537; 133).
static TopPlan top_plan(int N, int V, int k, int vec) {
  TopPlan p{};
  const long nv = ((long)V + vec - 1) / vec;
  const int cus = device_cus() > 0 ? device_cus() : 256;
  auto units = [&](int vectors) { return (nv < vectors ? nv : vectors) * vec / 8 >= 4 * k; };      // enough of them for k
  if (nv <= 256 && k <= 64) { p.W = 1; p.NVR = 4; }
  else if (nv <= 512 && k <= 64 && units(512)) { p.W = 1; p.NVR = 8; }
  else if (nv <= 1024 && k <= 128 && units(1024)) { p.W = 2; p.NVR = 8; }
  else {
    p.W = 4; p.NVR = 16;
    while (p.NVR > 4 && nv <= 256L * (p.NVR / 2)) p.NVR /= 2;
    if (nv > 256L * 16 && (long)N * ((nv + 256L * 16 - 1) / (256L * 16)) < 2L * cus) p.NVR = 8;
  }
  if (p.NVR > 4 && !units(64 * p.W * p.NVR)) p.NVR = 4;
  p.G = 4 * k <= 64 * p.W ? 1 : 4;
  const long held = 64L * p.W * p.NVR;
  p.S = (int)((nv + held - 1) / held);
  p.vps = (int)((nv + p.S - 1) / p.S);      // equal ones: a short last segment would have too few maxima for a bound
  p.ks = k + k / 2 + 32;        // (k and the few more that reach a bound)
  p.per = kMergeMax / p.ks;
  for (int n = p.S; n > 1;) { n = (n + p.per - 1) / p.per; p.count[p.levels++] = n; }
  return p;
}
static int64_t top_ws(const TopPlan& p, int N) {
  int64_t segs = p.S > 1 ? p.S : 0;
  for (int i = 0; i + 1 < p.levels; ++i) segs += p.count[i];
  return segs * N * ((int64_t)p.ks * 8 + 8);
}

template <typename E, int W, int NVR> static void top_rows(const TopArgs& a, int G, hipStream_t st) {
  const dim3 grid((unsigned)a.N, (unsigned)a.S);
  if (G == 1) VLN_LAUNCH((top_row_kernel<E, W, NVR, 1>), grid, dim3(64 * W), 0, st, a);
  else VLN_LAUNCH((top_row_kernel<E, W, NVR, 4>), grid, dim3(64 * W), 0, st, a);
}
template <typename E> static int top_launch(TopArgs a, const TopPlan& p, char* ws, hipStream_t st) {
  auto take = [&](int segs) {
    a.keys = reinterpret_cast<u64*>(ws);
    a.sums = reinterpret_cast<float2*>(ws + (int64_t)a.N * segs * a.ks * 8);
    ws += (int64_t)a.N * segs * (a.ks * 8 + 8);
  };
  a.S = p.S; a.ks = p.ks; a.vps = p.vps;
  if (a.S > 1) take(a.S);
  if (p.W == 1 && p.NVR == 4) top_rows<E, 1, 4>(a, p.G, st);
  else if (p.W == 1) top_rows<E, 1, 8>(a, p.G, st);
  else if (p.W == 2) top_rows<E, 2, 8>(a, p.G, st);
  else if (p.NVR == 4) top_rows<E, 4, 4>(a, p.G, st);
  else if (p.NVR == 8) top_rows<E, 4, 8>(a, p.G, st);
  else top_rows<E, 4, 16>(a, p.G, st);
  for (int i = 0; i < p.levels; ++i) {
    const TopArgs from = a;
    const bool last = p.count[i] == 1;
    if (!last) take(p.count[i]);
    VLN_LAUNCH((top_merge_kernel<E>), dim3((unsigned)a.N, (unsigned)p.count[i]), dim3(kMergeThreads), 0, st, from, p.per, last ? nullptr : a.keys,
               last ? nullptr : a.sums);
    a.S = p.count[i];
  }
  VLN_CHECK_LAUNCH("top_logits");
  return VLN_OK;
}

}  // namespace vln

extern "C" int64_t vln_top_logits_ws_bytes(int N, int V, int type, int k) {
  if (N <= 0 || V <= 0 || k <= 0 || k > VLN_TOP_LOGITS_MAX || (type != VLN_F32 && type != VLN_BF16)) return 0;
  return vln::top_ws(vln::top_plan(N, V, k, type == VLN_F32 ? 4 : 8), N);
}
extern "C" int vln_top_logits(const void* logits, int64_t ld, int type, int N, int V, int k, float temperature, void* values, int64_t* ids,
                              float* rest, void* ws, int64_t ws_bytes, vln_stream_t s) {
  if (!logits || !values || !ids || !rest || N <= 0 || V <= 0 || ld < V) { vln::set_error("vln_top_logits: bad args"); return VLN_ERR_ARG; }
  if (type != VLN_F32 && type != VLN_BF16) { vln::set_error("vln_top_logits: type must be fp32 or bf16"); return VLN_ERR_ARG; }
  if (k < 1 || k > V || k > VLN_TOP_LOGITS_MAX) { vln::set_error("vln_top_logits: k must be 1 .. min(V, %d)", VLN_TOP_LOGITS_MAX); return VLN_ERR_ARG; }
  if (!(temperature >= VLN_TEMPERATURE_MIN && temperature <= VLN_TEMPERATURE_MAX)) { vln::set_error("vln_top_logits: bad temperature"); return VLN_ERR_ARG; }
  const vln::TopPlan p = vln::top_plan(N, V, k, type == VLN_F32 ? 4 : 8);
  if (!vln::grid_fits(N, p.S > 1 ? vln::kMergeThreads : 64 * p.W, p.S)) { vln::set_error("vln_top_logits: too many or too long rows for one launch"); return VLN_ERR_ARG; }
  const int64_t need = vln::top_ws(p, N);
  if (need && (!ws || ws_bytes < need)) { vln::set_error("vln_top_logits: workspace too small"); return VLN_ERR_ARG; }
  vln::TopArgs a{};
  a.logits = logits; a.ld = ld; a.N = N; a.V = V; a.k = k;
  a.c = vln::kLog2e / temperature; a.invT = 1.f / temperature;
  a.values = values; a.ids = (long long*)ids; a.rest = rest;
  if (type == VLN_F32) return vln::top_launch<float>(a, p, static_cast<char*>(ws), (hipStream_t)s);
  return vln::top_launch<bf16_raw>(a, p, static_cast<char*>(ws), (hipStream_t)s);
}
