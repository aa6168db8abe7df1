// The k largest logits of every row, sorted, and the log-mass of all others (vln_top_logits): a teacher's targets for vln_distill_*,
// and with k = 1 the greedy word.  include/vln_hip.h states the contract.
//
// Bound: bytes for many rows (the row is read once, into registers: all its loads are in flight at once), the length of one workgroup's
// chain for few.  A workgroup of W waves holds a row, or one of S segments of it, as NVR vectors of 16 bytes per thread:
//   1. the largest element of every thread (G groups per thread, so that there are >= 4 k groups): at least k elements reach the k-th
//      largest of these group maxima, and hardly more than k do -- a bound that costs a bisection over 64 W G numbers;
//   2. one sweep over the registers: elements above the bound are candidates (an LDS list), all others go into the running (maximum,
//      sum) of exp(z / T) -- the others' mass is a sum of positive terms, never a difference;
//   3. a candidate's place is the number of larger ones; places from k on belong to the others.
// Elements are ordered by (order-preserving bits of the value, lower index first): all distinct, so ties fall to the lowest index and the
// order in which candidates were collected does not show.  Where more reach the bound than the list holds (constant or masked rows), the
// exact border is found by bisection over value and index.  Segments leave their k best, and one workgroup per row selects among them.
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
  int N, V, k, S;                  // S segments per row
  float c, invT;                   // log2(e) / T, 1 / T
  void* values; long long* ids; float* rest;
  u64* keys; float2* sums;         // S > 1: [N, S, k] (order bits << 32 | ~index; 0: none) and [N, S]
};

__device__ __forceinline__ float nan_max(float a, float b) { return __builtin_elementwise_maximum(a, b); }   // NaN wins (v_maximum3_f32)

// maximum over the wave by data-parallel moves (row shifts of 1, 2, 4, 8, then two broadcasts: lane 63 holds the result)
__device__ __forceinline__ unsigned wave_umax(unsigned v) {
#define VLN_DPP_MAX(ctrl) { const unsigned o = (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, 0xf, 0xf, false); v = o > v ? o : v; }
  VLN_DPP_MAX(0x111) VLN_DPP_MAX(0x112) VLN_DPP_MAX(0x114) VLN_DPP_MAX(0x118) VLN_DPP_MAX(0x142) VLN_DPP_MAX(0x143)
#undef VLN_DPP_MAX
  return (unsigned)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ unsigned wave_umin(unsigned v) { return ~wave_umax(~v); }

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

template <typename E> __device__ __forceinline__ void emit_row(const TopArgs& a, long n, int rank, unsigned order, unsigned idx) {
  Elt<E>::st(static_cast<E*>(a.values) + n * a.k + rank, order_value(order));
  a.ids[n * a.k + rank] = (long long)idx;
}
__device__ __forceinline__ float log_mass(float m, float s, float invT) {
  return s == 0.f ? -INFINITY : (m == INFINITY ? INFINITY : m * invT + logf(s));
}

// workgroups per CU that the registers are limited to: 4 waves per SIMD hold 64 KB rows, 8 the smaller ones
template <int W, int NVR> constexpr int row_groups() { return (NVR == 16 ? 4 : NVR == 8 ? 6 : 8) * 4 / W; }

template <typename E, int W, int NVR, int G> __global__ __launch_bounds__(64 * W, (row_groups<W, NVR>())) void top_row_kernel(TopArgs a) {
  constexpr int VEC = RowGeo<E>::VEC, T = 64 * W, CAP = W == 1 ? 256 : 1024, GU = NVR / G;
  __shared__ u64 cand[CAP];
  __shared__ unsigned gmax[T * G];
  __shared__ int count, part[2][W];
  __shared__ float bound;
  __shared__ float2 sums[W];
  const long n = blockIdx.x;
  const int s = blockIdx.y, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const E* p = static_cast<const E*>(a.logits) + n * a.ld;
  const RowGeo<E> g(p, a.V);
  const int v0 = min(g.nv, s * T * NVR), v1 = min(g.nv, v0 + T * NVR);
  uint4 raw[NVR];
#pragma unroll
  for (int u = 0; u < NVR; ++u) {
    raw[u] = make_uint4(0, 0, 0, 0);
    if (v0 + u * T + tid < v1) raw[u] = ld_vec<E>(p + g.head + (int64_t)(v0 + u * T + tid) * VEC);
  }
  // the single elements in front of the first and behind the last vector: threads of the first segment
  int scol = -1;
  if (s == 0) scol = tid < g.head ? tid : (tid >= VEC && tid - VEC < g.tail ? g.tail0() + tid - VEC : -1);
  const float sx = scol >= 0 ? Elt<E>::ld(p + scol) : -INFINITY;
  if (tid == 0) count = 0;
#pragma unroll
  for (int q = 0; q < G; ++q) {
    float m = -INFINITY;
    bool has = false;
#pragma unroll
    for (int u = q * GU; u < (q + 1) * GU; ++u) {
      asm volatile("" : "+v"(raw[u].x), "+v"(raw[u].y), "+v"(raw[u].z), "+v"(raw[u].w));
      float x[VEC];
      unpack16<E>(raw[u], x);
      float t = x[0];
#pragma unroll
      for (int j = 1; j < VEC; ++j) t = nan_max(t, x[j]);
      if (v0 + u * T + tid < v1) { m = nan_max(m, t); has = true; }
    }
    if (q == 0 && scol >= 0) { m = nan_max(m, sx); has = true; }
    gmax[q * T + tid] = has ? order_bits(m) : 0u;
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
    float t = __builtin_nanf("");              // fewer groups than k: every element is a candidate
    if (groups >= a.k) {
      bool exact;
      const unsigned th = bisect(wave_umin(least) + 1u, wave_umax(most), a.k, exact, [&](unsigned b) {
        int c = 0;
#pragma unroll
        for (int i = 0; i < W * G; ++i) c += __popcll(__ballot(gm[i] >= b));
        return c;
      });
      t = order_value(th == 0x80000000u ? th - 2 : th - 1);      // just below th (below +0 comes -0, which compares equal to it)
    }
    if (lane == 0) bound = t;
  }
  __syncthreads();
  const float tval = bound;
  OnlineSum others;
  bool exact = false;                          // only elements of order bits > th, or == th and complemented index >= tl, are candidates
  unsigned th = 0u, tl = 0u;
  while (true) {
    auto offer = [&](float x, int col) {       // false: one of the others
      const unsigned o = order_bits(x);
      if (exact && !(o > th || (o == th && ~(unsigned)col >= tl))) return false;
      const int at = atomicAdd(&count, 1);
      if (at < CAP) cand[at] = ((u64)o << 32) | (unsigned)~col;
      return true;
    };
#pragma unroll
    for (int u = 0; u < NVR; ++u) {
      int i = v0 + u * T + tid;
      if (v0 + u * T >= v1) continue;           // uniform
      // (unpacked again, and columns formed, where they are needed: prepared ahead for all vectors they would take three times the registers)
      asm volatile("" : "+v"(raw[u].x), "+v"(raw[u].y), "+v"(raw[u].z), "+v"(raw[u].w), "+v"(i));
      float x[VEC];
      unpack16<E>(raw[u], x);
      float mx = x[0];
#pragma unroll
      for (int j = 1; j < VEC; ++j) mx = nan_max(mx, x[j]);
      if (i >= v1) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) x[j] = -INFINITY;
        mx = -INFINITY;
      }
      if (__ballot(!(mx <= tval))) {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if (!(x[j] <= tval) && i < v1 && offer(x[j], g.head + i * VEC + j)) x[j] = -INFINITY;
        mx = x[0];
#pragma unroll
        for (int j = 1; j < VEC; ++j) mx = fmaxf(mx, x[j]);
      }
      others.add_max(x, mx, a.c);
    }
    if (scol >= 0 && ((sx <= tval) || !offer(sx, scol))) others.add1(sx, a.c);
    __syncthreads();
    if (count <= CAP || exact) break;
    // More reach the bound than the list holds: the exact border, counting the segment's elements per step (read again, from the caches).
    int turn = 0;
    auto block_count = [&](auto&& has) {       // has(order bits, complemented index)
      int c = 0;
      for (int i = v0 + tid; i < v1; i += T) {
        float x[VEC];
        unpack16<E>(ld_vec<E>(p + g.head + (int64_t)i * VEC), x);
        for (int j = 0; j < VEC; ++j) c += has(order_bits(x[j]), ~(unsigned)(g.head + i * VEC + j)) ? 1 : 0;
      }
      if (scol >= 0) c += has(order_bits(sx), ~(unsigned)scol) ? 1 : 0;
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) c += __shfl_xor(c, o, 64);
      if (lane == 0) part[turn][w] = c;
      __syncthreads();
      c = 0;
      for (int i = 0; i < W; ++i) c += part[turn][i];
      turn ^= 1;
      return c;
    };
    bool enough;
    th = bisect(1u, 0xffffffffu, a.k, enough, [&](unsigned t) { return block_count([&](unsigned h, unsigned) { return h >= t; }); });
    if (!enough) {
      const int need = a.k - block_count([&](unsigned h, unsigned) { return h > th; });
      bool e;
      tl = bisect(0u, 0xffffffffu, need, e, [&](unsigned t) { return block_count([&](unsigned h, unsigned l) { return h == th && l >= t; }); });
    }
    exact = true;
    __syncthreads();
    if (tid == 0) count = 0;
    others = OnlineSum();
    __syncthreads();
  }
  const int nc = count;
  u64* seg = a.S > 1 ? a.keys + (n * a.S + s) * a.k : nullptr;
  // every candidate to its place; what the places beyond k add to the others then depends on the values only
  u64 mine[CAP / T];
  int rank[CAP / T];
#pragma unroll
  for (int i = 0; i < CAP / T; ++i) {
    if (i * T >= nc) continue;
    mine[i] = i * T + tid < nc ? cand[i * T + tid] : 0ull;
    int r = 0;
    for (int j = 0; j < nc; ++j) r += cand[j] > mine[i] ? 1 : 0;
    rank[i] = r;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < CAP / T; ++i) if (i * T + tid < nc) cand[rank[i]] = mine[i];
  __syncthreads();
  for (int c = tid; c < nc; c += T) {
    const u64 v = cand[c];
    if (c >= a.k) others.add1(order_value((unsigned)(v >> 32)), a.c);
    else if (seg) seg[c] = v;
    else emit_row<E>(a, n, c, (unsigned)(v >> 32), ~(unsigned)v);
  }
  if (seg) for (int c = nc + tid; c < a.k; c += T) seg[c] = 0ull;
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

// One workgroup selects the k best of up to `per` segments' candidates: all of them in registers, the k-th best by bisection over the
// order bits (then, among equal values, over the indices), counting with one barrier per step.  A row with more segments is merged in
// levels: blockIdx.y is the group, its result one segment of the next level (last level: the row's result).
constexpr int kMergeThreads = 512, kMergeRegs = 16, kMergeMax = kMergeThreads * kMergeRegs;

template <typename E> __global__ __launch_bounds__(kMergeThreads) void top_merge_kernel(TopArgs a, int per, u64* keys_out, float2* sums_out) {
  constexpr int W = kMergeThreads / 64;
  __shared__ u64 best[VLN_TOP_LOGITS_MAX];
  __shared__ int part[2][W];
  __shared__ unsigned ends[2][W];
  __shared__ float2 sums[W];
  __shared__ int taken;
  const long n = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, s0 = blockIdx.y * per, segs = min(per, a.S - s0), total = segs * a.k;
  const u64* keys = a.keys + (n * a.S + s0) * a.k;
  OnlineSum others;
  for (int i = tid; i < segs; i += kMergeThreads) {
    const float2 o = a.sums[n * a.S + s0 + i];
    others.merge(o.x, o.y, a.c);
  }
  unsigned hi[kMergeRegs], lo[kMergeRegs], least = 0xffffffffu, most = 0;
  const int regs = (total + kMergeThreads - 1) / kMergeThreads;
#pragma unroll
  for (int i = 0; i < kMergeRegs; ++i) {
    const int at = i * kMergeThreads + tid;
    const u64 v = i < regs && at < total ? keys[at] : 0ull;
    hi[i] = (unsigned)(v >> 32); lo[i] = (unsigned)v;
    most = max(most, hi[i]);
    least = min(least, v ? hi[i] : 0xffffffffu);
  }
  if (tid == 0) taken = 0;
  if (tid < a.k) best[tid] = 0ull;
  least = wave_umin(least); most = wave_umax(most);
  if (lane == 0) { ends[0][w] = least; ends[1][w] = most; }
  __syncthreads();
  for (int i = 0; i < W; ++i) { least = min(least, ends[0][i]); most = max(most, ends[1][i]); }
  int turn = 0;
  auto block_count = [&](auto&& has) {
    int c = 0;
#pragma unroll
    for (int i = 0; i < kMergeRegs; ++i) if (i < regs) c += __popcll(__ballot(has(hi[i], lo[i])));
    if (lane == 0) part[turn][w] = c;
    __syncthreads();
    c = 0;
    for (int i = 0; i < W; ++i) c += part[turn][i];
    turn ^= 1;
    return c;
  };
  bool exact = true;
  unsigned th = 1u, tl = 0u;                 // (a group with no more than k elements keeps them all)
  if (block_count([&](unsigned h, unsigned) { return h != 0u; }) > a.k)
    th = bisect(least, most, a.k, exact, [&](unsigned t) { return block_count([&](unsigned h, unsigned) { return h >= t; }); });
  if (!exact) {
    const int need = a.k - block_count([&](unsigned h, unsigned) { return h > th; });
    bool e;
    tl = bisect(0u, 0xffffffffu, need, e, [&](unsigned t) { return block_count([&](unsigned h, unsigned l) { return h == th && l >= t; }); });
  }
#pragma unroll
  for (int i = 0; i < kMergeRegs; ++i) {
    if (i >= regs) continue;
    const bool keep = hi[i] > th || (hi[i] == th && lo[i] >= tl);
    const u64 mask = __ballot(keep);
    int base = 0;
    if (mask && lane == 0) base = atomicAdd(&taken, __popcll(mask));
    base = __builtin_amdgcn_readfirstlane(base);
    if (keep) best[base + lanes_below(mask)] = ((u64)hi[i] << 32) | lo[i];
    else if (hi[i]) others.add1(order_value(hi[i]), a.c);
  }
  others.wave(a.c);
  if (lane == 0) sums[w] = make_float2(others.m, others.s);
  __syncthreads();
  const long slot = n * gridDim.y + blockIdx.y;
  if (tid < a.k) {
    const u64 mine = best[tid];
    int rank = 0;
    for (int j = 0; j < a.k; ++j) rank += best[j] > mine ? 1 : 0;
    if (keys_out) keys_out[slot * a.k + tid] = mine;
    else emit_row<E>(a, n, rank, (unsigned)(mine >> 32), ~(unsigned)mine);
  }
  if (tid == 0) {
    OnlineSum o;
    for (int i = 0; i < W; ++i) o.merge(sums[i].x, sums[i].y, a.c);
    if (keys_out) sums_out[slot] = make_float2(o.m, o.s);
    else a.rest[n] = log_mass(o.m, o.s, a.invT);
  }
}

struct TopPlan {
  int W, NVR, G, S, per;        // waves, vectors per thread, groups per thread, segments, segments of one merge
  int levels; int count[8];     // segments left after each merge level
};
// Short rows (<= 256 vectors) with k <= 64: one wave, no barrier to wait for.  Otherwise four waves and the most vectors per thread (16:
// 64 KB of a row) that still give every CU two workgroups; more, smaller segments otherwise, at least 4 vectors per thread.
static TopPlan top_plan(int N, int V, int k, int vec) {
  TopPlan p{};
  const long nv = ((long)V + vec - 1) / vec;
  const int cus = device_cus() > 0 ? device_cus() : 256;
  if (nv <= 256 && k <= 64) { p.W = 1; p.NVR = 4; p.G = k <= 16 ? 1 : 4; }
  else {
    p.W = 4; p.NVR = 16; p.G = k <= 64 ? 1 : 4;
    while (p.NVR > 4 && (nv <= 256L * (p.NVR / 2) || (long)N * ((nv + 256L * p.NVR - 1) / (256L * p.NVR)) < 2L * cus)) p.NVR /= 2;
  }
  const long held = 64L * p.W * p.NVR;
  p.S = (int)((nv + held - 1) / held);
  p.per = kMergeMax / k;
  for (int n = p.S; n > 1;) { n = (n + p.per - 1) / p.per; p.count[p.levels++] = n; }
  return p;
}
static int64_t top_ws(const TopPlan& p, int N, int k) {
  int64_t segs = p.S > 1 ? p.S : 0;
  for (int i = 0; i + 1 < p.levels; ++i) segs += p.count[i];
  return segs * N * ((int64_t)k * 8 + 8);
}

template <typename E, int W, int NVR> static void top_rows(const TopArgs& a, int G, hipStream_t st) {
  const dim3 grid((unsigned)a.N, (unsigned)a.S);
  if (G == 1) VLN_LAUNCH((top_row_kernel<E, W, NVR, 1>), grid, dim3(64 * W), 0, st, a);
  else VLN_LAUNCH((top_row_kernel<E, W, NVR, 4>), grid, dim3(64 * W), 0, st, a);
}
template <typename E> static int top_launch(TopArgs a, const TopPlan& p, char* ws, hipStream_t st) {
  auto take = [&](int segs) {
    a.keys = reinterpret_cast<u64*>(ws);
    a.sums = reinterpret_cast<float2*>(ws + (int64_t)a.N * segs * a.k * 8);
    ws += (int64_t)a.N * segs * (a.k * 8 + 8);
  };
  a.S = p.S;
  if (a.S > 1) take(a.S);
  if (p.W == 1) top_rows<E, 1, 4>(a, p.G, st);
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
  return vln::top_ws(vln::top_plan(N, V, k, type == VLN_F32 ? 4 : 8), N, k);
}
extern "C" int vln_top_logits(const void* logits, int64_t ld, int type, int N, int V, int k, float temperature, void* values, int64_t* ids,
                              float* rest, void* ws, int64_t ws_bytes, vln_stream_t s) {
  if (!logits || !values || !ids || !rest || N <= 0 || V <= 0 || ld < V) { vln::set_error("vln_top_logits: bad args"); return VLN_ERR_ARG; }
  if (type != VLN_F32 && type != VLN_BF16) { vln::set_error("vln_top_logits: type must be fp32 or bf16"); return VLN_ERR_ARG; }
  if (k < 1 || k > V || k > VLN_TOP_LOGITS_MAX) { vln::set_error("vln_top_logits: k must be 1 .. min(V, %d)", VLN_TOP_LOGITS_MAX); return VLN_ERR_ARG; }
  if (!(temperature >= VLN_TEMPERATURE_MIN && temperature <= VLN_TEMPERATURE_MAX)) { vln::set_error("vln_top_logits: bad temperature"); return VLN_ERR_ARG; }
  const vln::TopPlan p = vln::top_plan(N, V, k, type == VLN_F32 ? 4 : 8);
  const int64_t need = vln::top_ws(p, N, k);
  if (need && (!ws || ws_bytes < need)) { vln::set_error("vln_top_logits: workspace too small"); return VLN_ERR_ARG; }
  vln::TopArgs a{};
  a.logits = logits; a.ld = ld; a.N = N; a.V = V; a.k = k;
  a.c = vln::kLog2e / temperature; a.invT = 1.f / temperature;
  a.values = values; a.ids = (long long*)ids; a.rest = rest;
  if (type == VLN_F32) return vln::top_launch<float>(a, p, static_cast<char*>(ws), (hipStream_t)s);
  return vln::top_launch<bf16_raw>(a, p, static_cast<char*>(ws), (hipStream_t)s);
}
