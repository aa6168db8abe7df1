// Distillation from a teacher's top logits (vln_distill_fwd / vln_distill_bwd): the loss of a row over the K words the teacher kept,
// optionally "any other word" as one more outcome, optionally mixed with the cross entropy of a hard target.  include/vln_hip.h states
// the formulas.
//
// Bound: bytes.  The forward reads the logits once (ONE WAVE per row, or per segment of a row when there are few rows: a running
// (maximum, sum) per lane, joined at the end, no workgroup barrier), the backward reads them again and writes the gradient: nothing of
// size N x V is kept between the two, only kStat floats per row.  With teacher_rest the sum runs over the words the teacher did NOT
// keep (a bitmap of the kept ones in LDS, one byte tested per 8 logits): the mass of the others is a sum of positive terms, never
// 1 - (sum of the kept), which cancels when the student is sure.  The kept words (<= VLN_DISTILL_MAX per row) are handled by their own
// lanes: loss terms in the forward, and in the backward their gradients overwrite what the streaming loop wrote there.
//
// Measured, us, forward / forward and backward: 8192 x 32000 bf16, K 64, T 2, hard targets 117 / 319 (4.5 and 4.9 TB/s of what is moved, a copy:
// 5.2); 1021 x 50001 bf16 with the rest 29 / 65; 5120 x 992 fp32 with the rest 14.6 / 24.5; 16 x 992: 6.3 / 11.4, of which three launches are
// most.  The backward reads the logits a second time rather than keep a gradient from the forward: with an upstream gradient of 1 the latter
// would move a third less, with any other a third more, and [N, V] would stay alive in between.
#include <type_traits>

#include "word_rows.h"
#include "../../include/vln_hip.h"

namespace vln {

constexpr int kStat = VLN_DISTILL_STATS;      // per row: see the enum
enum { ST_FLAGS = 0, ST_M, ST_S, ST_S1, ST_MR, ST_SR, ST_TM, ST_TS, ST_R };      // (finish_row writes them in this order)
enum { ROW_LIVE = 1, ROW_SOFT = 2, ROW_TWICE = 4 };      // counted; the teacher has mass; some kept word is listed twice

struct DistillArgs {
  const void* logits; int64_t ld;
  const long long* ids; int64_t ld_ids;
  const void* tvals; int64_t ld_t; int t_bf16;
  const float* t_rest;
  const long long* target;
  long ignore;
  int N, V, K, W, S, seg_vecs;
  float c, invT, T, alpha;
  float* rows; float* stats;
  float4* part;               // S > 1: [N, S]
  // backward
  void* dz; int64_t ldz; const float* g; long g_stride; const float* inv_count;
};

__device__ __forceinline__ float teacher_value(const DistillArgs& a, long n, int j) {
  return a.t_bf16 ? Elt<bf16_raw>::ld(static_cast<const bf16_raw*>(a.tvals) + n * a.ld_t + j)
                  : static_cast<const float*>(a.tvals)[n * a.ld_t + j];
}
// t / T; a finite value stays finite, so that a row masked with the type's lowest value is still a distribution
__device__ __forceinline__ float teacher_u(const DistillArgs& a, long n, int j) {
  const float t = teacher_value(a, n, j);
  return t == -INFINITY ? t : (t < 0.f ? fmaxf(t * a.invT, -FLT_MAX) : t * a.invT);
}
__device__ __forceinline__ bool row_ignored(const DistillArgs& a, long n) { return a.target && (long)a.target[n] == a.ignore; }

// The kept words of a row in registers, entry j of thread j % B: ids are asked for first, the student's logits at them as soon as they
// are there, so that neither waits behind the stream of the row.
template <int B> struct Kept {
  static constexpr int R = VLN_DISTILL_MAX / B;
  int id[R];             // -1: absent
  float u[R], z[R];      // t / T, the student's logit
  __device__ __forceinline__ void ask(const DistillArgs& a, long n, int tid) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      id[i] = -1;
      u[i] = z[i] = 0.f;
      const int j = i * B + tid;
      if (j < a.K) {
        const long long v = a.ids[n * a.ld_ids + j];
        id[i] = v >= 0 && v < a.V ? (int)v : -1;
        u[i] = teacher_u(a, n, j);
      }
    }
  }
  template <typename E> __device__ __forceinline__ void gather(const E* p) {
#pragma unroll
    for (int i = 0; i < R; ++i) if (id[i] >= 0) z[i] = Elt<E>::ld(p + id[i]);
  }
  template <typename F> __device__ __forceinline__ void each(F&& f) const {      // f(i): the entries present
#pragma unroll
    for (int i = 0; i < R; ++i) if (id[i] >= 0) f(i);
  }
};

// Everything of a row that does not need the whole row again, by one wave.  dense / s1: the (maximum, sum) over all words -- or, TAIL,
// over the words that are not kept -- at temperature T, and the sum at temperature 1 relative to the same maximum (hard targets).
// kid [K]: the row's word ids in LDS (-1: absent); twice: some word may be listed twice; zy: the student's logit at the target.
template <bool TAIL> __device__ __forceinline__ void finish_row(const DistillArgs& a, long n, const Kept<64>& k, OnlineSum dense, float s1,
                                                                const int* kid, bool twice, float rest, float zy, int lane) {
  const float c = a.c;
  // teacher: maximum and sum over the outcomes present
  float tm = -INFINITY;
  bool nan = false;                  // (no maximum takes a NaN: it enters through the sum, and the row's loss is NaN)
  auto outcome = [&](float u) { tm = fmaxf(tm, u); nan = nan || u != u; };
  if (TAIL) outcome(rest);
  k.each([&](int i) { outcome(k.u[i]); });
  tm = wave_fmax(tm);
  const bool soft = tm != -INFINITY || __any(nan);
  const float tref = tm != -INFINITY ? tm : 0.f;
  float ts = 0.f;
  k.each([&](int i) { ts += exp2_hw((k.u[i] - tref) * kLog2e); });
  const float er = TAIL ? exp2_hw((rest - tref) * kLog2e) : 0.f;
  ts = wave_fsum(ts) + er;
  // a word listed twice: only its first entry counts in the student's total
  bool again[Kept<64>::R] = {};
  if (twice) {
    twice = false;
    k.each([&](int i) {
      for (int j = 0; j < i * 64 + lane; ++j) again[i] = again[i] || kid[j] == k.id[i];
      twice = twice || again[i];
    });
    twice = __any(twice);
  }
  // student
  OnlineSum all = dense;
  if (TAIL) {
    float M = dense.m;
    k.each([&](int i) { M = fmaxf(M, k.z[i]); });
    M = wave_fmax(M);
    float t = 0.f, t1 = 0.f;
    k.each([&](int i) {
      if (again[i]) return;
      const float d = k.z[i] - M;
      t += exp2_hw(d * c);
      t1 += exp2_hw(d * kLog2e);
    });
    all.s = dense.s * exp2_hw((dense.m - M) * c) + wave_fsum(t);
    s1 = s1 * exp2_hw((dense.m - M) * kLog2e) + wave_fsum(t1);
    all.m = M;
  }
  const float log_s = logf(all.s), log_ts = logf(ts);
  float loss = 0.f;
  if (soft) {
    k.each([&](int i) {
      const float lq = (k.u[i] - tref) - log_ts, q = exp2_hw(lq * kLog2e);
      const float lp = k.z[i] == -INFINITY ? -INFINITY : (k.z[i] - all.m) * a.invT - log_s;
      if (q != 0.f) loss += q * (lq - lp);
    });
    if (TAIL && lane == 0 && er != 0.f) {
      const float lr = (rest - tref) - log_ts;
      const float lpr = dense.s == 0.f ? -INFINITY : (dense.m - all.m) * a.invT + logf(dense.s) - log_s;
      loss += exp2_hw(lr * kLog2e) * (lr - lpr);
    }
  }
  loss = wave_fsum(loss) * a.alpha * a.T * a.T;
  if (a.alpha == 0.f) loss = 0.f;
  const bool live = a.target ? true : soft;          // (ignored rows do not come here)
  if (a.target && a.alpha < 1.f) loss += (1.f - a.alpha) * (all.m - zy + logf(s1));
  if (lane == 0) {
    a.rows[n] = live ? loss : 0.f;
    float4* st = reinterpret_cast<float4*>(a.stats + n * kStat);
    st[0] = make_float4(__int_as_float((live ? ROW_LIVE : 0) | (soft ? ROW_SOFT : 0) | (twice ? ROW_TWICE : 0)), all.m, all.s, s1);
    st[1] = make_float4(dense.m, dense.s, tref, ts);
    st[2] = make_float4(soft ? er / ts : 0.f, 0.f, 0.f, 0.f);
  }
}
template <typename E> __device__ __forceinline__ float target_logit(const DistillArgs& a, long n, const E* p) {      // NaN: no such word
  if (!a.target || a.alpha >= 1.f) return 0.f;
  const long y = (long)a.target[n];
  return y >= 0 && y < a.V ? Elt<E>::ld(p + y) : __builtin_nanf("");
}
__device__ __forceinline__ void dead_row(const DistillArgs& a, long n, int lane) {
  if (lane == 0) { a.rows[n] = 0.f; a.stats[n * kStat] = __int_as_float(0); }
}
// one wave joins the (maximum, sum at T, sum at 1) of `count` parts, in their order per lane
__device__ __forceinline__ void join_parts(OnlineSum& o, float& s1, const float4* parts, int count, float c, int lane) {
  o = OnlineSum();
  s1 = 0.f;
  for (int i = lane; i < count; i += 64) {
    const float4 q = parts[i];
    const float M = fmaxf(o.m, q.x);
    s1 = s1 * exp2_hw((o.m - M) * kLog2e) + q.z * exp2_hw((q.x - M) * kLog2e);
    o.merge(q.x, q.y, c);
  }
  const float M = wave_fmax(o.m);
  s1 = wave_fsum(s1 * exp2_hw((o.m - M) * kLog2e));
  o.wave(c);
}
// kid <- the ids; true if two of the wave's entries may name the same word: their bits in a table of 2^14 meet (then the list is searched)
constexpr int kHashWords = 512;
__device__ __forceinline__ bool stage_ids(const DistillArgs& a, const Kept<64>& k, int* kid, unsigned* hash, int lane) {
  for (int i = lane; i < kHashWords; i += 64) hash[i] = 0u;
  wave_sync();
  bool met = false;
#pragma unroll
  for (int i = 0; i < Kept<64>::R; ++i) {
    if (i * 64 + lane < a.K) kid[i * 64 + lane] = k.id[i];
    if (k.id[i] >= 0) {
      const unsigned h = (unsigned)k.id[i] & (kHashWords * 32 - 1);
      met = met || ((atomicOr(&hash[h >> 5], 1u << (h & 31)) >> (h & 31)) & 1u);
    }
  }
  wave_sync();
  return __any(met);
}

// HARD: also the sum at temperature 1 (T != 1 and a hard target); otherwise s1 is the sum at T.  W: waves of a row (or segment).
template <typename E, bool TAIL, bool HARD, int W> __global__ __launch_bounds__(64 * W) void distill_fwd_kernel(DistillArgs a) {
  extern __shared__ unsigned lds[];
  constexpr int VEC = RowGeo<E>::VEC, U = 4, B = 64 * W;
  const long n = blockIdx.x;
  const int s = blockIdx.y, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  if (row_ignored(a, n)) { if (s == 0) dead_row(a, n, tid); return; }
  const E* p = static_cast<const E*>(a.logits) + n * a.ld;
  const RowGeo<E> g(p, a.V);
  const int v0 = min(g.nv, s * a.seg_vecs), v1 = min(g.nv, v0 + a.seg_vecs);
  const bool finishes = a.S == 1 && w == 0;
  Kept<64> k;
  if (finishes || (TAIL && w == 0)) k.ask(a, n, lane);
  float rest = 0.f, zy = 0.f;
  if (finishes) { rest = TAIL ? a.t_rest[n] : 0.f; zy = target_logit(a, n, p); }
  uint4 raw[U];
  auto fetch = [&](int v) {
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = ld_vec<E>(p + g.head + (int64_t)min(v + u * B, v1 - 1) * VEC);
  };
  if (v0 + tid < v1) fetch(v0 + tid);
  int* kid = reinterpret_cast<int*>(lds);
  unsigned* bm = lds + VLN_DISTILL_MAX + kHashWords;       // bit i: column i of the segment's vectors; then head, then tail (VEC bits each)
  const int nbits_v = a.seg_vecs * VEC;
  bool twice = false;
  if (TAIL) {
    const int nw = (nbits_v + 2 * VEC + 31) / 32;
    for (int i = tid; i < nw; i += B) bm[i] = 0u;
    __syncthreads();
  }
  if (finishes) {
    twice = stage_ids(a, k, kid, lds + VLN_DISTILL_MAX, lane);
    k.gather(p);
  }
  if (TAIL) {
    if (w == 0) k.each([&](int i) {
      const int id = k.id[i];
      int bit = -1;
      if (id < g.head) bit = nbits_v + id;
      else if (id >= g.tail0()) bit = nbits_v + VEC + (id - g.tail0());
      else { const int at = id - g.head - v0 * VEC; if (at >= 0 && at < (v1 - v0) * VEC) bit = at; }
      if (bit >= 0) atomicOr(&bm[bit >> 5], 1u << (bit & 31));
    });
    __syncthreads();
  }
  OnlineSum o;
  float s1 = 0.f;
  auto take = [&](const auto& x, float mx) {
    constexpr int N = sizeof(x) / sizeof(float);
    if (mx > o.m) {
      if (HARD) s1 *= exp2_hw((o.m - mx) * kLog2e);
      o.raise(mx, a.c);
    }
    float t = 0.f, t1 = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float d = x[i] - o.m;
      t += exp2_hw(d * a.c);
      if (HARD) t1 += exp2_hw(d * kLog2e);
    }
    o.s += t;
    if (HARD) s1 += t1;
  };
  if (s == 0) {
    int col = -1, bit = 0;
    if (tid < g.head) { col = tid; bit = nbits_v + tid; }
    else if (tid >= VEC && tid - VEC < g.tail) { col = g.tail0() + tid - VEC; bit = nbits_v + tid; }
    float x[1] = {col >= 0 ? Elt<E>::ld(p + col) : -INFINITY};
    if (TAIL && col >= 0 && ((bm[bit >> 5] >> (bit & 31)) & 1u)) x[0] = -INFINITY;
    take(x, x[0]);
  }
  for (int v = v0 + tid; v < v1; v += B * U) {
    float x[U * VEC];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      unpack16<E>(raw[u], x + u * VEC);
      unsigned out = 0u;             // bit j: element j does not count
      if (TAIL) { const int bit = (v + u * B - v0) * VEC; if (v + u * B < v1) out = (bm[bit >> 5] >> (bit & 31)) & ((1u << VEC) - 1u); }
      if (v + u * B >= v1) out = ~0u;
      if (out) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) if ((out >> j) & 1u) x[u * VEC + j] = -INFINITY;
      }
    }
    if (v + B * U < v1) fetch(v + B * U);
    float mx = x[0];
#pragma unroll
    for (int j = 1; j < U * VEC; ++j) mx = fmaxf(mx, x[j]);
    take(x, mx);
  }
  const float M = wave_fmax(o.m);
  if (HARD) s1 = wave_fsum(s1 * exp2_hw((o.m - M) * kLog2e));
  o.s = wave_fsum(o.s * exp2_hw((o.m - M) * a.c));
  o.m = M;
  if (!HARD) s1 = o.s;
  if (W > 1) {
    __shared__ float4 parts[W];
    if (lane == 0) parts[w] = make_float4(o.m, o.s, s1, 0.f);
    __syncthreads();
    if (w > 0) return;
    join_parts(o, s1, parts, W, a.c, lane);
  }
  if (finishes) finish_row<TAIL>(a, n, k, o, s1, kid, twice, rest, zy, lane);
  else if (lane == 0) a.part[n * a.S + s] = make_float4(o.m, o.s, s1, 0.f);
}

template <typename E, bool TAIL> __global__ __launch_bounds__(64) void distill_join_kernel(DistillArgs a) {
  __shared__ int kid[VLN_DISTILL_MAX];
  __shared__ unsigned hash[kHashWords];
  const long n = blockIdx.x;
  const int lane = threadIdx.x;
  if (row_ignored(a, n)) return;
  const E* p = static_cast<const E*>(a.logits) + n * a.ld;
  Kept<64> k;
  k.ask(a, n, lane);
  const float rest = TAIL ? a.t_rest[n] : 0.f, zy = target_logit(a, n, p);
  OnlineSum o;
  float s1;
  join_parts(o, s1, a.part + n * a.S, a.S, a.c, lane);
  const bool twice = stage_ids(a, k, kid, hash, lane);
  k.gather(p);
  __syncthreads();
  finish_row<TAIL>(a, n, k, o, s1, kid, twice, rest, zy, lane);
}

// sum or mean over the rows, in a fixed order; inv_count: what the backward multiplies every row's gradient with
__global__ __launch_bounds__(1024) void distill_reduce_kernel(const float* rows, const float* stats, int N, int mean, float* loss, float* inv_count) {
  __shared__ float part[16];
  __shared__ int cnt[16];
  float acc = 0.f;
  int n = 0;
  for (int i = threadIdx.x; i < N; i += 1024) {
    acc += rows[i];
    n += __float_as_int(stats[(long)i * kStat + ST_FLAGS]) & ROW_LIVE;
  }
  acc = wave_fsum(acc);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
  if ((threadIdx.x & 63) == 0) { part[threadIdx.x >> 6] = acc; cnt[threadIdx.x >> 6] = n; }
  __syncthreads();
  if (threadIdx.x == 0) {
    float t = 0.f;
    int c = 0;
    for (int i = 0; i < 16; ++i) { t += part[i]; c += cnt[i]; }
    loss[0] = mean ? t / (float)c : t;
    inv_count[0] = mean ? 1.f / (float)c : 1.f;
  }
}

// The gradient is written past the caches (nontemporal): 4096 x 32000 bf16 190 -> 171 us, 5120 x 992 fp32 unchanged.  Rows come in reverse
// order, those the forward read last first: 8192 x 32000 bf16 350 -> 329 us.
// d z_v = g [ alpha T (p_v - q_v) + (1 - alpha) (softmax(z)_v - [v = y]) ], p_v - r p_v / p_rest for the words the teacher did not keep.
// The streaming loop evaluates  A exp((z - M) / T) + H exp(z - M)  with one pair (A, H) per row: M is the maximum the exponentials of
// that loop are bounded by (TAIL: the others' maximum), so neither a sure student's tiny p_rest nor its kept words leave the range.
template <typename E, bool TAIL, bool HARD, int W> __global__ __launch_bounds__(64 * W) void distill_bwd_kernel(DistillArgs a) {
  extern __shared__ unsigned lds[];
  constexpr int VEC = RowGeo<E>::VEC, U = 4, B = 64 * W;
  __shared__ int y_kept;
  const long n = gridDim.x - 1 - blockIdx.x;
  const int s = blockIdx.y, tid = threadIdx.x;
  if (tid == 0) y_kept = 0;
  const E* p = static_cast<const E*>(a.logits) + n * a.ld;
  E* dz = static_cast<E*>(a.dz) + n * a.ldz;
  Kept<B> k;
  k.ask(a, n, tid);
  const float* st = a.stats + n * kStat;
  const int flags = __float_as_int(st[ST_FLAGS]);
  const RowGeo<E> g(dz, a.V);                 // the writes decide the alignment
  const bool same = ((reinterpret_cast<uintptr_t>(p) ^ reinterpret_cast<uintptr_t>(dz)) & 15) == 0;
  const int v0 = min(g.nv, s * a.seg_vecs), v1 = min(g.nv, v0 + a.seg_vecs);
  const bool single = s == 0 && (tid < g.head || (tid >= VEC && tid - VEC < g.tail));
  const int scol = tid < g.head ? tid : g.tail0() + tid - VEC;
  if (!(flags & ROW_LIVE)) {                  // an ignored row: zeros, whatever its logits hold
    if (single) Elt<E>::st(dz + scol, 0.f);
    for (int v = v0 + tid; v < v1; v += B) st_vec_nt<E>(dz + g.head + (int64_t)v * VEC, make_uint4(0, 0, 0, 0));
    return;
  }
  uint4 raw[U];
  auto fetch = [&](int v) {
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = ld_vec<E>(p + g.head + (int64_t)min(v + u * B, v1 - 1) * VEC);
  };
  if (same && v0 + tid < v1) fetch(v0 + tid);
  auto here = [&](int id) {                   // a column of this segment
    if (id < g.head || id >= g.tail0()) return s == 0;
    const int i = (id - g.head) / VEC;
    return i >= v0 && i < v1;
  };
  int* kid = reinterpret_cast<int*>(lds);
  if (flags & ROW_TWICE) {
#pragma unroll
    for (int i = 0; i < Kept<B>::R; ++i) if (i * B + tid < a.K) kid[i * B + tid] = k.id[i];
  }
  const float up = a.g[n * a.g_stride] * (a.inv_count ? a.inv_count[0] : 1.f);
  const bool soft = (flags & ROW_SOFT) != 0 && a.alpha != 0.f;
  const float m = st[ST_M], sum = st[ST_S], s1 = st[ST_S1], r = TAIL ? st[ST_R] : 0.f;
  const float M = TAIL ? st[ST_MR] : m, sr = st[ST_SR], tm = st[ST_TM], its = 1.f / st[ST_TS];
  const float gs = soft ? up * a.alpha * a.T : 0.f;                  // soft term's factor
  const bool hard = a.target != nullptr && a.alpha < 1.f;
  const float gh = hard ? up * (1.f - a.alpha) : 0.f;
  const float is = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum), is1 = s1 > 0.f ? 1.f / s1 : (s1 == 0.f ? 0.f : s1);
  float A = gs * (exp2_hw((M - m) * a.c) * is - (TAIL && sr > 0.f ? r / sr : 0.f));
  float H = gh * exp2_hw((M - m) * kLog2e) * is1;
  const long y = hard ? (long)a.target[n] : -1;
  const bool bad_y = hard && (y < 0 || y >= a.V);
  if (bad_y) H = __builtin_nanf("");
  if (!HARD) A += H;                          // temperature 1: one exponential serves both terms
  auto grad = [&](float z) {
    const float d = z - M;
    float v = A * exp2_hw(d * a.c);
    if (HARD) v += H * exp2_hw(d * kLog2e);
    return v;
  };
  // (kept words matter if they have a share of the gradient, or if the streaming loop's factors are not theirs)
  if (soft || TAIL) {
    k.gather(p);
    k.each([&](int i) { if (k.id[i] == y) y_kept = 1; });
  }
  if (single) Elt<E>::st(dz + scol, grad(Elt<E>::ld(p + scol)));
  if (same) {
    for (int v = v0 + tid; v < v1; v += B * U) {
      uint4 now[U];
#pragma unroll
      for (int u = 0; u < U; ++u) now[u] = raw[u];
      if (v + B * U < v1) fetch(v + B * U);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float x[VEC];
        unpack16<E>(now[u], x);
#pragma unroll
        for (int j = 0; j < VEC; ++j) x[j] = grad(x[j]);
        if (v + u * B < v1) st_vec_nt<E>(dz + g.head + (int64_t)(v + u * B) * VEC, pack16<E>(x));
      }
    }
  } else {                                    // rows that start at different distances from a 16-byte boundary
    for (int c = g.head + v0 * VEC + tid; c < g.head + v1 * VEC; c += B) Elt<E>::st(dz + c, grad(Elt<E>::ld(p + c)));
  }
  // the kept words and the target: their own values over what the loop wrote
  __syncthreads();
  if (soft || TAIL) k.each([&](int i) {
    const int id = k.id[i], j = i * B + tid;
    if (!here(id)) return;
    float q = soft ? exp2_hw((k.u[i] - tm) * kLog2e) * its : 0.f;
    if (soft && (flags & ROW_TWICE)) {        // listed more than once: the first entry writes the sum, in entry order
      for (int e = 0; e < j; ++e) if (kid[e] == id) return;
      for (int e = j + 1; e < a.K; ++e) if (kid[e] == id) q += exp2_hw((teacher_u(a, n, e) - tm) * kLog2e) * its;
    }
    const float d = k.z[i] - m;
    float v = gs * (exp2_hw(d * a.c) * is - q);
    if (hard) v += gh * (exp2_hw(d * kLog2e) * is1 - (id == y ? 1.f : 0.f));
    Elt<E>::st(dz + id, bad_y ? __builtin_nanf("") : v);
  });
  if (hard && !bad_y && !y_kept && tid == 0 && here((int)y)) Elt<E>::st(dz + y, grad(Elt<E>::ld(p + y)) - gh);
}

// Waves and segments per row: one wave for rows under 16 KB (5120 x 992 fp32, forward and backward: 23.9 us; four waves: 32.2), four for
// long ones -- a row is then read by one workgroup front to back, which the memory serves better than 4 x as many rows at once (8192 x
// 32000 bf16: 318; one wave: 347; at 16 KB the two meet).  Fewer rows than CUs are cut into segments, one workgroup per CU (64 x 131072
// bf16: 22 us; not cut: 39), none under two rounds of the workgroup's loads; more would only pay for the join (512 x 32000 bf16: 29; two
// segments: 33).
static void distill_split(int N, int V, int vec, int* W, int* S, int* seg_vecs) {
  const int cus = device_cus() > 0 ? device_cus() : 256;
  const int nv = (V + vec - 1) / vec;
  *W = nv >= 1024 ? 4 : 1;
  const int round = 64 * *W * 4;
  const int want = (cus + N - 1) / N, most = (nv + 2 * round - 1) / (2 * round);
  int n = want < most ? want : most;
  const int least = (nv + 32767) / 32768;                     // (a segment's bitmap stays at 32 KB of LDS)
  if (n < least) n = least;
  if (n < 1) n = 1;
  *seg_vecs = ((nv + n - 1) / n + 63) / 64 * 64;
  *S = (nv + *seg_vecs - 1) / *seg_vecs;
}

template <typename E, bool TAIL, int W> static int distill_fwd_launch(const DistillArgs& a, bool hard, int reduce, float* loss, float* inv_count, hipStream_t st) {
  const unsigned ids = (VLN_DISTILL_MAX + kHashWords) * 4;
  const unsigned bits = TAIL ? (unsigned)((a.seg_vecs * Elt<E>::kVec + 2 * Elt<E>::kVec + 31) / 32 * 4) : 0u;
  const dim3 grid((unsigned)a.N, (unsigned)a.S);
  if (hard) VLN_LAUNCH((distill_fwd_kernel<E, TAIL, true, W>), grid, dim3(64 * W), ids + bits, st, a);
  else VLN_LAUNCH((distill_fwd_kernel<E, TAIL, false, W>), grid, dim3(64 * W), ids + bits, st, a);
  if (a.S > 1) VLN_LAUNCH((distill_join_kernel<E, TAIL>), dim3((unsigned)a.N), dim3(64), 0, st, a);
  if (reduce) VLN_LAUNCH(distill_reduce_kernel, dim3(1), dim3(1024), 0, st, (const float*)a.rows, (const float*)a.stats, a.N, reduce == VLN_REDUCE_MEAN ? 1 : 0, loss, inv_count);
  VLN_CHECK_LAUNCH("distill_fwd");
  return VLN_OK;
}
template <typename E, bool TAIL, int W> static int distill_bwd_launch(const DistillArgs& a, bool hard, hipStream_t st) {
  const dim3 grid((unsigned)a.N, (unsigned)a.S);
  const unsigned ids = VLN_DISTILL_MAX * 4;
  if (hard) VLN_LAUNCH((distill_bwd_kernel<E, TAIL, true, W>), grid, dim3(64 * W), ids, st, a);
  else VLN_LAUNCH((distill_bwd_kernel<E, TAIL, false, W>), grid, dim3(64 * W), ids, st, a);
  VLN_CHECK_LAUNCH("distill_bwd");
  return VLN_OK;
}
template <typename F> static int distill_dispatch(const DistillArgs& a, int type, F&& f) {      // f(element, with rest, waves)
  auto waves = [&](auto e, auto tail) { return a.W == 4 ? f(e, tail, std::integral_constant<int, 4>()) : f(e, tail, std::integral_constant<int, 1>()); };
  auto rest = [&](auto e) { return a.t_rest ? waves(e, std::true_type()) : waves(e, std::false_type()); };
  return type == VLN_F32 ? rest(float()) : rest(bf16_raw());
}

static int distill_args(const vln_distill* p, DistillArgs& a, const char* who, bool backward) {
  if (!p) { set_error("%s: null pointer", who); return VLN_ERR_ARG; }
  if (p->N <= 0 || p->V <= 0 || !p->logits || p->ld < p->V) { set_error("%s: bad logits", who); return VLN_ERR_ARG; }
  if (p->K < 1 || p->K > VLN_DISTILL_MAX || !p->ids || !p->teacher || p->ld_ids < p->K || p->ld_teacher < p->K) {
    set_error("%s: the teacher keeps 1 .. %d words per row", who, VLN_DISTILL_MAX); return VLN_ERR_ARG;
  }
  if ((p->type != VLN_F32 && p->type != VLN_BF16) || (p->teacher_type != VLN_F32 && p->teacher_type != VLN_BF16)) {
    set_error("%s: types must be fp32 or bf16", who); return VLN_ERR_ARG;
  }
  if (!(p->temperature >= VLN_TEMPERATURE_MIN && p->temperature <= VLN_TEMPERATURE_MAX) || !(p->alpha >= 0.f && p->alpha <= 1.f)) {
    set_error("%s: bad temperature / alpha", who); return VLN_ERR_ARG;
  }
  if (p->alpha < 1.f && !p->target) { set_error("%s: alpha < 1 needs hard targets", who); return VLN_ERR_ARG; }
  if ((!p->rows && !backward) || !p->stats) { set_error("%s: rows / stats missing", who); return VLN_ERR_ARG; }
  a = DistillArgs{};
  a.logits = p->logits; a.ld = p->ld;
  a.ids = (const long long*)p->ids; a.ld_ids = p->ld_ids;
  a.tvals = p->teacher; a.ld_t = p->ld_teacher; a.t_bf16 = p->teacher_type == VLN_BF16;
  a.t_rest = p->teacher_rest;
  a.target = (const long long*)p->target; a.ignore = (long)p->ignore_index;
  a.N = p->N; a.V = p->V; a.K = p->K;
  a.c = kLog2e / p->temperature; a.invT = 1.f / p->temperature; a.T = p->temperature; a.alpha = p->alpha;
  a.rows = p->rows; a.stats = p->stats;
  distill_split(a.N, a.V, p->type == VLN_F32 ? 4 : 8, &a.W, &a.S, &a.seg_vecs);
  if (!grid_fits(a.N, 64 * a.W, a.S)) { set_error("%s: too many rows for one launch", who); return VLN_ERR_ARG; }
  return VLN_OK;
}

}  // namespace vln

extern "C" int64_t vln_distill_ws_bytes(int N, int V, int type) {
  if (N <= 0 || V <= 0 || (type != VLN_F32 && type != VLN_BF16)) return 0;
  int W, S, sv;
  vln::distill_split(N, V, type == VLN_F32 ? 4 : 8, &W, &S, &sv);
  return S > 1 ? (int64_t)N * S * 16 : 0;
}
extern "C" int vln_distill_fwd(const vln_distill* p, int reduction, float* loss, float* inv_count, void* ws, int64_t ws_bytes, vln_stream_t s) {
  vln::DistillArgs a;
  const int rc = vln::distill_args(p, a, "vln_distill_fwd", false);
  if (rc != VLN_OK) return rc;
  if ((reduction != VLN_REDUCE_NONE && reduction != VLN_REDUCE_SUM && reduction != VLN_REDUCE_MEAN) || (reduction != VLN_REDUCE_NONE && (!loss || !inv_count))) {
    vln::set_error("vln_distill_fwd: bad reduction"); return VLN_ERR_ARG;
  }
  if (a.S > 1) {
    if (!ws || ws_bytes < (int64_t)a.N * a.S * 16) { vln::set_error("vln_distill_fwd: workspace too small"); return VLN_ERR_ARG; }
    a.part = static_cast<float4*>(ws);
  }
  const bool hard = a.alpha < 1.f && a.T != 1.f;
  hipStream_t st = (hipStream_t)s;
  return vln::distill_dispatch(a, p->type, [&](auto e, auto tail, auto w) {
    return vln::distill_fwd_launch<decltype(e), decltype(tail)::value, decltype(w)::value>(a, hard, reduction, loss, inv_count, st);
  });
}
extern "C" int vln_distill_bwd(const vln_distill* p, const float* dloss, int64_t dloss_stride, const float* inv_count, void* dlogits, int64_t ld_dlogits,
                               vln_stream_t s) {
  vln::DistillArgs a;
  const int rc = vln::distill_args(p, a, "vln_distill_bwd", true);
  if (rc != VLN_OK) return rc;
  if (!dloss || (dloss_stride != 0 && dloss_stride != 1) || !dlogits || ld_dlogits < p->V) { vln::set_error("vln_distill_bwd: bad args"); return VLN_ERR_ARG; }
  a.g = dloss; a.g_stride = (long)dloss_stride; a.inv_count = inv_count; a.dz = dlogits; a.ldz = ld_dlogits;
  const bool hard = a.alpha < 1.f && a.T != 1.f;
  hipStream_t st = (hipStream_t)s;
  return vln::distill_dispatch(a, p->type, [&](auto e, auto tail, auto w) {
    return vln::distill_bwd_launch<decltype(e), decltype(tail)::value, decltype(w)::value>(a, hard, st);
  });
}
