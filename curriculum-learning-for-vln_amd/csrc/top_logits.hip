// The k largest logits of every row, sorted, and the log-mass of all others (vln_top_logits): a teacher's targets for vln_distill_*,
// and with k = 1 the greedy word.  include/vln_hip.h states the contract.
//
// Bound: bytes (the row is read once) for many rows; latency of one wave's chain for few.  ONE WAVE streams a row (or, with few
// rows, one of S segments of it) in chunks of 16 elements per lane and keeps the candidates in a small LDS buffer: no workgroup
// barrier anywhere.  Elements are compared as 64-bit keys (order-preserving bits of the value, complement of the index), all
// distinct, so ties fall to the lowest index and the result does not depend on the order in which candidates were collected.
//   * the first chunk's threshold is the k-th largest of the lanes' maxima (found bit by bit with ballots): at least k elements
//     reach it, and at most 16 k / (maxima per lane) do;
//   * afterwards an element enters the buffer only above the k-th best key so far; a full buffer is cut back to its k best;
//   * everything that is not kept goes into the running (maximum, sum) of exp(z / T), also what a cut throws out, so that the
//     others' mass is a sum of positive terms and never a difference.
// Segments leave k sorted keys each and a second launch merges them with the same buffer.
#include "word_rows.h"
#include "../../include/vln_hip.h"

namespace vln {

typedef unsigned long long u64;

// value <-> order-preserving bits; every NaN is the largest, -0 equals +0.  0 is no element's key.
__device__ __forceinline__ unsigned order_bits(float x) {
  const unsigned b = __float_as_uint(x + 0.f);
  if (x != x) return 0xffffffffu;
  return b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float order_value(unsigned o) {
  if (o == 0xffffffffu) return __builtin_nanf("");
  return __uint_as_float((o & 0x80000000u) ? (o ^ 0x80000000u) : ~o);
}
__device__ __forceinline__ u64 make_key(float x, unsigned idx) { return ((u64)order_bits(x) << 32) | (u64)(~idx); }

struct TopArgs {
  const void* logits; int64_t ld;
  int N, V, k, S, seg;             // seg: elements per segment (a multiple of the chunk), S segments per row
  float c, invT;                   // log2(e) / T, 1 / T
  void* values; long long* ids; float* rest;
  u64* keys; float2* sums;         // S > 1: [N, S, k] and [N, S]
};

__device__ __forceinline__ float nan_max(float a, float b) { return __builtin_elementwise_maximum(a, b); }   // NaN wins (v_maximum3_f32)

// A wave's candidates.  KB: k <= KB; NK registers per lane hold the whole buffer while it is cut.
template <int KB> struct Candidates {
  static constexpr int CAP = 2 * KB + 64, NK = CAP / 64;
  u64* buf;              // [CAP] LDS of this wave
  int cnt, k;
  u64 tkey;              // keys above it may enter
  float tval;            // an element with !(x <= tval) may be above tkey (NaN: all)
  OnlineSum others;      // per lane
  float c;
  int lane;

  __device__ __forceinline__ void init(u64* b, int k_, float c_, int lane_) {
    buf = b; cnt = 0; k = k_; tkey = 0; tval = __builtin_nanf(""); c = c_; lane = lane_;
  }
  // cut the buffer to its k best (call with cnt > k)
  __device__ __forceinline__ void cut() {
    unsigned hi[NK], lo[NK];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      const int at = i * 64 + lane;
      const u64 v = at < cnt ? buf[at] : 0;
      hi[i] = (unsigned)(v >> 32); lo[i] = (unsigned)v;
    }
    // the largest th with at least k keys of hi >= th, bit by bit; the search ends early where exactly k reach it
    unsigned th = 0, tl = 0;
    bool exact = false;
    for (int bit = 31; bit >= 0; --bit) {
      const unsigned t = th | (1u << bit);
      int n = 0;
#pragma unroll
      for (int i = 0; i < NK; ++i) n += __popcll(__ballot(hi[i] >= t));
      if (n >= k) { th = t; if (n == k) { exact = true; break; } }
    }
    if (!exact) {          // equal values at the border: of those, the `need` lowest indices (largest lo)
      int need = k;
#pragma unroll
      for (int i = 0; i < NK; ++i) need -= __popcll(__ballot(hi[i] > th));
      for (int bit = 31; bit >= 0; --bit) {
        const unsigned t = tl | (1u << bit);
        int n = 0;
#pragma unroll
        for (int i = 0; i < NK; ++i) n += __popcll(__ballot(hi[i] == th && lo[i] >= t));
        if (n >= need) tl = t;
      }
    }
    __syncthreads();
    int at = 0;
    u64 least = ~0ull;
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      const bool keep = hi[i] > th || (hi[i] == th && lo[i] >= tl);
      const bool real = i * 64 + lane < cnt;
      const u64 mask = __ballot(keep);
      if (keep) {
        const u64 v = ((u64)hi[i] << 32) | lo[i];
        buf[at + lanes_below(mask)] = v;
        least = v < least ? v : least;
      } else if (real) {
        others.add1(order_value(hi[i]), c);
      }
      at += __popcll(mask);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const u64 v = __shfl_xor(least, o, 64);
      least = v < least ? v : least;
    }
    cnt = k;
    tkey = least;
    const float t = order_value((unsigned)(least >> 32));
    tval = t != t ? INFINITY : t;
    __syncthreads();
  }
  // lanes with `has` offer a key; returns true where it was taken (what is not taken belongs to the others)
  __device__ __forceinline__ bool offer(u64 key, bool has) {
    bool in = has && key > tkey;
    u64 mask = __ballot(in);
    if (!mask) return false;
    if (cnt + __popcll(mask) > CAP) {
      cut();
      in = in && key > tkey;
      mask = __ballot(in);
    }
    if (in) buf[cnt + lanes_below(mask)] = key;
    cnt += __popcll(mask);
    return in;
  }
  // sort what is left (<= k keys): every key's rank is the number of larger ones
  template <typename F> __device__ __forceinline__ void finish(F&& emit) {
    if (cnt > k) cut();
    __syncthreads();
    u64 mine[KB / 64];
    int rank[KB / 64];
#pragma unroll
    for (int i = 0; i < KB / 64; ++i) { mine[i] = i * 64 + lane < cnt ? buf[i * 64 + lane] : 0; rank[i] = 0; }
    for (int j = 0; j < cnt; ++j) {
      const u64 v = buf[j];
#pragma unroll
      for (int i = 0; i < KB / 64; ++i) rank[i] += v > mine[i] ? 1 : 0;
    }
#pragma unroll
    for (int i = 0; i < KB / 64; ++i) if (i * 64 + lane < cnt) emit(rank[i], mine[i]);
    others.wave(c);
  }
};

template <typename E> __device__ __forceinline__ void emit_row(const TopArgs& a, long n, int rank, u64 key) {
  const float v = order_value((unsigned)(key >> 32));
  Elt<E>::st(static_cast<E*>(a.values) + n * a.k + rank, v);
  a.ids[n * a.k + rank] = (long long)(~(unsigned)key);
}
__device__ __forceinline__ float log_mass(const OnlineSum& o, float invT) {
  return o.s == 0.f ? -INFINITY : (o.m == INFINITY ? INFINITY : o.m * invT + logf(o.s));
}

template <typename E, int KB> __global__ __launch_bounds__(64) void top_scan_kernel(TopArgs a) {
  constexpr int VEC = RowGeo<E>::VEC, U = 16 / VEC, G = KB / 64;      // G maxima per lane for the first threshold
  __shared__ u64 buf[Candidates<KB>::CAP];
  const long n = blockIdx.x;
  const int s = blockIdx.y, lane = threadIdx.x;
  const E* p = static_cast<const E*>(a.logits) + n * a.ld;
  const RowGeo<E> g(p, a.V);
  Candidates<KB> cd;
  cd.init(buf, a.k, a.c, lane);
  const int segv = a.seg / VEC, v0 = min(g.nv, s * segv), v1 = s == a.S - 1 ? g.nv : min(g.nv, v0 + segv);
  auto single = [&](int col, bool has) {
    const float x = has ? Elt<E>::ld(p + col) : -INFINITY;
    const bool in = cd.offer(make_key(x, (unsigned)col), has);
    if (has && !in) cd.others.add1(x, a.c);
  };
  if (s == 0 && g.head) single(lane, lane < g.head);
  uint4 raw[U];
  auto fetch = [&](int v) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = v + u * 64 + lane;
      raw[u] = ld_vec<E>(p + g.head + (int64_t)(i < v1 ? i : v1 - 1) * VEC);
    }
  };
  if (v0 < v1) fetch(v0);
  for (int v = v0; v < v1; v += 64 * U) {
    float x[16];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      unpack16<E>(raw[u], x + u * VEC);
      if (v + u * 64 + lane >= v1) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) x[u * VEC + j] = -INFINITY;
      }
    }
    if (v + 64 * U < v1) fetch(v + 64 * U);
    float mx = x[0];
#pragma unroll
    for (int j = 1; j < 16; ++j) mx = nan_max(mx, x[j]);
    if (__any(!(mx <= cd.tval))) {
      if (v == v0) {
        // the k-th largest of 64 G group maxima (groups beyond the row's end do not count) is reached by at least k elements
        unsigned gm[G];
#pragma unroll
        for (int i = 0; i < G; ++i) {
          float m = x[i * (16 / G)];
#pragma unroll
          for (int j = 1; j < 16 / G; ++j) m = nan_max(m, x[i * (16 / G) + j]);
          const int u = i * (16 / G) / VEC;
          gm[i] = v + u * 64 + lane < v1 ? order_bits(m) : 0u;
        }
        unsigned th = 0;
        for (int bit = 31; bit >= 0; --bit) {
          const unsigned t = th | (1u << bit);
          int c = 0;
#pragma unroll
          for (int i = 0; i < G; ++i) c += __popcll(__ballot(gm[i] >= t));
          if (c >= a.k) { th = t; if (c == a.k) break; }
        }
        if (th) {
          const u64 t = ((u64)th << 32) - 1;
          if (t > cd.tkey) {
            cd.tkey = t;
            cd.tval = order_value(th == 0x80000000u ? th - 2 : th - 1);      // below +0 comes -0, which compares equal to it
          }
        }
      }
      // (the bound of the chunk's start: a cut in between raises tval to a value that elements of THIS chunk may share at a lower index)
      const float tval = cd.tval;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = v + u * 64 + lane;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const bool may = !(x[u * VEC + j] <= tval);
          if (__any(may)) {
            const bool in = cd.offer(make_key(x[u * VEC + j], (unsigned)(g.head + i * VEC + j)), may && i < v1);
            if (in) x[u * VEC + j] = -INFINITY;
          }
        }
      }
      // the exact border of what has been seen: later elements equal to it have higher indices and lose
      if (cd.cnt > cd.k && (v == v0 || cd.cnt > cd.k + KB / 2)) cd.cut();
      mx = x[0];
#pragma unroll
      for (int j = 1; j < 16; ++j) mx = fmaxf(mx, x[j]);
    }
    cd.others.add_max(x, mx, a.c);
  }
  if (s == a.S - 1 && g.tail) single(g.tail0() + lane, lane < g.tail);
  if (a.S == 1) {
    cd.finish([&](int rank, u64 key) { emit_row<E>(a, n, rank, key); });
    if (lane == 0) a.rest[n] = log_mass(cd.others, a.invT);
  } else {
    u64* o = a.keys + (n * a.S + s) * a.k;
    cd.finish([&](int rank, u64 key) { o[rank] = key; });
    for (int i = cd.cnt + lane; i < a.k; i += 64) o[i] = 0;
    if (lane == 0) a.sums[n * a.S + s] = make_float2(cd.others.m, cd.others.s);
  }
}

template <typename E, int KB> __global__ __launch_bounds__(64) void top_merge_kernel(TopArgs a) {
  __shared__ u64 buf[Candidates<KB>::CAP];
  const long n = blockIdx.x;
  const int lane = threadIdx.x, total = a.S * a.k;
  Candidates<KB> cd;
  cd.init(buf, a.k, a.c, lane);
  for (int i = lane; i < a.S; i += 64) {
    const float2 o = a.sums[n * a.S + i];
    cd.others.merge(o.x, o.y, a.c);
  }
  const u64* keys = a.keys + n * total;
  for (int i = 0; i < total; i += 64) {
    const bool has = i + lane < total;
    const u64 key = has ? keys[i + lane] : 0;
    const bool in = cd.offer(key, has && key);
    if (has && key && !in) cd.others.add1(order_value((unsigned)(key >> 32)), a.c);
  }
  cd.finish([&](int rank, u64 key) { emit_row<E>(a, n, rank, key); });
  if (lane == 0) a.rest[n] = log_mass(cd.others, a.invT);
}

// Segments per row: as many waves as keep every SIMD busy (16 per CU), but none shorter than four chunks -- each segment costs a
// threshold search and k keys of traffic.
static void top_split(int N, int V, int* S, int* seg) {
  const int cus = device_cus() > 0 ? device_cus() : 256;
  const int want = (16 * cus + N - 1) / N, most = (V + 4095) / 4096;
  int n = want < most ? want : most;
  if (n < 1) n = 1;
  *seg = ((V + n - 1) / n + 1023) / 1024 * 1024;
  *S = (V + *seg - 1) / *seg;
}

template <typename E, int KB> static int top_launch(const TopArgs& a, hipStream_t st) {
  VLN_LAUNCH((top_scan_kernel<E, KB>), dim3((unsigned)a.N, (unsigned)a.S), dim3(64), 0, st, a);
  if (a.S > 1) VLN_LAUNCH((top_merge_kernel<E, KB>), dim3((unsigned)a.N), dim3(64), 0, st, a);
  VLN_CHECK_LAUNCH("top_logits");
  return VLN_OK;
}
template <typename E> static int top_dispatch(const TopArgs& a, hipStream_t st) {
  if (a.k <= 64) return top_launch<E, 64>(a, st);
  if (a.k <= 128) return top_launch<E, 128>(a, st);
  return top_launch<E, 256>(a, st);
}

}  // namespace vln

extern "C" int64_t vln_top_logits_ws_bytes(int N, int V, int k) {
  if (N <= 0 || V <= 0 || k <= 0) return 0;
  int S, seg;
  vln::top_split(N, V, &S, &seg);
  return S > 1 ? (int64_t)N * S * ((int64_t)k * 8 + 8) : 0;
}
extern "C" int vln_top_logits(const void* logits, int64_t ld, int type, int N, int V, int k, float temperature, void* values, int64_t* ids,
                              float* rest, void* ws, int64_t ws_bytes, vln_stream_t s) {
  if (!logits || !values || !ids || !rest || N <= 0 || V <= 0 || ld < V) { vln::set_error("vln_top_logits: bad args"); return VLN_ERR_ARG; }
  if (k < 1 || k > V || k > VLN_TOP_LOGITS_MAX) { vln::set_error("vln_top_logits: k must be 1 .. min(V, %d)", VLN_TOP_LOGITS_MAX); return VLN_ERR_ARG; }
  if (!(temperature >= VLN_TEMPERATURE_MIN && temperature <= VLN_TEMPERATURE_MAX)) { vln::set_error("vln_top_logits: bad temperature"); return VLN_ERR_ARG; }
  vln::TopArgs a{};
  a.logits = logits; a.ld = ld; a.N = N; a.V = V; a.k = k;
  vln::top_split(N, V, &a.S, &a.seg);
  if (a.S > 1) {
    if (!ws || ws_bytes < vln_top_logits_ws_bytes(N, V, k)) { vln::set_error("vln_top_logits: workspace too small"); return VLN_ERR_ARG; }
    a.keys = static_cast<vln::u64*>(ws);
    a.sums = reinterpret_cast<float2*>(a.keys + (int64_t)N * a.S * k);
  }
  a.c = vln::kLog2e / temperature; a.invT = 1.f / temperature;
  a.values = values; a.ids = (long long*)ids; a.rest = rest;
  if (type == VLN_F32) return vln::top_dispatch<float>(a, (hipStream_t)s);
  if (type == VLN_BF16) return vln::top_dispatch<bf16_raw>(a, (hipStream_t)s);
  vln::set_error("vln_top_logits: type must be fp32 or bf16");
  return VLN_ERR_ARG;
}
