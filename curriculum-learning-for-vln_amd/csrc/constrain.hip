// Constraints on word logits before a word is drawn (vln_constrain_logits): penalties for words that stand in the history or the
// prompt, word biases, grammar masks.  include/vln_hip.h states the formula.
//
// Bound: bytes -- the row is read once and written once; everything per word is a handful of operations.  One workgroup takes one
// SEGMENT of a row's columns, up to VPT vectors of 16 bytes per thread:
//   1. the mask bits of the thread's vectors, then the vectors that are not banned altogether, all loads in flight before anything waits;
//   2. meanwhile how often each word of the segment stands in the history is counted into LDS (integer atomics: the order does not
//      matter), one 2-byte counter per column, and the segment's biases are collected and summed;
//   3. a vector's counters are one 16-byte LDS read: what nothing touches is copied (in place: left alone).
// Every segment reads the whole history (from L2), so segments are long unless there are too few rows to occupy the chip.
//
// Measured, us: 512 rows x 131072 bf16 54 (4.9 TB/s: the rate of a copy), with 4096 words of history per row 71, with grammar masks too 73,
// with 300 biases as well 80; in place 25 | 69 | 72 | 79.  What the lists add is latency: counting, a barrier, and the biases' gather, in
// workgroups of which four share a CU.  256 x 32001 bf16, 1024 words, masks and biases: 15.6; 1 x 992 fp32: 4.6, of which a launch is most.
// Four workgroups of 512 threads, 4 vectors each, are the best of the shapes tried (256 threads x 8 vectors: 94 us where this takes 84).
// New values scattered into the counters by the threads that hold the ids, so that the vectors need no arithmetic: 88 (a gather per word);
// workgroups that keep the ids and walk over a row's segments with the next one's loads in flight: 108 (128 registers, half the
// workgroups).  The result is stored through the caches: past them the kernel alone is faster (without lists 45 us), but whoever reads the
// logits next is slower by more (with vln_top_logits behind it 140 us, 134 like this).
#include "word_rows.h"
#include "../../include/vln_hip.h"

namespace vln {

constexpr int kCThreads = 512;
constexpr int kBiasMax = VLN_CONSTRAIN_MAX_BIAS;

struct ConstrainArgs {
  vln_constrain a;
  int seg_vecs;          // vectors of 16 bytes per segment, <= VPT x kCThreads
  int n_seg, xcds;       // xcds > 1: the segments of a row follow each other on one of `xcds` dies, whose L2 then serves the history
};

// a column's counter: times in the history | "in the prompt" in the top bit | "has a bias" in the next
template <typename CT> struct Counter {
  static constexpr unsigned kPrompt = 1u << (8 * sizeof(CT) - 1), kBias = kPrompt >> 1, kCount = kBias - 1;
  __device__ static __forceinline__ int shift(int i) { return sizeof(CT) == 2 ? (i & 1) * 16 : 0; }
  __device__ static __forceinline__ unsigned* word(unsigned* w, int i) { return &w[sizeof(CT) == 2 ? i >> 1 : i]; }
  __device__ static __forceinline__ void count(unsigned* w, int i) { atomicAdd(word(w, i), 1u << shift(i)); }
  __device__ static __forceinline__ bool flag(unsigned* w, int i, unsigned bit) { return (atomicOr(word(w, i), bit << shift(i)) >> shift(i)) & bit; }
  __device__ static __forceinline__ unsigned get(unsigned* w, int i) { return sizeof(CT) == 2 ? (*word(w, i) >> shift(i)) & 0xffffu : *word(w, i); }
};

struct Penalty { float r, ri, p, f; };      // ri: 1 / r

// x / r if z > 0, x * r otherwise.  The quotient is the product with 1 / r, corrected by its remainder: rounded like a division, at half
// its instructions (256 rows x 32001 bf16, 1024 words of history: 16.2 -> 15.6 us); r is a normal number.
__device__ __forceinline__ float repeated(float z, float x, const Penalty& q) {
  const float t = x * q.ri, e = fmaf(fmaf(-t, q.r, x), q.ri, t);
  return z > 0.f ? (fabsf(t) < INFINITY ? e : t) : x * q.r;
}
template <typename CT> __device__ __forceinline__ float penalised(float z, unsigned n, const Penalty& q) {
  typedef Counter<CT> Cn;
  if (n & (Cn::kPrompt | Cn::kCount)) z = repeated(z, z, q);
  const unsigned c = n & Cn::kCount;
  if (c) z -= q.f * (float)c + q.p;
  return z;
}

// E: logits; CT: counter; BWD: in = d out, out = d logits, `logits` = the forward's input (its sign decides the repetition factor)
template <typename E, typename CT, int VPT, bool BWD>
// (four workgroups per CU: 96 scalar registers, 64 vector registers)
__global__ __launch_bounds__(kCThreads, 4) __attribute__((amdgpu_num_sgpr(96))) void constrain_kernel(ConstrainArgs k) {
  extern __shared__ unsigned lds[];
  const vln_constrain& a = k.a;
  constexpr int VEC = RowGeo<E>::VEC;
  constexpr unsigned all = (1u << VEC) - 1u;
  typedef Counter<CT> Cn;
  const int turn = blockIdx.x / k.xcds, tid = threadIdx.x;
  const int b = turn / k.n_seg * k.xcds + blockIdx.x % k.xcds, seg = turn % k.n_seg;
  if (b >= a.B) return;
  const E* in = static_cast<const E*>(a.in) + (int64_t)b * a.ld_in;
  const E* zr = BWD ? static_cast<const E*>(a.logits) + (int64_t)b * a.ld_logits : in;
  E* out = static_cast<E*>(a.out) + (int64_t)b * a.ld_out;
  const RowGeo<E> g(in, a.V);
  const int v0 = min(g.nv, seg * k.seg_vecs), v1 = min(g.nv, v0 + k.seg_vecs);
  const bool in_place = !BWD && static_cast<const void*>(in) == static_cast<const void*>(out);
  // mask row: NULL = every word allowed; a row index outside [-1, G) bans every word (the grammar did not allow any)
  const unsigned* mk = nullptr;
  bool ban_all = false;
  if (a.allowed) {
    const long r = a.allowed_rows ? (long)a.allowed_rows[b] : (a.G == 1 ? 0L : (long)b);
    if (r >= 0 && r < a.G) mk = reinterpret_cast<const unsigned*>(a.allowed) + r * a.ld_allowed;
    else if (r != -1) ban_all = true;
  }
  const int last_word = (a.V - 1) >> 5;
  auto bits_at = [&](int c) -> unsigned {       // VEC mask bits of columns c .. c + VEC - 1
    if (ban_all) return 0u;
    if (!mk) return all;
    const int w = c >> 5, sh = c & 31;
    unsigned x = mk[w] >> sh;
    if (sh + VEC > 32 && w < last_word) x |= mk[w + 1] << (32 - sh);
    return x & all;
  };
  // Loads come back in order: the mask bits first, which say what logits are needed, then what the counting needs, then the logits.
  unsigned ok[VPT];
  uint4 raw[VPT];
#pragma unroll
  for (int u = 0; u < VPT; ++u) {
    const int i = v0 + u * kCThreads + tid;
    ok[u] = i < v1 ? bits_at(g.head + i * VEC) : 0u;
  }
  constexpr int HP = 8, PP = 2;
  const int64_t* prompt = a.prompt + (int64_t)b * a.ld_prompt;
  const int64_t* hist = a.history + (int64_t)b * a.ld_history;
  int64_t first_ids[HP];
#pragma unroll
  for (int t = 0; t < HP; ++t) first_ids[t] = t * kCThreads + tid < a.H ? hist[t * kCThreads + tid] : -1;
  int64_t prompt_ids[PP];
#pragma unroll
  for (int t = 0; t < PP; ++t) prompt_ids[t] = t * kCThreads + tid < a.P ? prompt[t * kCThreads + tid] : -1;
  int64_t bias_id = -1;
  float bias_val = 0.f;
  if (!BWD && tid < a.n_bias) {
    bias_id = a.bias_ids[(int64_t)b * a.ld_bias_ids + tid];
    bias_val = a.bias_values[(int64_t)b * a.ld_bias_values + tid];
  }
#pragma unroll
  for (int u = 0; u < VPT; ++u) {
    raw[u] = make_uint4(0, 0, 0, 0);
    if (ok[u] && !(in_place && ok[u] == all)) raw[u] = ld_vec<E>(in + g.head + (int64_t)(v0 + u * kCThreads + tid) * VEC);
  }

  // Counter slots: the segment's vectors in order, then (first segment only) the single columns of head and tail.
  const int nslot_v = k.seg_vecs * VEC, col0 = g.head + v0 * VEC, cols = (v1 - v0) * VEC;
  auto slot = [&](int64_t id) -> int {
    const int64_t i = id - col0;
    if (i >= 0 && i < cols) return (int)i;
    if (seg != 0) return -1;
    if (id >= 0 && id < g.head) return nslot_v + (int)id;
    if (id >= g.tail0() && id < a.V) return nslot_v + VEC + (int)(id - g.tail0());
    return -1;
  };
  const int nwords = ((nslot_v + 2 * VEC) * (int)sizeof(CT) + 15) / 16 * 4;
  for (int i = tid; i < nwords / 4; i += kCThreads) reinterpret_cast<uint4*>(lds)[i] = make_uint4(0, 0, 0, 0);
  __shared__ int n_here, n_twice;
  if (tid == 0) n_here = n_twice = 0;
  __syncthreads();
  auto length = [&](const int64_t* lens, int n) { return (int)(lens ? max((int64_t)0, min(lens[b], (int64_t)n)) : (int64_t)n); };
  const int hl = length(a.history_len, a.H);
#pragma unroll
  for (int t = 0; t < HP; ++t) {
    const int s = t * kCThreads + tid < hl ? slot(first_ids[t]) : -1;
    if (s >= 0) Cn::count(lds, s);
  }
  auto each = [&](const int64_t* row, int from, int len, auto&& f) {      // the ids that fall into this segment
    for (int64_t i = from + tid; i < len; i += 4 * kCThreads) {
      int64_t id[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) id[t] = i + t * kCThreads < len ? row[i + t * kCThreads] : -1;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int s = slot(id[t]);
        if (s >= 0) f(s);
      }
    }
  };
  each(hist, HP * kCThreads, hl, [&](int s) { Cn::count(lds, s); });
  if (a.P) {
    const int pl = length(a.prompt_len, a.P);
#pragma unroll
    for (int t = 0; t < PP; ++t) {
      const int s = t * kCThreads + tid < pl ? slot(prompt_ids[t]) : -1;
      if (s >= 0) Cn::flag(lds, s, Cn::kPrompt);
    }
    each(prompt, PP * kCThreads, pl, [&](int s) { Cn::flag(lds, s, Cn::kPrompt); });
  }
  // The segment's bias entries: slot, entry, value and the logit as it is before any of this row is written (in-place calls).
  int4* bias = reinterpret_cast<int4*>(lds + nwords);
  if (!BWD) {
    for (int j = tid; j < a.n_bias; j += kCThreads) {
      if (j != tid) {
        bias_id = a.bias_ids[(int64_t)b * a.ld_bias_ids + j];
        bias_val = a.bias_values[(int64_t)b * a.ld_bias_values + j];
      }
      const int s = slot(bias_id);
      if (s >= 0) {
        const float z = Elt<E>::ld(in + bias_id);
        const unsigned may = bits_at((int)bias_id) & 1u;                   // (a banned word's entry: slot with the top bit set)
        if (Cn::flag(lds, s, Cn::kBias)) n_twice = 1;
        bias[atomicAdd(&n_here, 1)] = make_int4(may ? s : s | (int)0x80000000, j, __float_as_int(bias_val), __float_as_int(z));
      }
    }
  }
  __syncthreads();

  Penalty q{a.repetition ? a.repetition[b] : a.repetition_all, 0.f, a.presence ? a.presence[b] : a.presence_all,
            a.frequency ? a.frequency[b] : a.frequency_all};
  q.ri = 1.f / q.r;
  // A word's biases are added up in entry order by its FIRST entry: the same bits whatever order the entries were collected in.
  constexpr int BPT = kBiasMax / kCThreads;
  int b_col[BPT];
  float b_out[BPT];
  const int nb = n_here;
  if (!BWD && nb) {
#pragma unroll
    for (int t = 0; t < BPT; ++t) {
      b_col[t] = -1;
      const int j = t * kCThreads + tid;
      if (j >= nb) continue;
      const int4 me = bias[j];
      float sum = __int_as_float(me.z);
      if (n_twice) {                              // some word of the segment has more than one entry
        int same = 0;
        bool first = true;
        for (int i = 0; i < nb; ++i) {
          const int2 o = *reinterpret_cast<const int2*>(&bias[i]);
          same += o.x == me.x ? 1 : 0;
          first = first && !(o.x == me.x && o.y < me.y);
        }
        if (!first) continue;
        for (int prev = me.y; --same > 0;) {
          int next = 0x7fffffff, at = 0;
          for (int i = 0; i < nb; ++i) if (bias[i].x == me.x && bias[i].y > prev && bias[i].y < next) { next = bias[i].y; at = i; }
          sum += __int_as_float(bias[at].z);
          prev = next;
        }
      }
      const int s = me.x & 0x7fffffff;
      b_col[t] = s < nslot_v ? col0 + s : (s < nslot_v + VEC ? s - nslot_v : g.tail0() + s - nslot_v - VEC);
      b_out[t] = penalised<CT>(__int_as_float(me.w), Cn::get(lds, s), q) + sum;
      if (me.x < 0) b_out[t] = -INFINITY;
    }
  }
  const float banned = BWD ? 0.f : -INFINITY;
  auto one = [&](float x, unsigned n, int c) -> float {          // one allowed column
    if (!BWD) return penalised<CT>(x, n, q);
    if (!(n & (Cn::kPrompt | Cn::kCount))) return x;
    return repeated(Elt<E>::ld(zr + c), x, q);
  };
  auto single = [&](int c, int s) {
    const bool may = bits_at(c) & 1u;
    Elt<E>::st(out + c, may ? one(Elt<E>::ld(in + c), Cn::get(lds, s), c) : banned);
  };
  if (seg == 0) {
    if (tid < g.head) single(tid, nslot_v + tid);
    else if (tid >= VEC && tid - VEC < g.tail) single(g.tail0() + tid - VEC, nslot_v + tid);
  }
  const bool vec_out = ((reinterpret_cast<uintptr_t>(in) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
#pragma unroll
  for (int u = 0; u < VPT; ++u) {
    const int i = v0 + u * kCThreads + tid;
    if (i >= v1) continue;
    const int c = g.head + i * VEC, s = (i - v0) * VEC;
    constexpr int CW = VEC * (int)sizeof(CT) / 4;      // counter words of a vector: 2 or 4 (u16), 4 or 8 (u32)
    unsigned cw[CW], any = 0;
#pragma unroll
    for (int w = 0; w < CW; ++w) { cw[w] = lds[s * (int)sizeof(CT) / 4 + w]; any |= cw[w]; }
    if (in_place && ok[u] == all) {
      if (!any) continue;
      raw[u] = ld_vec<E>(in + c);
    }
    float x[VEC];
    if (ok[u] != all || any) {
      unpack16<E>(raw[u], x);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const unsigned n = sizeof(CT) == 2 ? (cw[j / 2] >> ((j & 1) * 16)) & 0xffffu : cw[j * CW / VEC];
        x[j] = ((ok[u] >> j) & 1u) ? (n ? one(x[j], n, c + j) : x[j]) : banned;
      }
      raw[u] = pack16<E>(x);
    }
    if (vec_out) {
      st_vec<E>(out + c, raw[u]);
    } else {
      unpack16<E>(raw[u], x);
#pragma unroll
      for (int j = 0; j < VEC; ++j) Elt<E>::st(out + c + j, x[j]);
    }
  }
  if (BWD || !nb) return;
  __syncthreads();
#pragma unroll
  for (int t = 0; t < BPT; ++t) if (t * kCThreads + tid < nb && b_col[t] >= 0) Elt<E>::st(out + b_col[t], b_out[t]);
}

template <typename E, typename CT, int VPT> static int constrain_launch(const vln_constrain& a, hipStream_t st) {
  constexpr int VEC = Elt<E>::kVec;
  ConstrainArgs k;
  k.a = a;
  const int nv = (a.V + VEC - 1) / VEC;
  const int cus = device_cus() > 0 ? device_cus() : 256;
  int n_seg = (nv + VPT * kCThreads - 1) / (VPT * kCThreads);
  // two workgroups per CU, but at least a vector per thread (32 rows x 131072 bf16, 4096 words of history: 10.6 us; one: 12.4; four: 12.6)
  const int want = (2 * cus + a.B - 1) / a.B;
  const int finest = (nv + kCThreads - 1) / kCThreads;
  if (n_seg < want) n_seg = want < finest ? want : finest;
  const size_t lists = a.backward ? 0 : (size_t)a.n_bias * 16;
  const int fits = (int)((65536 - 64 - lists) / sizeof(CT)) / VEC - 2;      // 64 KB of LDS with the bias lists
  k.seg_vecs = (nv + n_seg - 1) / n_seg;
  if (k.seg_vecs > fits) k.seg_vecs = fits;
  k.n_seg = (nv + k.seg_vecs - 1) / k.seg_vecs;
  // Workgroups go to the 8 dies in turn.  With rows enough for all dies the segments of a row share one, and the history comes from memory
  // once (512 rows x 131072 bf16, 4096 words of history: 73 us; spread over all dies: 78; without a history 54 | 55).
  k.xcds = a.B >= 64 ? 8 : 1;
  const unsigned lds = (unsigned)(((k.seg_vecs * VEC + 2 * VEC) * sizeof(CT) + 15) / 16 * 16 + lists);
  const int64_t groups = ((int64_t)a.B + k.xcds - 1) / k.xcds * k.xcds * k.n_seg;
  if (!grid_fits(groups, kCThreads, 1)) { set_error("vln_constrain_logits: too many rows for one launch"); return VLN_ERR_ARG; }
  const dim3 grid((unsigned)groups);
  if (a.backward) VLN_LAUNCH((constrain_kernel<E, CT, VPT, true>), grid, dim3(kCThreads), lds, st, k);
  else VLN_LAUNCH((constrain_kernel<E, CT, VPT, false>), grid, dim3(kCThreads), lds, st, k);
  VLN_CHECK_LAUNCH("constrain_logits");
  return VLN_OK;
}

}  // namespace vln

extern "C" int vln_constrain_logits(const vln_constrain* p, vln_stream_t s) {
  if (!p) { vln::set_error("vln_constrain_logits: null pointer"); return VLN_ERR_ARG; }
  const vln_constrain& a = *p;
  if (a.B <= 0 || a.V <= 0 || a.H < 0 || a.P < 0 || a.n_bias < 0 || a.G < 0) { vln::set_error("vln_constrain_logits: bad sizes"); return VLN_ERR_ARG; }
  if (!a.in || !a.out || a.ld_in < a.V || a.ld_out < a.V) { vln::set_error("vln_constrain_logits: bad logits / out"); return VLN_ERR_ARG; }
  if (a.backward && (!a.logits || a.ld_logits < a.V)) { vln::set_error("vln_constrain_logits: the backward needs the forward's logits"); return VLN_ERR_ARG; }
  if ((a.H > 0 && !a.history) || (a.P > 0 && !a.prompt) || (a.n_bias > 0 && (!a.bias_ids || !a.bias_values))) {
    vln::set_error("vln_constrain_logits: a list without its pointer"); return VLN_ERR_ARG;
  }
  if (a.n_bias > vln::kBiasMax) { vln::set_error("vln_constrain_logits: at most %d biases per row", vln::kBiasMax); return VLN_ERR_ARG; }
  if (a.allowed && (a.G <= 0 || a.ld_allowed < (a.V + 31) / 32 || (!a.allowed_rows && a.G != 1 && a.G != a.B))) {
    vln::set_error("vln_constrain_logits: bad mask"); return VLN_ERR_ARG;
  }
  hipStream_t st = (hipStream_t)s;
  const bool small = a.H < 0x4000;          // 14 bits of count
  // (LDS of a segment: 32 KB of counters at most, and 16 bytes per bias of the row)
  if (a.type == VLN_F32) return small ? vln::constrain_launch<float, unsigned short, 4>(a, st) : vln::constrain_launch<float, unsigned, 4>(a, st);
  if (a.type == VLN_BF16) return small ? vln::constrain_launch<bf16_raw, unsigned short, 4>(a, st) : vln::constrain_launch<bf16_raw, unsigned, 2>(a, st);
  vln::set_error("vln_constrain_logits: type must be fp32 or bf16");
  return VLN_ERR_ARG;
}
