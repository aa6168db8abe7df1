// Constraints on word logits before a word is drawn (vln_constrain_logits): penalties for words that stand in the history or the
// prompt, word biases, grammar masks.  include/vln_hip.h states the formula.
//
// Bound: bytes -- the row is read once and written once; everything per word is a handful of operations.  One workgroup takes one
// SEGMENT of a row's columns.  How often each word of the segment stands in the history is counted into LDS (integer atomics: the
// order does not matter), one 2-byte counter per column, so the streaming loop tests 8 columns with one 16-byte LDS read and copies
// a vector that nothing touches.  A vector whose words are all banned is not even read, and an in-place call leaves an untouched
// vector alone.  Every segment reads the whole history (from L2), so segments are as long as the counters allow (kSegMax) unless
// there are too few rows to occupy the chip.
#include "word_rows.h"
#include "../../include/vln_hip.h"

namespace vln {

constexpr int kCThreads = 512;
constexpr int kSegMaxBytes = 32 * 1024;     // counters of a segment
constexpr int kBiasMax = VLN_CONSTRAIN_MAX_BIAS;

struct ConstrainArgs {
  vln_constrain a;
  int seg_vecs;          // vectors of 16 bytes per segment
  int n_seg;
};

template <typename CT> struct Counter;      // count | flag "in the prompt" in the top bit
template <> struct Counter<unsigned short> {
  static constexpr unsigned kFlag = 0x8000u;
  __device__ static __forceinline__ void count(unsigned* w, int i) { atomicAdd(&w[i >> 1], (i & 1) ? 0x10000u : 1u); }
  __device__ static __forceinline__ void flag(unsigned* w, int i) { atomicOr(&w[i >> 1], (i & 1) ? 0x80000000u : 0x8000u); }
  __device__ static __forceinline__ unsigned get(const unsigned* w, int i) { return (w[i >> 1] >> ((i & 1) * 16)) & 0xffffu; }
};
template <> struct Counter<unsigned> {
  static constexpr unsigned kFlag = 0x80000000u;
  __device__ static __forceinline__ void count(unsigned* w, int i) { atomicAdd(&w[i], 1u); }
  __device__ static __forceinline__ void flag(unsigned* w, int i) { atomicOr(&w[i], kFlag); }
  __device__ static __forceinline__ unsigned get(const unsigned* w, int i) { return w[i]; }
};

struct Penalty { float r, p, f; };

template <typename CT> __device__ __forceinline__ float penalised(float z, unsigned n, const Penalty& q) {
  if (n) z = z > 0.f ? z / q.r : z * q.r;
  const unsigned c = n & ~Counter<CT>::kFlag;
  if (c) z -= q.f * (float)c + q.p;
  return z;
}

// E: logits; CT: counter; BWD: in = d out, out = d logits, `logits` = the forward's input (its sign decides the repetition factor)
template <typename E, typename CT, bool BWD>
__global__ __launch_bounds__(kCThreads) void constrain_kernel(ConstrainArgs k) {
  extern __shared__ unsigned lds[];
  const vln_constrain& a = k.a;
  constexpr int VEC = RowGeo<E>::VEC;
  typedef Counter<CT> Cn;
  const int b = blockIdx.x, seg = blockIdx.y, tid = threadIdx.x;
  const E* in = static_cast<const E*>(a.in) + (int64_t)b * a.ld_in;
  const E* zr = BWD ? static_cast<const E*>(a.logits) + (int64_t)b * a.ld_logits : in;
  E* out = static_cast<E*>(a.out) + (int64_t)b * a.ld_out;
  const RowGeo<E> g(in, a.V);
  const int v0 = seg * k.seg_vecs, v1 = min(g.nv, v0 + k.seg_vecs);
  // Counter slots: the segment's vectors in order, then (first segment only) the single columns of head and tail.
  const int nslot_v = k.seg_vecs * VEC;
  auto slot = [&](long id) -> int {
    if (id < 0 || id >= a.V) return -1;
    const int c = (int)id;
    if (c < g.head) return seg == 0 ? nslot_v + c : -1;
    if (c >= g.tail0()) return seg == 0 ? nslot_v + VEC + (c - g.tail0()) : -1;
    const int i = c - g.head - v0 * VEC;
    return (i >= 0 && i < (v1 - v0) * VEC) ? i : -1;
  };
  const int nslots = nslot_v + 2 * VEC;
  const int nwords = (nslots * (int)sizeof(CT) + 15) / 16 * 4;
  for (int i = tid; i < nwords / 4; i += kCThreads) reinterpret_cast<uint4*>(lds)[i] = make_uint4(0, 0, 0, 0);
  __shared__ int n_here;
  if (tid == 0) n_here = 0;
  __syncthreads();
  const long hl = a.history ? (a.history_len ? min((long)a.history_len[b], (long)a.H) : (long)a.H) : 0;
  for (long i = tid; i < hl; i += kCThreads) {
    const int s = slot(a.history[(int64_t)b * a.ld_history + i]);
    if (s >= 0) Cn::count(lds, s);
  }
  const long pl = a.prompt ? (a.prompt_len ? min((long)a.prompt_len[b], (long)a.P) : (long)a.P) : 0;
  for (long i = tid; i < pl; i += kCThreads) {
    const int s = slot(a.prompt[(int64_t)b * a.ld_prompt + i]);
    if (s >= 0) Cn::flag(lds, s);
  }
  // The segment's bias entries: {slot, entry} pairs and the logit as it is before any of this row is written (in-place calls).
  int* b_slot = reinterpret_cast<int*>(lds + nwords);
  int* b_entry = b_slot + a.n_bias;
  float* b_z = reinterpret_cast<float*>(b_entry + a.n_bias);
  if (!BWD && a.n_bias) {
    for (int j = tid; j < a.n_bias; j += kCThreads) {
      const long id = a.bias_ids[(int64_t)b * a.ld_bias_ids + j];
      const int s = slot(id);
      if (s >= 0) {
        const int at = atomicAdd(&n_here, 1);
        b_slot[at] = s; b_entry[at] = j; b_z[at] = Elt<E>::ld(in + id);
      }
    }
  }
  __syncthreads();

  const Penalty q{a.repetition ? a.repetition[b] : a.repetition_all, a.presence ? a.presence[b] : a.presence_all,
                  a.frequency ? a.frequency[b] : a.frequency_all};
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
    constexpr unsigned all = (1u << VEC) - 1u;
    if (ban_all) return 0u;
    if (!mk) return all;
    const int w = c >> 5, sh = c & 31;
    unsigned x = mk[w] >> sh;
    if (sh + VEC > 32 && w < last_word) x |= mk[w + 1] << (32 - sh);
    return x & all;
  };
  const float banned = BWD ? 0.f : -INFINITY;
  auto one = [&](float x, unsigned n, int c) -> float {          // one allowed column
    if (!BWD) return penalised<CT>(x, n, q);
    if (!n) return x;
    return Elt<E>::ld(zr + c) > 0.f ? x / q.r : x * q.r;
  };
  auto single = [&](int c, int s) {
    const bool ok = bits_at(c) & 1u;
    Elt<E>::st(out + c, ok ? one(Elt<E>::ld(in + c), Cn::get(lds, s), c) : banned);
  };
  if (seg == 0) {
    if (tid < g.head) single(tid, nslot_v + tid);
    else if (tid >= VEC && tid - VEC < g.tail) single(g.tail0() + tid - VEC, nslot_v + tid);
  }
  const bool in_place = !BWD && static_cast<const void*>(in) == static_cast<const void*>(out);
  const bool vec_out = ((reinterpret_cast<uintptr_t>(in) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
  for (int i = v0 + tid; i < v1; i += kCThreads) {
    const int c = g.head + i * VEC, s = (i - v0) * VEC;
    constexpr int CW = VEC * (int)sizeof(CT) / 4;      // counter words of a vector: 2 or 4 (u16), 4 or 8 (u32)
    unsigned cw[CW], any = 0;
#pragma unroll
    for (int w = 0; w < CW; ++w) { cw[w] = lds[s * (int)sizeof(CT) / 4 + w]; any |= cw[w]; }
    const unsigned ok = bits_at(c);
    constexpr unsigned all = (1u << VEC) - 1u;
    if (in_place && ok == all && !any) continue;
    float x[VEC];
    uint4 raw = make_uint4(0, 0, 0, 0);
    if (ok) raw = ld_vec<E>(in + c);
    if (ok != all || any) {
      unpack16<E>(raw, x);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const unsigned n = sizeof(CT) == 2 ? (cw[j / 2] >> ((j & 1) * 16)) & 0xffffu : cw[j * CW / VEC];
        x[j] = ((ok >> j) & 1u) ? (n ? one(x[j], n, c + j) : x[j]) : banned;
      }
      raw = pack16<E>(x);
    }
    if (vec_out) {
      st_vec<E>(out + c, raw);
    } else {
      unpack16<E>(raw, x);
#pragma unroll
      for (int j = 0; j < VEC; ++j) Elt<E>::st(out + c + j, x[j]);
    }
  }
  if (BWD || !a.n_bias) return;
  __syncthreads();
  // A word's biases are added up in entry order by its FIRST entry: the same bits whatever order the entries were collected in.
  const int n = n_here;
  for (int j = tid; j < n; j += kCThreads) {
    const int s = b_slot[j], e = b_entry[j];
    bool first = true;
    for (int i = 0; i < n; ++i) first = first && !(b_slot[i] == s && b_entry[i] < e);
    if (!first) continue;
    float sum = 0.f;
    int prev = e - 1;
    while (true) {
      int next = 0x7fffffff;
      for (int i = 0; i < n; ++i) if (b_slot[i] == s && b_entry[i] > prev) next = min(next, b_entry[i]);
      if (next == 0x7fffffff) break;
      sum += a.bias_values[(int64_t)b * a.ld_bias_values + next];
      prev = next;
    }
    const int c = (int)a.bias_ids[(int64_t)b * a.ld_bias_ids + e];
    if (bits_at(c) & 1u) Elt<E>::st(out + c, penalised<CT>(b_z[j], Cn::get(lds, s), q) + sum);
  }
}

template <typename E, typename CT> static int constrain_launch(const vln_constrain& a, hipStream_t st) {
  constexpr int VEC = Elt<E>::kVec;
  ConstrainArgs k;
  k.a = a;
  const int nv = (a.V + VEC - 1) / VEC;
  const int cus = device_cus() > 0 ? device_cus() : 256;
  const int per_seg_max = kSegMaxBytes / (int)sizeof(CT) / VEC;             // vectors whose counters fit
  int n_seg = (nv + per_seg_max - 1) / per_seg_max;
  const int want = (2 * cus + a.B - 1) / a.B;                               // two workgroups per CU ...
  const int finest = (nv + kCThreads - 1) / kCThreads;                      // ... but at least a vector per thread
  if (n_seg < want) n_seg = want < finest ? want : finest;
  if (n_seg < 1) n_seg = 1;
  k.seg_vecs = (nv + n_seg - 1) / n_seg;
  if (k.seg_vecs < 1) k.seg_vecs = 1;
  k.n_seg = (nv + k.seg_vecs - 1) / k.seg_vecs;
  if (k.n_seg < 1) k.n_seg = 1;
  const int slots = k.seg_vecs * VEC + 2 * VEC;
  const unsigned lds = (unsigned)((slots * sizeof(CT) + 15) / 16 * 16 + (a.backward ? 0 : (size_t)a.n_bias * 12));
  const dim3 grid((unsigned)a.B, (unsigned)k.n_seg);
  if (a.backward) VLN_LAUNCH((constrain_kernel<E, CT, true>), grid, dim3(kCThreads), lds, st, k);
  else VLN_LAUNCH((constrain_kernel<E, CT, false>), grid, dim3(kCThreads), lds, st, k);
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
  const bool small = a.H < 0x8000;          // 15 bits of count
  if (a.type == VLN_F32) return small ? vln::constrain_launch<float, unsigned short>(a, st) : vln::constrain_launch<float, unsigned>(a, st);
  if (a.type == VLN_BF16) return small ? vln::constrain_launch<bf16_raw, unsigned short>(a, st) : vln::constrain_launch<bf16_raw, unsigned>(a, st);
  vln::set_error("vln_constrain_logits: type must be fp32 or bf16");
  return VLN_ERR_ARG;
}
