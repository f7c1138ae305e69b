// Losses over rows of a vocabulary softmax held in memory ([T][V] logits or log-probabilities, fp32 / bf16 / fp16), next to
// the NLL of a given text: per-token log-probability and entropy, distillation from a teacher's top logits, the clipped
// policy loss with a KL term, and the preference loss over pairs of answers, each with its gradient.
//
// With c = 1 / temperature, m = max_v z_v, s = sum_v exp(c (z_v - m)), p_v = exp(c (z_v - m)) / s:
//   log p_v = c (z_v - m) - ln s,   H = ln s - sum_v p_v c (z_v - m)
// and every gradient has the form  dz_v = e_v (a + b x_v) + [v in a short list] d_v,  x_v = c log2(e) (z_v - m), e_v = 2^x_v,
// with a, b and the list known once the row's statistics are.  All statistics, sums and coefficients are fp32 or fp64;
// only the gradient is rounded to the logits' type, once.
//
// Rows start at any element (an odd vocabulary puts every second row of a 16-bit type at an odd one), and are taken in 16-byte
// pieces from the first aligned one on (of the gradient's row where one is written); the up to N - 1 elements before it and
// behind the last piece go to one thread each.  gfx950 takes unaligned global accesses, so logits and gradient may be aligned
// differently; pieces at odd 2-byte addresses cost 15 to 18 % (V = 20003 against 20002, bf16).
#include "common.h"
#include "../../include/pevae_hip.h"

namespace {

constexpr int kTeacherMax = 256;        // teacher entries a row: four a lane of one wave
constexpr int kVocabMax = 1 << 24;      // indices of a row fit fp32 and int32 with room
constexpr long kRowsMax = (1L << 26) - 1;     // a wave a row: fewer than 2^32 threads a launch
constexpr long kPairsMax = (1L << 24) - 1;    // 256 threads a pair
constexpr float kFloorX = -2.0e4f;      // 2^kFloorX is 0: keeps 0 * (-inf) out of the entropy terms
constexpr float kDead = __builtin_inff();   // `m` of a row that is not computed (padding, empty teacher list)

enum { HEAD_TOKEN = 0, HEAD_POLICY = 1, HEAD_DISTILL = 2 };

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
struct __attribute__((packed, aligned(1))) piece_t { u32x4 v; };     // 16 bytes at any address
struct __attribute__((packed, aligned(1))) half_piece_t { uint32_t v[2]; };

// (a copy of the element: __builtin_bit_cast of an element of a vector register reads element 0)
__device__ __forceinline__ float as_float(uint32_t u) { return __builtin_bit_cast(float, u); }
__device__ __forceinline__ uint32_t as_uint(float f) { return __builtin_bit_cast(uint32_t, f); }

struct F32 {
  typedef float type;
  static constexpr int N = 4;              // elements of a piece
  static __device__ __forceinline__ u32x4 nothing() { return u32x4{0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u}; }
  static __device__ __forceinline__ float up(float x) { return x; }
  static __device__ __forceinline__ float down(float x) { return x; }
  static __device__ __forceinline__ void unpack(u32x4 r, float (&f)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = as_float(r[i]);
  }
  static __device__ __forceinline__ u32x4 pack(const float (&f)[4]) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = as_uint(f[i]);
    return r;
  }
};
struct BF16 {
  typedef bf16_t type;
  static constexpr int N = 8;
  static __device__ __forceinline__ u32x4 nothing() { return u32x4{0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u}; }
  static __device__ __forceinline__ float up(bf16_t x) { return bf2f(x); }
  static __device__ __forceinline__ bf16_t down(float x) { return f2bf(x); }
  static __device__ __forceinline__ void unpack(u32x4 r, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = as_float(r[i] << 16);
      f[2 * i + 1] = as_float(r[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ u32x4 pack(const float (&f)[8]) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = pack2bf(f[2 * i], f[2 * i + 1]);
    return r;
  }
};
struct F16 {
  typedef uint16_t type;
  static constexpr int N = 8;
  static __device__ __forceinline__ u32x4 nothing() { return u32x4{0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u}; }
  static __device__ __forceinline__ float up(uint16_t x) { return (float)__builtin_bit_cast(_Float16, x); }
  static __device__ __forceinline__ uint16_t down(float x) { return __builtin_bit_cast(uint16_t, (_Float16)x); }
  static __device__ __forceinline__ void unpack(u32x4 r, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = up((uint16_t)(r[i] & 0xffffu));
      f[2 * i + 1] = up((uint16_t)(r[i] >> 16));
    }
  }
  static __device__ __forceinline__ u32x4 pack(const float (&f)[8]) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = (uint32_t)down(f[2 * i]) | ((uint32_t)down(f[2 * i + 1]) << 16);
    return r;
  }
};

// the compiler forgets what it has unpacked from a piece: the packed form is what stays in registers
__device__ __forceinline__ void keep_packed(u32x4& r) { asm volatile("" : "+v"(r)); }
__device__ __forceinline__ u32x4 load_piece(const void* p) { return ((const piece_t*)p)->v; }
__device__ __forceinline__ void store_piece(void* p, u32x4 v) { ((piece_t*)p)->v = v; }
// how a row of V elements at `p` splits: `head` elements, `full` pieces, then the rest; the element of thread tid outside the
// pieces, or V where it has none
template <class E>
struct Split {
  int head, full;
  __device__ __forceinline__ Split(const void* p, int V) {
    head = (int)((16 - ((uintptr_t)p & 15)) & 15) / (int)sizeof(typename E::type);
    head = head < V ? head : V;
    full = (V - head) / E::N;
  }
  __device__ __forceinline__ int edge(int tid, int V) const {
    const int v = tid < head ? tid : tid + full * E::N;
    return v < V ? v : V;
  }
};
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor(x, o));
  return x;
}
__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
  return x;
}
__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
  return x;
}

// Softmax statistics of a part of a row: maximum, sum of e = 2^x, sum of e x (x in units of log2).  An empty part is
// {-inf, 0, 0}; a NaN among the elements makes s NaN (fmaxf alone would drop it).
struct Stat {
  float m, s, ex;
};
__device__ __forceinline__ float finite_max(float m) { return m == -__builtin_inff() ? 0.f : m; }
// the part seen from the maximum mm >= st.m (finite, or +inf / NaN that the result carries on)
__device__ __forceinline__ void rebase(Stat& st, float mm, float k) {
  const float d = (st.m - mm) * k, f = exp2_(d);
  st.ex = (st.ex + st.s * fmaxf(d, kFloorX)) * f;
  st.s *= f;
}
__device__ __forceinline__ Stat wave_stat(Stat st, float k) {
  const float m = wave_max(st.m);
  rebase(st, finite_max(m), k);
  return {m, wave_sum(st.s), wave_sum(st.ex)};
}

// e (a + b x) for w = {m, a, b, -}; B: b may differ from 0
template <bool B>
__device__ __forceinline__ float slope(float z, const float4& w, float k) {
  const float x = (z - w.x) * k, e = exp2_(x);
  return B ? e * (w.y + w.z * fmaxf(x, kFloorX)) : e * w.y;
}
// the N values of a piece of the input as elements of the output type O
template <class E, class O>
__device__ __forceinline__ void store_values(typename O::type* p, const float (&z)[E::N]) {
  if constexpr (E::N == O::N) {
    store_piece(p, O::pack(z));
  } else {                                         // four fp32 values to four bf16 ones
    half_piece_t h = {{pack2bf(z[0], z[1]), pack2bf(z[2], z[3])}};
    *(half_piece_t*)p = h;
  }
}
template <class E, class O>
__device__ __forceinline__ void store_zeros(typename O::type* p) {
  const float z[E::N] = {};
  store_values<E, O>(p, z);
}
// the gradient of one piece of a row whose first word is v, to out; y: the word that gets d on top (none: negative)
template <class E, class O, bool B>
__device__ __forceinline__ void slope_piece(typename O::type* out, u32x4 raw, int v, const float4& w, float k, int y, float d) {
  float z[E::N];
  E::unpack(raw, z);
#pragma unroll
  for (int n = 0; n < E::N; ++n) z[n] = slope<B>(z[n], w, k);
  if ((unsigned)(y - v) < (unsigned)E::N) {        // one piece of the row
#pragma unroll
    for (int n = 0; n < E::N; ++n) z[n] += v + n == y ? d : 0.f;
  }
  store_values<E, O>(out + v, z);
}

// x - ln(s) to about half a unit of the result: ln s = n ln2 + ln f with the two halves of ln2 kept apart, the rounding of
// the first difference carried into the second.
__device__ __forceinline__ float minus_log(float x, float s) {
  if (!(fabsf(x) < __builtin_inff()) || !(s > 0.f && s < __builtin_inff())) return x - logf(s);
  int n;
  float f = frexpf(s, &n);
  if (f < 0.70710678f) {
    f *= 2.f;
    n -= 1;
  }
  const float hi = (float)n * 0.693145751953125f;                  // 16 bits of ln2: exact times n
  const float lo = (float)n * 1.42860682e-6f + logf(f);
  const float t = x - hi, bb = t - x;
  const float err = (x - (t - bb)) + (-hi - bb);
  return t + (err - lo);
}
// e^d - 1 - d; its leading terms cancel for small d
__device__ __forceinline__ float exp_minus_1_minus(float d, float em1) {
  if (fabsf(d) >= 0.25f) return em1 - d;
  return d * d * (0.5f + d * (1.f / 6 + d * (1.f / 24 + d * (1.f / 120 + d * (1.f / 720 + d * (1.f / 5040))))));
}

// ---- arguments ---------------------------------------------------------------------------------------------------------
struct Rows {
  const void* logits;
  int n1, V;                 // row t = (t / n1, t % n1)
  long T, s0, s1;            // element strides of the two row indices
  float c, k;                // 1 / temperature, c * log2(e)
  const int64_t* labels;     // NULL: every row is live and there is no label
  int64_t ignore;
  const int64_t* perm;       // rows_once_kernel: row t of the logits is row perm[t] of everything else (NULL: t)
};
struct Policy {
  const float *old_lp, *ref_lp, *adv;      // ref_lp NULL: no KL term; adv [T] or [T / n1]
  int adv_per_row;
  float lo, hi, kl, ent;
};
struct Distill {
  const int64_t* ids;        // [T][K]
  const void* t_logits;      // [T][K]
  int K, dtype;
  float* psum;               // [T][K]: the teacher's probability of the entry's word, duplicates added up; -1: nothing to add
  float c, k;                // 1 / temperature of the loss and of the teacher, c * log2(e)
};
struct Scale {
  float weight;              // of the loss, divided by *count where count != NULL (at least 1)
  const float* count;
  __device__ __forceinline__ float get() const { return count ? weight / fmaxf(*count, 1.f) : weight; }
};

__device__ __forceinline__ uint32_t sequence_of(const Rows& a, long t) { return (uint32_t)t / (uint32_t)a.n1; }  // t < 2^31
template <class E>
__device__ __forceinline__ const typename E::type* row_of(const Rows& a, long t) {
  const uint32_t i = sequence_of(a, t), j = (uint32_t)t - i * (uint32_t)a.n1;
  return (const typename E::type*)a.logits + i * a.s0 + j * a.s1;
}

// what a row's loss needs besides its logits, asked for before the row itself: its latency passes behind the row's
struct RowIn {
  float old_lp, ref_lp, adv, scale;
};
template <int HEAD>
__device__ __forceinline__ RowIn load_row_in(const Rows& a, const Policy& h, const Scale& sc, long t) {
  if (HEAD == HEAD_TOKEN) return {0.f, 0.f, 0.f, 0.f};
  if (HEAD == HEAD_DISTILL) return {0.f, 0.f, 0.f, sc.get()};
  return {h.old_lp[t], h.ref_lp ? h.ref_lp[t] : 0.f, h.adv[h.adv_per_row ? t : (long)sequence_of(a, t)], sc.get()};
}
struct PolicyTerm {
  float pg, k3, cut, dlp;
};
// -min(r A, clip(r) A) with r = exp(lp - old), and kl times the estimate e^d - 1 - d, d = ref - lp, of the divergence
__device__ __forceinline__ PolicyTerm policy_term(const Policy& h, float lp, float old_lp, float ref_lp, float A) {
  const float r = expf(lp - old_lp);
  float u = r * A, w = fminf(fmaxf(r, h.lo), h.hi) * A;
  if (A == 0.f && r == r) u = w = 0.f;            // r may be infinite; a NaN stays
  PolicyTerm o;
  const bool cut = u > w;
  o.cut = cut ? 1.f : 0.f;
  o.pg = cut ? -w : -u;
  o.dlp = cut ? 0.f : -u;
  o.k3 = 0.f;
  if (h.ref_lp) {
    const float d = ref_lp - lp, em1 = expm1f(d);
    o.k3 = exp_minus_1_minus(d, em1);
    if (h.kl != 0.f) o.dlp -= h.kl * em1;         // (em1 may be infinite)
  }
  return o;
}

// The teacher's side of a row, by one wave: its softmax over the K entries (those of -inf do not count), the sum of
// p (log p - c (z - zref)) over the entries, and for each entry the probability of its word (duplicate words added up).
// empty: no entry counts.  bad: an entry that counts names a word outside the vocabulary.
// Its loads are asked for before the row's own (behind them they would arrive last, and the words' logits a latency later), and
// the words' logits are kept for the end of the row: V = 5003, bf16, K = 64, 20000 rows: 102 us, 122 without either and with a sum
// over the list for every entry of it.
struct Teacher {
  float acc, zref;
  bool empty, bad;
};
struct TeacherList {         // of a row, in shared memory
  int id[kTeacherMax];       // -1: no word of the vocabulary, or nothing to add to it
  float p[kTeacherMax], z[kTeacherMax], psum[kTeacherMax];     // of an entry: probability, its word's logit and probability
};
struct TeacherIn {           // an entry as it stands in memory
  uint32_t x;
  int64_t id;
};
__device__ __forceinline__ TeacherIn load_teacher(const Distill& h, long t, int j) {
  if (j >= h.K) return {0u, -1};
  const long at = t * h.K + j;
  return {h.dtype == PV_DTYPE_F32 ? ((const uint32_t*)h.t_logits)[at] : ((const uint16_t*)h.t_logits)[at], h.ids[at]};
}
__device__ __forceinline__ float teacher_value(const Distill& h, uint32_t x) {
  if (h.dtype == PV_DTYPE_F32) return as_float(x);
  return h.dtype == PV_DTYPE_BF16 ? bf2f((uint16_t)x) : F16::up((uint16_t)x);
}

// The smallest x ^ y over the lanes that lie FROM to TO places further round in each row of 16: 0 where two ids are equal.
template <int FROM, int TO>
__device__ __forceinline__ uint32_t meet(int x, int y) {
  uint32_t t = x ^ __builtin_amdgcn_update_dpp(0, y, 0x120 + FROM, 0xf, 0xf, true);      // row_ror
  if constexpr (FROM < TO) t = min(t, meet<FROM + 1, TO>(x, y));
  return t;
}
// Whether two of the first K <= 64 lanes hold the same id >= 0: all pairs, each in one direction or the other of the 8 nearest
// places of a row of 16 lanes, rows against each other the same way.  Lists without a word twice are the rule, and a sum over
// the list for every entry of it took 18 of 132 us at V = 1009, bf16, K = 64, 60000 rows.
__device__ __forceinline__ bool duplicates(int id, int lane, int K) {
  const int x = id >= 0 ? id : -1 - lane;
  uint32_t t = meet<1, 8>(x, x);
#pragma unroll
  for (int o = 16; o < 64; o += 16) {
    if (K <= (o < 32 ? 16 : 32)) break;
    const int y = __shfl_xor(x, o);
    t = min(t, min((uint32_t)(x ^ y), meet<1, 8>(x, y)));
  }
  return __ballot(t == 0) != 0;
}

// The same for longer lists, in shared memory: every entry writes its place into a table at its id's hash; one that finds
// another's place there either holds the same id or tries again with another hash.  Every round ends with fewer entries.
// (V = 5003, bf16, K = 200, 20000 rows: 155 us, with the sum for every entry 366.)
__device__ __forceinline__ bool duplicates(TeacherList& l, int lane, int K) {
  uint8_t* table = (uint8_t*)l.psum;               // 1024 places; kTeacherMax entries fit a byte
  uint32_t factor = 0x9e3779b1u;
  int todo = 0;                                    // entries lane, lane + 64, ...: a bit each
  for (int j = lane; j < K; j += 64) todo |= l.id[j] >= 0 ? 1 << (j >> 6) : 0;
  bool found = false;
  while (__ballot(todo != 0) && !__ballot(found)) {
    for (int j = lane; j < K; j += 64)
      if (todo >> (j >> 6) & 1) table[(uint32_t)l.id[j] * factor >> 22] = (uint8_t)j;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    for (int j = lane; j < K; j += 64)
      if (todo >> (j >> 6) & 1) {
        const int w = table[(uint32_t)l.id[j] * factor >> 22];
        if (w != j && l.id[w] == l.id[j]) found = true;
        if (w == j) todo &= ~(1 << (j >> 6));
      }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    factor += 0x3c6ef372u;                         // stays odd
  }
  return __ballot(found) != 0;
}

// in: entry `lane`
template <class E>
__device__ __forceinline__ Teacher teacher_row(const Rows& a, const Distill& h, long t, const typename E::type* row, int lane,
                                               TeacherIn in, TeacherList& l) {
  float mx = -__builtin_inff(), nan = 0.f;         // fmaxf drops a NaN: the sum keeps it
  for (int j = lane; j < h.K; j += 64) {
    if (j >= 64) in = load_teacher(h, t, j);
    const int id = in.id >= 0 && in.id < a.V ? (int)in.id : -1;
    const float x = teacher_value(h, in.x);
    l.z[j] = id >= 0 ? E::up(row[id]) : 0.f;
    l.id[j] = id;
    l.p[j] = x;
    mx = fmaxf(mx, x);
    nan += x != x ? x : 0.f;
  }
  mx = wave_max(mx) + wave_sum(nan);
  Teacher r;
  r.empty = mx == -__builtin_inff();
  float sum = 0.f, zr = -__builtin_inff(), bad = 0.f;
  for (int j = lane; j < h.K; j += 64) {
    const float x = l.p[j], p = x == -__builtin_inff() ? 0.f : exp2_((x - mx) * h.k);
    sum += p;
    if (p > 0.f) {
      if (l.id[j] < 0)
        bad = 1.f;
      else
        zr = fmaxf(zr, l.z[j]);
    }
  }
  sum = wave_sum(sum);
  r.bad = wave_sum(bad) > 0.f || sum != sum;       // (a NaN or +inf among the teacher's logits)
  r.zref = finite_max(wave_max(zr));
  const float inv = r.empty ? 0.f : 1.f / sum;
  float acc = 0.f;
  int id = -1;
  for (int j = lane; j < h.K; j += 64) {
    const float x = l.p[j], p = x == -__builtin_inff() ? 0.f : exp2_((x - mx) * h.k) * inv;
    id = p == 0.f ? -1 : l.id[j];
    if (p > 0.f && id >= 0) acc += p * (minus_log((x - mx) * h.c, sum) - a.c * (l.z[j] - r.zref));
    l.id[j] = id;
    l.p[j] = p;
  }
  r.acc = wave_sum(acc);
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");       // the lanes read each other's entries
  const bool twice = h.K > 64 ? duplicates(l, lane, h.K) : duplicates(id, lane, h.K);
  for (int j = lane; j < h.K; j += 64) {
    float ps = l.p[j];
    if (twice) {
      ps = 0.f;
      for (int q = 0; q < h.K; ++q) ps += l.id[q] == l.id[j] ? l.p[q] : 0.f;
    }
    l.psum[j] = ps;
    h.psum[t * h.K + j] = l.id[j] >= 0 ? ps : -1.f;
  }
  return r;
}

// ---- forward: statistics and losses of a row, one workgroup each ---------------------------------------------------------
struct FwdOut {
  float *logp, *ent;         // HEAD_TOKEN
  float4* rowout;            // HEAD_POLICY {pg, k3, cut, H}, HEAD_DISTILL {loss, -, -, -} of the row, unscaled
  float4* save;              // what the gradient pass starts from: HEAD_TOKEN {m, 1/s, ex/s, -}, else {m, a, b, d}
};

// running statistics of a thread over n elements held in registers (-inf where there is none)
template <int N, bool ENT>
__device__ __forceinline__ void accumulate(Stat& st, const float (&z)[N], float k) {
  float mb = z[0];
#pragma unroll
  for (int i = 1; i < N; ++i) mb = fmaxf(mb, z[i]);
  const float m = fmaxf(st.m, mb), mm = finite_max(m);
  const float d = (st.m - mm) * k, f = exp2_(d);
  float s = st.s * f, ex = ENT ? (st.ex + st.s * fmaxf(d, kFloorX)) * f : 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float x = (z[i] - mm) * k, e = exp2_(x);
    s += e;
    if (ENT) ex += e * fmaxf(x, kFloorX);
  }
  st = {m, s, ex};
}

// the row's loss terms (stored by one thread, where `first`) and {m, a, b, d}, the coefficients of its gradient
template <int HEAD>
__device__ __forceinline__ float4 finish_row(const Rows& a, const Policy& hp, float tau, const RowIn& in, const Teacher& te, const FwdOut& o,
                                             long t, Stat st, float zy, bool bad, bool first) {
  const float nan = __builtin_nanf("");
  const float inv = 1.f / st.s, ln2 = 0.69314718056f;
  if (st.m == kDead) st.m = nan;                   // a logit of +inf: no distribution
  if (HEAD == HEAD_TOKEN) {
    if (first) {
      o.logp[t] = bad ? nan : minus_log((zy - st.m) * a.c, st.s);
      if (o.ent) o.ent[t] = -minus_log(st.ex * inv * ln2, st.s);
    }
    return make_float4(bad ? nan : st.m, inv, st.ex * inv, 0.f);
  } else if (HEAD == HEAD_POLICY) {
    const float lp = bad ? nan : minus_log((zy - st.m) * a.c, st.s);
    const float H = -minus_log(st.ex * inv * ln2, st.s);
    const PolicyTerm q = policy_term(hp, lp, in.old_lp, in.ref_lp, in.adv);
    if (first) o.rowout[t] = make_float4(q.pg, q.k3, q.cut, H);
    // d(loss)/d(log p[y]) = g, d(loss)/dH = h: dz_v = c (g [v = y] - p_v (g + h (log p_v + H)))
    const float w = in.scale, g = w * q.dlp, h = -w * hp.ent;
    return make_float4(st.m, -a.c * inv * (g - h * ln2 * st.ex * inv), -a.c * inv * h * ln2, a.c * g);
  } else {
    if (first) {
      const float loss = te.bad ? nan : te.acc + (a.c * (st.m - te.zref) - minus_log(0.f, st.s));
      o.rowout[t] = make_float4(te.empty ? 0.f : tau * tau * loss, 0.f, 0.f, 0.f);
    }
    const float w = in.scale * tau * tau * a.c;
    return make_float4(te.empty ? kDead : st.m, te.bad ? nan : w * inv, 0.f, -w);
  }
}

// A row belongs to NT threads: a workgroup, or (NT = 64) one of the four waves of a workgroup, since launching a workgroup for
// every short row costs more than the row (V = 1009, bf16: 1.3 ns a row).
template <int NT>
struct Place {
  static constexpr int R = NT == 64 ? 4 : 1, W = NT / 64;       // rows of a workgroup, waves of a row
  static_assert((W & (W - 1)) == 0, "waves are joined by halving");
  static __device__ __forceinline__ long row() { return blockIdx.x * (long)R + (R > 1 ? threadIdx.x >> 6 : 0); }
  static __device__ __forceinline__ int slot() { return R > 1 ? threadIdx.x >> 6 : 0; }
  static __device__ __forceinline__ int tid() { return threadIdx.x & (NT - 1); }
  static __device__ __forceinline__ void sync() {
    if (W > 1)
      __syncthreads();
    else
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  // the row's statistics for all its threads, from those of the threads
  template <bool ENT>
  static __device__ __forceinline__ Stat join(Stat st, float k, Stat (*part)[W]) {
    st = wave_stat(st, k);
    if (W == 1) return st;
    if ((tid() & 63) == 0) part[0][tid() >> 6] = st;
    sync();
    st = part[0][threadIdx.x & (W - 1)];           // every group of W lanes holds all waves' parts
    float m = st.m;
#pragma unroll
    for (int i = W / 2; i > 0; i >>= 1) m = fmaxf(m, __shfl_xor(m, i));
    rebase(st, finite_max(m), k);
#pragma unroll
    for (int i = W / 2; i > 0; i >>= 1) {
      st.s += __shfl_xor(st.s, i);
      if (ENT) st.ex += __shfl_xor(st.ex, i);
    }
    st.m = m;
    return st;
  }
};

template <int HEAD>
__device__ __forceinline__ void dead_row(const FwdOut& o, long t) {
  if (HEAD == HEAD_TOKEN) {
    o.logp[t] = 0.f;
    if (o.ent) o.ent[t] = 0.f;
  } else {
    o.rowout[t] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  if (o.save) o.save[t] = make_float4(kDead, 0.f, 0.f, 0.f);
}

// running statistics of a thread over the pieces first, first + step, ... below end of a row, four in flight
template <class E, bool ENT>
__device__ __forceinline__ void sweep_pieces(Stat& st, const typename E::type* row, int first, int step, int end, float k) {
  for (int c = first; c < end; c += 4 * step) {
    u32x4 raw[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) raw[i] = c + i * step < end ? load_piece(row + (long)(c + i * step) * E::N) : E::nothing();
#pragma unroll
    for (int i = 0; i < 4; i += 2)
      if (c + i * step < end) {                    // two pieces: the maximum moves, and the sums are rescaled, once for both
        float f[E::N], z[2 * E::N];
        E::unpack(raw[i], f);
#pragma unroll
        for (int n = 0; n < E::N; ++n) z[n] = f[n];
        E::unpack(raw[i + 1], f);
#pragma unroll
        for (int n = 0; n < E::N; ++n) z[E::N + n] = f[n];
        accumulate<2 * E::N, ENT>(st, z, k);
      }
  }
}

template <class E, int HEAD, bool ENT, int NT>
__device__ __forceinline__ void forward_row(const Rows& a, const Policy& hp, const Distill& hd, const Scale& sc, const FwdOut& o,
                                            long t) {
  typedef Place<NT> P;
  const int tid = P::tid();
  const int64_t y = a.labels ? a.labels[t] : -1;
  if (a.labels && y == a.ignore) {
    if (tid == 0) dead_row<HEAD>(o, t);
    return;
  }
  const RowIn in = load_row_in<HEAD>(a, hp, sc, t);
  const typename E::type* row = row_of<E>(a, t);
  TeacherIn ti = {0u, -1};
  if (HEAD == HEAD_DISTILL && tid < 64) ti = load_teacher(hd, t, tid);
  const bool bad = HEAD != HEAD_DISTILL && (y < 0 || y >= a.V);
  const float zy = HEAD != HEAD_DISTILL && !bad ? E::up(row[y]) : 0.f;
  Teacher te = {0.f, 0.f, false, false};
  __shared__ TeacherList list[HEAD == HEAD_DISTILL ? P::R : 1];
  __shared__ Stat part[1][P::W];
  if (HEAD == HEAD_DISTILL && tid < 64) te = teacher_row<E>(a, hd, t, row, tid, ti, list[P::slot()]);
  Stat st = {-__builtin_inff(), 0.f, 0.f};
  const Split<E> sp(row, a.V);
  sweep_pieces<E, ENT>(st, row + sp.head, tid, NT, sp.full, a.k);
  const int rest = sp.edge(tid, a.V);
  if (rest < a.V) {
    const float z[1] = {E::up(row[rest])};
    accumulate<1, ENT>(st, z, a.k);
  }
  st = P::template join<ENT>(st, a.k, part);
  if (tid == 0) {
    const float4 w = finish_row<HEAD>(a, hp, 1.f / hd.c, in, te, o, t, st, zy, bad, true);
    if (o.save) o.save[t] = w;
  }
}
template <class E, int HEAD, bool ENT, int NT>
__global__ __launch_bounds__(NT == 64 ? 256 : NT) void rows_fwd_kernel(Rows a, Policy hp, Distill hd, Scale sc, FwdOut o) {
  const long t = Place<NT>::row();
  if (t < a.T) forward_row<E, HEAD, ENT, NT>(a, hp, hd, sc, o, t);
}
// the rows of two tensors of one type and vocabulary, one after the other: neither waits for the other's last rows (64 x 50 and
// 64 x 43 rows of V = 20004, bf16, half of them dead: 42 us in one launch, 26 + 22 in two; their gradients 72 us, 2 x 38)
template <class E, int NT>
__global__ __launch_bounds__(NT == 64 ? 256 : NT) void rows_fwd_pair_kernel(Rows a, Rows b, FwdOut oa, FwdOut ob) {
  const long t = Place<NT>::row();
  if (__builtin_amdgcn_readfirstlane(t < a.T))     // a wave has one row
    forward_row<E, HEAD_TOKEN, false, NT>(a, Policy{}, Distill{}, Scale{}, oa, t);
  else if (t - a.T < b.T)
    forward_row<E, HEAD_TOKEN, false, NT>(b, Policy{}, Distill{}, Scale{}, ob, t - a.T);
}

template <class E, class O, bool B, int NT, int CH>
__device__ __forceinline__ void write_once(u32x4 (&raw)[CH], typename O::type* out, int tid, const Split<E>& sp,
                                           const float4& w, float k, int y, float d) {
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int c = tid + i * NT;
    keep_packed(raw[i]);
    if (c < sp.full) slope_piece<E, O, B>(out, raw[i], sp.head + c * E::N, w, k, y, d);
  }
}
template <class E, class O>
__device__ __forceinline__ void zero_row(typename O::type* out, int tid, int step, const Split<E>& sp, int V) {
  for (int i = tid; i < sp.full; i += step) store_zeros<E, O>(out + sp.head + (long)i * E::N);
  const int rest = sp.edge(tid, V);
  if (rest < V) out[rest] = O::down(0.f);
}

// Loss and gradient of a row in one pass: the row stays in its threads' registers (CH pieces each) between its statistics and
// its gradient, so that it is read once and its gradient written once; a forward and a backward pass over memory would read it
// twice.  Each thread runs its own maximum and sums while its pieces arrive; one exchange through shared memory gives every
// wave the row's.  WAVES a SIMD bound the registers so that a CU holds several rows: while one waits for memory another one
// computes.
// The gradient has the logits' type E, or is bf16 for fp32 logits: the operand of the products behind a projection, whose rows
// are ldg elements apart with zeros behind the V words.
template <class E, class O, int HEAD, int NT, int CH, int WAVES>
__global__ __launch_bounds__(NT == 64 ? 256 : NT, WAVES) void rows_once_kernel(Rows a, Policy hp, Distill hd, Scale sc, FwdOut o,
                                                                           typename O::type* __restrict__ grad, long ldg) {
  typedef Place<NT> P;
  const long t = P::row();
  const int tid = P::tid();
  if (P::R > 1 && t >= a.T) return;
  typename O::type* out = grad + t * ldg;
  const Split<E> sp(E::N == O::N ? (const void*)out : (const void*)row_of<E>(a, t), a.V);
  const int full = sp.full, rest = sp.edge(tid, a.V);
  if (E::N != O::N && a.V + tid < ldg) out[a.V + tid] = O::down(0.f);      // fewer than 64 words
  const long src = a.perm ? a.perm[t] : t;
  const int64_t y = a.labels ? a.labels[src] : -1;
  if (a.labels && y == a.ignore) {
    zero_row<E, O>(out, tid, NT, sp, a.V);
    if (tid == 0) dead_row<HEAD>(o, t);
    return;
  }
  const RowIn in = load_row_in<HEAD>(a, hp, sc, src);
  TeacherIn ti = {0u, -1};
  if (HEAD == HEAD_DISTILL && tid < 64) ti = load_teacher(hd, src, tid);
  const typename E::type* row = row_of<E>(a, t);
  u32x4 raw[CH];
#pragma unroll
  for (int i = 0; i < CH; ++i)
    raw[i] = tid + i * NT < full ? load_piece(row + sp.head + (long)(tid + i * NT) * E::N) : E::nothing();
  const float zr = rest < a.V ? E::up(row[rest]) : -__builtin_inff();
  const bool bad = HEAD == HEAD_POLICY && (y < 0 || y >= a.V);
  const float zy = HEAD == HEAD_POLICY && !bad ? E::up(row[y]) : 0.f;
  __shared__ Stat part[1][P::W];
  __shared__ int flags[2];
  __shared__ TeacherList lists[HEAD == HEAD_DISTILL ? P::R : 1];
  TeacherList& list = lists[HEAD == HEAD_DISTILL ? P::slot() : 0];
  Teacher te = {0.f, 0.f, false, false};
  if (HEAD == HEAD_DISTILL && tid < 64) {
    te = teacher_row<E>(a, hd, src, row, tid, ti, list);
    if (P::W > 1 && tid == 0) {
      flags[0] = te.empty;
      flags[1] = te.bad;
    }
  }
  constexpr bool ENT = HEAD == HEAD_POLICY;
  Stat st = {-__builtin_inff(), 0.f, 0.f};
  {
    const float z[1] = {zr};
    accumulate<1, ENT>(st, z, a.k);
  }
#pragma unroll
  for (int i = 0; i < CH; ++i)
    if (tid + i * NT < full) {
      float z[E::N];
      E::unpack(raw[i], z);
      accumulate<E::N, ENT>(st, z, a.k);
    }
  st = P::template join<ENT>(st, a.k, part);
  if (HEAD == HEAD_DISTILL && P::W > 1) {
    te.empty = flags[0];
    te.bad = flags[1];
  }
  const float4 w = finish_row<HEAD>(a, hp, 1.f / hd.c, in, te, o, t, st, zy, bad, tid == 0);
  if (tid == 0) o.save[t] = w;
  if (HEAD == HEAD_DISTILL && w.x == kDead) {
    zero_row<E, O>(out, tid, NT, sp, a.V);
    return;
  }
  const int yy = HEAD == HEAD_POLICY ? (int)y : -1;
  if (HEAD == HEAD_POLICY && w.z != 0.f)
    write_once<E, O, true, NT, CH>(raw, out, tid, sp, w, a.k, yy, w.w);
  else
    write_once<E, O, false, NT, CH>(raw, out, tid, sp, w, a.k, yy, w.w);
  if (rest < a.V) out[rest] = O::down(slope<HEAD == HEAD_POLICY>(zr, w, a.k) + (rest == yy ? w.w : 0.f));
  if (HEAD == HEAD_DISTILL) {
    P::sync();                                     // the list's words are written again, after the sweep
    for (int j = tid; j < hd.K; j += NT) {
      const int id = list.id[j];
      if (id >= 0) out[id] = O::down(slope<false>(list.z[j], w, a.k) + w.w * list.psum[j]);
    }
  }
}

// ---- gradient: dz_v = g (e_v (a + b x_v) + d [v in the row's list]), pieces of rows dealt out to workgroups ----------------
struct Grad {
  const float4* save;
  const float *dlogp, *dent; // HEAD_TOKEN: upstream gradients a row,
  const float* slope;        // or, where not NULL, slope of the row's sequence times scale * *g
  float scale;
  const float* g;            // upstream gradient of the loss (device scalar)
  void* out;                 // [T][V]
  int ready;                 // out holds the gradient for *g = 1 already
};

// the pieces c, c + NT, ... below end of a row, four in flight
template <class E, bool B, int NT>
__device__ __forceinline__ void sweep_grad(const typename E::type* row, typename E::type* out, int head, int c, int end,
                                           const float4& w, float k, int y, float d) {
  for (; c < end; c += 4 * NT) {
    u32x4 raw[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (c + i * NT < end) raw[i] = load_piece(row + head + (long)(c + i * NT) * E::N);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (c + i * NT < end) slope_piece<E, E, B>(out, raw[i], head + (c + i * NT) * E::N, w, k, y, d);
  }
}

// NT threads (as above) take a row, or one of `blocks` equal shares of its pieces.  B: an entropy's gradient may be among it
template <class E, int HEAD, bool B, int NT>
__device__ __forceinline__ void gradient_item(const Rows& a, const Distill& hd, const Grad& q, float up, int blocks, uint32_t t,
                                              uint32_t share) {
  typedef Place<NT> P;
  const int tid = P::tid();
  typename E::type* out = (typename E::type*)q.out + (long)t * a.V;
  const Split<E> sp(out, a.V);
  const int each = (sp.full + blocks - 1) / blocks, c0 = (int)share * each;
  const int c1 = c0 + each < sp.full ? c0 + each : sp.full;
  const int rest = share == 0 ? sp.edge(tid, a.V) : a.V;        // the first share has the edges
  float4 w = q.save[t];
  float dy = 0.f;
  int y = -1;
  if (HEAD == HEAD_TOKEN) {
    const float g = q.slope ? up * q.scale * q.slope[sequence_of(a, t)] : q.dlogp ? q.dlogp[t] : 0.f;
    const float h = B && q.dent ? q.dent[t] : 0.f, ln2 = 0.69314718056f;
    if (w.x != kDead) {
      w = make_float4(w.x, -a.c * w.y * (g - h * ln2 * w.z), -a.c * w.y * h * ln2, 0.f);
      dy = a.c * g;
      y = (int)a.labels[t];
    }
  } else {
    w.y *= up;
    w.z *= up;
    dy = w.w * up;
    if (HEAD == HEAD_POLICY && w.x != kDead) y = (int)a.labels[t];
  }
  if (w.x == kDead) {
    for (int c = c0 + tid; c < c1; c += NT) store_zeros<E, E>(out + sp.head + (long)c * E::N);
    if (rest < a.V) out[rest] = E::down(0.f);
    return;
  }
  const typename E::type* row = row_of<E>(a, t);
  if (B && w.z != 0.f)
    sweep_grad<E, true, NT>(row, out, sp.head, c0 + tid, c1, w, a.k, y, dy);
  else
    sweep_grad<E, false, NT>(row, out, sp.head, c0 + tid, c1, w, a.k, y, dy);
  if (rest < a.V) out[rest] = E::down(slope<B>(E::up(row[rest]), w, a.k) + (rest == y ? dy : 0.f));
  if (HEAD == HEAD_DISTILL) {
    P::sync();                                     // the list's words are written again, after the sweep
    for (int j = tid; j < hd.K; j += NT) {
      const int64_t id = hd.ids[(long)t * hd.K + j];
      const float p = hd.psum[(long)t * hd.K + j];
      if (p < 0.f || id < 0 || id >= a.V) continue;
      const int piece = (int)id - sp.head;         // of this share: its pieces, and the edges with the first
      const bool mine = piece < 0 || piece >= sp.full * E::N ? share == 0 : piece >= c0 * E::N && piece < c1 * E::N;
      if (mine) out[id] = E::down(slope<false>(E::up(row[id]), w, a.k) + dy * p);
    }
    P::sync();
  }
}
template <class E, int HEAD, int NT>
__global__ __launch_bounds__(NT == 64 ? 256 : NT, 8) void rows_grad_kernel(Rows a, Distill hd, Grad q, int blocks, long items) {
  typedef Place<NT> P;
  const float up = q.g ? *q.g : 1.f;
  if (HEAD != HEAD_TOKEN && q.ready && up == 1.f) return;
  for (long it = P::row(); it < items; it += gridDim.x * (long)P::R) {
    const uint32_t t = (uint32_t)it / (uint32_t)blocks, share = (uint32_t)it - t * (uint32_t)blocks;   // items < 2^32
    gradient_item<E, HEAD, HEAD != HEAD_DISTILL, NT>(a, hd, q, up, blocks, t, share);
  }
}
// of two tensors of one type and vocabulary, as in the forward pass
template <class E, int NT>
__global__ __launch_bounds__(NT == 64 ? 256 : NT, 8) void rows_grad_pair_kernel(Rows a, Rows b, Grad qa, Grad qb, int blocks,
                                                                                long items) {
  typedef Place<NT> P;
  const float up = *qa.g;
  for (long it = P::row(); it < items; it += gridDim.x * (long)P::R) {
    const uint32_t t = (uint32_t)it / (uint32_t)blocks, share = (uint32_t)it - t * (uint32_t)blocks;   // items < 2^32
    if (__builtin_amdgcn_readfirstlane(t < (uint32_t)a.T))
      gradient_item<E, HEAD_TOKEN, false, NT>(a, Distill{}, qa, up, blocks, t, share);
    else
      gradient_item<E, HEAD_TOKEN, false, NT>(b, Distill{}, qb, up, blocks, t - (uint32_t)a.T, share);
  }
}

// ---- sums --------------------------------------------------------------------------------------------------------------
// Fixed order: a workgroup's threads take rows a stride apart, its tree is fixed, a second launch adds the workgroups' sums.
struct Sum5 {
  double v[5];
};
__device__ __forceinline__ void block_sum(double (&v)[5], double (*sh)[5]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
#pragma unroll
  for (int i = 0; i < 5; ++i) {
    v[i] = wave_sum(v[i]);
    if (lane == 0) sh[wave][i] = v[i];
  }
  __syncthreads();
  if (wave != 0) return;
#pragma unroll
  for (int i = 0; i < 5; ++i) {
    v[i] = lane < waves ? sh[lane][i] : 0.0;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v[i] += __shfl_xor(v[i], o);
  }
}
// what becomes of the sums of {pg, k3, cut, H, live}
struct Result {
  float kl, ent, weight;
  int word;
  float* loss;
  float* stats;              // [4] means over live rows; NULL: not wanted
  float* scale;              // what the rows' terms were multiplied by; NULL: not wanted
};
__device__ __forceinline__ void write_result(const double (&v)[5], const Result& r) {
  const double n = v[4] > 1.0 ? v[4] : 1.0;
  const double scale = r.word ? r.weight / n : r.weight;
  const double kl = r.kl != 0.f ? (double)r.kl * v[1] : 0.0;         // the term may be infinite where it only is reported
  *r.loss = (float)(scale * (v[0] + kl - (double)r.ent * v[3]));
  if (r.stats)
    for (int i = 0; i < 4; ++i) r.stats[i] = (float)(v[i] / n);
  if (r.scale) *r.scale = (float)scale;
}

__global__ __launch_bounds__(1024) void sum_rows_kernel(const float4* __restrict__ rows, const int64_t* __restrict__ labels,
                                                        int64_t ignore, long T, Sum5* __restrict__ part, Result r) {
  __shared__ double sh[16][5];
  double v[5] = {0, 0, 0, 0, 0};
  const long step = gridDim.x * 1024L;
  for (long t0 = blockIdx.x * 1024L + threadIdx.x; t0 < T; t0 += 8 * step) {
    float4 q[8];
    int64_t y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {                  // eight rows in flight
      const long t = t0 + i * step;
      q[i] = t < T ? rows[t] : make_float4(0.f, 0.f, 0.f, 0.f);
      y[i] = t < T && labels ? labels[t] : ignore;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[0] += q[i].x;
      v[1] += q[i].y;
      v[2] += q[i].z;
      v[3] += q[i].w;
      v[4] += labels ? y[i] != ignore : t0 + i * step < T;
    }
  }
  block_sum(v, sh);
  if (threadIdx.x == 0) {
    if (gridDim.x > 1) {
      for (int i = 0; i < 5; ++i) part[blockIdx.x].v[i] = v[i];
    } else {
      write_result(v, r);
    }
  }
}
__global__ __launch_bounds__(256) void sum_parts_kernel(const Sum5* __restrict__ part, int n, Result r) {
  __shared__ double sh[16][5];
  double v[5] = {0, 0, 0, 0, 0};
  for (int t = threadIdx.x; t < n; t += 256)
    for (int i = 0; i < 5; ++i) v[i] += part[t].v[i];
  block_sum(v, sh);
  if (threadIdx.x == 0) write_result(v, r);
}
constexpr int kSumGroups = 256;
inline int sum_groups(long T) {
  const long g = (T + 16383) / 16384;
  return (int)(g < 1 ? 1 : g > kSumGroups ? kSumGroups : g);
}

// live rows, before a pass that divides by them
__global__ __launch_bounds__(1024) void count_live_kernel(const int64_t* __restrict__ labels, int64_t ignore, long T,
                                                          float* __restrict__ part, float* __restrict__ out) {
  __shared__ int sh[16];
  int n = 0;
  const long step = gridDim.x * 1024L;
  for (long t0 = blockIdx.x * 1024L + threadIdx.x; t0 < T; t0 += 8 * step) {
    int64_t y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = t0 + i * step < T ? labels[t0 + i * step] : ignore;
#pragma unroll
    for (int i = 0; i < 8; ++i) n += y[i] != ignore ? 1 : 0;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = n;
  __syncthreads();
  if (threadIdx.x < 64) {
    n = threadIdx.x < 16 ? sh[threadIdx.x] : 0;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) n += __shfl_xor(n, o);
    if (threadIdx.x == 0) (gridDim.x > 1 ? part[blockIdx.x] : out[0]) = (float)n;
  }
}
__global__ __launch_bounds__(256) void add_counts_kernel(const float* __restrict__ part, int n, float* __restrict__ out) {
  __shared__ double sh[16][5];
  double v[5] = {(int)threadIdx.x < n ? (double)part[threadIdx.x] : 0.0, 0, 0, 0, 0};
  block_sum(v, sh);
  if (threadIdx.x == 0) out[0] = (float)v[0];
}

// ---- behind a projection: column sums of a bf16 gradient, results times a device scalar ------------------------------------
// Columns in pairs, 128 to a workgroup; its four waves take a quarter each of a share of the rows, and a second launch adds
// the shares in order.
constexpr int kColShares = 64;
__global__ __launch_bounds__(256) void colsum_part_kernel(const uint32_t* __restrict__ P, long ld2, long T, int V,
                                                          float* __restrict__ part) {
  __shared__ float2 sh[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, pair = blockIdx.x * 64 + lane;
  const long each = (T + gridDim.y - 1) / gridDim.y, t0 = blockIdx.y * each, t1 = t0 + each < T ? t0 + each : T;
  float2 s = make_float2(0.f, 0.f);
  if (2 * pair < V) {
    for (long t = t0 + wave; t < t1; t += 4 * 8) {
      uint32_t r[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) r[i] = t + 4 * i < t1 ? P[(t + 4 * i) * ld2 + pair] : 0u;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        s.x += as_float(r[i] << 16);
        s.y += as_float(r[i] & 0xffff0000u);
      }
    }
  }
  sh[wave][lane] = s;
  __syncthreads();
  if (wave != 0 || 2 * pair >= V) return;
  for (int w = 1; w < 4; ++w) {
    s.x += sh[w][lane].x;
    s.y += sh[w][lane].y;
  }
  part[blockIdx.y * (long)V + 2 * pair] = s.x;
  if (2 * pair + 1 < V) part[blockIdx.y * (long)V + 2 * pair + 1] = s.y;
}
__global__ __launch_bounds__(64) void colsum_join_kernel(const float* __restrict__ part, int V, const float* __restrict__ g,
                                                         float* __restrict__ out) {
  const int v = blockIdx.x * 64 + threadIdx.x;
  if (v >= V) return;
  float s = 0.f;
  for (int i0 = 0; i0 < kColShares; i0 += 16) {    // sixteen shares in flight
    float r[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) r[i] = part[(i0 + i) * (long)V + v];
#pragma unroll
    for (int i = 0; i < 16; ++i) s += r[i];
  }
  out[v] = s * *g;
}
__global__ __launch_bounds__(256) void scale_by_kernel(float4* __restrict__ x, long n4, const float* __restrict__ g) {
  const float w = *g;
  if (w == 1.f) return;
  for (long i = blockIdx.x * 256L + threadIdx.x; i < n4; i += gridDim.x * 256L) {
    float4 v = x[i];
    x[i] = make_float4(v.x * w, v.y * w, v.z * w, v.w * w);
  }
}

// Live rows of a bf16 matrix to the front, zeros behind them up to Tp rows: they meet the zero rows of the gradient in the
// weight gradient's product, and what stands in dead rows of the caller's, NaN included, must not.
__global__ __launch_bounds__(256) void gather_live_kernel(const uint4* __restrict__ h, const int64_t* __restrict__ perm,
                                                          const int* __restrict__ count, int pieces, long n, uint4* __restrict__ out) {
  const int live = *count;
  for (long i = blockIdx.x * 256L + threadIdx.x; i < n; i += gridDim.x * 256L) {
    const uint32_t row = (uint32_t)(i / pieces);
    out[i] = (int)row < live ? h[perm[row] * pieces + (i - (long)row * pieces)] : uint4{0u, 0u, 0u, 0u};
  }
}

// ---- policy loss from log-probabilities ------------------------------------------------------------------------------------
// Latency bound: a few bytes a token.  One launch up to 4096 tokens, and one more that adds the workgroups' sums beyond.
__global__ __launch_bounds__(1024) void policy_tokens_kernel(const float* __restrict__ logp, const int64_t* __restrict__ labels,
                                                             int64_t ignore, long T, int n1, Policy h, float* __restrict__ dlp,
                                                             Sum5* __restrict__ part, Result r) {
  __shared__ double sh[16][5];
  double v[5] = {0, 0, 0, 0, 0};
  const long step = gridDim.x * 1024L;
  for (long t0 = blockIdx.x * 1024L + threadIdx.x; t0 < T; t0 += 4 * step) {
    float lp[4], old[4], ref[4], adv[4];
    bool live[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {                  // four tokens in flight; a dead one's entries may hold anything
      const long t = t0 + i * step;
      if (t >= T) break;
      live[i] = labels[t] != ignore;
      lp[i] = logp[t];
      old[i] = h.old_lp[t];
      ref[i] = h.ref_lp ? h.ref_lp[t] : 0.f;
      adv[i] = h.adv[h.adv_per_row ? t : (long)((uint32_t)t / (uint32_t)n1)];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const long t = t0 + i * step;
      if (t >= T) break;
      float d = 0.f;
      if (live[i]) {
        const PolicyTerm q = policy_term(h, lp[i], old[i], ref[i], adv[i]);
        v[0] += q.pg;
        v[1] += q.k3;
        v[2] += q.cut;
        v[4] += 1.0;
        d = q.dlp;
      }
      if (dlp) dlp[t] = d;
    }
  }
  block_sum(v, sh);
  if (threadIdx.x == 0) {
    if (gridDim.x > 1) {
      for (int i = 0; i < 5; ++i) part[blockIdx.x].v[i] = v[i];
    } else {
      write_result(v, r);
    }
  }
}
// d logp = g * scale * dlp
__global__ __launch_bounds__(256) void policy_tokens_bwd_kernel(const float* __restrict__ dlp, const float* __restrict__ scale,
                                                                const float* __restrict__ g, long T, float* __restrict__ out) {
  const float w = *g * *scale;
  for (long t = blockIdx.x * 256L + threadIdx.x; t < T; t += gridDim.x * 256L) out[t] = w * dlp[t];
}

// ---- preference loss -----------------------------------------------------------------------------------------------------
struct Answers {
  const float *logp, *ref;   // [P][L]; ref NULL: no reference model
  const int64_t* labels;
  int L;
};
// sum over the live tokens of (log p - log p_ref), in fp64: long answers cancel
__device__ __forceinline__ double answer_sum(const Answers& a, int64_t ignore, long b) {
  double v = 0.0;
  for (int i0 = threadIdx.x; i0 < a.L; i0 += 4 * 256) {
    int64_t y[4];
    float lp[4], ref[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {                  // four tokens in flight; a dead one's entries may hold anything
      const long t = b * a.L + i0 + k * 256;
      const bool in = i0 + k * 256 < a.L;
      y[k] = in ? a.labels[t] : ignore;
      lp[k] = in ? a.logp[t] : 0.f;
      ref[k] = in && a.ref ? a.ref[t] : 0.f;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (y[k] != ignore) v += (double)lp[k] - (double)ref[k];
  }
  return v;
}
// One workgroup a pair: x = beta (sum_chosen - sum_rejected), loss = -(1 - e) ln sig(x) - e ln sig(-x), its slope.
__global__ __launch_bounds__(256) void preference_kernel(Answers c, Answers r, int64_t ignore, float beta, float smooth,
                                                         float* __restrict__ reward_c, float* __restrict__ reward_r,
                                                         float* __restrict__ slope, float4* __restrict__ rowout) {
  __shared__ double sh[4][2];
  const long b = blockIdx.x;
  double vc = wave_sum(answer_sum(c, ignore, b)), vr = wave_sum(answer_sum(r, ignore, b));
  if ((threadIdx.x & 63) == 0) {
    sh[threadIdx.x >> 6][0] = vc;
    sh[threadIdx.x >> 6][1] = vr;
  }
  __syncthreads();
  if (threadIdx.x != 0) return;
  vc = sh[0][0] + sh[1][0] + sh[2][0] + sh[3][0];
  vr = sh[0][1] + sh[1][1] + sh[2][1] + sh[3][1];
  reward_c[b] = (float)(beta * vc);
  reward_r[b] = (float)(beta * vr);
  const float x = (float)(beta * (vc - vr));
  const float q = expf(-fabsf(x)), l = log1pf(q);                    // -ln sig(|x|)
  const float up = x >= 0.f ? l : l - x, down = x >= 0.f ? l + x : l;   // -ln sig(x), -ln sig(-x)
  const float small = q / (1.f + q), large = 1.f / (1.f + q);           // sig(-|x|), sig(|x|)
  const float sig = x >= 0.f ? large : small, gis = x >= 0.f ? small : large;
  float loss = smooth != 1.f ? (1.f - smooth) * up : 0.f;               // up and down may be infinite
  if (smooth != 0.f) loss += smooth * down;
  rowout[b] = make_float4(x != x ? x : loss, 0.f, 0.f, 0.f);
  slope[b] = beta * (smooth * sig - (1.f - smooth) * gis);
}
// d logp of both answers of a pair: +- g * scale * slope on live tokens
__global__ __launch_bounds__(256) void preference_bwd_kernel(const int64_t* __restrict__ labels_c, int Lc, float* __restrict__ dc,
                                                             const int64_t* __restrict__ labels_r, int Lr, float* __restrict__ dr,
                                                             int64_t ignore, const float* __restrict__ slope, float scale,
                                                             const float* __restrict__ g) {
  const long b = blockIdx.x;
  const float w = *g * scale * slope[b];
  for (int i = threadIdx.x; i < Lc; i += 256) dc[b * Lc + i] = labels_c[b * Lc + i] != ignore ? w : 0.f;
  for (int i = threadIdx.x; i < Lr; i += 256) dr[b * Lr + i] = labels_r[b * Lr + i] != ignore ? -w : 0.f;
}

// ---- host side -----------------------------------------------------------------------------------------------------------
inline int pieces_of(int dtype, int V) { return V / (dtype == PV_DTYPE_F32 ? 4 : 8); }
// a launch has fewer than 2^32 threads; the ladders below give a row at most these
inline long threads_of(int dtype, int V) {
  const int pieces = pieces_of(dtype, V);
  return pieces <= 512 ? 64 : pieces <= 1024 ? 128 : pieces <= 2048 ? 256 : pieces <= 4096 ? 512 : 1024;
}
int check_rows(const char* who, const void* logits, int dtype, long n0, int n1, long s0, long s1, int V, float inv_temp) {
  PV_REQUIRE(logits && n0 > 0 && n1 > 0 && V > 0, "%s: null logits or an empty size", who);
  PV_REQUIRE(dtype == PV_DTYPE_F32 || dtype == PV_DTYPE_BF16 || dtype == PV_DTYPE_F16, "%s: unknown dtype %d", who, dtype);
  PV_REQUIRE(s0 >= 0 && s1 >= 0, "%s: negative stride", who);
  PV_REQUIRE(inv_temp > 0.f && inv_temp < __builtin_inff(), "%s: the inverse temperature must be positive and finite", who);
  PV_REQUIRE(((uintptr_t)logits & (dtype == PV_DTYPE_F32 ? 3 : 1)) == 0, "%s: logits not aligned to their elements", who);
  if (V > kVocabMax || n0 > kRowsMax || n0 * (long)n1 > kRowsMax) {
    pv_set_error("%s: %ld x %d rows of %d words are beyond the limit (%ld rows, 2^24 words)", who, n0, n1, V, kRowsMax);
    return PV_ERR_LIMIT;
  }
  if (n0 * (long)n1 * threads_of(dtype, V) >= 1L << 32) {
    pv_set_error("%s: %ld rows of %d words are more than a launch has threads for", who, n0 * (long)n1, V);
    return PV_ERR_LIMIT;
  }
  return PV_OK;
}
int check_count(const char* who, long n, long limit) {
  if (n <= limit) return PV_OK;
  pv_set_error("%s: %ld are beyond the limit of %ld", who, n, limit);
  return PV_ERR_LIMIT;
}
Rows make_rows(const void* logits, long n0, int n1, long s0, long s1, int V, const int64_t* labels, int64_t ignore, float c) {
  return {logits, n1, V, n0 * (long)n1, s0, s1, c, (float)((double)c * 1.4426950408889634), labels, ignore, nullptr};
}

// Answers of one type and vocabulary, whose rows fit a launch together too.
bool share_a_launch(int dtype_a, const Rows& a, int dtype_b, const Rows& b) {
  return dtype_a == dtype_b && a.V == b.V && a.T + b.T <= kRowsMax && (a.T + b.T) * threads_of(dtype_a, a.V) < 1L << 32;
}

// Threads a row of the pass that only reads: fewer for short rows, whose workgroups cost more than their words, and for many
// rows.  us at the borders, the side in front and the one behind (log-probabilities, half of the 12800 rows and none of the 400
// dead, bf16 / fp32):
//     256 pieces  T = 12800: 64  9.7 / 8.0, 256 14.9 / 12.9                   T = 400:  64 6.2 / 6.4, 256  6.5 / 6.1
//    1000         T = 12800: 64 27.0 / 22.7, 256 23.6 / 20.6 (512 pieces: 64 15.5 / 12.5, 256 17.9 / 15.3)
//    4096         T = 12800: 256 76.7 / 74.5, 512 73.1 / 72.8                 T = 400: 256 9.0 / 7.5, 1024 9.3 / 8.2
//    6100         T = 12800: 512 112 / 110, 1024 129 / 109; T = 600: 512 12.3 / 10.1, 1024 10.7 / 9.2
//    8000         T = 12800: 512 144 / 141, 1024 152 / 136; T = 600: 512 15.0 / 12.1, 1024 12.4 / 10.6
//   12000         T = 12800: 512 216 / 207, 1024 204 / 197
// and one row of V = 131071, fp32: 1024 10.4, 256 17.5.  Few rows take more threads each, which they leave idle otherwise (1000
// pieces, T = 400: 64 7.1, 256 6.6).  Splitting one row over workgroups and joining the parts in a second launch took 9.4 us for
// that row, and more than one launch everywhere else.
template <class E, int HEAD, bool ENT>
int launch_fwd_typed(const Rows& a, const Policy& hp, const Distill& hd, const Scale& sc, const FwdOut& o, hipStream_t st) {
  const int pieces = a.V / E::N;
  const unsigned T = (unsigned)a.T;
  if (pieces <= 256 || (pieces <= 1024 && T >= 512))
    rows_fwd_kernel<E, HEAD, ENT, 64><<<dim3((T + 3) / 4), dim3(256), 0, st>>>(a, hp, hd, sc, o);
  else if (pieces <= 4096)
    rows_fwd_kernel<E, HEAD, ENT, 256><<<dim3(T), dim3(256), 0, st>>>(a, hp, hd, sc, o);
  else if (pieces <= 6144 && T >= 512)
    rows_fwd_kernel<E, HEAD, ENT, 512><<<dim3(T), dim3(512), 0, st>>>(a, hp, hd, sc, o);
  else
    rows_fwd_kernel<E, HEAD, ENT, 1024><<<dim3(T), dim3(1024), 0, st>>>(a, hp, hd, sc, o);
  PV_LAUNCH_CHECK("rows_fwd_kernel");
  return PV_OK;
}
template <class E>
int launch_fwd_pair_typed(const Rows& a, const Rows& b, const FwdOut& oa, const FwdOut& ob, hipStream_t st) {
  const int pieces = a.V / E::N;
  const unsigned T = (unsigned)(a.T + b.T);
  if (pieces <= 256 || (pieces <= 1024 && T >= 512))
    rows_fwd_pair_kernel<E, 64><<<dim3((T + 3) / 4), dim3(256), 0, st>>>(a, b, oa, ob);
  else if (pieces <= 4096)
    rows_fwd_pair_kernel<E, 256><<<dim3(T), dim3(256), 0, st>>>(a, b, oa, ob);
  else if (pieces <= 6144 && T >= 512)
    rows_fwd_pair_kernel<E, 512><<<dim3(T), dim3(512), 0, st>>>(a, b, oa, ob);
  else
    rows_fwd_pair_kernel<E, 1024><<<dim3(T), dim3(1024), 0, st>>>(a, b, oa, ob);
  PV_LAUNCH_CHECK("rows_fwd_pair_kernel");
  return PV_OK;
}
template <int HEAD, bool ENT>
int launch_fwd(int dtype, const Rows& a, const Policy& hp, const Distill& hd, const Scale& sc, const FwdOut& o, hipStream_t st) {
  if (dtype == PV_DTYPE_F32) return launch_fwd_typed<F32, HEAD, ENT>(a, hp, hd, sc, o, st);
  if (dtype == PV_DTYPE_BF16) return launch_fwd_typed<BF16, HEAD, ENT>(a, hp, hd, sc, o, st);
  return launch_fwd_typed<F16, HEAD, ENT>(a, hp, hd, sc, o, st);
}

// The one-pass kernel takes the fewest threads that can hold a row: fewer threads with more pieces each keep more rows of a CU
// in flight.  TB/s of live reads and of writes at each border, the rung in front of it and the next ones (policy loss, half of
// the rows dead, odd numbers of words, bf16 / fp32):
//     256 pieces   64 x 4 3.88 / 3.93     128 x 8 3.74 / 4.06     256 x 8 2.84 / 3.22
//     512          64 x 8 3.95 / 4.05     128 x 8 4.08 / 4.13     256 x 8 4.13 / 4.30
//    1024         128 x 8 3.89 / 4.01     256 x 8 4.13 / 4.22     512 x 8 3.98 / 4.38
//    2048         256 x 8 4.10 / 4.28     512 x 8 4.40 / 4.37    1024 x 8 3.94 / 4.45
//    4000         512 x 8 4.19 / 4.35    1024 x 6 4.45 / 4.63
//    6144        1024 x 6 4.34 / 4.53    512 x 20 4.30 / 4.48
//    8000        1024 x 8 4.20 / 4.40    512 x 20 4.15 / 4.39   1024 x 12 3.72 / 4.54
//   10000        512 x 20 3.96 / 4.20   1024 x 12 3.73 / 4.40
// The upper end of a rung would gain 0 to 11 % by the next one, its lower end loses more (500 pieces: 512 x 6 2.8 / 3.3).
// At one number of threads, pieces that a row does not fill cost registers, and with them rows of a CU (two full rungs against
// one that the row fits): 64 x 8 for 4 up to 20 %, 512 x 8 for 6 7 to 9 % with a bf16 gradient of fp32 rows, 1024 x 8 for 6 3 to
// 7 % there and in the distillation of 16-bit rows, 1024 x 16 for 12 3 to 5 % in their policy loss, 20 for 16 1 to 3 %.  (64 x 2
// and 256 x 6 gave 1 and 2 % at most and are not kept.)  Beyond 10 240 pieces a CU holds one row,
// which still beats two passes over memory: at the last border 3.7 / 4.4 TB/s (distillation, K = 64) and 3.6 / 4.35 (policy), behind
// it 3.3 / 3.4 and 3.0 / 3.2.  Keeping part of such rows in shared memory to hold two of them gained nothing
// (512 x 23 + 9: 3.6, its registers spill).
constexpr int kOncePieces = 1024 * 20;            // of a row that the one-pass kernel holds
template <class E, class O, int HEAD>
int launch_once_typed(const Rows& a, const Policy& hp, const Distill& hd, const Scale& sc, const FwdOut& o, void* grad, long ldg,
                      hipStream_t st) {
  const int pieces = a.V / E::N;
  typename O::type* g = (typename O::type*)grad;
#define PV_ONCE(NT, CH, WAVES)                                                                                  \
  if (pieces <= NT * CH) {                                                                                      \
    typedef Place<NT> P;                                                                                        \
    rows_once_kernel<E, O, HEAD, NT, CH, WAVES>                                                                 \
        <<<dim3((unsigned)((a.T + P::R - 1) / P::R)), dim3(NT * P::R), 0, st>>>(a, hp, hd, sc, o, g, ldg);       \
    PV_LAUNCH_CHECK("rows_once_kernel");                                                                        \
    return PV_OK;                                                                                               \
  }
  PV_ONCE(64, 4, 8)
  PV_ONCE(64, 8, 6)
  PV_ONCE(128, 8, 7)
  PV_ONCE(256, 8, 7)
  PV_ONCE(512, 6, 8)
  PV_ONCE(512, 8, 6)
  PV_ONCE(1024, 6, 8)
  PV_ONCE(1024, 8, 8)
  PV_ONCE(512, 20, 4)
  PV_ONCE(1024, 12, 4)
  PV_ONCE(1024, 16, 4)
  PV_ONCE(1024, 20, 4)
#undef PV_ONCE
  pv_set_error("rows_once_kernel: a row of %d words does not fit", a.V);
  return PV_ERR_LIMIT;
}
template <int HEAD>
int launch_once(int dtype, const Rows& a, const Policy& hp, const Distill& hd, const Scale& sc, const FwdOut& o, void* grad,
                long ldg, hipStream_t st) {
  if (ldg > 0) return launch_once_typed<F32, BF16, HEAD>(a, hp, hd, sc, o, grad, ldg, st);
  if (dtype == PV_DTYPE_F32) return launch_once_typed<F32, F32, HEAD>(a, hp, hd, sc, o, grad, a.V, st);
  if (dtype == PV_DTYPE_BF16) return launch_once_typed<BF16, BF16, HEAD>(a, hp, hd, sc, o, grad, a.V, st);
  return launch_once_typed<F16, F16, HEAD>(a, hp, hd, sc, o, grad, a.V, st);
}
int check_gradient(const char* who, int dtype, int V, const void* save, const void* dlogits, long ld_bf16, const void* perm) {
  PV_REQUIRE(!perm || ld_bf16 > 0, "%s: an order of the rows goes with a bf16 gradient", who);
  PV_REQUIRE(!dlogits || (save && pv_vocab_rows_one_pass(dtype, V)), "%s: no gradient in the forward pass here", who);
  PV_REQUIRE(ld_bf16 == 0 || (dlogits && dtype == PV_DTYPE_F32 && ld_bf16 >= V && ld_bf16 - V < 64),
             "%s: a bf16 gradient needs fp32 logits and rows of V to V + 63 words", who);
  return PV_OK;
}

// The gradient pass: a wave a row for short ones, 256 threads for 1024 pieces of a longer one.  us, half of the rows dead, the
// shapes of 0.3 GB or 60000 rows (bf16 / fp32): 100 pieces 64 33 / 29, 256 80 / 75; 200 49 / 47, 95 / 89; 300 96 / 95, 110 / 106;
// 512 95 / 95, 97 / 95; 1100 102 / 99, 106 / 103, but with 600 rows 8.6 / 7.5, 6.7 / 6.2.  Shares of 512 and 2048 pieces: 2500
// pieces 102 / 99, 107 / 103, of 1024 103 / 100; 16384 97 / 95, 96 / 95, of 1024 94 / 92.  2048 workgroups: a launch that finds the
// gradient ready ends in 5 us with 512 as well, and one that does not takes 97 to 141 us with 512 or 1024, 85 with 2048 (V = 5003,
// bf16, 20000 rows).
template <class E, int HEAD>
int launch_grad_typed(const Rows& a, const Distill& hd, const Grad& q, hipStream_t st) {
  const int pieces = a.V / E::N;
  if (pieces <= 512) {                             // a wave a row
    const long quads = (a.T + 3) / 4;
    rows_grad_kernel<E, HEAD, 64><<<dim3((unsigned)(quads < 2048 ? quads : 2048)), dim3(256), 0, st>>>(a, hd, q, 1, a.T);
  } else {
    const int blocks = cdiv(pieces, 256 * 4);
    const long items = a.T * blocks;
    rows_grad_kernel<E, HEAD, 256><<<dim3((unsigned)(items < 2048 ? items : 2048)), dim3(256), 0, st>>>(a, hd, q, blocks, items);
  }
  PV_LAUNCH_CHECK("rows_grad_kernel");
  return PV_OK;
}
template <class E>
int launch_grad_pair_typed(const Rows& a, const Rows& b, const Grad& qa, const Grad& qb, hipStream_t st) {
  const int pieces = a.V / E::N;
  const long T = a.T + b.T;
  if (pieces <= 512) {
    const long quads = (T + 3) / 4;
    rows_grad_pair_kernel<E, 64><<<dim3((unsigned)(quads < 2048 ? quads : 2048)), dim3(256), 0, st>>>(a, b, qa, qb, 1, T);
  } else {
    const int blocks = cdiv(pieces, 256 * 4);
    const long items = T * blocks;
    rows_grad_pair_kernel<E, 256><<<dim3((unsigned)(items < 2048 ? items : 2048)), dim3(256), 0, st>>>(a, b, qa, qb, blocks, items);
  }
  PV_LAUNCH_CHECK("rows_grad_pair_kernel");
  return PV_OK;
}
template <int HEAD>
int launch_grad(int dtype, const Rows& a, const Distill& hd, const Grad& q, hipStream_t st) {
  if (dtype == PV_DTYPE_F32) return launch_grad_typed<F32, HEAD>(a, hd, q, st);
  if (dtype == PV_DTYPE_BF16) return launch_grad_typed<BF16, HEAD>(a, hd, q, st);
  return launch_grad_typed<F16, HEAD>(a, hd, q, st);
}

int launch_count(const int64_t* labels, int64_t ignore, long T, float* part, float* out, hipStream_t st) {
  const int g = sum_groups(T);
  count_live_kernel<<<dim3(g), dim3(1024), 0, st>>>(labels, ignore, T, part, out);
  PV_LAUNCH_CHECK("count_live_kernel");
  if (g > 1) {
    add_counts_kernel<<<dim3(1), dim3(256), 0, st>>>(part, g, out);
    PV_LAUNCH_CHECK("add_counts_kernel");
  }
  return PV_OK;
}
int launch_sum(const float4* rows, const int64_t* labels, int64_t ignore, long T, Sum5* part, const Result& r, hipStream_t st) {
  const int g = sum_groups(T);
  sum_rows_kernel<<<dim3(g), dim3(1024), 0, st>>>(rows, labels, ignore, T, part, r);
  PV_LAUNCH_CHECK("sum_rows_kernel");
  if (g > 1) {
    sum_parts_kernel<<<dim3(1), dim3(256), 0, st>>>(part, g, r);
    PV_LAUNCH_CHECK("sum_parts_kernel");
  }
  return PV_OK;
}

}  // namespace

extern "C" {

// {the rows' terms, the sums' parts, the count}
size_t pv_vocab_rows_ws_bytes(long rows) {
  return rows < 0 ? 0 : (size_t)rows * sizeof(float4) + kSumGroups * sizeof(Sum5) + sizeof(float);
}

int pv_vocab_rows_one_pass(int dtype, int V) {
  return V > 0 && pieces_of(dtype, V) <= kOncePieces;
}

int pv_token_logp_fwd(const void* logits, int dtype, long n0, int n1, long s0, long s1, int V, const int64_t* tokens,
                      int64_t ignore, float inv_temp, float* logp, float* entropy, float* save, void* stream) {
  const int rc = check_rows("pv_token_logp_fwd", logits, dtype, n0, n1, s0, s1, V, inv_temp);
  if (rc != PV_OK) return rc;
  PV_REQUIRE(tokens && logp, "pv_token_logp_fwd: null argument");
  const Rows a = make_rows(logits, n0, n1, s0, s1, V, tokens, ignore, inv_temp);
  const FwdOut o = {logp, entropy, nullptr, (float4*)save};
  if (entropy) return launch_fwd<HEAD_TOKEN, true>(dtype, a, Policy{}, Distill{}, Scale{}, o, (hipStream_t)stream);
  return launch_fwd<HEAD_TOKEN, false>(dtype, a, Policy{}, Distill{}, Scale{}, o, (hipStream_t)stream);
}

int pv_token_logp_bwd(const void* logits, int dtype, long n0, int n1, long s0, long s1, int V, const int64_t* tokens,
                      int64_t ignore, float inv_temp, const float* save, const float* dlogp, const float* dentropy,
                      void* dlogits, void* stream) {
  const int rc = check_rows("pv_token_logp_bwd", logits, dtype, n0, n1, s0, s1, V, inv_temp);
  if (rc != PV_OK) return rc;
  PV_REQUIRE(tokens && save && dlogits && (dlogp || dentropy), "pv_token_logp_bwd: null argument");
  const Rows a = make_rows(logits, n0, n1, s0, s1, V, tokens, ignore, inv_temp);
  return launch_grad<HEAD_TOKEN>(dtype, a, Distill{}, Grad{(const float4*)save, dlogp, dentropy, nullptr, 0.f, nullptr, dlogits, 0},
                                 (hipStream_t)stream);
}

int pv_policy_rows_fwd(const void* logits, int dtype, long n0, int n1, long s0, long s1, int V, const int64_t* tokens,
                       int64_t ignore, float inv_temp, const float* old_logp, const float* ref_logp, const float* adv,
                       int adv_per_token, float clip_lo, float clip_hi, float kl_coef, float ent_coef, float weight, int word,
                       float* loss, float* stats, float* save, void* dlogits, long ld_bf16,
                       const int64_t* perm, void* ws, void* stream) {
  int rc = check_rows("pv_policy_rows_fwd", logits, dtype, n0, n1, s0, s1, V, inv_temp);
  if (rc == PV_OK) rc = check_gradient("pv_policy_rows_fwd", dtype, V, save, dlogits, ld_bf16, perm);
  if (rc != PV_OK) return rc;
  PV_REQUIRE(tokens && old_logp && adv && loss && stats && ws, "pv_policy_rows_fwd: null argument");
  PV_REQUIRE(clip_lo <= clip_hi, "pv_policy_rows_fwd: the clip range is empty");
  hipStream_t st = (hipStream_t)stream;
  Rows a = make_rows(logits, n0, n1, s0, s1, V, tokens, ignore, inv_temp);
  a.perm = perm;
  float4* rowout = (float4*)ws;
  Sum5* part = (Sum5*)(rowout + a.T);
  Scale sc = {weight, nullptr};
  if (word && save) {
    float* count = (float*)(part + kSumGroups);
    const int r = launch_count(tokens, ignore, a.T, (float*)part, count, st);
    if (r != PV_OK) return r;
    sc.count = count;
  }
  const Policy hp = {old_logp, ref_logp, adv, adv_per_token, clip_lo, clip_hi, kl_coef, ent_coef};
  const FwdOut o = {nullptr, nullptr, rowout, (float4*)save};
  const int r = dlogits ? launch_once<HEAD_POLICY>(dtype, a, hp, Distill{}, sc, o, dlogits, ld_bf16, st)
                        : launch_fwd<HEAD_POLICY, true>(dtype, a, hp, Distill{}, sc, o, st);
  if (r != PV_OK) return r;
  return launch_sum(rowout, tokens, ignore, a.T, part, Result{kl_coef, ent_coef, weight, word, loss, stats, nullptr}, st);
}

int pv_policy_rows_bwd(const void* logits, int dtype, long n0, int n1, long s0, long s1, int V, const int64_t* tokens,
                       int64_t ignore, float inv_temp, const float* save, const float* g, int ready, void* dlogits, void* stream) {
  const int rc = check_rows("pv_policy_rows_bwd", logits, dtype, n0, n1, s0, s1, V, inv_temp);
  if (rc != PV_OK) return rc;
  PV_REQUIRE(tokens && save && g && dlogits, "pv_policy_rows_bwd: null argument");
  const Rows a = make_rows(logits, n0, n1, s0, s1, V, tokens, ignore, inv_temp);
  return launch_grad<HEAD_POLICY>(dtype, a, Distill{}, Grad{(const float4*)save, nullptr, nullptr, nullptr, 0.f, g, dlogits, ready},
                                  (hipStream_t)stream);
}

int pv_distill_max_entries(void) { return kTeacherMax; }

int pv_distill_rows_fwd(const void* logits, int dtype, long n0, int n1, long s0, long s1, int V, const int64_t* labels,
                        int64_t ignore, float inv_temp, float t_inv_temp, const int64_t* t_ids, const void* t_logits, int t_dtype,
                        int K, float weight, int word, float* loss, float* save, float* psum, void* dlogits, long ld_bf16,
                        const int64_t* perm, void* ws, void* stream) {
  int rc = check_rows("pv_distill_rows_fwd", logits, dtype, n0, n1, s0, s1, V, inv_temp);
  if (rc == PV_OK) rc = check_gradient("pv_distill_rows_fwd", dtype, V, save, dlogits, ld_bf16, perm);
  if (rc != PV_OK) return rc;
  PV_REQUIRE(t_ids && t_logits && loss && psum && ws, "pv_distill_rows_fwd: null argument");
  PV_REQUIRE(t_dtype == PV_DTYPE_F32 || t_dtype == PV_DTYPE_BF16 || t_dtype == PV_DTYPE_F16,
             "pv_distill_rows_fwd: unknown teacher dtype %d", t_dtype);
  PV_REQUIRE(K > 0, "pv_distill_rows_fwd: no teacher entries");
  PV_REQUIRE(t_inv_temp > 0.f && t_inv_temp < __builtin_inff(), "pv_distill_rows_fwd: the teacher's inverse temperature must be positive and finite");
  if (K > kTeacherMax) {
    pv_set_error("pv_distill_rows_fwd: %d teacher entries are beyond the limit of %d", K, kTeacherMax);
    return PV_ERR_LIMIT;
  }
  hipStream_t st = (hipStream_t)stream;
  Rows a = make_rows(logits, n0, n1, s0, s1, V, labels, ignore, inv_temp);
  a.perm = perm;
  float4* rowout = (float4*)ws;
  Sum5* part = (Sum5*)(rowout + a.T);
  Scale sc = {weight, nullptr};
  if (word && !labels) sc.weight = weight / (float)a.T;
  if (word && labels && save) {
    float* count = (float*)(part + kSumGroups);
    const int r = launch_count(labels, ignore, a.T, (float*)part, count, st);
    if (r != PV_OK) return r;
    sc.count = count;
  }
  const Distill hd = {t_ids, t_logits, K, t_dtype, psum, t_inv_temp, (float)((double)t_inv_temp * 1.4426950408889634)};
  const FwdOut o = {nullptr, nullptr, rowout, (float4*)save};
  const int r = dlogits ? launch_once<HEAD_DISTILL>(dtype, a, Policy{}, hd, sc, o, dlogits, ld_bf16, st)
                        : launch_fwd<HEAD_DISTILL, false>(dtype, a, Policy{}, hd, sc, o, st);
  if (r != PV_OK) return r;
  return launch_sum(rowout, labels, ignore, a.T, part, Result{0.f, 0.f, weight, word, loss, nullptr, nullptr}, st);
}

int pv_distill_rows_bwd(const void* logits, int dtype, long n0, int n1, long s0, long s1, int V, float inv_temp,
                        const int64_t* t_ids, int K, const float* save, const float* psum, const float* g, int ready,
                        void* dlogits, void* stream) {
  const int rc = check_rows("pv_distill_rows_bwd", logits, dtype, n0, n1, s0, s1, V, inv_temp);
  if (rc != PV_OK) return rc;
  PV_REQUIRE(t_ids && save && psum && g && dlogits && K > 0 && K <= kTeacherMax, "pv_distill_rows_bwd: bad argument");
  const Rows a = make_rows(logits, n0, n1, s0, s1, V, nullptr, 0, inv_temp);
  return launch_grad<HEAD_DISTILL>(dtype, a, Distill{t_ids, nullptr, K, 0, (float*)psum, 0.f, 0.f},
                                   Grad{(const float4*)save, nullptr, nullptr, nullptr, 0.f, g, dlogits, ready}, (hipStream_t)stream);
}

size_t pv_colsum_scaled_ws_bytes(int V) { return V > 0 ? (size_t)kColShares * V * sizeof(float) : 0; }

int pv_colsum_scaled_bf16(const void* P, long ld, long T, int V, const float* g, float* out, void* ws, void* stream) {
  PV_REQUIRE(P && g && out && ws && T > 0 && V > 0 && ld >= V, "pv_colsum_scaled_bf16: bad argument");
  PV_REQUIRE(ld % 2 == 0 && ((uintptr_t)P & 3) == 0, "pv_colsum_scaled_bf16: rows must start at even elements");
  hipStream_t st = (hipStream_t)stream;
  colsum_part_kernel<<<dim3(cdiv(V, 128), kColShares), dim3(256), 0, st>>>((const uint32_t*)P, ld / 2, T, V, (float*)ws);
  PV_LAUNCH_CHECK("colsum_part_kernel");
  colsum_join_kernel<<<dim3(cdiv(V, 64)), dim3(64), 0, st>>>((const float*)ws, V, g, out);
  PV_LAUNCH_CHECK("colsum_join_kernel");
  return PV_OK;
}

int pv_gather_live_rows_bf16(const void* h, const int64_t* perm, const int* count, long rows, int H, void* out, void* stream) {
  PV_REQUIRE(h && perm && count && out && rows > 0 && rows <= 0x7fffffffL && H > 0, "pv_gather_live_rows_bf16: bad argument");
  PV_REQUIRE(H % 8 == 0 && ((uintptr_t)h & 15) == 0 && ((uintptr_t)out & 15) == 0,
             "pv_gather_live_rows_bf16: rows must be 16-byte aligned");
  const long n = rows * (H / 8), want = (n + 255) / 256;
  gather_live_kernel<<<dim3((unsigned)(want > 4096 ? 4096 : want)), dim3(256), 0, (hipStream_t)stream>>>(
      (const uint4*)h, perm, count, H / 8, n, (uint4*)out);
  PV_LAUNCH_CHECK("gather_live_kernel");
  return PV_OK;
}

int pv_scale_by_f32(float* x, long n, const float* g, void* stream) {
  PV_REQUIRE(x && g && n >= 0 && n % 4 == 0 && ((uintptr_t)x & 15) == 0, "pv_scale_by_f32: n must be a multiple of 4, x 16-byte aligned");
  if (n == 0) return PV_OK;
  const long want = (n / 4 + 255) / 256;
  scale_by_kernel<<<dim3((unsigned)(want > 1024 ? 1024 : want)), dim3(256), 0, (hipStream_t)stream>>>((float4*)x, n / 4, g);
  PV_LAUNCH_CHECK("scale_by_kernel");
  return PV_OK;
}

int pv_policy_tokens_fwd(const float* logp, const int64_t* tokens, int64_t ignore, long n0, int n1, const float* old_logp,
                         const float* ref_logp, const float* adv, int adv_per_token, float clip_lo, float clip_hi,
                         float kl_coef, float weight, int word, float* loss, float* stats, float* dlogp, void* ws, void* stream) {
  PV_REQUIRE(logp && tokens && old_logp && adv && loss && stats && ws && n0 > 0 && n1 > 0, "pv_policy_tokens_fwd: bad argument");
  PV_REQUIRE(clip_lo <= clip_hi, "pv_policy_tokens_fwd: the clip range is empty");
  hipStream_t st = (hipStream_t)stream;
  const long T = n0 * (long)n1;
  if (check_count("pv_policy_tokens_fwd", n0 > 0x7fffffffL ? n0 : T, 0x7fffffffL) != PV_OK) return PV_ERR_LIMIT;
  const Policy h = {old_logp, ref_logp, adv, adv_per_token, clip_lo, clip_hi, kl_coef, 0.f};
  const Result r = {kl_coef, 0.f, weight, word, loss, stats, dlogp ? dlogp + T : nullptr};
  const long want = T <= 4096 ? 1 : (T + 1023) / 1024;
  const int g = (int)(want > kSumGroups ? kSumGroups : want);
  policy_tokens_kernel<<<dim3(g), dim3(1024), 0, st>>>(logp, tokens, ignore, T, n1, h, dlogp, (Sum5*)ws, r);
  PV_LAUNCH_CHECK("policy_tokens_kernel");
  if (g > 1) {
    sum_parts_kernel<<<dim3(1), dim3(256), 0, st>>>((const Sum5*)ws, g, r);
    PV_LAUNCH_CHECK("sum_parts_kernel");
  }
  return PV_OK;
}

int pv_policy_tokens_bwd(const float* dlogp, const float* g, long n, float* d, void* stream) {
  PV_REQUIRE(dlogp && g && d && n > 0, "pv_policy_tokens_bwd: bad argument");
  const long want = (n + 255) / 256;
  policy_tokens_bwd_kernel<<<dim3((unsigned)(want > 2048 ? 2048 : want)), dim3(256), 0, (hipStream_t)stream>>>(
      dlogp, dlogp + n, g, n, d);
  PV_LAUNCH_CHECK("policy_tokens_bwd_kernel");
  return PV_OK;
}

int pv_preference_fwd(const float* logp_c, const float* ref_c, const int64_t* labels_c, int Lc, const float* logp_r,
                      const float* ref_r, const int64_t* labels_r, int Lr, long pairs, int64_t ignore, float beta,
                      float smoothing, float weight, float* loss, float* rewards, float* slope, void* ws, void* stream) {
  PV_REQUIRE(loss && rewards && slope && ws && pairs > 0 && Lc >= 0 && Lr >= 0, "pv_preference_fwd: bad argument");
  PV_REQUIRE((Lc == 0 || (logp_c && labels_c)) && (Lr == 0 || (logp_r && labels_r)), "pv_preference_fwd: null argument");
  if (check_count("pv_preference_fwd", pairs, kPairsMax) != PV_OK) return PV_ERR_LIMIT;
  hipStream_t st = (hipStream_t)stream;
  float4* rowout = (float4*)ws;
  preference_kernel<<<dim3((unsigned)pairs), dim3(256), 0, st>>>(Answers{logp_c, ref_c, labels_c, Lc},
                                                                 Answers{logp_r, ref_r, labels_r, Lr}, ignore, beta, smoothing,
                                                                 rewards, rewards + pairs, slope, rowout);
  PV_LAUNCH_CHECK("preference_kernel");
  return launch_sum(rowout, nullptr, 0, pairs, (Sum5*)(rowout + pairs), Result{0.f, 0.f, weight, 0, loss, nullptr, nullptr}, st);
}

int pv_preference_rows_fwd(const void* logits_c, int dtype_c, long pairs, int Lc, long s0c, long s1c, int Vc,
                           const int64_t* labels_c, const float* ref_c, const void* logits_r, int dtype_r, int Lr, long s0r,
                           long s1r, int Vr, const int64_t* labels_r, const float* ref_r, int64_t ignore, float inv_temp,
                           float beta, float smoothing, float weight, float* loss, float* rewards, float* slope, float* save_c,
                           float* save_r, void* ws, void* stream) {
  int rc = check_rows("pv_preference_rows_fwd", logits_c, dtype_c, pairs, Lc, s0c, s1c, Vc, inv_temp);
  if (rc == PV_OK) rc = check_rows("pv_preference_rows_fwd", logits_r, dtype_r, pairs, Lr, s0r, s1r, Vr, inv_temp);
  if (rc != PV_OK) return rc;
  PV_REQUIRE(labels_c && labels_r && loss && rewards && slope && ws, "pv_preference_rows_fwd: null argument");
  float* lp_c = (float*)((char*)ws + pv_vocab_rows_ws_bytes(pairs));
  float* lp_r = lp_c + pairs * Lc;
  const Rows c = make_rows(logits_c, pairs, Lc, s0c, s1c, Vc, labels_c, ignore, inv_temp);
  const Rows r = make_rows(logits_r, pairs, Lr, s0r, s1r, Vr, labels_r, ignore, inv_temp);
  const FwdOut oc = {lp_c, nullptr, nullptr, (float4*)save_c}, orr = {lp_r, nullptr, nullptr, (float4*)save_r};
  hipStream_t st = (hipStream_t)stream;
  if (share_a_launch(dtype_c, c, dtype_r, r)) {
    rc = dtype_c == PV_DTYPE_F32    ? launch_fwd_pair_typed<F32>(c, r, oc, orr, st)
         : dtype_c == PV_DTYPE_BF16 ? launch_fwd_pair_typed<BF16>(c, r, oc, orr, st)
                                    : launch_fwd_pair_typed<F16>(c, r, oc, orr, st);
  } else {
    rc = launch_fwd<HEAD_TOKEN, false>(dtype_c, c, Policy{}, Distill{}, Scale{}, oc, st);
    if (rc == PV_OK) rc = launch_fwd<HEAD_TOKEN, false>(dtype_r, r, Policy{}, Distill{}, Scale{}, orr, st);
  }
  if (rc != PV_OK) return rc;
  return pv_preference_fwd(lp_c, ref_c, labels_c, Lc, lp_r, ref_r, labels_r, Lr, pairs, ignore, beta, smoothing, weight, loss,
                           rewards, slope, ws, stream);
}

int pv_preference_rows_bwd(const void* logits_c, int dtype_c, long pairs, int Lc, long s0c, long s1c, int Vc,
                           const int64_t* labels_c, const void* logits_r, int dtype_r, int Lr, long s0r, long s1r, int Vr,
                           const int64_t* labels_r, int64_t ignore, float inv_temp, const float* save_c, const float* save_r,
                           const float* slope, float weight, const float* g, void* dlogits_c, void* dlogits_r, void* stream) {
  PV_REQUIRE(slope && g && (dlogits_c || dlogits_r), "pv_preference_rows_bwd: null argument");
  int rc = dlogits_c ? check_rows("pv_preference_rows_bwd", logits_c, dtype_c, pairs, Lc, s0c, s1c, Vc, inv_temp) : PV_OK;
  if (rc == PV_OK && dlogits_r) rc = check_rows("pv_preference_rows_bwd", logits_r, dtype_r, pairs, Lr, s0r, s1r, Vr, inv_temp);
  if (rc != PV_OK) return rc;
  PV_REQUIRE((!dlogits_c || (labels_c && save_c)) && (!dlogits_r || (labels_r && save_r)), "pv_preference_rows_bwd: null argument");
  const Rows c = make_rows(logits_c, pairs, Lc, s0c, s1c, Vc, labels_c, ignore, inv_temp);
  const Rows r = make_rows(logits_r, pairs, Lr, s0r, s1r, Vr, labels_r, ignore, inv_temp);
  const Grad qc = {(const float4*)save_c, nullptr, nullptr, slope, weight, g, dlogits_c, 0};
  const Grad qr = {(const float4*)save_r, nullptr, nullptr, slope, -weight, g, dlogits_r, 0};
  hipStream_t st = (hipStream_t)stream;
  if (dlogits_c && dlogits_r && share_a_launch(dtype_c, c, dtype_r, r))
    return dtype_c == PV_DTYPE_F32    ? launch_grad_pair_typed<F32>(c, r, qc, qr, st)
           : dtype_c == PV_DTYPE_BF16 ? launch_grad_pair_typed<BF16>(c, r, qc, qr, st)
                                      : launch_grad_pair_typed<F16>(c, r, qc, qr, st);
  if (dlogits_c) rc = launch_grad<HEAD_TOKEN>(dtype_c, c, Distill{}, qc, st);
  if (rc == PV_OK && dlogits_r) rc = launch_grad<HEAD_TOKEN>(dtype_r, r, Distill{}, qr, st);
  return rc;
}

int pv_preference_bwd(const int64_t* labels_c, int Lc, const int64_t* labels_r, int Lr, long pairs, int64_t ignore,
                      const float* slope, float weight, const float* g, float* dlogp_c, float* dlogp_r, void* stream) {
  PV_REQUIRE(slope && g && pairs > 0 && Lc >= 0 && Lr >= 0, "pv_preference_bwd: bad argument");
  PV_REQUIRE((Lc == 0 || (labels_c && dlogp_c)) && (Lr == 0 || (labels_r && dlogp_r)), "pv_preference_bwd: null argument");
  if (check_count("pv_preference_bwd", pairs, kPairsMax) != PV_OK) return PV_ERR_LIMIT;
  preference_bwd_kernel<<<dim3((unsigned)pairs), dim3(256), 0, (hipStream_t)stream>>>(labels_c, Lc, dlogp_c, labels_r, Lr, dlogp_r,
                                                                                      ignore, slope, weight, g);
  PV_LAUNCH_CHECK("preference_bwd_kernel");
  return PV_OK;
}

}  // extern "C"
