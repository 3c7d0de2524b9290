// KL divergence of one vocabulary row between a teacher known by a list of tokens and the student's full
// softmax q of x / T: the list, the student's sum without it, and the loss with its derivatives.
//
//   kind            loss                                                     dL/dz_listed      dL/dz_other
//   forward, tail   sum p (log p - log q) + t (log t - log s)                (P+t) q - p       (P+t - t/s) q
//   forward         sum w (log w - log q),  w = p / P                        q - w             q
//   reverse, tail   sum q (log q - log p) + s (log s - log t)                q (r - L)         q (log s/t - L)
//
// with P = sum p, t = 1 - P (at least 0; in the reverse form at least 2^-24, what a sum of fp32
// probabilities resolves), s the student's mass outside the list, r = log q - log p, z = x / T. The
// gradient of every other element is one number times q: the backward is a softmax pass and a patch of
// the listed elements. The row is summed without the listed elements, which join it in fp64: s is never
// 1 - sum q, which for a student that is sure of the listed tokens would be rounding noise, and log s, t / s
// and -log q with it (a loss of 1e-4 was off by 4e-4 where an fp32 sum held the listed elements too).
#pragma once
#include "list_rows.h"

namespace orlhf {

constexpr int kMaxList = 128;                 // two entries per lane of one wave
constexpr int64_t kMaxDistillVocab = 520192;  // a bit per element in 64 KiB of LDS, less the static part
constexpr double kTinyTail = 5.9604644775390625e-08;  // 2^-24
constexpr double kTinyRest = 1.1754943508222875e-38;       // 2^-126: the student's tail mass is taken to be at least that
constexpr double kLogTinyRest = -87.33654475055310898657;  // its logarithm

__device__ __forceinline__ double wave_max(double v) {
#pragma unroll
  for (int o = kWave / 2; o > 0; o >>= 1) {
    const double other = __shfl_xor(v, o, kWave);
    v = other > v ? other : v;
  }
  return v;
}

// Teacher's list of one row and the student's logits there, held by one wave: entry lane + 64 i. An entry
// with a negative id or a log-prob of -inf is absent, one past the vocabulary is absent and makes the
// loss NaN, an id that comes twice counts once with the sum of its probabilities.
struct ListEntries {
  int id[2];     // -1: absent
  float x[2];    // the student's logit
  double lp[2];  // the teacher's log-prob; where the list is renormalised relative to its largest value
  bool bad;
};

struct ListSource {
  const int64_t* ids;
  const float* teacher;
  int k;
  double inv_teacher_t;
  bool renormalise;  // the values are to go through a softmax: logits of any size
};

// The row's list as it stands in memory.
struct RawList {
  int64_t id[2];
  float value[2];
};
__device__ __forceinline__ RawList fetch_list(const ListSource& src, int64_t row_i) {
  RawList raw;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int at = (int)(threadIdx.x & (kWave - 1)) + i * kWave;
    raw.id[i] = at < src.k ? src.ids[row_i * src.k + at] : -1;
    raw.value[i] = at < src.k ? src.teacher[row_i * src.k + at] : -INFINITY;
  }
  return raw;
}

template <int DT>
__device__ __forceinline__ ListEntries settle_list(const RawList& raw, const ListSource& src, const char* row, int64_t vocab) {
  using E = Elt<DT>;
  const int lane = threadIdx.x & (kWave - 1);
  ListEntries e;
  e.bad = false;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const bool given = raw.id[i] >= 0 && raw.value[i] != -INFINITY;
    e.bad = e.bad || (given && raw.id[i] >= vocab);
    e.id[i] = given && raw.id[i] < vocab ? (int)raw.id[i] : -1;
    e.lp[i] = (double)raw.value[i] * src.inv_teacher_t;
    e.x[i] = e.id[i] >= 0 ? E::load1(row + (int64_t)e.id[i] * E::kSize) : 0.0f;
  }
  e.bad = __ballot(e.bad) != 0ull;
  if (src.renormalise) {  // the largest value comes off before anything is exponentiated
    const double a = e.id[0] >= 0 ? e.lp[0] : -INFINITY, b = e.id[1] >= 0 ? e.lp[1] : -INFINITY;
    const double top = wave_max(a > b ? a : b);
    e.lp[0] -= top, e.lp[1] -= top;
  }
  return e;
}

// Whether an id stands in the list more than once.
__device__ __forceinline__ bool list_repeats(const ListEntries& e, int k) {
  const int lane = threadIdx.x & (kWave - 1);
  bool again = false;
#pragma unroll 1
  for (int j = 0; j < k - 1; ++j) {
    const int other = j < kWave ? __builtin_amdgcn_readlane(e.id[0], j) : __builtin_amdgcn_readlane(e.id[1], j - kWave);
#pragma unroll
    for (int i = 0; i < 2; ++i) again = again || (e.id[i] == other && other >= 0 && lane + i * kWave > j);
  }
  return __ballot(again) != 0ull;
}

// Adds the probabilities of an id's later entries to its first, in their order, and drops them. Relative to the
// largest of them: the values may be logits of any size.
__device__ __forceinline__ void join_repeats(ListEntries& e, int k) {
  const int lane = threadIdx.x & (kWave - 1);
  auto each_twin = [&](auto&& f) {
#pragma unroll 1
    for (int j = 0; j < k; ++j) {
      const bool second = j >= kWave;
      const int other = __shfl(second ? e.id[1] : e.id[0], j & (kWave - 1), kWave);
      const double lp = __shfl(second ? e.lp[1] : e.lp[0], j & (kWave - 1), kWave);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int at = lane + i * kWave;
        if (other >= 0 && e.id[i] == other && at != j) f(i, at < j, lp);
      }
    }
  };
  double top[2] = {e.lp[0], e.lp[1]};
  bool more[2] = {false, false}, again[2] = {false, false};
  each_twin([&](int i, bool later, double lp) {
    if (later) more[i] = true;
    if (!later) again[i] = true;
    top[i] = lp > top[i] ? lp : top[i];
  });
  double sum[2] = {exp(e.lp[0] - top[0]), exp(e.lp[1] - top[1])};
  each_twin([&](int i, bool later, double lp) {
    if (later) sum[i] += exp(lp - top[i]);
  });
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (more[i]) e.lp[i] = top[i] + log(sum[i]);
    if (again[i]) e.id[i] = -1;
  }
}

template <int DT>
__device__ __forceinline__ ListEntries load_list(const ListSource& src, int64_t row_i, const char* row, int64_t vocab) {
  ListEntries e = settle_list<DT>(fetch_list(src, row_i), src, row, vocab);
  if (list_repeats(e, src.k)) join_repeats(e, src.k);
  return e;
}

// One bit per element of a row (or segment), set for the listed ones, in the order of the body's
// elements: a vector of 8 elements is a byte, one of 4 half a byte. The scalars at the row's ends have
// bits of their own behind it.
template <int DT>
struct ListMap {
  static constexpr int EPV = Elt<DT>::kPerVec;
  uint32_t* words;
  uint32_t* ends;  // one word
  static __host__ __device__ int64_t bytes(int64_t len) { return ((len + 127) / 128) * 16; }
  __device__ __forceinline__ void clear(const RowGeom& g, int threads) const {
    const uint32_t n16 = (g.nvec * EPV + 127u) / 128u;
    for (uint32_t i = threadIdx.x; i < n16; i += threads) ((u32x4*)words)[i] = u32x4{0u, 0u, 0u, 0u};
    if (threadIdx.x == 0) *ends = 0u;
  }
  __device__ __forceinline__ void set(const RowGeom& g, int64_t e, int64_t len) const {
    if (e < 0 || e >= len) return;
    const uint32_t i = (uint32_t)e, body = g.nvec * EPV;
    if (i < g.head) {
      atomicOr(ends, 1u << i);
    } else if (i - g.head >= body) {
      atomicOr(ends, 1u << (i - body));
    } else {
      atomicOr(words + (i - g.head) / 32u, 1u << ((i - g.head) % 32u));
    }
  }
  // Takes an element's bit, and those around it, out again (all bits set are taken out this way).
  __device__ __forceinline__ void drop(const RowGeom& g, uint32_t i) const {
    if (i >= g.head && i - g.head < g.nvec * EPV) words[(i - g.head) / 32u] = 0u;
  }
  __device__ __forceinline__ uint32_t vec(uint32_t v) const { return vec(v, 0u); }
  // Of vector v + step, step a known even number: it stays an offset in the instruction.
  __device__ __forceinline__ uint32_t vec(uint32_t v, uint32_t step) const {
    const uint8_t* b = (const uint8_t*)words;
    return EPV == 8 ? (b + v)[step] : (uint32_t)((b + (v >> 1))[step >> 1] >> ((v & 1u) * 4u)) & 0xfu;
  }
  __device__ __forceinline__ bool scalar(uint32_t s) const { return (*ends >> s & 1u) != 0u; }
};

// Takes the listed elements out of the sums: their weight becomes that of -inf.
template <int DT>
struct WithoutListed {
  ListMap<DT> map;
  template <int N>
  __device__ __forceinline__ void vec(float (&x)[N], uint32_t v, uint32_t step = 0u) const {
    const uint32_t bits = map.vec(v, step);
    if (__ballot(bits != 0u) != 0ull) {  // a branch of the wave, hardly ever taken
#pragma unroll
      for (int j = 0; j < N; ++j) x[j] = (bits >> j & 1u) != 0u ? -INFINITY : x[j];
    }
  }
  __device__ __forceinline__ void one(float& x, uint32_t s) const {
    if (map.scalar(s)) x = -INFINITY;
  }
};

// What the loss takes from the teacher alone and from the student's listed logits alone: each one wave's
// work that does not wait for the row.
struct TeacherTerms {
  double p[2];  // of this lane's entries, 0 where absent; for the kind without a tail up to the factor 1 / mass
  double mass, t, log_t, log_mass;
  int n_on;
};
__device__ __forceinline__ TeacherTerms teacher_terms(const ListEntries& e, int kind, int64_t vocab) {
  TeacherTerms r;
  r.n_on = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    r.n_on += __popcll(__ballot(e.id[i] >= 0));
    r.p[i] = e.id[i] >= 0 ? exp(e.lp[i]) : 0.0;
  }
  r.mass = wave_sum(r.p[0] + r.p[1]);
  const bool tail = kind != ORLHF_DISTILL_FORWARD && r.n_on < vocab;
  r.t = tail ? fmax(1.0 - r.mass, kind == ORLHF_DISTILL_REVERSE_TAIL ? kTinyTail : 0.0) : 0.0;
  r.log_t = log(r.t);  // used where t > 0
  r.log_mass = kind == ORLHF_DISTILL_FORWARD ? log(r.mass) : 0.0;
  return r;
}

struct StudentTerms {
  double top, sum;  // sum exp(x / T - top) over the list
};
__device__ __forceinline__ StudentTerms student_terms(const ListEntries& e, double inv_t) {
  double z[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) z[i] = e.id[i] >= 0 ? (double)e.x[i] * inv_t : -INFINITY;
  StudentTerms r;
  r.top = wave_max(z[0] > z[1] ? z[0] : z[1]);
  double own = 0.0;
#pragma unroll
  for (int i = 0; i < 2; ++i) own += e.id[i] >= 0 ? (z[i] == r.top ? 1.0 : exp(z[i] - r.top)) : 0.0;
  r.sum = wave_sum(own);
  return r;
}

// The backward of the unlisted elements goes by r = q / s, the softmax outside the list: its weights are in
// range however small s is. By q, a student that is sure by more than 75 nats lost the pull of the teacher's
// tail, t r, to weights below 2^-126.
struct ListTerms {
  double loss, other;  // the loss and dL/dz / r of an element that is not listed
  double grad[2];      // dL/dz of this lane's entries (0 where absent)
  float centre, l2;    // r = 2^((x - centre) cT - l2)
};

// One wave. `sum`: the student's softmax sum without the listed elements. fp64: a few hundred operations of
// one wave per row.
__device__ __forceinline__ ListTerms list_terms(const ListEntries& e, const TeacherTerms& teacher, const StudentTerms& student,
                                                const RowTotals& sum, int kind, double temperature, int64_t vocab) {
  ListTerms r;
  const double inv_t = 1.0 / temperature;
  const bool tail = kind != ORLHF_DISTILL_FORWARD;
  const bool some = sum.sT > 0.0 || sum.sT != sum.sT;  // anything of weight outside the list
  const double rest_base = some ? sum.base_t : -INFINITY, base = student.top > rest_base ? student.top : rest_base;
  const double listed = student.sum * (student.top == base ? 1.0 : exp(student.top - base));
  const double total =
      (some ? sum.sT * (rest_base == base ? 1.0 : exp(rest_base - base)) : 0.0) + (teacher.n_on > 0 ? listed : 0.0);
  const double log_total = sum.nan ? (double)NAN : log(total);
  double lq[2], q[2], part[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    lq[i] = ((double)e.x[i] * inv_t - base) - log_total;
    q[i] = e.id[i] >= 0 ? exp(lq[i]) : 0.0;
  }
  const double log_rest = log(sum.sT);
  double log_s = some ? (sum.base_t - base) + log_rest - log_total : -INFINITY;
  const double s = exp(log_s), t = teacher.t;
  double pull = t;  // t q / s at the least s, in units of r
  if (log_s < kLogTinyRest) pull = t * exp(log_s - kLogTinyRest), log_s = kLogTinyRest;
  if (kind == ORLHF_DISTILL_REVERSE_TAIL) {
#pragma unroll
    for (int i = 0; i < 2; ++i) part[i] = e.id[i] >= 0 && q[i] != 0.0 ? q[i] * (lq[i] - e.lp[i]) : 0.0;
    r.loss = wave_sum(part[0] + part[1]) + (t > 0.0 ? fmax(s, kTinyRest) * (log_s - teacher.log_t) : 0.0);
    r.other = s * ((log_s - teacher.log_t) - r.loss);
#pragma unroll
    for (int i = 0; i < 2; ++i) r.grad[i] = part[i] - q[i] * r.loss;
  } else {
    const double scale = tail ? 1.0 : 1.0 / teacher.mass, all = tail ? teacher.mass + t : 1.0;
    r.other = all * s - pull;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const double p = teacher.p[i] * scale;
      part[i] = p != 0.0 ? p * (e.lp[i] - teacher.log_mass - lq[i]) : 0.0;
      r.grad[i] = e.id[i] >= 0 ? all * q[i] - p : 0.0;
    }
    r.loss = wave_sum(part[0] + part[1]) + (t > 0.0 ? t * (teacher.log_t - log_s) : 0.0);
  }
  const double at = sum.base_t * temperature;
  r.centre = (float)at;
  r.l2 = (float)((log_rest + (at - (double)r.centre) * inv_t) * 1.4426950408889634);
  if (teacher.n_on == 0) r.loss = 0.0;  // nothing to learn from: no loss, no gradient
  if (teacher.n_on == 0 || !some) {
    r.centre = INFINITY;  // every weight of the backward 0
    r.l2 = 0.0f;
    r.other = teacher.n_on > 0 && base == -INFINITY ? NAN : 0.0;  // nothing but -inf in the row: no softmax
  }
  if (e.bad) r.loss = NAN;
  return r;
}

// All of it at once.
__device__ __forceinline__ ListTerms list_terms(const ListEntries& e, const RowTotals& sum, int kind, double temperature,
                                                int64_t vocab) {
  return list_terms(e, teacher_terms(e, kind, vocab), student_terms(e, 1.0 / temperature), sum, kind, temperature, vocab);
}

// Coefficient of the softmax weight in an element's gradient. A weight that is 0 has to stay 0.
__device__ __forceinline__ float grad_coef(double upstream, double other, double temperature) {
  const double a = upstream * other / temperature;
  return (float)(a > 3.0e38 ? 3.0e38 : (a < -3.0e38 ? -3.0e38 : a));
}

// ---------------------------------------------------------------- host side
inline int check_distill(const char* what, int dtype, int64_t n_rows, int64_t vocab, int64_t row_stride, int64_t k,
                         double temperature) {
  ORLHF_CHECK_ARG(n_rows >= 0 && vocab > 0, "%s: n_rows=%lld vocab=%lld", what, (long long)n_rows, (long long)vocab);
  ORLHF_CHECK_ARG(row_stride >= vocab, "%s: row_stride %lld < vocab %lld", what, (long long)row_stride, (long long)vocab);
  if (vocab > kMaxDistillVocab)
    return fail(ORLHF_ERR_UNSUPPORTED, "%s: vocab %lld, rows beyond %lld elements are not implemented", what,
                (long long)vocab, (long long)kMaxDistillVocab);
  ORLHF_CHECK_ARG(temperature > 0.0 && temperature < INFINITY, "%s: temperature must be > 0 and finite", what);
  ORLHF_CHECK_ARG(dtype == ORLHF_F32 || dtype == ORLHF_BF16 || dtype == ORLHF_F16, "%s: unknown dtype %d", what, dtype);
  ORLHF_CHECK_ARG(k >= 1 && k <= kMaxList, "%s: k=%lld must lie in 1..%d", what, (long long)k, kMaxList);
  return ORLHF_OK;
}

inline int check_kind(const char* what, int kind, double teacher_temperature) {
  ORLHF_CHECK_ARG(kind >= ORLHF_DISTILL_FORWARD_TAIL && kind <= ORLHF_DISTILL_REVERSE_TAIL, "%s: unknown kind %d", what, kind);
  ORLHF_CHECK_ARG(teacher_temperature > 0.0 && teacher_temperature < INFINITY,
                  "%s: teacher_temperature must be > 0 and finite", what);
  ORLHF_CHECK_ARG(kind == ORLHF_DISTILL_FORWARD || teacher_temperature == 1.0,
                  "%s: a kind with a tail takes log-probs as they are (teacher_temperature 1)", what);
  return ORLHF_OK;
}

}  // namespace orlhf
