// Shared pieces of the vocabulary-row kernels: element traits (bf16 / fp16 / fp32 as 16-byte
// vectors), row geometry, statistic modes, the per-element gradient, and the streaming pass of one
// 256-thread workgroup over a row with its softmax accumulators.
#pragma once
#include "common.h"

#ifndef ORLHF_NT_LOAD
#define ORLHF_NT_LOAD 1
#endif
#ifndef ORLHF_ROW_UNROLL
#define ORLHF_ROW_UNROLL 8
#endif
#ifndef ORLHF_NT_STORE
#define ORLHF_NT_STORE 1
#endif

namespace orlhf {

constexpr int64_t kIgnoredLabel = -100;  // its log-prob is the constant 0, without a gradient

// ---------------------------------------------------------------- element traits
template <int DT>
struct Elt;

template <>
struct Elt<ORLHF_BF16> {
  static constexpr int kSize = 2;
  static constexpr int kPerVec = 8;
  static __device__ __forceinline__ void unpack(const u32x4& r, float (&x)[8]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      x[2 * k] = bf16_lo(r[k]);
      x[2 * k + 1] = bf16_hi(r[k]);
    }
  }
  static __device__ __forceinline__ u32x4 pack(const float (&x)[8]) {
    u32x4 r;
#pragma unroll
    for (int k = 0; k < 4; ++k) r[k] = pack_bf16(x[2 * k], x[2 * k + 1]);
    return r;
  }
  static __device__ __forceinline__ float load1(const char* p) {
    return __builtin_bit_cast(float, (uint32_t)(*(const uint16_t*)p) << 16);
  }
  static __device__ __forceinline__ void store1(char* p, float v) {
    *(uint16_t*)p = (uint16_t)(pack_bf16(v, 0.0f) & 0xffffu);
  }
  static __device__ __forceinline__ float round(float v) { return bf16_lo(pack_bf16(v, 0.0f)); }
};

template <>
struct Elt<ORLHF_F16> {
  static constexpr int kSize = 2;
  static constexpr int kPerVec = 8;
  static __device__ __forceinline__ void unpack(const u32x4& r, float (&x)[8]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t w = r[k];  // by value: a vector lane is not addressable
      f16x2 h = __builtin_bit_cast(f16x2, w);
      x[2 * k] = (float)h[0];
      x[2 * k + 1] = (float)h[1];
    }
  }
  static __device__ __forceinline__ u32x4 pack(const float (&x)[8]) {
    u32x4 r;
#pragma unroll
    for (int k = 0; k < 4; ++k) r[k] = pack_f16(x[2 * k], x[2 * k + 1]);
    return r;
  }
  static __device__ __forceinline__ float load1(const char* p) { return (float)(*(const _Float16*)p); }
  static __device__ __forceinline__ void store1(char* p, float v) { *(_Float16*)p = (_Float16)v; }
  static __device__ __forceinline__ float round(float v) { return (float)(_Float16)v; }
};

template <>
struct Elt<ORLHF_F32> {
  static constexpr int kSize = 4;
  static constexpr int kPerVec = 4;
  static __device__ __forceinline__ void unpack(const u32x4& r, float (&x)[4]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = as_float(r[k]);  // by value: a vector lane is not addressable
  }
  static __device__ __forceinline__ u32x4 pack(const float (&x)[4]) {
    u32x4 r;
#pragma unroll
    for (int k = 0; k < 4; ++k) r[k] = as_uint(x[k]);
    return r;
  }
  static __device__ __forceinline__ float load1(const char* p) { return *(const float*)p; }
  static __device__ __forceinline__ void store1(char* p, float v) { *(float*)p = v; }
  static __device__ __forceinline__ float round(float v) { return v; }
};

__device__ __forceinline__ u32x4 load_vec(const char* p) {
#if ORLHF_NT_LOAD
  return __builtin_nontemporal_load((const u32x4*)p);
#else
  return *(const u32x4*)p;
#endif
}
__device__ __forceinline__ void store_vec(char* p, const u32x4& v) {
#if ORLHF_NT_STORE
  __builtin_nontemporal_store(v, (u32x4*)p);
#else
  *(u32x4*)p = v;
#endif
}

// ---------------------------------------------------------------- row geometry + traversal
// A row is split into a scalar head (elements before the first 16-byte boundary), a body of
// 16-byte vectors and a scalar tail, so any vocab size, row stride and base alignment works.
// `scalar_only` (host decision: input and output rows are misaligned differently) turns the
// whole row into the scalar part.
struct RowGeom {
  uint32_t head, nvec, tail;  // element / vector counts; a row is < 2 GiB (host check)
};

template <int DT>
__device__ __forceinline__ RowGeom row_geom(const char* row, int64_t vocab, bool scalar_only) {
  using E = Elt<DT>;
  RowGeom g;
  if (scalar_only) {
    g.head = (uint32_t)vocab;
    g.nvec = 0;
    g.tail = 0;
    return g;
  }
  const uint32_t mis = (uint32_t)((uintptr_t)row & 15u);
  uint32_t head = mis ? (16u - mis) / E::kSize : 0u;
  if (head > (uint32_t)vocab) head = (uint32_t)vocab;
  g.head = head;
  g.nvec = ((uint32_t)vocab - head) / E::kPerVec;
  g.tail = (uint32_t)vocab - head - g.nvec * E::kPerVec;
  return g;
}

// ---------------------------------------------------------------- forward accumulators
// Modes: which statistics a row needs.
//   kLpOnly   : sum exp(z - m)                      z = x / T
//   kEntOnly  : sum exp(x - m), sum exp(x - m) * x
//   kBothT1   : T == 1, one shared set
//   kBothT    : T != 1, scaled set for the log-prob and unscaled set for the entropy
enum FwdMode { kLpOnly = 0, kEntOnly = 1, kBothT1 = 2, kBothT = 3 };

template <int MODE>
struct ModeTraits {
  static constexpr bool kScaledSet = (MODE == kLpOnly || MODE == kBothT);  // separate x/T set
  static constexpr bool kPlainSet = (MODE != kLpOnly);                     // unscaled set (+ sum e*x)
};

// ---------------------------------------------------------------- gradient of one element
enum BwdMode { kBwdLp = 0, kBwdEnt = 1, kBwdBothT1 = 2, kBwdBothT = 3 };

template <int MODE>
struct GradFn {
  float cT, negLT, c1, negL1;  // exponents: x*c - lse*log2e
  float a_lp;                  // -g_lp / T          (coefficient of softmax(z))
  float gh, k1;                // entropy term p*(k1 - gh*x); k1 = gh*E (- g_lp when T == 1)
  float onehot;                // g_lp / T
  uint32_t label_vec;          // body vector holding the label (0xffffffff: none)
  uint32_t label_lane;         // its position inside that vector
  uint32_t label_elem;         // the label as an element index (0xffffffff: out of range)
  __device__ __forceinline__ float elem(float x) const {
    if (MODE == kBwdLp) return fast_exp2(fmaf(x, cT, negLT)) * a_lp;
    if (MODE == kBwdEnt || MODE == kBwdBothT1) return fast_exp2(fmaf(x, c1, negL1)) * fmaf(-gh, x, k1);
    const float pt = fast_exp2(fmaf(x, cT, negLT));
    const float p1 = fast_exp2(fmaf(x, c1, negL1));
    return fmaf(pt, a_lp, p1 * fmaf(-gh, x, k1));
  }
  template <int N>
  __device__ __forceinline__ void vec(float (&x)[N], uint32_t v) const {
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = elem(x[j]);
    if (MODE != kBwdEnt && v == label_vec) {
#pragma unroll
      for (int j = 0; j < N; ++j) x[j] += ((uint32_t)j == label_lane) ? onehot : 0.0f;
    }
  }
  __device__ __forceinline__ void one(float& x, uint32_t e) const {
    x = elem(x);
    if (MODE != kBwdEnt && e == label_elem) x += onehot;
  }
  __device__ __forceinline__ void set_label(int64_t label, int64_t vocab, const RowGeom& g, int epv) {
    label_vec = label_lane = label_elem = 0xffffffffu;
    if (label < 0 || label >= vocab) return;
    label_elem = (uint32_t)label;
    if (label_elem >= g.head && label_elem < g.head + g.nvec * (uint32_t)epv) {
      label_vec = (label_elem - g.head) / (uint32_t)epv;
      label_lane = (label_elem - g.head) % (uint32_t)epv;
    }
  }
};

// ---------------------------------------------------------------- streaming pass over a row
// Visits every element of a row exactly once. f.vec(x, v) gets the kPerVec consecutive elements
// of body vector v (element index head + v*kPerVec); f.one(x, e) gets element e. With STORE the
// (modified) values are written to out_row at the same element positions in the same dtype.
// All in-row offsets are 32-bit: the row base stays in scalar registers.
template <int DT, bool STORE, typename F>
__device__ __forceinline__ void traverse_row(const char* row, char* out_row, const RowGeom& g,
                                             F& f) {
  using E = Elt<DT>;
  constexpr uint32_t U = ORLHF_ROW_UNROLL;
  constexpr uint32_t EPV = E::kPerVec;
  const uint32_t tid = threadIdx.x;
  const char* body = row + g.head * E::kSize;
  char* obody = STORE ? out_row + g.head * E::kSize : nullptr;

  const uint32_t nbatch = g.nvec / (kBlock * U);
  uint32_t v0 = tid;
  for (uint32_t b = 0; b < nbatch; ++b, v0 += kBlock * U) {
    u32x4 buf[U];
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) buf[u] = load_vec(body + (v0 + u * kBlock) * 16u);
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      float x[EPV];
      E::unpack(buf[u], x);
      f.vec(x, v0 + u * kBlock);
      if (STORE) store_vec(obody + (v0 + u * kBlock) * 16u, E::pack(x));
    }
  }
  if (v0 < g.nvec) {  // last, partial batch: same loads in flight, predicated per vector
    u32x4 buf[U];
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      const uint32_t v = v0 + u * kBlock;
      if (v < g.nvec) buf[u] = load_vec(body + v * 16u);
    }
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      const uint32_t v = v0 + u * kBlock;
      if (v < g.nvec) {
        float x[EPV];
        E::unpack(buf[u], x);
        f.vec(x, v);
        if (STORE) store_vec(obody + v * 16u, E::pack(x));
      }
    }
  }
  // scalar head + tail (at most 2*(kPerVec-1) elements unless scalar_only)
  const uint32_t nscalar = g.head + g.tail;
  for (uint32_t k = tid; k < nscalar; k += kBlock) {
    const uint32_t e = k < g.head ? k : g.head + g.nvec * EPV + (k - g.head);
    float x = E::load1(row + e * E::kSize);
    f.one(x, e);
    if (STORE) E::store1(out_row + e * E::kSize, x);
  }
}

constexpr int kAcc = 4;  // independent accumulators per lane

// Fast path: exponent = x*c - M with a wave-uniform reference M (no running maximum).
template <int MODE, int ACC = kAcc>
struct FastAcc {
  float cT, negMT, c1, negM1;
  float sT[ACC], s1[ACC], t1[ACC];
  __device__ __forceinline__ void init(float m_ref, float c_scaled, float c_plain) {
    cT = c_scaled;
    c1 = c_plain;
    negMT = -(m_ref * c_scaled);
    negM1 = -(m_ref * c_plain);
#pragma unroll
    for (int k = 0; k < ACC; ++k) sT[k] = s1[k] = t1[k] = 0.0f;
  }
  __device__ __forceinline__ void elem(float x, int k) {
    if (ModeTraits<MODE>::kScaledSet) sT[k] += fast_exp2(fmaf(x, cT, negMT));
    if (ModeTraits<MODE>::kPlainSet) {
      const float e = fast_exp2(fmaf(x, c1, negM1));
      s1[k] += e;
      t1[k] = fmaf(e, x, t1[k]);
    }
  }
  template <int N>
  __device__ __forceinline__ void vec(float (&x)[N], uint32_t) {
#pragma unroll
    for (int j = 0; j < N; ++j) elem(x[j], j % ACC);
  }
  __device__ __forceinline__ void one(float& x, uint32_t) { elem(x, 0); }
  __device__ __forceinline__ void fold(float& st, float& s, float& t) const {
    static_assert(ACC == 2 || ACC == 4, "fold adds pairs");
    if (ACC == 4) {
      st = (sT[0] + sT[1]) + (sT[ACC - 2] + sT[ACC - 1]);
      s = (s1[0] + s1[1]) + (s1[ACC - 2] + s1[ACC - 1]);
      t = (t1[0] + t1[1]) + (t1[ACC - 2] + t1[ACC - 1]);
    } else {
      st = sT[0] + sT[1];
      s = s1[0] + s1[1];
      t = t1[0] + t1[1];
    }
  }
};

// Safe path: per-lane running maximum m (raw logit units), sums relative to it.
template <int MODE>
struct SafeAcc {
  float cT, c1;
  float m, sT, s1, t1;
  __device__ __forceinline__ void init(float c_scaled, float c_plain) {
    cT = c_scaled;
    c1 = c_plain;
    m = -INFINITY;
    sT = s1 = t1 = 0.0f;
  }
  __device__ __forceinline__ void raise(float cm) {
    if (cm > m) {  // also true for the first finite element (m == -inf)
      if (m != -INFINITY) {
        const float d = m - cm;  // < 0, or -inf when cm == +inf
        if (ModeTraits<MODE>::kScaledSet) sT *= fast_exp2(d * cT);
        if (ModeTraits<MODE>::kPlainSet) {
          const float r = fast_exp2(d * c1);
          s1 *= r;
          t1 *= r;
        }
      }
      m = cm;
    }
  }
  __device__ __forceinline__ void elem(float x) {
    if (m == -INFINITY) {
      // only -inf (or NaN) seen so far: exp() contributes 0 to the sums, but the reference's
      // softmax(x)*x is 0 * -inf = NaN for such an element (a NaN logit poisons everything).
      if (ModeTraits<MODE>::kPlainSet) t1 = NAN;
      if (x != x) sT = s1 = NAN;
      return;
    }
    // x == m covers m == +inf (inf - inf would be NaN): such an element counts as exp(0),
    // which makes logsumexp +inf and the entropy NaN, as in the reference
    const float d = (x == m) ? 0.0f : x - m;
    if (ModeTraits<MODE>::kScaledSet) sT += fast_exp2(d * cT);
    if (ModeTraits<MODE>::kPlainSet) {
      const float e = fast_exp2(d * c1);
      s1 += e;
      t1 = fmaf(e, x, t1);
    }
  }
  template <int N>
  __device__ __forceinline__ void vec(float (&x)[N], uint32_t) {
    float cm = x[0];
#pragma unroll
    for (int j = 1; j < N; ++j) cm = fmaxf(cm, x[j]);
    raise(cm);
#pragma unroll
    for (int j = 0; j < N; ++j) elem(x[j]);
  }
  __device__ __forceinline__ void one(float& x, uint32_t) {
    raise(x);
    elem(x);
  }
};

// Workgroup-combined sums. Fast pass: exponents were x*c - M, MT / M1 hold M (log2 units).
// Safe pass: exponents were (x - m)*c, MT and M1 both hold the row maximum m (logit units).
struct RowSums {
  float MT, sT, M1, s1, t1;
};

__device__ __forceinline__ bool sums_usable(float s) { return s > 0.0f && s < INFINITY; }

// Zero-fills a row without reading it.
template <int DT>
__device__ __forceinline__ void zero_row(char* out_row, const RowGeom& g) {
  using E = Elt<DT>;
  const uint32_t tid = threadIdx.x;
  char* obody = out_row + g.head * E::kSize;
  const u32x4 z = {0u, 0u, 0u, 0u};
  for (uint32_t v = tid; v < g.nvec; v += kBlock) store_vec(obody + v * 16u, z);
  const uint32_t nscalar = g.head + g.tail;
  for (uint32_t k = tid; k < nscalar; k += kBlock) {
    const uint32_t e = k < g.head ? k : g.head + g.nvec * E::kPerVec + (k - g.head);
    E::store1(out_row + e * E::kSize, 0.0f);
  }
}

inline int grid_for_rows(int64_t n_rows) {
  // one workgroup per row; cap the grid and stride over rows beyond it
  const int64_t cap = 1 << 20;
  return (int)(n_rows < cap ? n_rows : cap);
}

}  // namespace orlhf
