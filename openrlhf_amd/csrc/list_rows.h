// What the operators over vocabulary rows with a list of tokens share: the softmax of a row (fast pass,
// exact pass, fp64 epilogue), the gradient of an element, and rows cut into segments.
#pragma once
#include "vocab_rows.h"

namespace orlhf {

// One workgroup per row (or segment) and no loop over rows in the kernels: a loop makes the compiler keep the
// constants of the whole body (of the logarithms above all) in registers, 20 to 30 per lane.
constexpr int64_t kGridX = 1 << 20;
inline dim3 row_grid(int64_t n_rows) {
  return dim3((unsigned)(n_rows < kGridX ? n_rows : kGridX), (unsigned)((n_rows + kGridX - 1) / kGridX));
}
__device__ __forceinline__ int64_t grid_row() { return (int64_t)blockIdx.y * kGridX + blockIdx.x; }

// The softmax of a row as what its outputs and its backward need: base + log_sum is the
// log-sum-exp of x / T (kept apart: base may be so large that the sum would be lost in it), `centre`
// a logit near base * T that every later difference starts from, entropy and E[x] - centre those of
// the unscaled logits.
struct RowSoftmax {
  double base, log_sum, entropy;
  float centre, l2_t, l2_1, ex;  // the backward's statistics: softmax(x / T) = 2^((x - centre) cT - l2_t)
};

// Two accumulators per sum: the waves of six workgroups per CU hide the rest of the adders' latency, and
// the registers of a third and fourth would cost one of the six.
template <int MODE>
struct ListAcc : FastAcc<MODE, 2> {
  // The sums so far are taken as used here, by no instruction: the compiler otherwise moves the
  // exponentials of several vectors behind the next branch and keeps all their elements until then.
  __device__ __forceinline__ void settle() {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (ModeTraits<MODE>::kScaledSet) asm volatile("" : "+v"(this->sT[k]));
      if (ModeTraits<MODE>::kPlainSet) asm volatile("" : "+v"(this->s1[k]), "+v"(this->t1[k]));
    }
  }
};

// Fast pass: per wave sums against its reference, folded over the workgroup.
template <int MODE>
__device__ __forceinline__ RowSums combine_fast(const ListAcc<MODE>& acc, float (*lds)[8]) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  float st, s, t;
  acc.fold(st, s, t);
  st = wave_sum(st);
  s = wave_sum(s);
  t = wave_sum(t);
  if (lane == 0) {
    lds[wave][0] = -acc.negMT;
    lds[wave][1] = st;
    lds[wave][2] = -acc.negM1;
    lds[wave][3] = s;
    lds[wave][4] = t;
  }
  __syncthreads();
  RowSums r;
  r.MT = lds[0][0], r.M1 = lds[0][2];
#pragma unroll
  for (int w = 1; w < kWavesPerBlock; ++w) {
    r.MT = fmaxf(r.MT, lds[w][0]);
    r.M1 = fmaxf(r.M1, lds[w][2]);
  }
  r.sT = r.s1 = r.t1 = 0.0f;
#pragma unroll
  for (int w = 0; w < kWavesPerBlock; ++w) {
    r.sT = fmaf(lds[w][1], fast_exp2(lds[w][0] - r.MT), r.sT);
    const float q = fast_exp2(lds[w][2] - r.M1);
    r.s1 = fmaf(lds[w][3], q, r.s1);
    r.t1 = fmaf(lds[w][4], q, r.t1);
  }
  __syncthreads();
  return r;
}

// The fast pass of a workgroup over a row. The loads of the next step are in flight while one is worked
// on: two steps of registers, 16 KiB asked for ahead by each workgroup at any time. The vectors past the
// last whole step come first, so that the loop has no predicated step (after one the compiler waits for
// every load before it issues the next). The wave's exponent reference is the maximum of its lanes' first
// vectors. `watch` sees every vector before the sums do (and may change it), the scalars at a row's ends,
// and, where it wants them, the maxima of each step; ready() is called once the first loads are on their way.
constexpr uint32_t kStepVecs = 4;  // vectors per lane and step

template <int DT, int MODE, typename W>
__device__ __forceinline__ void stream_row(const char* row, const RowGeom& g, float c_scaled, ListAcc<MODE>& acc, W& watch) {
  using E = Elt<DT>;
  constexpr int EPV = E::kPerVec;
  constexpr uint32_t kStep = kStepVecs * kBlock;
  const uint32_t tid = threadIdx.x;
  const char* body = row + g.head * E::kSize;
  const uint32_t whole = g.nvec / kStep, rest = g.nvec - whole * kStep;
  auto load = [&](u32x4 (&raw)[kStepVecs], uint32_t step) {
    const uint32_t at = step * (kStep * 16u) + tid * 16u;
#pragma unroll
    for (uint32_t u = 0; u < kStepVecs; ++u) raw[u] = load_vec(body + (at + u * (kBlock * 16u)));
    __builtin_amdgcn_sched_barrier(0);  // all of them issued before the work on the step at hand
  };
  auto unpacked = [&](const u32x4& raw, float (&x)[EPV], uint32_t v) {
    uint32_t w0 = raw[0], w1 = raw[1], w2 = raw[2], w3 = raw[3];
    asm volatile("" : "+v"(w0), "+v"(w1), "+v"(w2), "+v"(w3));  // unpacked here, not ahead for several vectors
    E::unpack(u32x4{w0, w1, w2, w3}, x);
    watch.vec(x, v);
  };
  auto take = [&](const u32x4& raw, float& m, uint32_t v) {
    float x[EPV];
    unpacked(raw, x, v);
    if (W::kMaxima) {
#pragma unroll
      for (int j = 0; j < EPV; ++j) m = fmaxf(m, x[j]);
    }
    acc.vec(x, 0);
    acc.settle();  // one vector's values at a time: registers decide how many rows a CU holds
  };
  auto consume = [&](const u32x4 (&raw)[kStepVecs], uint32_t step) {
    float m[kStepVecs] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (uint32_t u = 0; u < kStepVecs; ++u) take(raw[u], m[u], step * kStep + u * kBlock + tid);
    if constexpr (W::kMaxima) watch.note(step, whole, rest, m);
  };

  u32x4 ping[kStepVecs], pong[kStepVecs];
#pragma unroll
  for (uint32_t u = 0; u < kStepVecs; ++u)
    if (u * kBlock + tid < rest) pong[u] = load_vec(body + (whole * kStep + u * kBlock + tid) * 16u);
  if (whole > 0) load(ping, 0);
  // head and tail of a row off the 16-byte grid: at most one element per thread
  const uint32_t nscalar = g.head + g.tail;
  float xs = -INFINITY;
  if (tid < nscalar) xs = E::load1(row + (tid < g.head ? tid : g.nvec * EPV + tid) * E::kSize);
  watch.ready();
  if (tid < nscalar) watch.one(xs, tid);
  float m_ref = xs;
  auto raise = [&](const u32x4& raw, uint32_t v) {
    float x[EPV];
    unpacked(raw, x, v);
#pragma unroll
    for (int j = 0; j < EPV; ++j) m_ref = fmaxf(m_ref, x[j]);
  };
  if (tid < rest) raise(pong[0], whole * kStep + tid);
  if (whole > 0) raise(ping[0], tid);
  acc.init(wave_max(m_ref), c_scaled, kLog2e);
  if (tid < nscalar) acc.one(xs, 0);
  if (rest > 0) {
    float m[kStepVecs] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (uint32_t u = 0; u < kStepVecs; ++u)
      if (u * kBlock + tid < rest) take(pong[u], m[u], whole * kStep + u * kBlock + tid);
    if constexpr (W::kMaxima) watch.note(whole, whole, rest, m);
  }
  if (whole == 0) return;
  uint32_t step = 0;
  for (; step + 2 < whole; step += 2) {
    load(pong, step + 1);
    consume(ping, step);
    load(ping, step + 2);
    consume(pong, step + 1);
  }
  if (step + 1 < whole) {
    load(pong, step + 1);
    consume(ping, step);
    consume(pong, step + 1);
  } else {
    consume(ping, step);
  }
}

// Rows whose fast sums are not usable (an element some 88 nats above the references, logits at the
// lowest values of their type, inf, NaN) or would lose digits (references so far from 0 that the
// roundings of x c, which grow with |x|, reach 2^-16 and the entropy's with it): the exact maximum
// first, then sums of the differences to it.
constexpr float kFarReference = 256.0f;  // log2 units

struct MaxAcc {
  float m;
  bool nan;
  __device__ __forceinline__ void one(float& x, uint32_t) {
    m = fmaxf(m, x);
    nan = nan || x != x;
  }
  template <int N>
  __device__ __forceinline__ void vec(float (&x)[N], uint32_t v) {
#pragma unroll
    for (int j = 0; j < N; ++j) one(x[j], v);
  }
};
template <int MODE>
struct ExactAcc {
  float m, cT, c1, sT, s1, t1;  // t1: sum of e (x - m); an element of weight 0 adds 0, also at -inf
  __device__ __forceinline__ void one(float& x, uint32_t) {
    const float d = x == m ? 0.0f : x - m;  // also for m = +-inf
    if (ModeTraits<MODE>::kScaledSet) sT += fast_exp2(d * cT);
    if (ModeTraits<MODE>::kPlainSet) {
      const float e = fast_exp2(d * c1);
      s1 += e;
      t1 += e > 0.0f ? e * d : 0.0f;
    }
  }
  template <int N>
  __device__ __forceinline__ void vec(float (&x)[N], uint32_t v) {
#pragma unroll
    for (int j = 0; j < N; ++j) one(x[j], v);
  }
};

// The sums of a row, or of a segment of one, in fp64 and natural units: sT = sum exp(x / T - base_t),
// s1 = sum exp(x - base_1), u1 = sum exp(x - base_1) (x - base_1). Nothing of weight: sums 0, base -inf.
struct RowTotals {
  double base_t, base_1, sT, s1, u1;
  bool nan;
};

template <int MODE>
__device__ __forceinline__ RowTotals fast_totals(const RowSums& s) {
  const double base_1 = (double)s.M1 * kLn2d;
  return {(double)s.MT * kLn2d, base_1, (double)s.sT, (double)s.s1, (double)s.t1 - base_1 * (double)s.s1, false};
}

template <int MODE>
__device__ __forceinline__ bool fast_usable(const RowSums& s) {
  using MT = ModeTraits<MODE>;
  bool ok = true;
  if (MT::kScaledSet) ok = ok && sums_usable(s.sT) && fabsf(s.MT) < kFarReference;
  if (MT::kPlainSet) ok = ok && sums_usable(s.s1) && fabsf(s.t1) < INFINITY && fabsf(s.M1) < kFarReference;
  return ok;
}

// What a walk does to the elements before it hands them on: nothing.
struct EveryElement {
  template <int N>
  __device__ __forceinline__ void vec(float (&)[N], uint32_t) const {}
  __device__ __forceinline__ void one(float&, uint32_t) const {}
};

// One vector per step: what only rare rows run must not cost the others their registers.
template <int DT, typename F, typename P>
__device__ __forceinline__ void walk_row(const char* row, const RowGeom& g, const P& prepare, F& f) {
  using E = Elt<DT>;
  const uint32_t tid = threadIdx.x;
  const char* body = row + g.head * E::kSize;
#pragma unroll 1
  for (uint32_t v = tid; v < g.nvec; v += kBlock) {
    float x[E::kPerVec];
    E::unpack(*(const u32x4*)(body + v * 16u), x);
    prepare.vec(x, v);
    f.vec(x, v);
  }
  if (tid < g.head + g.tail) {
    const uint32_t e = tid < g.head ? tid : g.nvec * E::kPerVec + tid;
    float x = E::load1(row + e * E::kSize);
    prepare.one(x, tid);
    f.one(x, e);
  }
}

template <int DT, int MODE, typename P>
__device__ __forceinline__ RowTotals exact_totals(const char* row, const RowGeom& g, const P& prepare, double temperature,
                                                  float (*lds)[8]) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  MaxAcc top{-INFINITY, false};
  walk_row<DT>(row, g, prepare, top);
  const float m_w = wave_max(top.m);
  const bool nan_w = __ballot(top.nan) != 0ull;
  if (lane == 0) {
    lds[wave][0] = m_w;
    lds[wave][1] = nan_w ? 1.0f : 0.0f;
  }
  __syncthreads();
  float m = lds[0][0], nans = lds[0][1];
#pragma unroll
  for (int w = 1; w < kWavesPerBlock; ++w) {
    m = fmaxf(m, lds[w][0]);
    nans += lds[w][1];
  }
  __syncthreads();
  ExactAcc<MODE> acc{m, (float)(1.4426950408889634 / temperature), kLog2e, 0.0f, 0.0f, 0.0f};
  if (m != -INFINITY) walk_row<DT>(row, g, prepare, acc);
  const float st = wave_sum(acc.sT), s = wave_sum(acc.s1), t = wave_sum(acc.t1);
  if (lane == 0) {
    lds[wave][0] = st;
    lds[wave][1] = s;
    lds[wave][2] = t;
  }
  __syncthreads();
  RowTotals r = {(double)m / temperature, (double)m, 0.0, 0.0, 0.0, nans != 0.0f};
#pragma unroll
  for (int w = 0; w < kWavesPerBlock; ++w) {
    r.sT += (double)lds[w][0];
    r.s1 += (double)lds[w][1];
    r.u1 += (double)lds[w][2];
  }
  __syncthreads();
  if (m == INFINITY) r.u1 = NAN;
  return r;
}

template <int MODE>
__device__ __forceinline__ RowSoftmax finish_row(const RowTotals& t, double temperature) {
  using MT = ModeTraits<MODE>;
  RowSoftmax r;
  const double scale = MT::kScaledSet ? temperature : 1.0;  // one set serves both where T = 1
  const double log_1 = MT::kPlainSet ? log(t.s1) : 0.0, ex = MT::kPlainSet ? t.u1 / t.s1 : 0.0;
  r.base = MT::kScaledSet ? t.base_t : t.base_1;
  r.log_sum = t.nan ? (double)NAN : (MT::kScaledSet ? log(t.sT) : log_1);
  const double at = r.base * scale;
  r.centre = (float)at;
  r.l2_t = (float)((r.log_sum + (at - (double)r.centre) / scale) * 1.4426950408889634);
  r.entropy = t.nan ? (double)NAN : log_1 - ex;
  const double rest = t.base_1 - (double)r.centre;
  r.l2_1 = MT::kPlainSet ? (float)((log_1 + rest) * 1.4426950408889634) : 0.0f;
  r.ex = MT::kPlainSet ? (float)(ex + rest) : 0.0f;
  return r;
}

__device__ __forceinline__ float logprob_of(float x, double temperature, const RowSoftmax& r) {
  return (float)(((double)x / temperature - r.base) - r.log_sum);
}

// ---------------------------------------------------------------- gradient of one element
// Gradient of one element from the saved statistics. d = x - centre instead of x: the exponent then
// carries the rounding of a difference, not of two large numbers, and a row at the lowest values of
// its type is an ordinary row. The lower bound on d keeps 0 * d at 0 for masked logits.
template <int MODE>
struct ListGrad {
  float centre, cT, negLT, negL1;
  float a_all;   // -(sum of the upstream gradients of all log-probs) / T
  float gh, k1;  // entropy term p (k1 - gh d), k1 = gh (E[x] - centre) (+ a_all where T = 1 shares the softmax)
  float onehot;
  uint32_t label_vec, label_lane, label_elem;
  __device__ __forceinline__ float elem(float x) const {
    const float d = fmaxf(x - centre, -1.0e30f);
    if (MODE == kBwdLp) return fast_exp2(fmaf(d, cT, negLT)) * a_all;
    if (MODE == kBwdBothT1) return fast_exp2(fmaf(d, cT, negLT)) * fmaf(-gh, d, k1);
    return fmaf(fast_exp2(fmaf(d, cT, negLT)), a_all, fast_exp2(fmaf(d, kLog2e, negL1)) * fmaf(-gh, d, k1));
  }
  __device__ __forceinline__ void one(float& x, uint32_t e) const {
    x = elem(x);
    if (e == label_elem) x += onehot;
  }
  template <int N>
  __device__ __forceinline__ void vec(float (&x)[N], uint32_t v) const {
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = elem(x[j]);
    if (v == label_vec) {
#pragma unroll
      for (int j = 0; j < N; ++j) x[j] += (uint32_t)j == label_lane ? onehot : 0.0f;
    }
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

// ---------------------------------------------------------------- rows cut into segments
// A launch with too few rows to fill the GPU cuts them into n segments of seg_elems elements (a
// multiple of 16, so that a segment starts on its row's 16-byte phase; the last one is shorter), one
// workgroup each. A segment writes a record, the workgroup that draws the row's last ticket merges
// the records in segment order, whichever came when: the result does not depend on it. Nobody waits.
constexpr int kMaxSegments = 64;  // a wave merges them, one per lane
struct ListSplit {
  int n;
  uint32_t seg_elems;
};
struct Segment {
  int64_t row;
  int index;
  uint32_t first;
  int64_t len;
};
__device__ __forceinline__ Segment segment_of(int64_t work, const ListSplit& split, int64_t vocab) {
  if (split.n == 1) return {work, 0, 0u, vocab};
  const int64_t row = work / split.n;
  const int index = (int)(work - row * split.n);
  const uint32_t first = (uint32_t)index * split.seg_elems;
  const int64_t left = vocab - first;
  return {row, index, first, left < (int64_t)split.seg_elems ? left : (int64_t)split.seg_elems};
}

// Records and tickets pass the caches that the compute dies do not share: device-scope accesses.
__device__ __forceinline__ void put64(uint64_t* p, uint64_t v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <bool FRESH>
__device__ __forceinline__ uint64_t get64(const uint64_t* p) {
  return FRESH ? __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : *p;
}
__device__ __forceinline__ uint64_t as_u64(double d) { return __builtin_bit_cast(uint64_t, d); }
__device__ __forceinline__ double as_double(uint64_t u) { return __builtin_bit_cast(double, u); }

constexpr int kTotalsWords = 6;  // a record's head: the totals, the label's logit and the NaN flag
__device__ __forceinline__ void put_totals(uint64_t* rec, const RowTotals& t, float x_label) {
  put64(rec + 0, as_u64(t.base_t));
  put64(rec + 1, as_u64(t.base_1));
  put64(rec + 2, as_u64(t.sT));
  put64(rec + 3, as_u64(t.s1));
  put64(rec + 4, as_u64(t.u1));
  put64(rec + 5, (uint64_t)as_uint(x_label) | (uint64_t)(t.nan ? 1u : 0u) << 32);
}

// One wave: the totals of a row from its segments' records (`stride` words apart), and the logit of
// the segment `label_segment` (-1: none).
template <bool FRESH>
__device__ __forceinline__ RowTotals merge_totals(const uint64_t* rec, int64_t stride, int n, int label_segment,
                                                  float& x_label) {
  const int lane = threadIdx.x & (kWave - 1);
  RowTotals t = {-INFINITY, -INFINITY, 0.0, 0.0, 0.0, false};
  float xl = 0.0f;
  if (lane < n) {
    const uint64_t* r = rec + lane * stride;
    t.base_t = as_double(get64<FRESH>(r + 0));
    t.base_1 = as_double(get64<FRESH>(r + 1));
    t.sT = as_double(get64<FRESH>(r + 2));
    t.s1 = as_double(get64<FRESH>(r + 3));
    t.u1 = as_double(get64<FRESH>(r + 4));
    const uint64_t w = get64<FRESH>(r + 5);
    t.nan = (w >> 32) != 0u;
    if (lane == label_segment) xl = as_float((uint32_t)w);
  }
  x_label = __shfl(xl, label_segment < 0 ? 0 : label_segment, kWave);
  double mt = t.base_t, m1 = t.base_1;
#pragma unroll
  for (int o = kWave / 2; o > 0; o >>= 1) {
    const double ot = __shfl_xor(mt, o, kWave), o1 = __shfl_xor(m1, o, kWave);
    mt = ot > mt ? ot : mt;
    m1 = o1 > m1 ? o1 : m1;
  }
  const double qt = t.base_t == mt ? 1.0 : exp(t.base_t - mt), q1 = t.base_1 == m1 ? 1.0 : exp(t.base_1 - m1);
  const double shift = t.base_1 == m1 || t.s1 == 0.0 ? 0.0 : (t.base_1 - m1) * t.s1;
  RowTotals r;
  r.base_t = mt, r.base_1 = m1;
  r.sT = wave_sum(t.sT * qt);
  r.s1 = wave_sum(t.s1 * q1);
  r.u1 = wave_sum(q1 == 0.0 ? 0.0 : q1 * (t.u1 + shift));
  r.nan = __ballot(t.nan) != 0ull;
  return r;
}

// True in the workgroup that finishes the last segment of its row. Every thread calls it, after its
// own stores to the record; the ticket is back at zero when it returns true.
__device__ __forceinline__ bool last_segment(int32_t* ticket, int n) {
  __shared__ int drawn;
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
  __builtin_amdgcn_s_waitcnt(0);  // this wave's stores have been acknowledged
  __syncthreads();
  if (threadIdx.x == 0) {
    drawn = __hip_atomic_fetch_add(ticket, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (drawn == n - 1) __hip_atomic_store(ticket, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  return drawn == n - 1;
}

// The cut depends on the shape only, so results do not depend on the device.
inline ListSplit list_split(int64_t n_rows, int64_t vocab, int esize) {
  constexpr int64_t kWholeRowsFrom = 512, kItems = 1024, kMinSegBytes = 16384;
  ListSplit split{1, (uint32_t)vocab};
  if (n_rows >= kWholeRowsFrom) return split;
  int64_t n = (kItems + n_rows - 1) / n_rows;
  if (n > kMaxSegments) n = kMaxSegments;
  if (n > vocab * esize / kMinSegBytes) n = vocab * esize / kMinSegBytes;
  if (n <= 1) return split;
  const int64_t seg = (((vocab + n - 1) / n) + 15) & ~(int64_t)15;
  split.n = (int)((vocab + seg - 1) / seg);
  split.seg_elems = (uint32_t)seg;
  return split;
}

}  // namespace orlhf
