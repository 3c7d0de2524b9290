// Log-prob of a given token, entropy and the K most likely tokens of every vocabulary row.
//
//   logprob = x_label / T - lse(x / T)            entropy = lse(x) - sum softmax(x) x
//   top     = the K largest x of the row, descending, equal values by ascending id,
//             each with x / T - lse(x / T)
//
// An element is one 64-bit key for the selection: the logit as an unsigned integer of the same
// order in the high half, the complement of its id in the low half. Keys are unique, "greater"
// means "ranked before", and a NaN (which has no order) ranks before everything.
#include "vocab_rows.h"

namespace orlhf {

constexpr int kMaxTop = 128;   // longest list of alternatives
constexpr int kCap = 1024;     // candidate keys a workgroup holds; a list and a round of pushes fit

__device__ __forceinline__ uint32_t ordered_bits(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = as_uint(x + 0.0f);  // -0 and +0 are equal
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float ordered_value(uint32_t o) {
  return as_float(o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ uint64_t make_key(float x, uint32_t id) {
  return (uint64_t)ordered_bits(x) << 32 | (0xffffffffu - id);
}
__device__ __forceinline__ uint32_t key_id(uint64_t key) { return 0xffffffffu - (uint32_t)key; }

struct Candidates {
  uint64_t key[kCap];
  int count;
};

// How many of the n candidates rank before each of this thread's (at threadIdx.x + i * kBlock).
template <int MINE>
__device__ __forceinline__ void rank_candidates(const Candidates& c, int n, uint64_t (&mine)[MINE], int (&rank)[MINE]) {
#pragma unroll
  for (int i = 0; i < MINE; ++i) {
    const int at = (int)threadIdx.x + i * kBlock;
    mine[i] = at < n ? c.key[at] : 0ull;
    rank[i] = 0;
  }
  if ((int)(threadIdx.x & ~(kWave - 1u)) >= n) return;  // a wave without a candidate
#pragma unroll 4
  for (int j = 0; j < n; ++j) {
    const uint64_t other = c.key[j];
#pragma unroll
    for (int i = 0; i < MINE; ++i) rank[i] += other > mine[i] ? 1 : 0;
  }
}

// Keeps the k best candidates, sorted, and returns the k-th (0 while there are fewer). The whole
// workgroup calls it with the candidates in place behind a barrier; another one ends it.
__device__ __forceinline__ uint64_t keep_best(Candidates& c, int k) {
  constexpr int kMine = kCap / kBlock;
  const int n = c.count;
  uint64_t mine[kMine];
  int rank[kMine];
  rank_candidates<kMine>(c, n, mine, rank);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const int at = (int)threadIdx.x + i * kBlock;
    if (at < n && rank[i] < k) c.key[rank[i]] = mine[i];
  }
  if (threadIdx.x == 0) c.count = n < k ? n : k;
  __syncthreads();
  return n < k ? 0ull : c.key[k - 1];
}

// Adds at most one key per thread, those above `least`; thins the candidates first when a whole
// round might not fit. Called by the whole workgroup.
__device__ __forceinline__ void push_round(Candidates& c, uint64_t key, int k, uint64_t& least) {
  __syncthreads();
  const int n = c.count;
  __syncthreads();
  if (n + kBlock > kCap) least = keep_best(c, k);
  if (key > least) c.key[atomicAdd(&c.count, 1)] = key;
}

// Every element of the row through the candidates, in ascending order of the ids: right for any
// row (equal values, -inf, NaN), whatever the threshold `least` it starts from.
template <int DT>
__device__ __forceinline__ void collect_row(const char* row, const RowGeom& g, uint32_t first, int k, uint64_t least,
                                            Candidates& c) {
  using E = Elt<DT>;
  constexpr int EPV = E::kPerVec;
  const uint32_t tid = threadIdx.x;
  const char* body = row + g.head * E::kSize;
  for (uint32_t v0 = 0; v0 < g.nvec; v0 += kBlock) {
    const uint32_t v = v0 + tid;
    uint64_t key[EPV];
    bool any = false;
    float x[EPV];
    if (v < g.nvec) E::unpack(*(const u32x4*)(body + v * 16u), x);
#pragma unroll
    for (int j = 0; j < EPV; ++j) {
      key[j] = v < g.nvec ? make_key(x[j], first + g.head + v * EPV + j) : 0ull;
      any = any || key[j] > least;
    }
    if (__syncthreads_or(any)) {
#pragma unroll
      for (int j = 0; j < EPV; ++j) push_round(c, key[j], k, least);
    }
  }
  const uint32_t nscalar = g.head + g.tail;
  for (uint32_t s0 = 0; s0 < nscalar; s0 += kBlock) {
    const uint32_t s = s0 + tid;
    const uint32_t e = s < g.head ? s : g.head + g.nvec * EPV + (s - g.head);
    push_round(c, s < nscalar ? make_key(E::load1(row + e * E::kSize), first + e) : 0ull, k, least);
  }
  __syncthreads();
}

struct TopArgs {
  const char* logits;
  int64_t n_rows, vocab, row_stride_bytes;
  const int64_t* labels;  // NULL: no log-prob
  double temperature;
  int k;
  float *logprob, *entropy, *top_logprob, *row_stats;  // logprob, entropy, row_stats may be NULL
  int64_t* top_ids;
  const uint8_t* row_mask;
  int shift;  // of the selection's blocks
};

__device__ __forceinline__ void write_skipped_row(const TopArgs& a, int64_t row_i) {
  for (int i = threadIdx.x; i < a.k; i += kBlock) {
    a.top_ids[row_i * a.k + i] = -1;
    a.top_logprob[row_i * a.k + i] = 0.0f;
  }
  if (threadIdx.x == 0) {
    if (a.logprob != nullptr) a.logprob[row_i] = 0.0f;
    if (a.entropy != nullptr) a.entropy[row_i] = 0.0f;
    if (a.row_stats != nullptr) *(f32x4*)(a.row_stats + row_i * 4) = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
}

// Wave reference of the fast pass: the maximum of the first vector (or scalar) of each lane.
template <int DT>
__device__ __forceinline__ float wave_reference(const char* row, const RowGeom& g, uint32_t len) {
  using E = Elt<DT>;
  float m = -INFINITY;
  if (g.nvec > 0) {
    const uint32_t v = threadIdx.x < g.nvec ? threadIdx.x : g.nvec - 1;
    float x[E::kPerVec];
    E::unpack(*(const u32x4*)(row + g.head * E::kSize + v * 16u), x);
#pragma unroll
    for (int j = 0; j < E::kPerVec; ++j) m = fmaxf(m, x[j]);
  } else {
    m = E::load1(row + (threadIdx.x < len ? threadIdx.x : len - 1) * E::kSize);
  }
  return wave_max(m);
}

// The softmax of a row as what its outputs and its backward need: base + log_sum is the
// log-sum-exp of x / T (kept apart: base may be so large that the sum would be lost in it), `centre`
// a logit near base * T that every later difference starts from, entropy and E[x] - centre those of
// the unscaled logits.
struct RowSoftmax {
  double base, log_sum, entropy;
  float centre, l2_t, l2_1, ex;  // the backward's statistics: softmax(x / T) = 2^((x - centre) cT - l2_t)
  bool nan;
};

// Fast pass: per wave sums against its reference, folded over the workgroup.
template <int MODE>
__device__ __forceinline__ RowSums combine_fast(const FastAcc<MODE>& acc, float (*lds)[8]) {
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

// All threads of the workgroup get the same result. T = 1 (and entropy-free) modes keep one set.
template <int DT, int MODE>
__device__ __forceinline__ RowSoftmax row_softmax(const char* row, const RowGeom& g, RowSums sums, float c_scaled,
                                                  double temperature, float (*lds)[8]) {
  using MT = ModeTraits<MODE>;
  RowSoftmax r;
  bool ok = true;
  if (MT::kScaledSet) ok = ok && sums_usable(sums.sT) && fabsf(sums.MT) < kFarReference;
  if (MT::kPlainSet) ok = ok && sums_usable(sums.s1) && fabsf(sums.t1) < INFINITY && fabsf(sums.M1) < kFarReference;
  r.nan = false;
  double base_1, log_1, ex;  // of the unscaled logits; ex = E[x] - base_1
  if (ok) {
    r.base = (double)(MT::kScaledSet ? sums.MT : sums.M1) * kLn2d;
    r.log_sum = log((double)(MT::kScaledSet ? sums.sT : sums.s1));
    base_1 = (double)sums.M1 * kLn2d;
    log_1 = MT::kPlainSet ? log((double)sums.s1) : 0.0;
    ex = MT::kPlainSet ? (double)sums.t1 / (double)sums.s1 - base_1 : 0.0;
  } else {
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    MaxAcc top{-INFINITY, false};
    traverse_row<DT, false>(row, nullptr, g, top);
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
    r.nan = nans != 0.0f;
    __syncthreads();
    ExactAcc<MODE> acc{m, c_scaled, kLog2e, 0.0f, 0.0f, 0.0f};
    traverse_row<DT, false>(row, nullptr, g, acc);
    const float st = wave_sum(acc.sT), s = wave_sum(acc.s1), t = wave_sum(acc.t1);
    if (lane == 0) {
      lds[wave][0] = st;
      lds[wave][1] = s;
      lds[wave][2] = t;
    }
    __syncthreads();
    double sT = 0.0, s1 = 0.0, t1 = 0.0;
#pragma unroll
    for (int w = 0; w < kWavesPerBlock; ++w) {
      sT += (double)lds[w][0];
      s1 += (double)lds[w][1];
      t1 += (double)lds[w][2];
    }
    __syncthreads();
    if (r.nan || m == -INFINITY) sT = s1 = NAN;
    if (m == INFINITY) t1 = NAN;
    base_1 = (double)m;
    r.base = (double)m / temperature;
    r.log_sum = log(MT::kScaledSet ? sT : s1);
    log_1 = log(s1);
    ex = t1 / s1;
  }
  const double at = r.base * (MT::kScaledSet ? temperature : 1.0);
  r.centre = (float)at;
  const double shift = at - (double)r.centre;
  r.l2_t = (float)((r.log_sum + shift / (MT::kScaledSet ? temperature : 1.0)) * 1.4426950408889634);
  r.entropy = log_1 - ex;
  const double rest = base_1 - (double)r.centre;
  r.l2_1 = MT::kPlainSet ? (float)((log_1 + rest) * 1.4426950408889634) : 0.0f;
  r.ex = MT::kPlainSet ? (float)(ex + rest) : 0.0f;
  return r;
}

__device__ __forceinline__ float logprob_of(float x, double temperature, const RowSoftmax& r) {
  return (float)(((double)x / temperature - r.base) - r.log_sum);
}

// ---------------------------------------------------------------- selection
// The streaming pass leaves, beside the sums, the maximum of every BLOCK of a thread's elements in
// LDS (a block: 4 vectors, or 4 << shift where a row has more than kMaxBlocks such blocks per
// thread) and the maximum of all of them in a register: half an operation per element. The k-th
// largest of the 256 thread maxima is a lower bound of the row's k-th largest logit that few more
// than k elements pass (expected -256 ln(1 - k/256): 20 for k = 20, 177 for k = 128), so only the
// blocks that reach it are read again, a few KiB per row, and their elements that reach it become
// candidates. A row that has more of them than fit (many equal logits), or a NaN, goes through
// collect_row instead.
constexpr int kMaxBlocks = 32;
constexpr uint32_t kBlockVecs = 4;  // vectors of one thread in a block (shift 0)

template <int DT, int MODE>
__device__ __forceinline__ float stream_row(const char* row, const RowGeom& g, FastAcc<MODE>& acc, float* block_max,
                                            int shift) {
  using E = Elt<DT>;
  constexpr uint32_t U = ORLHF_ROW_UNROLL;
  static_assert(U % kBlockVecs == 0, "a batch holds whole blocks");
  const uint32_t tid = threadIdx.x;
  const char* body = row + g.head * E::kSize;
  float thread_max = -INFINITY;
  auto take = [&](const u32x4& raw, float& bm, uint32_t v) {
    float x[E::kPerVec];
    E::unpack(raw, x);
#pragma unroll
    for (int j = 0; j < E::kPerVec; ++j) bm = fmaxf(bm, x[j]);
    acc.vec(x, v);
  };
  auto note = [&](uint32_t part, float bm) {  // part: which group of kBlockVecs vectors of the thread
    float* slot = block_max + (part >> shift) * kBlock + tid;
    *slot = (part & ((1u << shift) - 1u)) == 0u ? bm : fmaxf(*slot, bm);
    thread_max = fmaxf(thread_max, bm);
  };
  const uint32_t nbatch = g.nvec / (kBlock * U);
  uint32_t v0 = tid, part = 0;
  for (uint32_t b = 0; b < nbatch; ++b, v0 += kBlock * U) {
    u32x4 buf[U];
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) buf[u] = load_vec(body + (v0 + u * kBlock) * 16u);
#pragma unroll
    for (uint32_t h = 0; h < U; h += kBlockVecs) {
      float bm = -INFINITY;
#pragma unroll
      for (uint32_t u = h; u < h + kBlockVecs; ++u) take(buf[u], bm, v0 + u * kBlock);
      note(part++, bm);
    }
  }
  if (nbatch * kBlock * U < g.nvec) {  // the last, partial batch
    u32x4 buf[U];
#pragma unroll
    for (uint32_t u = 0; u < U; ++u)
      if (v0 + u * kBlock < g.nvec) buf[u] = load_vec(body + (v0 + u * kBlock) * 16u);
#pragma unroll
    for (uint32_t h = 0; h < U; h += kBlockVecs) {
      if ((nbatch * U + h) * kBlock < g.nvec) {
        float bm = -INFINITY;
#pragma unroll
        for (uint32_t u = h; u < h + kBlockVecs; ++u)
          if (v0 + u * kBlock < g.nvec) take(buf[u], bm, v0 + u * kBlock);
        note(part++, bm);
      }
    }
  }
  const uint32_t nscalar = g.head + g.tail;
  for (uint32_t k = tid; k < nscalar; k += kBlock) {
    const uint32_t e = k < g.head ? k : g.head + g.nvec * E::kPerVec + (k - g.head);
    float x = E::load1(row + e * E::kSize);
    acc.one(x, e);
  }
  return thread_max;
}

// The largest value of 16 leading bits that at least k of the 256 maxima reach, as ordered bits: one
// wave, four maxima per lane, one counting step per bit.
__device__ __forceinline__ uint32_t kth_maximum(const float* thread_max, int k) {
  const int lane = threadIdx.x & (kWave - 1);
  const f32x4 m = *(const f32x4*)(thread_max + lane * 4);
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = ordered_bits(m[i]);
  uint32_t found = 0;
#pragma unroll
  for (int bit = 31; bit >= 16; --bit) {
    const uint32_t probe = found | (1u << bit);
    int n = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) n += __popcll(__ballot(o[i] >= probe));
    if (n >= k) found = probe;
  }
  return found;
}

// The elements that reach `bar` in the blocks that do, into the candidates (their count may pass
// kCap: then not all are there).
template <int DT>
__device__ __forceinline__ void collect_blocks(const char* row, const RowGeom& g, uint32_t first, const float* block_max,
                                               int shift, float bar, float thread_max, Candidates& c) {
  using E = Elt<DT>;
  const uint32_t tid = threadIdx.x;
  const char* body = row + g.head * E::kSize;
  auto push = [&](float x, uint32_t id) {
    if (x >= bar) {
      const int at = atomicAdd(&c.count, 1);
      if (at < kCap) c.key[at] = make_key(x, id);
    }
  };
  if (thread_max >= bar) {
    const uint32_t parts = (g.nvec + kBlockVecs * kBlock - 1) / (kBlockVecs * kBlock);
    const uint32_t blocks = (parts + (1u << shift) - 1u) >> shift;
    uint32_t wanted = 0;
    for (uint32_t b = 0; b < blocks; ++b) wanted |= (block_max[b * kBlock + tid] >= bar ? 1u : 0u) << b;
    while (wanted != 0u) {
      const uint32_t b = (uint32_t)__builtin_ctz(wanted);
      wanted &= wanted - 1u;
      for (uint32_t part = b << shift; part < (b + 1u) << shift; ++part) {
        u32x4 raw[kBlockVecs];
        const uint32_t v0 = part * (kBlockVecs * kBlock) + tid;
#pragma unroll
        for (uint32_t u = 0; u < kBlockVecs; ++u)
          if (v0 + u * kBlock < g.nvec) raw[u] = *(const u32x4*)(body + (v0 + u * kBlock) * 16u);
#pragma unroll
        for (uint32_t u = 0; u < kBlockVecs; ++u) {
          const uint32_t v = v0 + u * kBlock;
          if (v < g.nvec) {
            float x[E::kPerVec];
            E::unpack(raw[u], x);
#pragma unroll
            for (int j = 0; j < E::kPerVec; ++j) push(x[j], first + g.head + v * E::kPerVec + j);
          }
        }
      }
    }
  }
  const uint32_t nscalar = g.head + g.tail;
  for (uint32_t k = tid; k < nscalar; k += kBlock) {
    const uint32_t e = k < g.head ? k : g.head + g.nvec * E::kPerVec + (k - g.head);
    push(E::load1(row + e * E::kSize), first + e);
  }
}

template <int DT, int MODE>
__global__ __launch_bounds__(kBlock, 4) void top_logprobs_fwd_kernel(TopArgs a) {
  using E = Elt<DT>;
  __shared__ float lds[kWavesPerBlock][8];
  __shared__ Candidates cand;
  __shared__ alignas(16) float thread_maxima[kBlock];
  __shared__ uint32_t bar_bits;
  extern __shared__ float block_max[];
  const int tid = threadIdx.x;
  const float c_scaled = (float)(1.4426950408889634 / a.temperature);
  for (int64_t row_i = blockIdx.x; row_i < a.n_rows; row_i += gridDim.x) {
    if (a.row_mask != nullptr && a.row_mask[row_i] == 0) {
      write_skipped_row(a, row_i);
      continue;
    }
    const char* row = a.logits + row_i * a.row_stride_bytes;
    const RowGeom g = row_geom<DT>(row, a.vocab, false);
    if (tid == 0) cand.count = 0;
    // the label and its logit are asked for now and used by the row's last instructions
    int64_t label = -1;
    float x_label = 0.0f;
    if (a.logprob != nullptr && tid == 0) {
      label = a.labels[row_i];
      if (label >= 0 && label < a.vocab) x_label = E::load1(row + label * E::kSize);
    }
    FastAcc<MODE> acc;
    acc.init(wave_reference<DT>(row, g, (uint32_t)a.vocab), c_scaled, kLog2e);
    const float thread_max = stream_row<DT, MODE>(row, g, acc, block_max, a.shift);
    thread_maxima[tid] = thread_max;
    const RowSums sums = combine_fast<MODE>(acc, lds);  // its barriers also publish the maxima
    if (tid < kWave) {
      const uint32_t bits = kth_maximum(thread_maxima, a.k);
      if (tid == 0) bar_bits = bits;
    }
    const RowSoftmax mine = row_softmax<DT, MODE>(row, g, sums, c_scaled, a.temperature, lds);
    __syncthreads();
    const uint32_t bits = bar_bits;
    const float bar = bits <= ordered_bits(-INFINITY) ? -INFINITY : ordered_value(bits);
    collect_blocks<DT>(row, g, 0u, block_max, a.shift, bar, thread_max, cand);
    __syncthreads();
    int n = cand.count;
    if (n > kCap || mine.nan) {
      __syncthreads();
      if (tid == 0) cand.count = 0;
      collect_row<DT>(row, g, 0u, a.k, bits != 0u ? ((uint64_t)bits << 32) - 1u : 0ull, cand);
      n = cand.count;
    }
    auto out = [&](uint64_t key, int at) {
      a.top_ids[row_i * a.k + at] = (int64_t)key_id(key);
      a.top_logprob[row_i * a.k + at] = logprob_of(ordered_value((uint32_t)(key >> 32)), a.temperature, mine);
    };
    if (n <= kBlock) {
      uint64_t key[1];
      int rank[1];
      rank_candidates<1>(cand, n, key, rank);
      if (tid < n && rank[0] < a.k) out(key[0], rank[0]);
    } else {
      keep_best(cand, a.k);
      if (tid < a.k) out(cand.key[tid], tid);
    }
    if (tid == 0) {
      if (a.logprob != nullptr)
        a.logprob[row_i] = label >= 0 && label < a.vocab ? logprob_of(x_label, a.temperature, mine) : (label == -100 ? 0.0f : NAN);
      if (ModeTraits<MODE>::kPlainSet && a.entropy != nullptr) a.entropy[row_i] = (float)mine.entropy;
      if (a.row_stats != nullptr) *(f32x4*)(a.row_stats + row_i * 4) = f32x4{mine.centre, mine.l2_t, mine.l2_1, mine.ex};
    }
    __syncthreads();  // the candidates are read until here
  }
}

// ---------------------------------------------------------------- backward
struct TopBwdArgs {
  const char* logits;
  char* grad;
  int64_t n_rows, vocab, row_stride_bytes, grad_stride_bytes;
  const int64_t *labels, *top_ids;
  double temperature;
  int k;
  const float *g_logprob, *g_entropy, *g_top, *row_stats;  // gradients may be NULL: zero
  const uint8_t* row_mask;
  int scalar_only;
};

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

// grad_j = [ g_lp 1(j = label) + sum_k g_k 1(j = id_k) - (g_lp + sum_k g_k) softmax(x / T)_j ] / T
//          + g_H softmax(x)_j (E[x] - x_j)
// The listed elements' gradients are worked out before the row is touched (the row may be
// overwritten in place) and stored over the row pass's values behind a barrier.
template <int DT, int MODE>
__global__ __launch_bounds__(kBlock) void top_logprobs_bwd_kernel(TopBwdArgs a) {
  using E = Elt<DT>;
  __shared__ float lds[kWavesPerBlock];
  const int tid = threadIdx.x;
  const double inv_t = 1.0 / a.temperature;
  for (int64_t row_i = blockIdx.x; row_i < a.n_rows; row_i += gridDim.x) {
    const char* row = a.logits + row_i * a.row_stride_bytes;
    char* out_row = a.grad + row_i * a.grad_stride_bytes;
    const RowGeom g = row_geom<DT>(row, a.vocab, a.scalar_only != 0);
    const bool skipped = a.row_mask != nullptr && a.row_mask[row_i] == 0;
    const bool mine = !skipped && tid < a.k && a.g_top != nullptr;
    const float gk = mine ? a.g_top[row_i * a.k + tid] : 0.0f;
    const int64_t id = mine ? a.top_ids[row_i * a.k + tid] : -1;
    const float w = wave_sum(gk);
    const bool wave_on = __ballot(gk != 0.0f) != 0ull;  // NaN counts as on
    if ((tid & (kWave - 1)) == 0) lds[tid / kWave] = w;
    const bool top_on = __syncthreads_or(wave_on);
    float sum_top = 0.0f;
#pragma unroll
    for (int i = 0; i < kWavesPerBlock; ++i) sum_top += lds[i];
    __syncthreads();
    const float glp = a.g_logprob != nullptr ? a.g_logprob[row_i] : 0.0f;
    const float gh = MODE != kBwdLp ? a.g_entropy[row_i] : 0.0f;
    if (skipped || (glp == 0.0f && gh == 0.0f && !top_on)) {
      zero_row<DT>(out_row, g);
      continue;
    }
    const f32x4 st = *(const f32x4*)(a.row_stats + row_i * 4);
    const double all = (double)glp + (double)sum_top;
    ListGrad<MODE> fn;
    fn.centre = st[0];
    fn.cT = (float)(1.4426950408889634 * inv_t);
    fn.negLT = -st[1];
    fn.negL1 = -st[2];
    fn.a_all = -(float)(all * inv_t);
    fn.onehot = (float)((double)glp * inv_t);
    fn.gh = gh;
    fn.k1 = gh * st[3] + (MODE == kBwdBothT1 ? fn.a_all : 0.0f);
    const int64_t label = a.g_logprob != nullptr ? a.labels[row_i] : -1;
    fn.set_label(label, a.vocab, g, E::kPerVec);
    const bool patch = mine && id >= 0 && id < a.vocab;
    float val = 0.0f;
    if (patch) {
      val = E::load1(row + id * E::kSize);
      fn.one(val, (uint32_t)id);
      val += (float)((double)gk * inv_t);
    }
    if (a.g_top != nullptr) __syncthreads();  // the listed logits are read before any is overwritten
    traverse_row<DT, true>(row, out_row, g, fn);
    if (a.g_top != nullptr) {
      __syncthreads();
      if (patch) E::store1(out_row + id * E::kSize, val);
      __syncthreads();
    }
  }
}

template <int DT>
static int launch_top_fwd(TopArgs a, hipStream_t stream) {
  const bool t1 = a.temperature == 1.0;
  const int64_t parts = (a.vocab / Elt<DT>::kPerVec + kBlockVecs * kBlock - 1) / (kBlockVecs * kBlock);
  while ((parts + (1 << a.shift) - 1) >> a.shift > kMaxBlocks) ++a.shift;
  const int64_t blocks = (parts + (1 << a.shift) - 1) >> a.shift;
  const size_t lds = (size_t)(blocks > 0 ? blocks : 1) * kBlock * sizeof(float);
  const dim3 grid(grid_for_rows(a.n_rows)), block(kBlock);
  if (a.entropy == nullptr)
    hipLaunchKernelGGL((top_logprobs_fwd_kernel<DT, kLpOnly>), grid, block, lds, stream, a);
  else if (t1)
    hipLaunchKernelGGL((top_logprobs_fwd_kernel<DT, kBothT1>), grid, block, lds, stream, a);
  else
    hipLaunchKernelGGL((top_logprobs_fwd_kernel<DT, kBothT>), grid, block, lds, stream, a);
  ORLHF_CHECK_LAUNCH("orlhf_top_logprobs_fwd");
  return ORLHF_OK;
}

template <int DT>
static int launch_top_bwd(const TopBwdArgs& a, hipStream_t stream) {
  const dim3 grid(grid_for_rows(a.n_rows)), block(kBlock);
  if (a.g_entropy == nullptr)
    hipLaunchKernelGGL((top_logprobs_bwd_kernel<DT, kBwdLp>), grid, block, 0, stream, a);
  else if (a.temperature == 1.0)
    hipLaunchKernelGGL((top_logprobs_bwd_kernel<DT, kBwdBothT1>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((top_logprobs_bwd_kernel<DT, kBwdBothT>), grid, block, 0, stream, a);
  ORLHF_CHECK_LAUNCH("orlhf_top_logprobs_bwd");
  return ORLHF_OK;
}

static int check_top(const char* what, int dtype, int64_t n_rows, int64_t vocab, int64_t row_stride, double temperature,
                     int64_t k) {
  ORLHF_CHECK_ARG(n_rows >= 0 && vocab > 0, "%s: n_rows=%lld vocab=%lld", what, (long long)n_rows, (long long)vocab);
  ORLHF_CHECK_ARG(row_stride >= vocab, "%s: row_stride %lld < vocab %lld", what, (long long)row_stride, (long long)vocab);
  ORLHF_CHECK_ARG(vocab < (1ll << 29), "%s: vocab %lld too large (row must stay below 2 GiB)", what, (long long)vocab);
  ORLHF_CHECK_ARG(temperature > 0.0 && temperature < INFINITY, "%s: temperature must be > 0 and finite", what);
  ORLHF_CHECK_ARG(dtype == ORLHF_F32 || dtype == ORLHF_BF16 || dtype == ORLHF_F16, "%s: unknown dtype %d", what, dtype);
  ORLHF_CHECK_ARG(k >= 1 && k <= kMaxTop && k <= vocab, "%s: k=%lld must lie in 1..%d and not exceed vocab %lld", what,
                  (long long)k, kMaxTop, (long long)vocab);
  return ORLHF_OK;
}

}  // namespace orlhf

using namespace orlhf;

extern "C" int orlhf_top_logprobs_fwd(const void* logits, int dtype, int64_t n_rows, int64_t vocab, int64_t row_stride,
                                      const int64_t* labels, double temperature, int64_t k, float* logprob,
                                      float* entropy, float* top_logprob, int64_t* top_ids, float* row_stats,
                                      const uint8_t* row_mask, orlhf_stream_t stream) {
  const int bad = check_top("top_logprobs_fwd", dtype, n_rows, vocab, row_stride, temperature, k);
  if (bad != ORLHF_OK) return bad;
  if (n_rows == 0) return ORLHF_OK;  // nothing to launch; empty arrays may well be NULL
  ORLHF_CHECK_ARG(logits != nullptr && top_logprob != nullptr && top_ids != nullptr,
                  "top_logprobs_fwd: NULL logits / top_logprob / top_ids");
  ORLHF_CHECK_ARG(logprob == nullptr || labels != nullptr, "top_logprobs_fwd: labels is NULL");
  ORLHF_CHECK_ARG(((uintptr_t)logits & (dtype == ORLHF_F32 ? 3u : 1u)) == 0,
                  "top_logprobs_fwd: logits not aligned to the element size");
  const int64_t esize = dtype == ORLHF_F32 ? 4 : 2;
  const TopArgs a = {(const char*)logits, n_rows, vocab, row_stride * esize, labels, temperature, (int)k, logprob,
                     entropy, top_logprob, row_stats, top_ids, row_mask, 0};
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case ORLHF_F32: return launch_top_fwd<ORLHF_F32>(a, s);
    case ORLHF_BF16: return launch_top_fwd<ORLHF_BF16>(a, s);
    default: return launch_top_fwd<ORLHF_F16>(a, s);
  }
}

extern "C" int orlhf_top_logprobs_bwd(const void* logits, void* grad_logits, int dtype, int64_t n_rows, int64_t vocab,
                                      int64_t row_stride, int64_t grad_row_stride, const int64_t* labels,
                                      double temperature, int64_t k, const int64_t* top_ids, const float* g_logprob,
                                      const float* g_entropy, const float* g_top_logprob, const float* row_stats,
                                      const uint8_t* row_mask, orlhf_stream_t stream) {
  const int bad = check_top("top_logprobs_bwd", dtype, n_rows, vocab, row_stride, temperature, k);
  if (bad != ORLHF_OK) return bad;
  ORLHF_CHECK_ARG(grad_row_stride >= vocab, "top_logprobs_bwd: grad_row_stride %lld < vocab %lld",
                  (long long)grad_row_stride, (long long)vocab);
  if (n_rows == 0) return ORLHF_OK;
  ORLHF_CHECK_ARG(g_logprob != nullptr || g_entropy != nullptr || g_top_logprob != nullptr,
                  "top_logprobs_bwd: every upstream gradient is NULL");
  ORLHF_CHECK_ARG(logits != nullptr && grad_logits != nullptr && row_stats != nullptr,
                  "top_logprobs_bwd: NULL logits / grad_logits / row_stats");
  ORLHF_CHECK_ARG(g_logprob == nullptr || labels != nullptr, "top_logprobs_bwd: labels is NULL");
  ORLHF_CHECK_ARG(g_top_logprob == nullptr || top_ids != nullptr, "top_logprobs_bwd: top_ids is NULL");
  const int64_t esize = dtype == ORLHF_F32 ? 4 : 2;
  ORLHF_CHECK_ARG((((uintptr_t)logits | (uintptr_t)grad_logits) & (uintptr_t)(esize - 1)) == 0,
                  "top_logprobs_bwd: pointers not aligned to the element size");
  const bool same_phase = (((uintptr_t)logits ^ (uintptr_t)grad_logits) & 15u) == 0 &&
                          (((row_stride - grad_row_stride) * esize) & 15) == 0;
  const TopBwdArgs a = {(const char*)logits, (char*)grad_logits, n_rows, vocab, row_stride * esize, grad_row_stride * esize,
                        labels, top_ids, temperature, (int)k, g_logprob, g_entropy, g_top_logprob, row_stats, row_mask,
                        same_phase ? 0 : 1};
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case ORLHF_F32: return launch_top_bwd<ORLHF_F32>(a, s);
    case ORLHF_BF16: return launch_top_bwd<ORLHF_BF16>(a, s);
    default: return launch_top_bwd<ORLHF_F16>(a, s);
  }
}
