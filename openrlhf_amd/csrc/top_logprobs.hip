// Log-prob of a given token, entropy and the K most likely tokens of every vocabulary row.
//
//   logprob = x_label / T - lse(x / T)            entropy = lse(x) - sum softmax(x) x
//   top     = the K largest x of the row, descending, equal values by ascending id,
//             each with x / T - lse(x / T)
//
// An element is one 64-bit key for the selection: the logit as an unsigned integer of the same
// order in the high half, the complement of its id in the low half. Keys are unique, "greater"
// means "ranked before", and a NaN (which has no order) ranks before everything.
#include <type_traits>

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
  uint64_t* key;  // [kCap], LDS
  int& count;
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
__device__ __forceinline__ uint64_t keep_best(const Candidates& c, int k) {
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
__device__ __forceinline__ void push_round(const Candidates& c, uint64_t key, int k, uint64_t& least) {
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
                                            const Candidates& c) {
  using E = Elt<DT>;
  constexpr int EPV = E::kPerVec;
  const uint32_t tid = threadIdx.x;
  const char* body = row + g.head * E::kSize;
#pragma unroll 1
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
#pragma unroll 1
      for (int j = 0; j < EPV; ++j) {  // not unrolled: the candidates' thinning is a large piece of code
        uint64_t mine = 0;
#pragma unroll
        for (int i = 0; i < EPV; ++i) mine = i == j ? key[i] : mine;
        push_round(c, mine, k, least);
      }
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

// One workgroup per row and no loop over rows in the kernels: a loop makes the compiler keep the
// constants of the whole body (of the logarithms above all) in registers, 20 to 30 per lane.
constexpr int64_t kGridX = 1 << 20;
inline dim3 row_grid(int64_t n_rows) {
  return dim3((unsigned)(n_rows < kGridX ? n_rows : kGridX), (unsigned)((n_rows + kGridX - 1) / kGridX));
}
__device__ __forceinline__ int64_t grid_row() { return (int64_t)blockIdx.y * kGridX + blockIdx.x; }

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

// The softmax of a row as what its outputs and its backward need: base + log_sum is the
// log-sum-exp of x / T (kept apart: base may be so large that the sum would be lost in it), `centre`
// a logit near base * T that every later difference starts from, entropy and E[x] - centre those of
// the unscaled logits.
struct RowSoftmax {
  double base, log_sum, entropy;
  float centre, l2_t, l2_1, ex;  // the backward's statistics: softmax(x / T) = 2^((x - centre) cT - l2_t)
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

// The sums of a row in the form that finish_row takes: of 2^((x - ref) c), with the reference in log2
// units after the fast pass and as a logit after the exact one.
struct RowTotals {
  float ref_t, ref_1;
  double sT, s1, t1;  // t1: sum of e x (fast) or of e (x - ref) (exact)
  bool fast, nan;
};

template <int MODE>
__device__ __forceinline__ bool fast_usable(const RowSums& s) {
  using MT = ModeTraits<MODE>;
  bool ok = true;
  if (MT::kScaledSet) ok = ok && sums_usable(s.sT) && fabsf(s.MT) < kFarReference;
  if (MT::kPlainSet) ok = ok && sums_usable(s.s1) && fabsf(s.t1) < INFINITY && fabsf(s.M1) < kFarReference;
  return ok;
}

// One vector per step: what only rare rows run must not cost the others their registers.
template <int DT, typename F>
__device__ __forceinline__ void walk_row(const char* row, const RowGeom& g, F& f) {
  using E = Elt<DT>;
  const uint32_t tid = threadIdx.x;
  const char* body = row + g.head * E::kSize;
#pragma unroll 1
  for (uint32_t v = tid; v < g.nvec; v += kBlock) {
    float x[E::kPerVec];
    E::unpack(*(const u32x4*)(body + v * 16u), x);
    f.vec(x, v);
  }
  if (tid < g.head + g.tail) {
    const uint32_t e = tid < g.head ? tid : g.nvec * E::kPerVec + tid;
    float x = E::load1(row + e * E::kSize);
    f.one(x, e);
  }
}

template <int DT, int MODE>
__device__ __forceinline__ RowTotals exact_totals(const char* row, const RowGeom& g, float c_scaled, float (*lds)[8]) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  MaxAcc top{-INFINITY, false};
  walk_row<DT>(row, g, top);
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
  ExactAcc<MODE> acc{m, c_scaled, kLog2e, 0.0f, 0.0f, 0.0f};
  walk_row<DT>(row, g, acc);
  const float st = wave_sum(acc.sT), s = wave_sum(acc.s1), t = wave_sum(acc.t1);
  if (lane == 0) {
    lds[wave][0] = st;
    lds[wave][1] = s;
    lds[wave][2] = t;
  }
  __syncthreads();
  RowTotals r = {m, m, 0.0, 0.0, 0.0, false, nans != 0.0f};
#pragma unroll
  for (int w = 0; w < kWavesPerBlock; ++w) {
    r.sT += (double)lds[w][0];
    r.s1 += (double)lds[w][1];
    r.t1 += (double)lds[w][2];
  }
  __syncthreads();
  if (r.nan || m == -INFINITY) r.sT = r.s1 = NAN;
  if (m == INFINITY) r.t1 = NAN;
  return r;
}

template <int MODE>
__device__ __forceinline__ RowSoftmax finish_row(const RowTotals& t, double temperature) {
  using MT = ModeTraits<MODE>;
  RowSoftmax r;
  const double scale = MT::kScaledSet ? temperature : 1.0;  // one set serves both where T = 1
  const double base_1 = t.fast ? (double)t.ref_1 * kLn2d : (double)t.ref_1;
  double log_1 = 0.0, ex = 0.0;  // of the unscaled logits; ex = E[x] - base_1
  if (MT::kPlainSet) {
    log_1 = log(t.s1);
    ex = t.t1 / t.s1 - (t.fast ? base_1 : 0.0);
  }
  r.base = MT::kScaledSet ? (t.fast ? (double)t.ref_t * kLn2d : (double)t.ref_t / temperature) : base_1;
  r.log_sum = MT::kScaledSet ? log(t.sT) : log_1;
  const double at = r.base * scale;
  r.centre = (float)at;
  r.l2_t = (float)((r.log_sum + (at - (double)r.centre) / scale) * 1.4426950408889634);
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
// The streaming pass leaves, beside the sums, the maximum of every BLOCK of the row in LDS and the
// maximum of all blocks of a thread in a register. A block is 64 consecutive bytes, the vectors that
// four neighbouring lanes load with one instruction (64 << shift bytes in pieces where a row has more
// than kMaxBlocks of them per thread); the four lanes exchange their maxima so that each keeps one of
// the four blocks of a step: 0.8 operations per element in all. The k-th largest of the 256 thread
// maxima is a lower bound of the row's k-th largest logit that few more than k elements pass
// (expected -256 ln(1 - k/256): 20 for k = 20, 177 for k = 128), so only the blocks that reach it are
// read again, about 64 k bytes per row, and their elements that reach it become candidates. (Blocks of
// one lane's four vectors need no exchange but lie 4 KiB apart, and reading them again fetched an
// eighth of the row: 221 against 197 us at 4096 x 151936 bf16, k = 64.) A row that has more candidates
// than fit (many equal logits), or a NaN, goes through collect_row instead.
constexpr int kMaxBlocks = 32;
constexpr uint32_t kBlockVecs = 4;  // vectors in a block, and a thread's loads per step

// Lane j of four gets the maximum over the four lanes of m[j].
__device__ __forceinline__ float quad_maxima(const float (&m)[4]) {
  const bool odd = (threadIdx.x & 1u) != 0u, high = (threadIdx.x & 2u) != 0u;
  auto with_neighbour = [](float keep, float give, auto ctrl) {
    constexpr int kCtrl = decltype(ctrl)::value;
    return fmaxf(keep, as_float((uint32_t)__builtin_amdgcn_mov_dpp((int)as_uint(give), kCtrl, 0xf, 0xf, true)));
  };
  constexpr std::integral_constant<int, 0xB1> kSwap1{};  // quad_perm [1, 0, 3, 2]
  constexpr std::integral_constant<int, 0x4E> kSwap2{};  // quad_perm [2, 3, 0, 1]
  const float lo = with_neighbour(odd ? m[1] : m[0], odd ? m[0] : m[1], kSwap1);
  const float hi = with_neighbour(odd ? m[3] : m[2], odd ? m[2] : m[3], kSwap1);
  return with_neighbour(high ? hi : lo, high ? lo : hi, kSwap2);
}

// The loads of the next block are in flight while one is worked on: two blocks of registers, 16 KiB
// asked for ahead by each workgroup at any time. The wave's exponent reference is the maximum of its
// lanes' first blocks.
template <int DT, int MODE>
__device__ __forceinline__ float stream_row(const char* row, const RowGeom& g, float c_scaled, FastAcc<MODE>& acc,
                                            float* block_max, int shift) {
  using E = Elt<DT>;
  constexpr int EPV = E::kPerVec;
  constexpr uint32_t kStep = kBlockVecs * kBlock;
  const uint32_t tid = threadIdx.x;
  const char* body = row + g.head * E::kSize;
  float thread_max = -INFINITY;
  const uint32_t parts = (g.nvec + kStep - 1) / kStep;
  auto load = [&](u32x4 (&raw)[kBlockVecs], uint32_t part) {  // past the end: the last vector again, not used
#pragma unroll
    for (uint32_t u = 0; u < kBlockVecs; ++u) {
      const uint32_t v = part * kStep + u * kBlock + tid;
      raw[u] = load_vec(body + (v < g.nvec ? v : g.nvec - 1) * 16u);
    }
  };
  auto consume = [&](const u32x4 (&raw)[kBlockVecs], uint32_t part) {
    float m[kBlockVecs] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    const uint32_t v0 = part * kStep + tid;
    auto take = [&](uint32_t u) {
      float x[EPV];
      E::unpack(raw[u], x);
#pragma unroll
      for (int j = 0; j < EPV; ++j) m[u] = fmaxf(m[u], x[j]);
      acc.vec(x, 0);
    };
    if ((part + 1) * kStep <= g.nvec) {
#pragma unroll
      for (uint32_t u = 0; u < kBlockVecs; ++u) take(u);
    } else {
#pragma unroll
      for (uint32_t u = 0; u < kBlockVecs; ++u)
        if (v0 + u * kBlock < g.nvec) take(u);
    }
    const float bm = quad_maxima(m);
    float* slot = block_max + (part >> shift) * kBlock + tid;
    *slot = (part & ((1u << shift) - 1u)) == 0u ? bm : fmaxf(*slot, bm);
    thread_max = fmaxf(thread_max, bm);
  };
  u32x4 ping[kBlockVecs], pong[kBlockVecs];
  if (parts > 0) load(ping, 0);
  // head and tail of a row off the 16-byte grid: at most one element per thread
  const uint32_t nscalar = g.head + g.tail;
  float xs = -INFINITY;
  if (tid < nscalar) xs = E::load1(row + (tid < g.head ? tid : g.nvec * EPV + tid) * E::kSize);
  float m_ref = xs;
  if (parts > 0) {
#pragma unroll
    for (uint32_t u = 0; u < kBlockVecs; ++u) {
      float x[EPV];
      E::unpack(ping[u], x);
#pragma unroll
      for (int j = 0; j < EPV; ++j) m_ref = fmaxf(m_ref, x[j]);
    }
  }
  acc.init(wave_max(m_ref), c_scaled, kLog2e);
  if (tid < nscalar) acc.one(xs, 0);
  for (uint32_t part = 0; part < parts;) {
    if (part + 1 < parts) load(pong, part + 1);
    consume(ping, part);
    if (++part >= parts) break;
    if (part + 1 < parts) load(ping, part + 1);
    consume(pong, part);
    ++part;
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

// The elements that reach `bar` in the blocks that do, into the candidates. The blocks are listed
// first, so that their vectors spread over the whole workgroup and all are asked for at once (each
// thread reading its own blocks one after the other costs a memory latency per block: 260 against
// 238 us at 4096 x 151936 bf16, k = 64). Counts beyond kListed or kCap mean that not everything is there.
constexpr int kListed = 1024;
struct BlockList {
  uint16_t block[kListed];  // block number * 256 + thread
  int count;
};
static_assert(kMaxBlocks * kBlock <= 65536, "a listed block fits 16 bits");

template <int DT>
__device__ __forceinline__ void collect_blocks(const char* row, const RowGeom& g, uint32_t first, const float* block_max,
                                               int shift, float bar, float thread_max, BlockList& list, const Candidates& c) {
  using E = Elt<DT>;
  constexpr int EPV = E::kPerVec;
  constexpr uint32_t kStep = kBlockVecs * kBlock;
  const uint32_t tid = threadIdx.x;
  const char* body = row + g.head * E::kSize;
  if (thread_max >= bar) {
    const uint32_t parts = (g.nvec + kStep - 1) / kStep;
    const uint32_t blocks = (parts + (1u << shift) - 1u) >> shift;
    for (uint32_t b = 0; b < blocks; ++b) {
      if (block_max[b * kBlock + tid] >= bar) {
        const int at = atomicAdd(&list.count, 1);
        if (at < kListed) list.block[at] = (uint16_t)(b * kBlock + tid);
      }
    }
  }
  auto push = [&](float x, uint32_t id) {
    const int at = atomicAdd(&c.count, 1);
    if (at < kCap) c.key[at] = make_key(x, id);
  };
  __syncthreads();  // from here on the candidates take the place of the block maxima
  const int listed = list.count;
  const uint32_t nscalar = g.head + g.tail;
  if (tid < nscalar) {
    const uint32_t e = tid < g.head ? tid : g.nvec * EPV + tid;
    const float x = E::load1(row + e * E::kSize);
    if (x >= bar) push(x, first + e);
  }
  const uint32_t per_shift = 2u + (uint32_t)shift;  // log2 of the vectors in a block
  static_assert(kBlockVecs == 4, "per_shift");
  if (listed <= kListed) {
    for (uint32_t i = tid; i < (uint32_t)listed << per_shift; i += kBlock) {
      const uint32_t blk = list.block[i >> per_shift];
      const uint32_t t = blk % kBlock, in = i & ((1u << per_shift) - 1u);
      const uint32_t v = (((blk / kBlock) << shift) + in / kBlockVecs) * kStep + t % 4u * kBlock + (t & ~3u) + in % kBlockVecs;
      if (v < g.nvec) {
        float x[EPV];
        E::unpack(*(const u32x4*)(body + v * 16u), x);
        float m = x[0];
#pragma unroll
        for (int j = 1; j < EPV; ++j) m = fmaxf(m, x[j]);
        if (m >= bar) {
#pragma unroll
          for (int j = 0; j < EPV; ++j)
            if (x[j] >= bar) push(x[j], first + g.head + v * EPV + j);
        }
      }
    }
  }
}

template <int DT, int MODE>
__global__ __launch_bounds__(kBlock) void top_logprobs_fwd_kernel(TopArgs a) {
  using E = Elt<DT>;
  __shared__ float lds[kWavesPerBlock][8];
  __shared__ int n_cand;
  __shared__ BlockList list;
  __shared__ alignas(16) float thread_maxima[kBlock];
  __shared__ uint32_t bar_bits;
  __shared__ RowSoftmax softmax;
  extern __shared__ uint64_t shared[];  // block maxima while the row streams by, candidates afterwards
  float* const block_max = (float*)shared;
  const Candidates cand = {shared, n_cand};
  const int tid = threadIdx.x;
  const float c_scaled = (float)(1.4426950408889634 / a.temperature);
  const int64_t row_i = grid_row();
  if (row_i >= a.n_rows) return;
  if (a.row_mask != nullptr && a.row_mask[row_i] == 0) {
    write_skipped_row(a, row_i);
    return;
  }
  const char* row = a.logits + row_i * a.row_stride_bytes;
  const RowGeom g = row_geom<DT>(row, a.vocab, false);
  if (tid == 0) n_cand = list.count = 0;
  // the label and its logit are asked for now and used by the row's last instructions
  int64_t label = -1;
  float x_label = 0.0f;
  if (a.logprob != nullptr && tid == 0) {
    label = a.labels[row_i];
    if (label >= 0 && label < a.vocab) x_label = E::load1(row + label * E::kSize);
  }
  FastAcc<MODE> acc;
  const float thread_max = stream_row<DT, MODE>(row, g, c_scaled, acc, block_max, a.shift);
  thread_maxima[tid] = thread_max;
  const RowSums sums = combine_fast<MODE>(acc, lds);  // its barriers also publish the maxima
  const bool fast = fast_usable<MODE>(sums);
  RowTotals totals = {sums.MT, sums.M1, sums.sT, sums.s1, sums.t1, true, false};
  if (!fast) totals = exact_totals<DT, MODE>(row, g, c_scaled, lds);
  const bool nan = totals.nan;
  if (tid < kWave) {  // one wave finds the bar, another takes the logarithms
    const uint32_t bits = kth_maximum(thread_maxima, a.k);
    if (tid == 0) bar_bits = bits;
  } else if (tid < 2 * kWave) {
    const RowSoftmax r = finish_row<MODE>(totals, a.temperature);
    if (tid == kWave) softmax = r;
  }
  __syncthreads();
  const uint32_t bits = bar_bits;
  const float bar = bits <= ordered_bits(-INFINITY) ? -INFINITY : ordered_value(bits);
  collect_blocks<DT>(row, g, 0u, block_max, a.shift, bar, thread_max, list, cand);
  __syncthreads();
  int n = cand.count;
  if (n > kCap || list.count > kListed || nan) {
    __syncthreads();
    if (tid == 0) cand.count = 0;
    collect_row<DT>(row, g, 0u, a.k, bits != 0u ? ((uint64_t)bits << 32) - 1u : 0ull, cand);
    n = cand.count;
  }
  auto out = [&](uint64_t key, int at) {
    a.top_ids[row_i * a.k + at] = (int64_t)key_id(key);
    a.top_logprob[row_i * a.k + at] = logprob_of(ordered_value((uint32_t)(key >> 32)), a.temperature, softmax);
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
      a.logprob[row_i] = label >= 0 && label < a.vocab ? logprob_of(x_label, a.temperature, softmax) : (label == -100 ? 0.0f : NAN);
    if (ModeTraits<MODE>::kPlainSet && a.entropy != nullptr) a.entropy[row_i] = (float)softmax.entropy;
    if (a.row_stats != nullptr) *(f32x4*)(a.row_stats + row_i * 4) = f32x4{softmax.centre, softmax.l2_t, softmax.l2_1, softmax.ex};
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
  const int64_t row_i = grid_row();
  if (row_i >= a.n_rows) return;
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
    return;
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
  }
}

template <int DT>
static int launch_top_fwd(TopArgs a, hipStream_t stream) {
  const bool t1 = a.temperature == 1.0;
  const int64_t parts = (a.vocab / Elt<DT>::kPerVec + kBlockVecs * kBlock - 1) / (kBlockVecs * kBlock);
  while ((parts + (1 << a.shift) - 1) >> a.shift > kMaxBlocks) ++a.shift;
  const int64_t blocks = (parts + (1 << a.shift) - 1) >> a.shift;
  const size_t maxima = (size_t)blocks * kBlock * sizeof(float), keys = kCap * sizeof(uint64_t);
  const size_t lds = maxima > keys ? maxima : keys;
  const dim3 grid = row_grid(a.n_rows), block(kBlock);
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
  const dim3 grid = row_grid(a.n_rows), block(kBlock);
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
