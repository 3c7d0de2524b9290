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

#include "list_rows.h"

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

// How many of the n candidates rank before each of this thread's (at threadIdx.x + i * kBlock). The
// candidates are read two by two, all lanes the same: a broadcast.
typedef uint64_t u64x2 __attribute__((ext_vector_type(2)));
template <int MINE>
__device__ __forceinline__ void rank_candidates(const Candidates& c, int n, uint64_t (&mine)[MINE], int (&rank)[MINE]) {
#pragma unroll
  for (int i = 0; i < MINE; ++i) {
    const int at = (int)threadIdx.x + i * kBlock;
    mine[i] = at < n ? c.key[at] : 0ull;
    rank[i] = 0;
  }
  if ((int)(threadIdx.x & ~(kWave - 1u)) >= n) return;  // a wave without a candidate
  auto count = [&](uint64_t other) {
#pragma unroll
    for (int i = 0; i < MINE; ++i) rank[i] += other > mine[i] ? 1 : 0;
  };
  constexpr int kAhead = MINE == 1 ? 4 : 1;  // more of them in registers where the usual rows come by
  int j = 0;
  for (; j + 2 * kAhead <= n; j += 2 * kAhead) {
    u64x2 two[kAhead];
#pragma unroll
    for (int q = 0; q < kAhead; ++q) two[q] = *(const u64x2*)(c.key + j + 2 * q);
#pragma unroll
    for (int q = 0; q < kAhead; ++q) count(two[q][0]), count(two[q][1]);
  }
  for (; j < n; ++j) count(c.key[j]);
}

template <int MINE>
__device__ __forceinline__ void sort_best(const Candidates& c, int n, int k) {
  uint64_t mine[MINE];
  int rank[MINE];
  rank_candidates<MINE>(c, n, mine, rank);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < MINE; ++i) {
    const int at = (int)threadIdx.x + i * kBlock;
    if (at < n && rank[i] < k) c.key[rank[i]] = mine[i];
  }
}

// Keeps the k best candidates, sorted, and returns the k-th (0 while there are fewer). The whole
// workgroup calls it with the candidates in place behind a barrier; another one ends it.
__device__ __forceinline__ uint64_t keep_best(const Candidates& c, int k) {
  const int n = c.count;
  if (n <= 2 * kBlock) {
    sort_best<2>(c, n, k);
  } else {
    sort_best<kCap / kBlock>(c, n, k);
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
    const uint32_t v = v0 + tid, id = first + g.head + v * EPV;
    bool any = false;
    if (v < g.nvec) {
      float x[EPV];
      E::unpack(*(const u32x4*)(body + v * 16u), x);
#pragma unroll
      for (int j = 0; j < EPV; ++j) any = any || make_key(x[j], id + j) > least;
    }
    if (__syncthreads_or(any)) {
#pragma unroll 1
      for (int j = 0; j < EPV; ++j)  // rare rows: read once more rather than held in registers
        push_round(c, v < g.nvec ? make_key(E::load1(body + v * 16u + j * E::kSize), id + j) : 0ull, k, least);
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
  ListSplit split;
  uint64_t* records;  // split rows: kTotalsWords + k words per (row, segment)
  int32_t* tickets;   // split rows: one per row, zero between launches; NULL: a second launch merges
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
// eighth of the row: 221 against 208 us at 4096 x 151936 bf16, k = 64.) A row that has more candidates
// than fit (many equal logits), or a NaN, goes through collect_row instead.
constexpr int kMaxBlocks = 32;
constexpr uint32_t kBlockVecs = kStepVecs;  // vectors in a block: as many as a step gives each lane

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

struct BlockMaxima {
  static constexpr bool kMaxima = true;
  float* block_max;
  int shift;
  float thread_max;
  __device__ __forceinline__ void ready() const {}
  template <int N>
  __device__ __forceinline__ void vec(float (&)[N], uint32_t) const {}
  __device__ __forceinline__ void one(float&, uint32_t) const {}
  // Maxima of a step's vectors. The remainder (step == whole) is noted first: it opens its slot, the
  // others of the slot add to it.
  __device__ __forceinline__ void note(uint32_t step, uint32_t whole, uint32_t rest, const float (&m)[kStepVecs]) {
    const float bm = quad_maxima(m);
    float* slot = block_max + (step >> shift) * kBlock + threadIdx.x;
    const bool opens = (step & ((1u << shift) - 1u)) == 0u && (shift == 0 || rest == 0u || (step >> shift) != (whole >> shift));
    *slot = opens || step == whole ? bm : fmaxf(*slot, bm);
    thread_max = fmaxf(thread_max, bm);
  }
};

// The largest value of 16 leading bits that at least k of the 256 values reach: one wave, four values
// per lane, one counting step per bit.
__device__ __forceinline__ uint32_t kth_largest(const uint32_t* values, int k) {
  const int lane = threadIdx.x & (kWave - 1);
  const u32x4 o = *(const u32x4*)(values + lane * 4);
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

struct TopShared {
  float lds[kWavesPerBlock][8];
  int n_cand;
  BlockList list;
  alignas(16) uint32_t best[kBlock];  // ordered bits of the largest value each thread has seen
  uint32_t bar_bits;
  RowSoftmax softmax;
};

// The row's outputs from its candidates (in place behind a barrier) and its softmax.
template <int MODE>
__device__ __forceinline__ void write_row(const TopArgs& a, int64_t row_i, const Candidates& cand, int64_t label,
                                          float x_label, const RowSoftmax& softmax) {
  const int tid = threadIdx.x, n = cand.count;
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
      a.logprob[row_i] = label >= 0 && label < a.vocab ? logprob_of(x_label, a.temperature, softmax) : (label == kIgnoredLabel ? 0.0f : NAN);
    if (ModeTraits<MODE>::kPlainSet && a.entropy != nullptr) a.entropy[row_i] = (float)softmax.entropy;
    if (a.row_stats != nullptr) *(f32x4*)(a.row_stats + row_i * 4) = f32x4{softmax.centre, softmax.l2_t, softmax.l2_1, softmax.ex};
  }
}

// A cut row from its segments' records: the k best of their lists, the merged softmax.
template <int MODE, bool FRESH>
__device__ __forceinline__ void merge_top_row(const TopArgs& a, int64_t row_i, const Candidates& cand, TopShared& sh) {
  const int tid = threadIdx.x, stride = kTotalsWords + a.k, total = a.split.n * a.k;
  const uint64_t* rec = a.records + row_i * a.split.n * stride;
  const int64_t label = a.logprob != nullptr ? a.labels[row_i] : -1;
  float x_label = 0.0f;
  if (tid < kWave) {
    const int at = label >= 0 && label < a.vocab ? (int)(label / a.split.seg_elems) : -1;
    const RowTotals t = merge_totals<FRESH>(rec, stride, a.split.n, at, x_label);
    const RowSoftmax r = finish_row<MODE>(t, a.temperature);
    if (tid == 0) sh.softmax = r;
  }
  auto key_at = [&](int i) { return get64<FRESH>(rec + (int64_t)(i / a.k) * stride + kTotalsWords + i % a.k); };
  // a bar as in the rows themselves: the k-th largest of the threads' best keys (absent keys are 0)
  uint64_t best = 0;
#pragma unroll 1
  for (int i = tid; i < total; i += kBlock) {
    const uint64_t key = key_at(i);
    if (i < kCap) cand.key[i] = key;
    best = key > best ? key : best;
  }
  sh.best[tid] = (uint32_t)(best >> 32);
  if (tid == 0) sh.n_cand = 0;
  __syncthreads();
  if (tid < kWave) {
    const uint32_t bits = kth_largest(sh.best, a.k);
    if (tid == 0) sh.bar_bits = bits;
  }
  __syncthreads();
  const uint32_t bits = sh.bar_bits;
  const uint64_t least = bits != 0u ? ((uint64_t)bits << 32) - 1u : 0ull;
  uint64_t mine[kCap / kBlock];
#pragma unroll
  for (int i = 0; i < kCap / kBlock; ++i) mine[i] = tid + i * kBlock < total ? cand.key[tid + i * kBlock] : 0ull;
  __syncthreads();
  if (total <= kCap) {
#pragma unroll
    for (int i = 0; i < kCap / kBlock; ++i)
      if (mine[i] > least) cand.key[atomicAdd(&sh.n_cand, 1)] = mine[i];
  } else {
    uint64_t above = least;
#pragma unroll 1
    for (int i = tid; i - tid < total; i += kBlock) push_round(cand, i < total ? key_at(i) : 0ull, a.k, above);
  }
  __syncthreads();
  write_row<MODE>(a, row_i, cand, label, x_label, sh.softmax);
}

template <int DT, int MODE>
__global__ __launch_bounds__(kBlock) void top_logprobs_fwd_kernel(TopArgs a) {
  using E = Elt<DT>;
  __shared__ TopShared sh;
  extern __shared__ __align__(16) uint64_t shared[];  // block maxima while the row streams by, candidates afterwards
  float* const block_max = (float*)shared;
  const Candidates cand = {shared, sh.n_cand};
  const int tid = threadIdx.x;
  const Segment seg = segment_of(grid_row(), a.split, a.vocab);
  const int64_t row_i = seg.row;
  if (row_i >= a.n_rows) return;
  if (a.row_mask != nullptr && a.row_mask[row_i] == 0) {
    if (seg.index == 0) write_skipped_row(a, row_i);
    return;
  }
  const char* row = a.logits + row_i * a.row_stride_bytes + (int64_t)seg.first * E::kSize;
  const RowGeom g = row_geom<DT>(row, seg.len, false);
  if (tid == 0) sh.n_cand = sh.list.count = 0;
  // the label and its logit are asked for now and used by the row's last instructions
  int64_t label = -1;
  float x_label = 0.0f;
  if (a.logprob != nullptr && tid == 0) {
    label = a.labels[row_i];
    const int64_t at = label - (int64_t)seg.first;
    if (at >= 0 && at < seg.len) x_label = E::load1(row + at * E::kSize);
  }
  ListAcc<MODE> acc;
  BlockMaxima maxima = {block_max, a.shift, -INFINITY};
  stream_row<DT, MODE>(row, g, (float)(1.4426950408889634 / a.temperature), acc, maxima);
  sh.best[tid] = ordered_bits(maxima.thread_max);
  const RowSums sums = combine_fast<MODE>(acc, sh.lds);  // its barriers also publish the maxima
  RowTotals totals;
  if (fast_usable<MODE>(sums)) {
    totals = fast_totals<MODE>(sums);
  } else {
    totals = exact_totals<DT, MODE>(row, g, EveryElement{}, a.temperature, sh.lds);
  }
  const bool nan = totals.nan;
  if (tid < kWave) {  // one wave finds the bar, another takes the logarithms
    const uint32_t bits = kth_largest(sh.best, a.k);
    if (tid == 0) sh.bar_bits = bits;
  } else if (tid < 2 * kWave && a.split.n == 1) {
    const RowSoftmax r = finish_row<MODE>(totals, a.temperature);
    if (tid == kWave) sh.softmax = r;
  }
  __syncthreads();
  const uint32_t bits = sh.bar_bits;
  const float bar = bits <= ordered_bits(-INFINITY) ? -INFINITY : ordered_value(bits);
  collect_blocks<DT>(row, g, seg.first, block_max, a.shift, bar, maxima.thread_max, sh.list, cand);
  __syncthreads();
  int n = cand.count;
  if (n > kCap || sh.list.count > kListed || nan) {
    __syncthreads();
    if (tid == 0) sh.n_cand = 0;
    collect_row<DT>(row, g, seg.first, a.k, bits != 0u ? ((uint64_t)bits << 32) - 1u : 0ull, cand);
    n = cand.count;
  }
  if (a.split.n == 1) {
    write_row<MODE>(a, row_i, cand, label, x_label, sh.softmax);
    return;
  }
  uint64_t* rec = a.records + (row_i * a.split.n + seg.index) * (kTotalsWords + a.k);
  if (n > kBlock) {
    keep_best(cand, a.k);
    n = cand.count;
  }
  uint64_t key[1];
  int rank[1];
  rank_candidates<1>(cand, n, key, rank);
  if (tid < n && rank[0] < a.k) put64(rec + kTotalsWords + rank[0], key[0]);
  if (tid >= n && tid < a.k) put64(rec + kTotalsWords + tid, 0ull);
  if (tid == 0) put_totals(rec, totals, x_label);
  if (a.tickets != nullptr && last_segment(a.tickets + row_i, a.split.n)) merge_top_row<MODE, true>(a, row_i, cand, sh);
}

// The merge as a launch of its own, for callers without tickets.
template <int MODE>
__global__ __launch_bounds__(kBlock) void top_logprobs_merge_kernel(TopArgs a) {
  __shared__ TopShared sh;
  __shared__ __align__(16) uint64_t keys[kCap];
  const int64_t row_i = grid_row();
  if (row_i >= a.n_rows || (a.row_mask != nullptr && a.row_mask[row_i] == 0)) return;
  const Candidates cand = {keys, sh.n_cand};
  merge_top_row<MODE, false>(a, row_i, cand, sh);
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
  ListSplit split;
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
  const Segment seg = segment_of(grid_row(), a.split, a.vocab);
  const int64_t row_i = seg.row;
  if (row_i >= a.n_rows) return;
  const char* row = a.logits + row_i * a.row_stride_bytes + (int64_t)seg.first * E::kSize;
  char* out_row = a.grad + row_i * a.grad_stride_bytes + (int64_t)seg.first * E::kSize;
  const RowGeom g = row_geom<DT>(row, seg.len, a.scalar_only != 0);
  const bool skipped = a.row_mask != nullptr && a.row_mask[row_i] == 0;
  const bool mine = !skipped && tid < a.k && a.g_top != nullptr;
  const float gk = mine ? a.g_top[row_i * a.k + tid] : 0.0f;
  const int64_t id = mine ? a.top_ids[row_i * a.k + tid] - (int64_t)seg.first : -1;  // within the segment
  const float w = wave_sum(gk);
  const bool wave_on = __ballot(gk != 0.0f) != 0ull;  // NaN counts as on
  if ((tid & (kWave - 1)) == 0) lds[tid / kWave] = w;
  const bool top_on = __syncthreads_or(wave_on);
  float sum_top = 0.0f;
#pragma unroll
  for (int i = 0; i < kWavesPerBlock; ++i) sum_top += lds[i];
  __syncthreads();
  const int64_t label = a.g_logprob != nullptr ? a.labels[row_i] : -1;
  const float glp = a.g_logprob != nullptr && label != kIgnoredLabel ? a.g_logprob[row_i] : 0.0f;  // ignored: a constant
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
  fn.set_label(label >= 0 && label < a.vocab ? label - (int64_t)seg.first : -1, seg.len, g, E::kPerVec);
  const bool patch = mine && id >= 0 && id < seg.len;
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

template <int DT, int MODE>
static int launch_top_mode(const TopArgs& a, size_t lds, hipStream_t stream) {
  hipLaunchKernelGGL((top_logprobs_fwd_kernel<DT, MODE>), row_grid(a.n_rows * a.split.n), dim3(kBlock), lds, stream, a);
  ORLHF_CHECK_LAUNCH("orlhf_top_logprobs_fwd");
  if (a.split.n > 1 && a.tickets == nullptr) {
    hipLaunchKernelGGL((top_logprobs_merge_kernel<MODE>), row_grid(a.n_rows), dim3(kBlock), 0, stream, a);
    ORLHF_CHECK_LAUNCH("orlhf_top_logprobs_fwd(merge)");
  }
  return ORLHF_OK;
}

template <int DT>
static int launch_top_fwd(TopArgs a, hipStream_t stream) {
  const int64_t len = a.split.n == 1 ? a.vocab : (int64_t)a.split.seg_elems;
  const int64_t parts = (len / Elt<DT>::kPerVec + kBlockVecs * kBlock - 1) / (kBlockVecs * kBlock);
  while ((parts + (1 << a.shift) - 1) >> a.shift > kMaxBlocks) ++a.shift;
  const int64_t blocks = (parts + (1 << a.shift) - 1) >> a.shift;
  const size_t maxima = (size_t)blocks * kBlock * sizeof(float), keys = kCap * sizeof(uint64_t);
  const size_t lds = maxima > keys ? maxima : keys;
  if (a.entropy == nullptr) return launch_top_mode<DT, kLpOnly>(a, lds, stream);
  if (a.temperature == 1.0) return launch_top_mode<DT, kBothT1>(a, lds, stream);
  return launch_top_mode<DT, kBothT>(a, lds, stream);
}

template <int DT>
static int launch_top_bwd(const TopBwdArgs& a, hipStream_t stream) {
  const dim3 grid = row_grid(a.n_rows * a.split.n), block(kBlock);
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

extern "C" int64_t orlhf_top_logprobs_workspace_bytes(int dtype, int64_t n_rows, int64_t vocab, int64_t k) {
  if (n_rows <= 0 || vocab <= 0 || vocab >= (1ll << 29) || k < 1 || k > kMaxTop) return 0;
  const ListSplit split = list_split(n_rows, vocab, dtype == ORLHF_F32 ? 4 : 2);
  return split.n > 1 ? n_rows * split.n * (kTotalsWords + k) * (int64_t)sizeof(uint64_t) : 0;
}

extern "C" int orlhf_top_logprobs_fwd(const void* logits, int dtype, int64_t n_rows, int64_t vocab, int64_t row_stride,
                                      const int64_t* labels, double temperature, int64_t k, float* logprob,
                                      float* entropy, float* top_logprob, int64_t* top_ids, float* row_stats,
                                      const uint8_t* row_mask, void* workspace, int64_t workspace_bytes,
                                      int32_t* tickets, orlhf_stream_t stream) {
  const int bad = check_top("top_logprobs_fwd", dtype, n_rows, vocab, row_stride, temperature, k);
  if (bad != ORLHF_OK) return bad;
  if (n_rows == 0) return ORLHF_OK;  // nothing to launch; empty arrays may well be NULL
  ORLHF_CHECK_ARG(logits != nullptr && top_logprob != nullptr && top_ids != nullptr,
                  "top_logprobs_fwd: NULL logits / top_logprob / top_ids");
  ORLHF_CHECK_ARG(logprob == nullptr || labels != nullptr, "top_logprobs_fwd: labels is NULL");
  ORLHF_CHECK_ARG(((uintptr_t)logits & (dtype == ORLHF_F32 ? 3u : 1u)) == 0,
                  "top_logprobs_fwd: logits not aligned to the element size");
  const int64_t esize = dtype == ORLHF_F32 ? 4 : 2;
  const int64_t need = orlhf_top_logprobs_workspace_bytes(dtype, n_rows, vocab, k);
  ORLHF_CHECK_ARG(need == 0 || (workspace != nullptr && workspace_bytes >= need && ((uintptr_t)workspace & 7u) == 0),
                  "top_logprobs_fwd: this shape needs %lld bytes of 8-byte aligned workspace, got %lld", (long long)need,
                  (long long)workspace_bytes);
  ORLHF_CHECK_ARG(((uintptr_t)tickets & 3u) == 0, "top_logprobs_fwd: tickets not 4-byte aligned");
  const TopArgs a = {(const char*)logits, n_rows, vocab, row_stride * esize, labels, temperature, (int)k, logprob,
                     entropy, top_logprob, row_stats, top_ids, row_mask, 0, list_split(n_rows, vocab, (int)esize),
                     (uint64_t*)workspace, tickets};
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
                        same_phase ? 0 : 1, list_split(n_rows, vocab, (int)esize)};
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case ORLHF_F32: return launch_top_bwd<ORLHF_F32>(a, s);
    case ORLHF_BF16: return launch_top_bwd<ORLHF_BF16>(a, s);
    default: return launch_top_bwd<ORLHF_F16>(a, s);
  }
}
