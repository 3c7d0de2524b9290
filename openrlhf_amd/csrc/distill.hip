// Distillation from a teacher's top tokens over vocabulary rows: forward and its streaming backward
// (mathematics in distill_terms.h).
//
// The forward reads the row once: the softmax sum of the elements outside the list, with the list as one
// bit per element in LDS (a byte per 16-byte vector of 8: one byte read and one branch per vector, where
// a search of the list would be work per element). One wave holds the list and finishes the row in fp64.
// The backward reads the row and writes its gradient, then stores the listed elements' gradients, which
// the forward has left per entry, over the row pass's values.
#include "distill_terms.h"

namespace orlhf {

struct DistillArgs {
  const char* logits;
  int64_t n_rows, vocab, row_stride_bytes;
  ListSource list;
  double temperature;
  int kind;
  float *loss, *row_stats, *list_grad;  // row_stats, list_grad, list_at: for the backward, NULL together
  int32_t* list_at;
  const uint8_t* row_mask;
  ListSplit split;
  uint64_t* records;
  int32_t* tickets;
};

__device__ __forceinline__ void write_list_row(const DistillArgs& a, int64_t row_i, const ListEntries& e, const ListTerms& t) {
  const int lane = threadIdx.x & (kWave - 1);
  if (lane == 0) a.loss[row_i] = (float)t.loss;
  if (a.row_stats == nullptr) return;
  if (lane == 0) *(f32x4*)(a.row_stats + row_i * 4) = f32x4{t.centre, t.l2, (float)t.other, (float)t.loss};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int at = lane + i * kWave;
    if (at < a.list.k) {
      a.list_at[row_i * a.list.k + at] = e.id[i];
      a.list_grad[row_i * a.list.k + at] = (float)t.grad[i];
    }
  }
}

__device__ __forceinline__ void write_skipped_list_row(const DistillArgs& a, int64_t row_i) {
  if (threadIdx.x == 0) a.loss[row_i] = 0.0f;
  if (a.row_stats == nullptr) return;
  if (threadIdx.x == 0) *(f32x4*)(a.row_stats + row_i * 4) = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  for (int at = threadIdx.x; at < a.list.k; at += blockDim.x) {
    a.list_at[row_i * a.list.k + at] = -1;
    a.list_grad[row_i * a.list.k + at] = 0.0f;
  }
}

// The list is fetched and marked while the row's first loads are on their way.
template <int DT>
struct ListWatch : WithoutListed<DT> {
  static constexpr bool kMaxima = false;
  const DistillArgs* a;
  RowGeom g;
  Segment seg;
  const char* row0;  // the whole row
  ListEntries* entries;  // of wave 0
  __device__ __forceinline__ void ready() const {
    this->map.clear(g, kBlock);
    __syncthreads();
    if (threadIdx.x < kWave) {
      *entries = load_list<DT>(a->list, seg.row, row0, a->vocab);
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (entries->id[i] >= 0) this->map.set(g, entries->id[i] - (int64_t)seg.first, seg.len);
    }
    __syncthreads();
  }
};

template <int DT>
__global__ __launch_bounds__(kBlock) void distill_fwd_kernel(DistillArgs a) {
  using E = Elt<DT>;
  __shared__ float lds[kWavesPerBlock][8];
  __shared__ uint32_t ends;
  extern __shared__ u32x4 map_words[];
  const int tid = threadIdx.x;
  const Segment seg = segment_of(grid_row(), a.split, a.vocab);
  if (seg.row >= a.n_rows) return;
  if (a.row_mask != nullptr && a.row_mask[seg.row] == 0) {
    if (seg.index == 0) write_skipped_list_row(a, seg.row);
    return;
  }
  const char* row0 = a.logits + seg.row * a.row_stride_bytes;
  const char* row = row0 + (int64_t)seg.first * E::kSize;
  const RowGeom g = row_geom<DT>(row, seg.len, false);
  ListEntries entries;
  ListWatch<DT> watch;
  watch.map = {(uint32_t*)map_words, &ends};
  watch.a = &a, watch.g = g, watch.seg = seg, watch.row0 = row0, watch.entries = &entries;
  ListAcc<kLpOnly> acc;
  stream_row<DT, kLpOnly>(row, g, (float)(1.4426950408889634 / a.temperature), acc, watch);
  const RowSums sums = combine_fast<kLpOnly>(acc, lds);
  RowTotals totals;
  if (fast_usable<kLpOnly>(sums)) {
    totals = fast_totals<kLpOnly>(sums);
  } else {
    totals = exact_totals<DT, kLpOnly>(row, g, watch, a.temperature, lds);
  }
  if (a.split.n > 1) {
    if (tid == 0) put_totals(a.records + (seg.row * a.split.n + seg.index) * kTotalsWords, totals, 0.0f);
    if (a.tickets == nullptr || !last_segment(a.tickets + seg.row, a.split.n)) return;
    if (tid < kWave) {
      float unused;
      totals = merge_totals<true>(a.records + seg.row * a.split.n * kTotalsWords, kTotalsWords, a.split.n, -1, unused);
    }
  }
  if (tid < kWave) write_list_row(a, seg.row, entries, list_terms(entries, totals, a.kind, a.temperature, a.vocab));
}

// The merge as a launch of its own, one wave per row, for callers without tickets.
template <int DT>
__global__ __launch_bounds__(kWave) void distill_merge_kernel(DistillArgs a) {
  const int64_t row_i = grid_row();
  if (row_i >= a.n_rows || (a.row_mask != nullptr && a.row_mask[row_i] == 0)) return;
  const ListEntries e = load_list<DT>(a.list, row_i, a.logits + row_i * a.row_stride_bytes, a.vocab);
  float unused;
  const RowTotals totals =
      merge_totals<false>(a.records + row_i * a.split.n * kTotalsWords, kTotalsWords, a.split.n, -1, unused);
  write_list_row(a, row_i, e, list_terms(e, totals, a.kind, a.temperature, a.vocab));
}

struct DistillBwdArgs {
  const char* logits;
  char* grad;
  int64_t n_rows, vocab, row_stride_bytes, grad_stride_bytes;
  int k;
  double temperature;
  const float *g_loss, *row_stats, *list_grad;
  const int32_t* list_at;
  const uint8_t* row_mask;
  int scalar_only;
  ListSplit split;
};

template <int DT>
__global__ __launch_bounds__(kBlock) void distill_bwd_kernel(DistillBwdArgs a) {
  using E = Elt<DT>;
  const int tid = threadIdx.x;
  const Segment seg = segment_of(grid_row(), a.split, a.vocab);
  if (seg.row >= a.n_rows) return;
  const char* row = a.logits + seg.row * a.row_stride_bytes + (int64_t)seg.first * E::kSize;
  char* out_row = a.grad + seg.row * a.grad_stride_bytes + (int64_t)seg.first * E::kSize;
  const RowGeom g = row_geom<DT>(row, seg.len, a.scalar_only != 0);
  const float gl = a.g_loss[seg.row];
  if (gl == 0.0f || (a.row_mask != nullptr && a.row_mask[seg.row] == 0)) {
    zero_row<DT>(out_row, g);
    return;
  }
  const int64_t at = tid < a.k ? (int64_t)a.list_at[seg.row * a.k + tid] : -1;
  const bool patch = at >= (int64_t)seg.first && at < (int64_t)seg.first + seg.len;
  const float val = patch ? (float)((double)gl * (double)a.list_grad[seg.row * a.k + tid] / a.temperature) : 0.0f;
  const f32x4 st = *(const f32x4*)(a.row_stats + seg.row * 4);
  ListGrad<kBwdLp> fn = {};
  fn.centre = st[0];
  fn.cT = (float)(1.4426950408889634 / a.temperature);
  fn.negLT = -st[1];
  fn.a_all = grad_coef((double)gl, (double)st[2], a.temperature);
  fn.set_label(-1, seg.len, g, E::kPerVec);
  traverse_row<DT, true>(row, out_row, g, fn);
  __syncthreads();  // the row pass's values are in place
  if (patch) E::store1(out_row + (at - (int64_t)seg.first) * E::kSize, val);
}

template <int DT>
static int launch_distill_fwd(const DistillArgs& a, hipStream_t stream) {
  const dim3 grid = row_grid(a.n_rows * a.split.n), block(kBlock);
  const int64_t len = a.split.n == 1 ? a.vocab : (int64_t)a.split.seg_elems;
  hipLaunchKernelGGL((distill_fwd_kernel<DT>), grid, block, (size_t)ListMap<DT>::bytes(len), stream, a);
  ORLHF_CHECK_LAUNCH("orlhf_distill_kl_fwd");
  if (a.split.n > 1 && a.tickets == nullptr) {
    hipLaunchKernelGGL((distill_merge_kernel<DT>), row_grid(a.n_rows), dim3(kWave), 0, stream, a);
    ORLHF_CHECK_LAUNCH("orlhf_distill_kl_fwd(merge)");
  }
  return ORLHF_OK;
}

template <int DT>
static int launch_distill_bwd(const DistillBwdArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL((distill_bwd_kernel<DT>), row_grid(a.n_rows * a.split.n), dim3(kBlock), 0, stream, a);
  ORLHF_CHECK_LAUNCH("orlhf_distill_kl_bwd");
  return ORLHF_OK;
}

}  // namespace orlhf

using namespace orlhf;

extern "C" int64_t orlhf_distill_kl_workspace_bytes(int dtype, int64_t n_rows, int64_t vocab) {
  if (n_rows <= 0 || vocab <= 0 || vocab > kMaxDistillVocab) return 0;
  const ListSplit split = list_split(n_rows, vocab, dtype == ORLHF_F32 ? 4 : 2);
  return split.n > 1 ? n_rows * split.n * kTotalsWords * (int64_t)sizeof(uint64_t) : 0;
}

extern "C" int orlhf_distill_kl_fwd(const void* logits, int dtype, int64_t n_rows, int64_t vocab, int64_t row_stride,
                                    const int64_t* teacher_ids, const float* teacher_logprob, int64_t k, double temperature,
                                    double teacher_temperature, int kind, float* loss, float* row_stats, float* list_grad,
                                    int32_t* list_at, const uint8_t* row_mask, void* workspace, int64_t workspace_bytes,
                                    int32_t* tickets, orlhf_stream_t stream) {
  int bad = check_distill("distill_kl_fwd", dtype, n_rows, vocab, row_stride, k, temperature);
  if (bad == ORLHF_OK) bad = check_kind("distill_kl_fwd", kind, teacher_temperature);
  if (bad != ORLHF_OK) return bad;
  if (n_rows == 0) return ORLHF_OK;  // nothing to launch; empty arrays may well be NULL
  ORLHF_CHECK_ARG(logits != nullptr && teacher_ids != nullptr && teacher_logprob != nullptr && loss != nullptr,
                  "distill_kl_fwd: NULL logits / teacher_ids / teacher_logprob / loss");
  ORLHF_CHECK_ARG((row_stats == nullptr) == (list_grad == nullptr) && (row_stats == nullptr) == (list_at == nullptr),
                  "distill_kl_fwd: row_stats, list_grad and list_at go together");
  const int64_t esize = dtype == ORLHF_F32 ? 4 : 2;
  ORLHF_CHECK_ARG(((uintptr_t)logits & (uintptr_t)(esize - 1)) == 0, "distill_kl_fwd: logits not aligned to the element size");
  const int64_t need = orlhf_distill_kl_workspace_bytes(dtype, n_rows, vocab);
  ORLHF_CHECK_ARG(need == 0 || (workspace != nullptr && workspace_bytes >= need && ((uintptr_t)workspace & 7u) == 0),
                  "distill_kl_fwd: this shape needs %lld bytes of 8-byte aligned workspace, got %lld", (long long)need,
                  (long long)workspace_bytes);
  ORLHF_CHECK_ARG(((uintptr_t)tickets & 3u) == 0, "distill_kl_fwd: tickets not 4-byte aligned");
  const DistillArgs a = {(const char*)logits, n_rows, vocab, row_stride * esize,
                         {teacher_ids, teacher_logprob, (int)k, 1.0 / teacher_temperature, kind == ORLHF_DISTILL_FORWARD},
                         temperature, kind, loss, row_stats, list_grad, list_at, row_mask,
                         list_split(n_rows, vocab, (int)esize), (uint64_t*)workspace, tickets};
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case ORLHF_F32: return launch_distill_fwd<ORLHF_F32>(a, s);
    case ORLHF_BF16: return launch_distill_fwd<ORLHF_BF16>(a, s);
    default: return launch_distill_fwd<ORLHF_F16>(a, s);
  }
}

extern "C" int orlhf_distill_kl_bwd(const void* logits, void* grad_logits, int dtype, int64_t n_rows, int64_t vocab,
                                    int64_t row_stride, int64_t grad_row_stride, int64_t k, double temperature,
                                    const float* g_loss, const float* row_stats, const float* list_grad,
                                    const int32_t* list_at, const uint8_t* row_mask, orlhf_stream_t stream) {
  const int bad = check_distill("distill_kl_bwd", dtype, n_rows, vocab, row_stride, k, temperature);
  if (bad != ORLHF_OK) return bad;
  ORLHF_CHECK_ARG(grad_row_stride >= vocab, "distill_kl_bwd: grad_row_stride %lld < vocab %lld", (long long)grad_row_stride,
                  (long long)vocab);
  if (n_rows == 0) return ORLHF_OK;
  ORLHF_CHECK_ARG(logits != nullptr && grad_logits != nullptr && g_loss != nullptr && row_stats != nullptr &&
                      list_grad != nullptr && list_at != nullptr,
                  "distill_kl_bwd: NULL logits / grad_logits / g_loss / row_stats / list_grad / list_at");
  const int64_t esize = dtype == ORLHF_F32 ? 4 : 2;
  ORLHF_CHECK_ARG((((uintptr_t)logits | (uintptr_t)grad_logits) & (uintptr_t)(esize - 1)) == 0,
                  "distill_kl_bwd: pointers not aligned to the element size");
  const bool same_phase = (((uintptr_t)logits ^ (uintptr_t)grad_logits) & 15u) == 0 &&
                          (((row_stride - grad_row_stride) * esize) & 15) == 0;
  const DistillBwdArgs a = {(const char*)logits, (char*)grad_logits, n_rows, vocab, row_stride * esize,
                            grad_row_stride * esize, (int)k, temperature, g_loss, row_stats, list_grad, list_at, row_mask,
                            same_phase ? 0 : 1, list_split(n_rows, vocab, (int)esize)};
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case ORLHF_F32: return launch_distill_bwd<ORLHF_F32>(a, s);
    case ORLHF_BF16: return launch_distill_bwd<ORLHF_BF16>(a, s);
    default: return launch_distill_bwd<ORLHF_F16>(a, s);
  }
}
