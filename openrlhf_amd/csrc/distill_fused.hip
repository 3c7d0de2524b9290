// Distillation, forward and backward in one pass for callers that know the upstream weights when the
// forward runs (loss = sum_i weight[i] * KL_i): every vocabulary row is read once, kept on chip and its
// gradient written once.
//
// A row of 151936 bf16 logits is 297 KiB; the vector registers of one CU are 512 KiB. One 512-thread
// workgroup owns a CU and a row: every lane keeps 38 16-byte chunks of it in registers (rows up to 155648
// 16-bit or 77824 fp32 elements); a longer row keeps its first 32 chunks per lane and streams the rest
// twice, once for the sum and once, mostly from the caches, for the gradient. While chunk c of a row is
// turned into its gradient and stored, chunk c of the workgroup's next row is loaded into the registers
// that it leaves.
//
// The list: a bit per element in LDS marks the listed elements, so that the sum leaves them out and the
// gradient pass puts their own gradients in place as it goes (id and value from a small hash table in
// LDS): no second store to them, and so no wait for the first. One wave fetches, checks and marks the list of the next row
// while that row's loads are in flight; map and table are double.
#include <type_traits>

#include "distill_terms.h"

namespace orlhf {

constexpr int kOneBlock = 512;
constexpr int kOneWaves = kOneBlock / kWave;
constexpr int kChunks = 38;      // 16-byte chunks of the row per lane
constexpr int kChunksLong = 32;  // the same for rows that do not fit: the rest is streamed twice
constexpr int kMaxFactor = 4;    // longest row: 4 x the resident part, and two maps of it fit LDS
constexpr int64_t kMaxMapped = 376832;
constexpr int kSlots = 256;      // of the hash table: twice the longest list
// Chunks of a lane that wait in LDS (its own 16 bytes each, no barrier) from the sum to the gradient: the
// fp64 arithmetic of the list in between needs their registers (without: 34 registers of the fp32 body spilled).
constexpr int kParked = 6;

struct OneArgs {
  const char* logits;
  char* grad;
  int64_t n_rows, vocab, row_stride_bytes, grad_stride_bytes;
  ListSource list;
  double temperature;
  int kind;
  const float* weight;
  float* loss;
  const uint8_t* row_mask;
  uint32_t map_words;  // of one map, a multiple of 4
};

// id -> gradient of the listed elements.
struct ListTable {
  int* key;  // [kSlots], -1: free
  float* value;
  static __device__ __forceinline__ uint32_t slot_of(int id) { return ((uint32_t)id * 2654435761u) >> 24; }
  // The slot of an id: its own, where another lane has put the same id already (`repeated`).
  __device__ __forceinline__ int insert(int id, bool& repeated) const {
    uint32_t s = slot_of(id);
#pragma unroll 1
    for (int n = 0; n < kSlots; ++n) {  // 128 of 256 taken at most
      const int was = atomicCAS(key + s, -1, id);
      repeated = was == id;
      if (was == -1 || repeated) break;
      s = (s + 1u) % kSlots;
    }
    return (int)s;
  }
  __device__ __forceinline__ float find(int id) const {
    uint32_t s = slot_of(id);
#pragma unroll 1
    for (int n = 0; n < kSlots && key[s] != id; ++n) s = (s + 1u) % kSlots;  // only marked ids are looked up: it is there
    return value[s];
  }
};

// A row's list while the row is on chip: one wave's, kept in LDS because the row has the registers.
struct ListState {
  double lp[kMaxList], p[kMaxList];
  float x[kMaxList];
  int id[kMaxList], slot[kMaxList];
  double mass, t, log_t, log_mass, top, sum;  // TeacherTerms, StudentTerms
  uint32_t head, nvec;                        // of the row
  float weight;
  int n_on, bad;
};

// The workgroup's static LDS; the dynamic part holds the two maps and the parked chunks.
struct OneShared {
  float lds[kOneWaves][4];
  float bcast[4];
  uint32_t ends[2];
  int keys[2][kSlots];
  float values[2][kSlots];
  ListState state[2];
  uint32_t dirty[2][kOneBlock][2];
};
constexpr int64_t kLdsBytes = 160 * 1024;  // of a CU
static_assert((int64_t)sizeof(OneShared) + 2 * ((kMaxMapped + 127) / 128 * 16) + kParked * kOneBlock * 16 <= kLdsBytes,
              "the longest row's maps fit");

// Workgroup barrier for what passes through LDS: loads and stores of device memory stay in flight.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

__device__ __forceinline__ u32x4 pinned(const u32x4& v) {  // unpacked anew in every pass, not kept as eight floats
  uint32_t a = v[0], b = v[1], c = v[2], d = v[3];
  asm volatile("" : "+v"(a), "+v"(b), "+v"(c), "+v"(d));
  return u32x4{a, b, c, d};
}

template <int DT>
__device__ __forceinline__ u32x4 minus_inf_vec() {
  const uint32_t w = DT == ORLHF_F32 ? 0xff800000u : (DT == ORLHF_BF16 ? 0xff80ff80u : 0xfc00fc00u);
  return u32x4{w, w, w, w};
}

template <int DT, int CHUNKS, bool LONG>
__global__ __launch_bounds__(kOneBlock) void distill_one_pass_kernel(OneArgs a) {
  using E = Elt<DT>;
  constexpr int EPV = E::kPerVec;
  __shared__ OneShared sh;
  auto& lds = sh.lds;
  auto& bcast = sh.bcast;
  auto& ends = sh.ends;
  auto& keys = sh.keys;
  auto& values = sh.values;
  auto& state = sh.state;
  auto& dirty = sh.dirty;
  extern __shared__ u32x4 maps[];  // two maps, then the parked chunks
  u32x4(*const park)[kOneBlock] = (u32x4(*)[kOneBlock])(maps + a.map_words / 2);
  const uint32_t tid = threadIdx.x, tid16 = tid * 16u, lane = tid % kWave, wave = tid / kWave;
  const double inv_t = 1.0 / a.temperature;
  const float cT = (float)(1.4426950408889634 * inv_t);

  // next row of this workgroup that is wanted; `write`: unwanted rows on the way get their zeros
  auto next_active = [&](int64_t r, bool write) -> int64_t {
    while (r < a.n_rows && a.row_mask != nullptr && a.row_mask[r] == 0) {
      if (write) {
        char* out = a.grad + r * a.grad_stride_bytes;
        const RowGeom z = row_geom<DT>(a.logits + r * a.row_stride_bytes, a.vocab, false);
        for (uint32_t v = tid; v < z.nvec; v += kOneBlock) store_vec(out + z.head * E::kSize + v * 16u, u32x4{0u, 0u, 0u, 0u});
        if (tid < z.head + z.tail) E::store1(out + (tid < z.head ? tid : z.nvec * EPV + tid) * E::kSize, 0.0f);
        if (tid == 0) a.loss[r] = 0.0f;
      }
      r += gridDim.x;
    }
    return r;
  };

  for (uint32_t i = tid; i < a.map_words / 2; i += kOneBlock) maps[i] = u32x4{0u, 0u, 0u, 0u};  // both maps
  for (uint32_t i = tid; i < 2 * kSlots; i += kOneBlock) keys[0][i] = -1;
  if (tid < 2) ends[tid] = 0u;
  if (tid < 2 * kMaxList) state[tid / kMaxList].id[tid % kMaxList] = -1;
  dirty[0][tid][0] = dirty[0][tid][1] = dirty[1][tid][0] = dirty[1][tid][1] = 0u;

  // Whether this lane's chunk c lies in a row of n vectors; written so that no register per chunk is kept for it.
  auto within = [&](int c, uint32_t n) { return (int)tid < (int)n - c * kOneBlock; };

  u32x4 buf[CHUNKS];
  float xs = -INFINITY;
  int64_t row_i = next_active(blockIdx.x, true);
  RowGeom g = {0, 0, 0};
  int side = 0;

  // The lane's chunk that holds an element of the body, 63 for all that are streamed, and its flag word.
  auto chunk_of = [&](const RowGeom& r, uint32_t e) -> uint32_t {
    const uint32_t c = (e - r.head) / EPV / kOneBlock;
    return c < (uint32_t)CHUNKS ? c : 63u;
  };
  auto dirty_of = [&](int to, const RowGeom& r, uint32_t e) -> uint32_t* {
    if (e < r.head || e - r.head >= r.nvec * EPV) return nullptr;
    return &dirty[to][(e - r.head) / EPV % kOneBlock][chunk_of(r, e) / 32u];
  };

  // Wave 0: a row's list into the map, table and state of side `to`, which the list of two rows ago leaves.
  auto mark = [&](const RawList& raw, int64_t row, const RowGeom& gn, int to) {
    const ListMap<DT> map = {(uint32_t*)maps + to * a.map_words, ends + to};
    const ListTable table = {keys[to], values[to]};
    ListState& st = state[to];
    ListEntries e = settle_list<DT>(raw, a.list, a.logits + row * a.row_stride_bytes, a.vocab);
    const float weight = a.weight[row];
    const RowGeom old = {st.head, st.nvec, 0u};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int id = st.id[lane + i * kWave];
      if (id >= 0) {
        map.drop(old, (uint32_t)id);
        table.key[st.slot[lane + i * kWave]] = -1;
        uint32_t* d = dirty_of(to, old, (uint32_t)id);
        if (d != nullptr) d[0] = 0u;
      }
    }
    if (lane == 0) *map.ends = 0u;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the old entries are out before the new ones go in
    bool repeated = false;
    int slot[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int id = e.id[i];
      if (id >= 0) {
        bool again;
        slot[i] = table.insert(id, again);
        repeated = repeated || again;
        map.set(gn, id, a.vocab);
        uint32_t* d = dirty_of(to, gn, (uint32_t)id);
        if (d != nullptr) atomicOr(d, 1u << (chunk_of(gn, (uint32_t)id) % 32u));
      }
    }
    if (__ballot(repeated) != 0ull) join_repeats(e, a.list.k);
    const TeacherTerms t = teacher_terms(e, a.kind, a.vocab);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int at = (int)lane + i * kWave;
      st.id[at] = e.id[i];
      st.slot[at] = slot[i];
      st.x[at] = e.x[i];
      st.lp[at] = e.lp[i];
      st.p[at] = t.p[i];
    }
    if (lane == 0) {
      st.mass = t.mass, st.t = t.t, st.log_t = t.log_t, st.log_mass = t.log_mass, st.n_on = t.n_on;
      st.head = gn.head, st.nvec = gn.nvec;
      st.weight = weight;
      st.bad = e.bad ? 1 : 0;
    }
  };
  auto listed = [&](int at) {  // of one wave
    ListEntries e;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      e.id[i] = state[at].id[lane + i * kWave];
      e.x[i] = state[at].x[lane + i * kWave];
      e.lp[i] = state[at].lp[lane + i * kWave];
    }
    e.bad = state[at].bad != 0;
    return e;
  };

  if (row_i < a.n_rows) {  // prologue: the first row's loads, then its list
    const char* row = a.logits + row_i * a.row_stride_bytes;
    g = row_geom<DT>(row, a.vocab, false);
    const char* body = row + g.head * E::kSize;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
      buf[c] = within(c, g.nvec) ? load_vec(body + (uint32_t)c * (kOneBlock * 16u) + tid16) : minus_inf_vec<DT>();
    if (tid < g.head + g.tail) xs = E::load1(row + (tid < g.head ? tid : g.nvec * EPV + tid) * E::kSize);
  }
  __syncthreads();  // the empty maps and tables
  if (row_i < a.n_rows && wave == 0) mark(fetch_list(a.list, row_i), row_i, g, 0);
  lds_barrier();

  while (row_i < a.n_rows) {
    const char* row = a.logits + row_i * a.row_stride_bytes;
    char* out_row = a.grad + row_i * a.grad_stride_bytes;
    const ListMap<DT> map = {(uint32_t*)maps + side * a.map_words, ends + side};
    const ListTable table = {keys[side], values[side]};
    const WithoutListed<DT> without = {map};
    const uint32_t nscalar = g.head + g.tail;
    const char* tail_body = row + g.head * E::kSize;
    constexpr uint32_t kResident = (uint32_t)CHUNKS * kOneBlock;

    // chunks of this lane with a listed element (the last bit: any of the streamed ones)
    const uint32_t dirty_lo = dirty[side][tid][0], dirty_hi = dirty[side][tid][1];
    auto mine = [&](int c) { return ((c < 32 ? dirty_lo : dirty_hi) >> (c % 32) & 1u) != 0u; };
    // what of the row the sum sees: all but the listed elements
    auto each = [&](auto&& f, auto&& settle, auto parked) {
      constexpr bool kFromLds = decltype(parked)::value;
      if (tid < nscalar) {
        float x = xs;
        without.one(x, tid);
        f(x, 0);
      }
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) {
        float x[EPV];
        E::unpack(pinned(kFromLds && c >= CHUNKS - kParked ? park[c - (CHUNKS - kParked)][tid] : buf[c]), x);
        if (mine(c)) without.vec(x, tid, (uint32_t)c * kOneBlock);  // never past the row, where the map ends
#pragma unroll
        for (int j = 0; j < EPV; ++j) f(x[j], j & 1);
        settle();
      }
      if (LONG) {
#pragma unroll 1
        for (uint32_t v = kResident + tid; v < g.nvec; v += kOneBlock) {
          float x[EPV];
          E::unpack(*(const u32x4*)(tail_body + v * 16u), x);
          without.vec(x, v);
#pragma unroll
          for (int j = 0; j < EPV; ++j) f(x[j], j & 1);
        }
      }
    };

    if (wave == 1) {  // the listed logits' own sum, while the row's loads land
      const StudentTerms t = student_terms(listed(side), inv_t);
      if (lane == 0) state[side].top = t.top, state[side].sum = t.sum;
    }

    // ---- sum against the wave maximum of each lane's first chunk (it lands first)
    float ref;
    {
      float x[EPV];
      E::unpack(pinned(buf[0]), x);
      if (mine(0)) without.vec(x, tid);
      ref = x[0];
#pragma unroll
      for (int j = 1; j < EPV; ++j) ref = fmaxf(ref, x[j]);
      ref = wave_max(ref) * cT;
    }
    // A wave past the end of a short row has nothing to refer to: reference 0 for its sum of nothing. (Another
    // wave without a finite first chunk gives NaN here, and the row takes the exact sums below.)
    const bool idle = wave != 0u && wave * kWave >= g.nvec;
    float acc[2] = {0.0f, 0.0f};
    {
      const float neg = idle ? 0.0f : -ref;
      each([&](float x, int k) { acc[k] += fast_exp2(fmaf(x, cT, neg)); },
           [&] { asm volatile("" : "+v"(acc[0]), "+v"(acc[1])); }, std::false_type{});
    }
#pragma unroll
    for (int c = CHUNKS - kParked; c < CHUNKS; ++c) park[c - (CHUNKS - kParked)][tid] = buf[c];
    const float ws = wave_sum(acc[0] + acc[1]);
    if (lane == 0) {
      lds[wave][0] = ref;
      lds[wave][1] = ws;
    }
    lds_barrier();
    float top = lds[0][0];
#pragma unroll
    for (int w = 1; w < kOneWaves; ++w) top = fmaxf(top, lds[w][0]);
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kOneWaves; ++w) sum = fmaf(lds[w][1], fast_exp2(lds[w][0] - top), sum);
    RowTotals totals = {(double)top * kLn2d, 0.0, (double)sum, 0.0, 0.0, false};
    if (!(sums_usable(sum) && fabsf(top) < kFarReference)) {  // rare, the same in every thread: exact maximum, then differences
      float m = -INFINITY;
      float odd = 0.0f;
      each([&](float x, int) {
        m = fmaxf(m, x);
        odd += x != x ? 1.0f : 0.0f;
      }, [&] { asm volatile("" : "+v"(m), "+v"(odd)); }, std::true_type{});
      m = wave_max(m);
      const bool nan = __ballot(odd != 0.0f) != 0ull;
      lds_barrier();
      if (lane == 0) {
        lds[wave][0] = m;
        lds[wave][1] = nan ? 1.0f : 0.0f;
      }
      lds_barrier();
      float nans = 0.0f;
#pragma unroll
      for (int w = 0; w < kOneWaves; ++w) {
        m = fmaxf(m, lds[w][0]);
        nans += lds[w][1];
      }
      float s = 0.0f;
      if (m != -INFINITY) each([&](float x, int) { s += fast_exp2((x == m ? 0.0f : x - m) * cT); }, [&] { asm volatile("" : "+v"(s)); }, std::true_type{});
      s = wave_sum(s);
      lds_barrier();
      if (lane == 0) lds[wave][1] = s;
      lds_barrier();
      totals = {(double)m / a.temperature, 0.0, 0.0, 0.0, 0.0, nans != 0.0f};
#pragma unroll
      for (int w = 0; w < kOneWaves; ++w) totals.sT += (double)lds[w][1];
    }

    // ---- the row's loss and gradient coefficients (one wave, fp64)
    const int64_t next_i = next_active(row_i + gridDim.x, false);
    if (wave == 0) {
      const ListState& st = state[side];
      const float w = st.weight;
      const ListEntries list = listed(side);
      const TeacherTerms teacher = {{st.p[lane], st.p[lane + kWave]}, st.mass, st.t, st.log_t, st.log_mass, st.n_on};
      const ListTerms t = list_terms(list, teacher, StudentTerms{st.top, st.sum}, totals, a.kind, a.temperature, a.vocab);
      if (lane == 0) {
        a.loss[row_i] = (float)t.loss;
        bcast[0] = w == 0.0f ? INFINITY : t.centre;  // weight 0: every exponent -inf, every gradient 0
        bcast[1] = w == 0.0f ? 0.0f : t.l2;
        bcast[2] = w == 0.0f ? 0.0f : grad_coef((double)w, t.other, a.temperature);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (list.id[i] >= 0) table.value[state[side].slot[lane + i * kWave]] = w == 0.0f ? 0.0f : (float)((double)w * t.grad[i] / a.temperature);
    }
    lds_barrier();
    const float centre = bcast[0], neg_l2 = -bcast[1], coef = bcast[2];
    auto grad_of = [&](float x) { return fast_exp2(fmaf(fmaxf(x - centre, -1.0e30f), cT, neg_l2)) * coef; };
    auto grad_vec = [&](float (&x)[EPV], uint32_t v, uint32_t step, int c) {
#pragma unroll
      for (int j = 0; j < EPV; ++j) x[j] = grad_of(x[j]);
      if (mine(c)) {
        // one loop over the set bits: unrolled per element the look-ups made half a megabyte of code
        uint32_t bits = map.vec(v, step);
#pragma unroll 1
        while (bits != 0u) {
          const int at = __builtin_ctz(bits);
          bits &= bits - 1u;
          const float value = table.find((int)(g.head + (v + step) * EPV + at));
#pragma unroll
          for (int j = 0; j < EPV; ++j) x[j] = j == at ? value : x[j];
        }
      }
    };

    // ---- gradient of this row out, next row in, chunk by chunk through the same registers
    RawList raw;
    if (next_i < a.n_rows && wave == 0) raw = fetch_list(a.list, next_i);
    if (a.row_mask != nullptr) next_active(row_i + gridDim.x, true);
    const bool has_next = next_i < a.n_rows;
    const char* nrow = a.logits + (has_next ? next_i : row_i) * a.row_stride_bytes;
    const RowGeom gn = has_next ? row_geom<DT>(nrow, a.vocab, false) : RowGeom{0, 0, 0};
    const char* nbody = nrow + gn.head * E::kSize;
    char* obody = out_row + g.head * E::kSize;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      if (within(c, g.nvec)) {
        float x[EPV];
        E::unpack(pinned(c >= CHUNKS - kParked ? park[c - (CHUNKS - kParked)][tid] : buf[c]), x);
        grad_vec(x, tid, (uint32_t)c * kOneBlock, c);
        store_vec(obody + (uint32_t)c * (kOneBlock * 16u) + tid16, E::pack(x));
      }
      buf[c] = within(c, gn.nvec) ? load_vec(nbody + (uint32_t)c * (kOneBlock * 16u) + tid16) : minus_inf_vec<DT>();
    }
    if (LONG) {
#pragma unroll 2
      for (uint32_t v = kResident + tid; v < g.nvec; v += kOneBlock) {
        float x[EPV];
        E::unpack(*(const u32x4*)(tail_body + v * 16u), x);
        grad_vec(x, v, 0u, 63);
        store_vec(obody + v * 16u, E::pack(x));
      }
    }
    if (tid < nscalar) {
      const uint32_t e = tid < g.head ? tid : g.nvec * EPV + tid;
      E::store1(out_row + e * E::kSize, map.scalar(tid) ? table.find((int)e) : grad_of(xs));
    }
    xs = -INFINITY;
    if (tid < gn.head + gn.tail) xs = E::load1(nrow + (tid < gn.head ? tid : gn.nvec * EPV + tid) * E::kSize);
    if (has_next && wave == 0) mark(raw, next_i, gn, side ^ 1);
    lds_barrier();
    row_i = next_i;
    g = gn;
    side ^= 1;
  }
}

static int64_t one_pass_max_vocab(int dtype) {
  if (dtype != ORLHF_F32 && dtype != ORLHF_BF16 && dtype != ORLHF_F16) return 0;
  const int64_t most = (int64_t)kMaxFactor * kChunksLong * kOneBlock * (dtype == ORLHF_F32 ? 4 : 8);
  return most < kMaxMapped ? most : kMaxMapped;
}

template <int DT, int CHUNKS, bool LONG>
static int launch_one_pass(const OneArgs& a, unsigned blocks, hipStream_t stream) {
  const size_t lds = (size_t)a.map_words * 4 * 2 + (size_t)kParked * kOneBlock * 16;
  // more than the 64 KiB that a launch may ask for by itself
  const hipError_t e = hipFuncSetAttribute((const void*)distill_one_pass_kernel<DT, CHUNKS, LONG>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
  if (e != hipSuccess) return fail(ORLHF_ERR_LAUNCH, "distill_kl_fwd_bwd: %zu bytes of LDS: %s", lds, hipGetErrorString(e));
  hipLaunchKernelGGL((distill_one_pass_kernel<DT, CHUNKS, LONG>), dim3(blocks), dim3(kOneBlock), lds, stream, a);
  ORLHF_CHECK_LAUNCH("orlhf_distill_kl_fwd_bwd");
  return ORLHF_OK;
}

template <int DT>
static int launch_one_pass_for(const OneArgs& a, unsigned blocks, hipStream_t stream) {
  if (a.vocab > (int64_t)kChunks * kOneBlock * Elt<DT>::kPerVec) return launch_one_pass<DT, kChunksLong, true>(a, blocks, stream);
  return launch_one_pass<DT, kChunks, false>(a, blocks, stream);
}

}  // namespace orlhf

using namespace orlhf;

extern "C" int64_t orlhf_distill_kl_fwd_bwd_max_vocab(int dtype) { return one_pass_max_vocab(dtype); }

extern "C" int orlhf_distill_kl_fwd_bwd(const void* logits, void* grad_logits, int dtype, int64_t n_rows, int64_t vocab,
                                        int64_t row_stride, int64_t grad_row_stride, const int64_t* teacher_ids,
                                        const float* teacher_logprob, int64_t k, double temperature,
                                        double teacher_temperature, int kind, const float* weight, float* loss,
                                        const uint8_t* row_mask, orlhf_stream_t stream) {
  int bad = check_distill("distill_kl_fwd_bwd", dtype, n_rows, vocab, row_stride, k, temperature);
  if (bad == ORLHF_OK) bad = check_kind("distill_kl_fwd_bwd", kind, teacher_temperature);
  if (bad != ORLHF_OK) return bad;
  ORLHF_CHECK_ARG(grad_row_stride >= vocab, "distill_kl_fwd_bwd: grad_row_stride %lld < vocab %lld",
                  (long long)grad_row_stride, (long long)vocab);
  if (n_rows == 0) return ORLHF_OK;  // nothing to launch; empty arrays may well be NULL
  ORLHF_CHECK_ARG(logits != nullptr && grad_logits != nullptr && teacher_ids != nullptr && teacher_logprob != nullptr &&
                      weight != nullptr && loss != nullptr,
                  "distill_kl_fwd_bwd: NULL logits / grad_logits / teacher_ids / teacher_logprob / weight / loss");
  const int64_t esize = dtype == ORLHF_F32 ? 4 : 2;
  ORLHF_CHECK_ARG((((uintptr_t)logits | (uintptr_t)grad_logits) & (uintptr_t)(esize - 1)) == 0,
                  "distill_kl_fwd_bwd: pointers not aligned to the element size");
  if (vocab > one_pass_max_vocab(dtype))
    return fail(ORLHF_ERR_UNSUPPORTED,
                "distill_kl_fwd_bwd: a row of %lld elements is too long for the one-pass kernel (max %lld); use the "
                "separate forward and backward",
                (long long)vocab, (long long)one_pass_max_vocab(dtype));
  if ((((uintptr_t)logits ^ (uintptr_t)grad_logits) & 15u) != 0 || (((row_stride - grad_row_stride) * esize) & 15) != 0)
    return fail(ORLHF_ERR_UNSUPPORTED,
                "distill_kl_fwd_bwd: logits and grad rows sit on different 16-byte phases; use the separate forward and "
                "backward");
  int device = 0, n_cu = 256;
  if (hipGetDevice(&device) == hipSuccess) {
    int v = 0;
    if (hipDeviceGetAttribute(&v, hipDeviceAttributeMultiprocessorCount, device) == hipSuccess && v > 0) n_cu = v;
  }
  OneArgs a = {(const char*)logits, (char*)grad_logits, n_rows, vocab, row_stride * esize, grad_row_stride * esize,
               {teacher_ids, teacher_logprob, (int)k, 1.0 / teacher_temperature, kind == ORLHF_DISTILL_FORWARD},
               temperature, kind, weight, loss, row_mask, (uint32_t)(ListMap<ORLHF_BF16>::bytes(vocab) / 4)};
  const unsigned blocks = (unsigned)(n_rows < n_cu ? n_rows : n_cu);  // a workgroup takes a CU's register file
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case ORLHF_F32: return launch_one_pass_for<ORLHF_F32>(a, blocks, s);
    case ORLHF_BF16: return launch_one_pass_for<ORLHF_BF16>(a, blocks, s);
    default: return launch_one_pass_for<ORLHF_F16>(a, blocks, s);
  }
}
