// step_ops.hip -- the operators around a step that brings several tokens per
// sequence: its page tables and slot maps, and the verification of drafted
// tokens.
#include <hip/hip_runtime.h>

#include "../../include/rstr_hip.h"
#include "device_math.h"
#include "kv4.h"

namespace rstr {

namespace {

// ---- step maps ------------------------------------------------------------------------
// Prefix sums over the sequences (pages wanted, then rows granted) and an
// element-wise fill of rows and new table entries.  Every workgroup computes the
// prefix sums of all sequences in its own LDS (8 bytes a sequence), so one launch
// does it without a wait between workgroups; workgroup 0 writes what is per
// sequence, and all share the fill.  Bound by its chain of waits (what is asked, the two scans, table
// entries): 5 us for 5 sequences, 13 for 1000 with about 64 thousand rows.
constexpr int kMapsThreads = 512;

// Inclusive sum over the workgroup's threads; `tmp` holds one value a wave.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* tmp, int64_t* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  v = wave_scan_i64(v);
  if (lane == 63) tmp[wave] = v;
  __syncthreads();
  int64_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kMapsThreads / 64; w++) {
    if (w < wave) before += tmp[w];
    all += tmp[w];
  }
  __syncthreads();
  *total = all;
  return v + before;
}

// The largest i in [0, n) with a[i] <= x (a[0] <= x, a does not decrease).
__device__ __forceinline__ int last_not_above(const int32_t* a, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kMapsThreads) k_step_maps(StepMaps a) {
  extern __shared__ int32_t lds[];
  int32_t *row0 = lds, *page0 = lds + a.batch;  // first row and first new page of each sequence
  __shared__ int64_t tmp[kMapsThreads / 64];
  __shared__ int64_t smax[2];
  const int tid = threadIdx.x, per = (a.batch + kMapsThreads - 1) / kMapsThreads;
  const int b0 = min(tid * per, a.batch), b1 = min(b0 + per, a.batch);
  const int64_t cap = min((int64_t)a.pps * a.page_size, (int64_t)0x7FFFFFFF);
  const auto pages_of = [&](uint32_t n) {
    const uint32_t p = n / (uint32_t)a.page_size;
    return (int)(p + (n != p * (uint32_t)a.page_size ? 1 : 0));
  };
  // what each sequence asks for: pages and rows
  int64_t sum = 0, total;
  for (int b = b0; b < b1; b++) {
    const int n = a.lengths[b], c = a.counts[b];
    const int m = n < 0 || c < 0 || (int64_t)n + c > cap ? 0 : c;
    const int need = m == 0 ? 0 : pages_of((uint32_t)n + (uint32_t)m) - pages_of((uint32_t)n);
    page0[b] = need;
    row0[b] = m;
    sum += need;
  }
  // pages: a sequence is served while the list of free pages lasts
  int64_t at = block_scan(sum, tmp, &total) - sum;
  int64_t rows = 0;
  for (int b = b0; b < b1; b++) {
    const int need = page0[b];
    page0[b] = (int)min(at, (int64_t)a.n_free);
    at += need;
    if (need != 0 && at > a.n_free) row0[b] = 0;
    rows += row0[b];
  }
  // rows: and while the row arrays do.  A sequence with rows has its pages up to where the
  // next sequence's begin.
  if (tid < 2) smax[tid] = 0;
  int64_t r = block_scan(rows, tmp, &total) - rows;
  int64_t granted_rows = 0, granted_pages = 0;
  for (int b = b0; b < b1; b++) {
    const int m = row0[b], end = b + 1 < b1 ? page0[b + 1] : (int)min(at, (int64_t)a.n_free);
    row0[b] = (int)min(r, (int64_t)a.rows);
    if (m > 0 && r + m <= a.rows) {
      granted_rows = r + m;
      if (end > page0[b]) granted_pages = end;
    }
    r += m;
  }
  if (granted_rows) atomicMax((unsigned long long*)&smax[0], (unsigned long long)granted_rows);
  if (granted_pages) atomicMax((unsigned long long*)&smax[1], (unsigned long long)granted_pages);
  __syncthreads();
  const int n_rows = (int)smax[0], n_pages = (int)smax[1];
  // a refused sequence has no rows: its first row is where the next granted one begins
  for (int b = b0; b < b1; b++) row0[b] = min(row0[b], n_rows);
  __syncthreads();
  if (blockIdx.x == 0) {
    for (int b = b0; b < b1; b++) {
      const int first = row0[b], next = b + 1 < a.batch ? row0[b + 1] : n_rows;
      a.row_offsets[b] = first;
      a.new_lengths[b] = a.lengths[b] + (next - first);
    }
    if (tid == 0) {
      a.row_offsets[a.batch] = n_rows;
      *a.taken = n_pages;
    }
  }
  const int64_t step = (int64_t)gridDim.x * kMapsThreads;
  for (int64_t i = (int64_t)blockIdx.x * kMapsThreads + tid; i < a.rows; i += step) {
    int pos = 0, slot = -1;
    if (i < n_rows) {
      const int b = last_not_above(row0, a.batch, (int)i);
      const int have = a.lengths[b], t = have + ((int)i - row0[b]);
      const int old = pages_of((uint32_t)have), pg = (int)((uint32_t)t / (uint32_t)a.page_size);
      const int page = pg < old ? a.page_table[(int64_t)b * a.pps + pg] : a.free_pages[page0[b] + (pg - old)];
      pos = t + (a.starts ? a.starts[b] : 0);
      const int64_t at = (int64_t)page * a.page_size + (t - pg * a.page_size);
      slot = at < 0 || at > 0x7FFFFFFF ? -1 : (int)at;
    }
    a.positions[i] = pos;
    a.slots[i] = slot;
  }
  for (int64_t e = (int64_t)blockIdx.x * kMapsThreads + tid; e < n_pages; e += step) {
    const int b = last_not_above(page0, a.batch, (int)e);
    const int old = pages_of((uint32_t)a.lengths[b]);
    a.page_table[(int64_t)b * a.pps + old + ((int)e - page0[b])] = a.free_pages[e];
  }
}

// ---- draft verification -----------------------------------------------------------------
// Target probabilities p = softmax(x / T) of every row, in 64 bits: a drawn number
// is compared with sums over the vocabulary, and 1e-7 of such a sum covers as many
// borders between tokens as the vocabulary has.  The exponentials are good to 1e-12, and
// so are the sums: one draw in ten million meets a border that two forms see differently.
//   1. k_verify_rows: per (row, chunk of the vocabulary) the maximum, its first
//      index and the sum of exp((x - max) / T).
//   2. k_verify_pick: per (sequence, chunk): every row's sums joined, the first
//      draft that is refused, and the chunk's sum of what a token is then drawn
//      from: max(p - q, 0), or p after the last draft.
//   3. k_verify_token: per sequence: the chunk where the running sum passes u, and
//      the token inside it.
// Three launches, as each needs sums over all that the one before it wrote.  64 sequences of up to six
// fp32 rows over 128256 tokens, with drafts' probabilities: 27 us, 4.3 TB/s, bound by memory; 19 for
// the picked rows and their drafts' probabilities (66 MB); 10, which three sequences take too: a wait for the
// chunks' sums, one for the chunk's elements, and their exponentials.
constexpr int kChunk = 4096, kVT = 256, kPer = kChunk / kVT;

// 2^t for t <= 0, to 3e-13 of itself: t = n + f with |f| <= 1/2, and the series of 2^f
// (coefficients ln(2)^k / k!) to the tenth power, whose rest is below 2^-41.
__device__ __forceinline__ double pow2(double t) {
  t = fmax(t, -1100.0);  // 0, and -infinity - -infinity is none
  const double n = __builtin_rint(t), f = t - n;
  double p = 7.0549116208011233e-09;
  p = __builtin_fma(p, f, 1.0178086009239699e-07);
  p = __builtin_fma(p, f, 1.3215486790144309e-06);
  p = __builtin_fma(p, f, 1.5252733804059840e-05);
  p = __builtin_fma(p, f, 1.5403530393381610e-04);
  p = __builtin_fma(p, f, 1.3333558146428443e-03);
  p = __builtin_fma(p, f, 9.6181291076284772e-03);
  p = __builtin_fma(p, f, 5.5504108664821580e-02);
  p = __builtin_fma(p, f, 2.4022650695910072e-01);
  p = __builtin_fma(p, f, 6.9314718055994531e-01);
  p = __builtin_fma(p, f, 1.0);
  return __builtin_amdgcn_ldexp(p, (int)n);
}
constexpr double kLog2e = 1.4426950408889634;

struct RowStat {
  double sum;   // of exp((x - top) / T) over the chunk; 0 where T <= 0
  float top;    // NaN if the chunk holds one
  int32_t at;   // first index of top (of the first NaN)
};
struct SeqPick {
  double top, z, scale;  // p(v) = 2^((x_v - top) * scale) / z
  int32_t row;           // the row the token is drawn from; -1: the sequence has none
  int32_t draft;         // >= 0: that token's probability is left out (a draft without probabilities)
  int32_t greedy;        // >= 0: the token itself
  int32_t from_probs;    // 1: max(p - q, 0) of the draft's probabilities
};

struct LF32 { typedef float T; static __device__ __forceinline__ float get(T x) { return x; } };
struct LF16 { typedef _Float16 T; static __device__ __forceinline__ float get(T x) { return (float)x; } };
struct LBF16 { typedef uint16_t T; static __device__ __forceinline__ float get(T x) { return __uint_as_float((uint32_t)x << 16); } };

// The last sequence that begins at or before a row: all offsets at once, one a lane, where
// they are few (one wait for memory instead of one for every halving).
__device__ __forceinline__ int seq_of(const Verify& a, int row) {
  if (a.batch <= 512) {
    int n = 0;
    for (int b = 0; b < a.batch; b += 64) {
      const int i = b + (threadIdx.x & 63);
      n += __popcll(__ballot(i < a.batch && a.row_offsets[i] <= row));
    }
    return max(n - 1, 0);
  }
  int lo = 0, hi = a.batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.row_offsets[mid] <= row) lo = mid; else hi = mid;
  }
  return lo;
}

// A temperature that draws; anything else (0, below, not finite) is greedy.
__device__ __forceinline__ bool draws(float T) { return T > 0.0f && T < INFINITY; }

// Sum over the wave's lanes, without the LDS crossbar (see wave_tree_sum).
template <int CTRL>
__device__ __forceinline__ double dpp64(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u, CTRL, 0xF, 0xF, true);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(u >> 32), CTRL, 0xF, 0xF, true);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
template <int M>
__device__ __forceinline__ double swap_add64(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  float l0, l1, h0, h1;
  lane_pair<M>(__uint_as_float((uint32_t)u), l0, l1);
  lane_pair<M>(__uint_as_float((uint32_t)(u >> 32)), h0, h1);
  return __builtin_bit_cast(double, (uint64_t)__float_as_uint(h0) << 32 | __float_as_uint(l0)) +
         __builtin_bit_cast(double, (uint64_t)__float_as_uint(h1) << 32 | __float_as_uint(l1));
}
__device__ __forceinline__ double wave_sum64(double v) {
  v += dpp64<0xB1>(v);
  v += dpp64<0x4E>(v);
  v += dpp64<0x141>(v);
  v += dpp64<0x128>(v);
  return swap_add64<32>(swap_add64<16>(v));
}

// The elements that a thread takes of a chunk: 16 bytes at a time, neighbours for
// neighbouring threads.  token_of(v0, i): the token of a thread's i-th element.
template <class E>
__device__ __forceinline__ int token_of(int v0, int i) {
  constexpr int PER = 16 / sizeof(typename E::T);
  return v0 + ((i / PER) * kVT + (int)threadIdx.x) * PER + i % PER;
}
template <class E>
__device__ __forceinline__ void load_chunk(const typename E::T* x, int v0, int v1, float (&val)[kPer]) {
  typedef typename E::T T;
  constexpr int PER = 16 / sizeof(T);
  if (v1 - v0 == kChunk && ((uintptr_t)(x + v0) % 16) == 0) {
    T t[kPer];
#pragma unroll
    for (int i = 0; i < kPer / PER; i++) ((u32x4*)t)[i] = *(const u32x4*)(x + v0 + (i * kVT + (int)threadIdx.x) * PER);
#pragma unroll
    for (int i = 0; i < kPer; i++) val[i] = E::get(t[i]);
  } else {
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      const int v = token_of<E>(v0, i);
      val[i] = v < v1 ? E::get(x[v]) : -INFINITY;
    }
  }
}

// kPer neighbours from v0 on.
template <class E>
__device__ __forceinline__ void load_run(const typename E::T* x, int v0, int v1, float (&val)[kPer]) {
  typedef typename E::T T;
  constexpr int PER = 16 / sizeof(T);
  if (v1 - v0 >= kPer && ((uintptr_t)(x + v0) % 16) == 0) {
    T t[kPer];
#pragma unroll
    for (int i = 0; i < kPer / PER; i++) ((u32x4*)t)[i] = ((const u32x4*)(x + v0))[i];
#pragma unroll
    for (int i = 0; i < kPer; i++) val[i] = E::get(t[i]);
  } else {
#pragma unroll
    for (int i = 0; i < kPer; i++) val[i] = v0 + i < v1 ? E::get(x[v0 + i]) : 0.0f;
  }
}

template <class E>
__global__ void __launch_bounds__(kVT) k_verify_rows(Verify a, RowStat* __restrict__ stats) {
  const int row = blockIdx.x, chunk = blockIdx.y, tid = threadIdx.x, chunks = gridDim.y;
  const int b = seq_of(a, row);
  if (row < a.row_offsets[b] || row >= a.row_offsets[b + 1]) return;  // behind the last sequence
  const float T = a.temperature[b];
  const typename E::T* x = (const typename E::T*)a.logits + (int64_t)row * a.logits_row;
  const int v0 = chunk * kChunk, v1 = min(v0 + kChunk, a.vocab);
  float val[kPer];
  float top = -INFINITY;
  int at = 0x7FFFFFFF;
  load_chunk<E>(x, v0, v1, val);
  __shared__ float st[kVT / 64];
  __shared__ int si[kVT / 64];
  __shared__ double ss[kVT / 64];
  const int wave = tid >> 6;
#pragma unroll
  for (int i = 0; i < kPer; i++) top = __builtin_elementwise_maximum(top, val[i]);  // NaN if there is one
  bool nan = top != top;
  top = wave_max(top);  // of the other lanes
  nan = __ballot(nan) != 0;
  if ((tid & 63) == 0) st[wave] = nan ? __builtin_nanf("") : top;
  __syncthreads();
  top = st[0];
#pragma unroll
  for (int w = 1; w < kVT / 64; w++) top = __builtin_elementwise_maximum(top, st[w]);
  if (!draws(T) || !(top > -INFINITY && top < INFINITY)) {  // greedy: where the maximum is first
#pragma unroll
    for (int i = kPer - 1; i >= 0; i--) {
      const int v = token_of<E>(v0, i);
      if (v < v1 && (val[i] == top || (val[i] != val[i] && top != top))) at = min(at, v);
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) at = min(at, __shfl_xor(at, d, 64));
    if ((tid & 63) == 0) si[wave] = at;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kVT / 64; w++) at = min(at, si[w]);
  }
  double sum = 0.0;
  if (draws(T) && top > -INFINITY && top < INFINITY) {
    const double k = kLog2e / (double)T, t = (double)top;
#pragma unroll
    for (int i = 0; i < kPer; i++) sum += pow2(((double)val[i] - t) * k);
  }
  sum = wave_sum64(sum);
  if ((tid & 63) == 0) ss[wave] = sum;
  __syncthreads();
  if (tid == 0) stats[(int64_t)row * chunks + chunk] = RowStat{ss[0] + ss[1] + ss[2] + ss[3], top, at};
}

// A row's chunks joined by one wave: maximum and normaliser, and where the row is greedy
// the maximum's first index.
__device__ __forceinline__ void join_row(const RowStat* s, int chunks, double k, float& top, int& at, double& z, bool& cold) {
  const int lane = threadIdx.x & 63;
  top = -INFINITY;
  for (int c = lane; c < chunks; c += 64) top = __builtin_elementwise_maximum(top, s[c].top);
  const bool nan = __ballot(top != top) != 0;
  top = nan ? __builtin_nanf("") : wave_max(top);
  cold = k == 0.0 || !(top > -INFINITY && top < INFINITY);
  at = 0x7FFFFFFF;
  z = 0.0;
  if (cold) {
    for (int c = lane; c < chunks; c += 64)
      if (s[c].top == top || (nan && s[c].top != s[c].top)) at = min(at, s[c].at);
#pragma unroll
    for (int d = 32; d; d >>= 1) at = min(at, __shfl_xor(at, d, 64));
    return;
  }
  for (int c = lane; c < chunks; c += 64)
    if (s[c].sum > 0.0) z += s[c].sum * pow2(((double)s[c].top - (double)top) * k);
  z = wave_sum64(z);
}

// What a token of logit x and draft probability q weighs in the picked row, times z.
__device__ __forceinline__ double weight(const SeqPick& s, float x, float q, int v) {
  const double e = pow2(((double)x - s.top) * s.scale);
  if (s.from_probs) {
    const double w = e - (double)q * s.z;
    return w > 0.0 ? w : 0.0;
  }
  return v == s.draft ? 0.0 : e;
}

template <class E>
__global__ void __launch_bounds__(kVT) k_verify_pick(Verify a, const RowStat* __restrict__ stats, SeqPick* __restrict__ picks,
                                                     double* __restrict__ sums) {
  const int b = blockIdx.x, chunk = blockIdx.y, chunks = gridDim.y, tid = threadIdx.x, wave = tid >> 6;
  const int r0 = max(a.row_offsets[b], 0), r1 = min(a.row_offsets[b + 1], a.rows);
  if (r1 <= r0) {
    if (chunk == 0 && tid == 0) {
      a.accepted[b] = 0;
      picks[b].row = -1;
    }
    return;
  }
  const float T = a.temperature[b];
  const double k = draws(T) ? kLog2e / (double)T : 0.0;
  __shared__ SeqPick pick;
  __shared__ int refused[kVT / 64], kept;
  __shared__ double ss[kVT / 64];
  // the first row, four at a time, whose draft is refused; the last row ends the search
  for (int base = r0;; base += kVT / 64) {
    const int row = base + wave;
    bool stop = false;
    SeqPick mine = {};
    if (row < r1) {
      // what the draft's test reads, asked for before the row's chunks are joined
      const bool last = row == r1 - 1;
      const int d = last ? -1 : a.drafts[row];
      const bool inside = d >= 0 && d < a.vocab;
      float u = 0.0f, q = 1.0f, x = 0.0f;
      if (inside) {
        u = a.u_accept[row];
        x = E::get(((const typename E::T*)a.logits)[(int64_t)row * a.logits_row + d]);
        if (a.probs) q = a.probs[(int64_t)row * a.probs_row + d];
      }
      float top;
      int at;
      double z;
      bool cold;
      join_row(stats + (int64_t)row * chunks, chunks, k, top, at, z, cold);
      mine = SeqPick{(double)top, z, k, row, -1, cold ? at : -1, 0};
      stop = true;
      if (!last) {
        bool ok = false;
        if (cold) ok = d == at;
        else if (inside) ok = (double)u * (double)q < pow2(((double)x - (double)top) * k) / z;
        stop = !ok;
        mine.draft = a.probs ? -1 : d;
        mine.from_probs = a.probs ? 1 : 0;
      }
    }
    if ((tid & 63) == 0) refused[wave] = stop;
    __syncthreads();
    int first = -1;
#pragma unroll
    for (int w = kVT / 64 - 1; w >= 0; w--)
      if (refused[w]) first = w;
    if (first == wave && (tid & 63) == 0) pick = mine;
    if (first >= 0) {
      if (tid == 0) kept = base + first;
      __syncthreads();
      break;
    }
    __syncthreads();
  }
  if (chunk == 0) {
    if (tid == 0) {
      picks[b] = pick;
      a.accepted[b] = kept - r0;
    }
    for (int r = r0 + tid; r < r1; r += kVT)
      if (r != kept) a.tokens[r] = r < kept ? a.drafts[r] : -1;
  }
  if (pick.greedy >= 0) return;
  double sum = 0.0;
  const int v0 = chunk * kChunk, v1 = min(v0 + kChunk, a.vocab);
  const SeqPick s = pick;
  float val[kPer], q[kPer];
  load_chunk<E>((const typename E::T*)a.logits + (int64_t)s.row * a.logits_row, v0, v1, val);
  if (s.from_probs) {
    const float* p = a.probs + (int64_t)s.row * a.probs_row;
    if constexpr (sizeof(typename E::T) == 4) {
      load_chunk<LF32>(p, v0, v1, q);
    } else {
#pragma unroll
      for (int i = 0; i < kPer; i++) q[i] = token_of<E>(v0, i) < v1 ? p[token_of<E>(v0, i)] : 0.0f;
    }
  }
#pragma unroll
  for (int i = 0; i < kPer; i++) {
    const int v = token_of<E>(v0, i);
    if (v < v1) sum += weight(s, val[i], s.from_probs ? q[i] : 0.0f, v);
  }
  sum = wave_sum64(sum);
  if ((tid & 63) == 0) ss[wave] = sum;
  __syncthreads();
  if (tid == 0) sums[(int64_t)b * chunks + chunk] = ss[0] + ss[1] + ss[2] + ss[3];
}

template <class E>
__global__ void __launch_bounds__(kVT) k_verify_token(Verify a, const RowStat* __restrict__ stats, const SeqPick* __restrict__ picks,
                                                      const double* __restrict__ sums, int chunks) {
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  // the first 64 chunks' sums (most vocabularies have no more), asked for beside the pick
  const double* c = sums + (int64_t)b * chunks;
  const double c0 = lane < chunks ? c[lane] : 0.0;
  SeqPick s = picks[b];
  if (s.row < 0) return;
  if (s.greedy >= 0) {
    if (tid == 0) a.tokens[s.row] = s.greedy;
    return;
  }
  __shared__ double wsum[kVT / 64], target, before;
  __shared__ int chosen, last, found;
  bool plain = false;  // nothing is left of p - q: the token comes from p
  if (wave == 0) {
    const double u = (double)a.u_sample[b];
    double total = c0;
    for (int i = lane + 64; i < chunks; i += 64) total += c[i];
    total = wave_sum64(total);
    plain = !(total > 0.0);
    const RowStat* st = stats + (int64_t)s.row * chunks;
    const auto mass = [&](int i) {
      if (!plain) return i < 64 ? c0 : c[i];
      return st[i].sum > 0.0 ? st[i].sum * pow2(((double)st[i].top - s.top) * s.scale) : 0.0;
    };
    if (plain) total = s.z;
    const double t = u * total;
    double run = 0.0, b4 = 0.0;
    int pickc = -1, lastc = 0;
    double lastb = 0.0;
    for (int i0 = 0; i0 < chunks && pickc < 0; i0 += 64) {
      const double w = i0 + lane < chunks ? mass(i0 + lane) : 0.0;
      const double in = wave_scan_f64(w);
      const uint64_t over = __ballot(w > 0.0 && run + in > t), some = __ballot(w > 0.0);
      if (over) {
        const int f = __ffsll((unsigned long long)over) - 1;
        pickc = i0 + f;
        b4 = run + __shfl(in - w, f, 64);
      } else if (some) {
        const int f = 63 - __clzll((long long)some);
        lastc = i0 + f;
        lastb = run + __shfl(in - w, f, 64);
      }
      run += __shfl(in, 63, 64);
    }
    if (lane == 0) {
      chosen = (pickc >= 0 ? pickc : lastc) | (plain ? 1 << 30 : 0);
      before = pickc >= 0 ? b4 : lastb;
      target = t;
      found = 0x7FFFFFFF;
      last = -1;
    }
  }
  __syncthreads();
  const int chunk = chosen & ~(1 << 30);
  if (chosen >> 30) { s.from_probs = 0; s.draft = -1; }
  const int v0 = chunk * kChunk + tid * kPer, v1 = min(chunk * kChunk + kChunk, a.vocab);
  double w[kPer], sum = 0.0;
  float x[kPer], q[kPer];
  load_run<E>((const typename E::T*)a.logits + (int64_t)s.row * a.logits_row, v0, v1, x);
  if (s.from_probs) load_run<LF32>(a.probs + (int64_t)s.row * a.probs_row, v0, v1, q);
#pragma unroll
  for (int i = 0; i < kPer; i++) {
    w[i] = v0 + i < v1 ? weight(s, x[i], s.from_probs ? q[i] : 0.0f, v0 + i) : 0.0;
    sum += w[i];
  }
  const double in = wave_scan_f64(sum);
  if (lane == 63) wsum[wave] = in;
  __syncthreads();
  double run = before + (in - sum);
  for (int i = 0; i < wave; i++) run += wsum[i];
  int hit = 0x7FFFFFFF, end = -1;
#pragma unroll
  for (int i = 0; i < kPer; i++) {
    run += w[i];
    if (w[i] > 0.0) {
      end = v0 + i;
      if (run > target && hit == 0x7FFFFFFF) hit = v0 + i;
    }
  }
  if (hit != 0x7FFFFFFF) atomicMin(&found, hit);
  if (end >= 0) atomicMax(&last, end);
  __syncthreads();
  if (tid == 0) a.tokens[s.row] = found != 0x7FFFFFFF ? found : last;  // rounding may leave the target just behind the last one
}

inline int verify_chunks(int vocab) { return (vocab + kChunk - 1) / kChunk; }
inline size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

template <class E>
hipError_t verify_type(hipStream_t st, const Verify& a) {
  const int chunks = verify_chunks(a.vocab);
  char* w = (char*)a.ws;
  RowStat* stats = (RowStat*)w;
  w += align256(sizeof(RowStat) * (size_t)a.rows * chunks);
  SeqPick* picks = (SeqPick*)w;
  w += align256(sizeof(SeqPick) * (size_t)a.batch);
  double* sums = (double*)w;
  if (a.rows > 0) {
    hipLaunchKernelGGL(k_verify_rows<E>, dim3((unsigned)a.rows, (unsigned)chunks), dim3(kVT), 0, st, a, stats);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(k_verify_pick<E>, dim3((unsigned)a.batch, (unsigned)chunks), dim3(kVT), 0, st, a, stats, picks, sums);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(k_verify_token<E>, dim3((unsigned)a.batch), dim3(kVT), 0, st, a, stats, picks, sums, chunks);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_step_maps(hipStream_t st, const StepMaps& m) {
  // rows and new pages are shared out over as many workgroups as they fill
  const int64_t work = (int64_t)m.rows > m.n_free ? m.rows : m.n_free;
  const int64_t groups = (work + kMapsThreads - 1) / kMapsThreads;
  const unsigned grid = (unsigned)(groups < 1 ? 1 : groups > 256 ? 256 : groups);
  hipLaunchKernelGGL(k_step_maps, dim3(grid), dim3(kMapsThreads), (size_t)8 * m.batch, st, m);
  return hipGetLastError();
}

size_t verify_workspace(int batch, int rows, int vocab) {
  const size_t chunks = (size_t)verify_chunks(vocab);
  return align256(sizeof(RowStat) * rows * chunks) + align256(sizeof(SeqPick) * batch) + sizeof(double) * batch * chunks;
}

hipError_t launch_verify(hipStream_t st, int dtype, const Verify& v) {
  if (v.batch == 0) return hipSuccess;
  if (dtype == RSTR_F32) return verify_type<LF32>(st, v);
  if (dtype == RSTR_F16) return verify_type<LF16>(st, v);
  return verify_type<LBF16>(st, v);
}

}  // namespace rstr
