// attn_line.h -- device code that the attention kernels over paged caches share: element types and their
// loads, the line of work as a wave walks it, and the pieces of items that several waves leave.
#pragma once
#include <hip/hip_runtime.h>

#include <atomic>

#include "device_math.h"
#include "kv4.h"
#include "kv4_line.h"

namespace rstr {
namespace {

typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));

// ---- element types ----------------------------------------------------------------
struct F32 {
  typedef float T;
  static __device__ __forceinline__ float get(T x) { return x; }
  static __device__ __forceinline__ T put(float x) { return x; }
};
struct F16 {
  typedef _Float16 T;
  static __device__ __forceinline__ float get(T x) { return (float)x; }
  static __device__ __forceinline__ T put(float x) { return (T)x; }
};
struct BF16 {
  typedef uint16_t T;
  static __device__ __forceinline__ float get(T x) { return __uint_as_float((uint32_t)x << 16); }
  static __device__ __forceinline__ T put(float x) { return __builtin_bit_cast(T, (__bf16)x); }
};

template <class E, bool VEC>
__device__ __forceinline__ void load8(const typename E::T* p, float (&x)[8]) {
  typename E::T t[8];
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(t) / 16; i++) ((u32x4*)t)[i] = ((const u32x4*)p)[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) t[i] = p[i];
  }
#pragma unroll
  for (int i = 0; i < 8; i++) x[i] = E::get(t[i]);
}
template <class E, bool VEC>
__device__ __forceinline__ void store8(typename E::T* p, const float (&x)[8]) {
  typename E::T t[8];
#pragma unroll
  for (int i = 0; i < 8; i++) t[i] = E::put(x[i]);
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(t) / 16; i++) ((u32x4*)p)[i] = ((u32x4*)t)[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) p[i] = t[i];
  }
}

__host__ __device__ inline bool vec_rows(const Rows& r, int size) {
  return ((uintptr_t)r.p % 16) == 0 && (r.row * size) % 16 == 0 && (r.head * size) % 16 == 0;
}

// ---- the line of work ---------------------------------------------------------------
// The value of one lane, the same for all.
__device__ __forceinline__ int64_t lane64(int64_t v, int lane) {
  return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)v, lane));
}
__device__ __forceinline__ int wave_sum_i32(int v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d, 64);
  return v;
}
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Pieces of items that several waves share: two a wave (the end of an item
// that an earlier wave began, the beginning of one that later waves end).  The wave
// that begins an item leaves what the merge needs to know of it.
struct Begun {
  int b, h, ct, w, pieces;  // w: the wave; pieces: 0 where it ended the item too
};
struct Pieces {
  int* n_items;
  Begun* begun;  // [items]
  float2* ml;   // [2 * workers][cols] (mref, l)
  float* acc;   // [2 * workers][cols][D]
};

// a / b of numbers of units without the loop that 64-bit division is.  (The reciprocal instruction
// gives an estimate, good to about 2^-23.)
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) { return quotient_from(a, b, __builtin_amdgcn_rcp((double)b)); }

// The parts of items that a wave (or a workgroup) works on, in their order.  A wave holds the sequences
// 64 at a time, one a lane.
struct Line {
  const Lines& L;
  int batch, w;
  int64_t part, u, u_end;
  // the part that next() came to: its item, and n of the item's units from `at` on
  Seq s;
  int b, h, ct, at, n, item, pieces;  // pieces of the item, 0 where there is one
  bool begins, ends;

  __device__ __forceinline__ Line(const Lines& lines, int n_seqs, int worker, int workers, int least) : L(lines), batch(n_seqs), w(worker) {
    seqs = chunk_of(0);
    int64_t in = wave_scan_i64(seqs.units), total = lane64(in, 63);
    ordered = seqs.ordered;
    if (batch > 64) {
      int64_t mine = 0;
      for (int i = 64; i < batch; i += 64) {
        const Seq x = chunk_of(i);
        mine += x.units;
        ordered = ordered && x.ordered;
      }
      total += lane64(wave_scan_i64(mine), 63);
    }
    ordered = __ballot(!ordered) == 0;
    if (!ordered) total = 0;
    part = quotient(total + workers - 1, workers);
    part = part > least ? part : least;
    u = (int64_t)w * part;
    u_end = min(u + part, total);
    if (u >= u_end) return;
    for (int64_t run = 0;;) {
      const uint64_t over = __ballot(run + in > u);
      const int f = over ? __ffsll((unsigned long long)over) - 1 : 64;
      if (!L.whole && (f > 0)) item0 = uniform(item0 + wave_sum_i32((int)(threadIdx.x & 63) < f ? L.n_kv * seqs.nct : 0));
      if (over) {
        at_seq = uniform(f);
        first = run + lane64(in - seqs.units, at_seq);
        return;
      }
      run += lane64(in, 63);
      b0 += 64;
      seqs = chunk_of(b0);
      in = wave_scan_i64(seqs.units);
    }
  }

  // Items of the call.
  __device__ __forceinline__ int items() const {
    if (!ordered) return 0;
    int n = 0;
    for (int i = 0; i < batch; i += 64) n += L.n_kv * chunk_of(i).nct;
    return wave_sum_i32(n);
  }

  __device__ __forceinline__ bool next() {
    while (u < u_end) {
      const auto of = [&](int v) { return __builtin_amdgcn_readlane(v, at_seq); };
      s = Seq{of(seqs.r0), of(seqs.m), of(seqs.len), of(seqs.lo), of(seqs.tiles), of(seqs.nct), true, 0};
      const int per_item = L.per_item(s.tiles);
      const int64_t units = (int64_t)L.n_kv * s.nct * per_item;
      if (u < first + units) {
        b = b0 + at_seq;
        const int64_t rel = u - first, i = quotient(rel, per_item);
        at = (int)(rel - i * per_item);
        h = (int)i / s.nct;
        ct = (int)(i - (int64_t)h * s.nct);
        item = item0 + (int)i;
        n = (int)min((int64_t)(per_item - at), u_end - u);
        begins = at == 0;
        ends = at + n == per_item;
        pieces = ends ? 0 : pieces_to(quotient(u + per_item - 1, part), w);
        u += n;
        return true;
      }
      first += units;  // behind it: the next sequence that has units
      item0 += L.n_kv * s.nct;
      for (int from = at_seq + 1;; from = 0) {
        const uint64_t some = from < 64 ? __ballot(seqs.units > 0) >> from << from : 0;
        if (some) {
          at_seq = uniform(__ffsll((unsigned long long)some) - 1);
          break;
        }
        b0 += 64;
        seqs = chunk_of(b0);
      }
    }
    return false;
  }

 private:
  Seq seqs;
  bool ordered;  // all sequences are
  int b0 = 0, at_seq = 0, item0 = 0;  // the sequence that unit u lies in (of seqs), its first item and unit
  int64_t first = 0;
  __device__ __forceinline__ Seq chunk_of(int from) const {
    const int at = from + (int)(threadIdx.x & 63);
    Seq x = sequence(L, min(at, batch - 1));
    if (at >= batch) x.nct = 0, x.units = 0;
    return x;
  }
};

// Is a lane of the own column among these?
__device__ __forceinline__ bool of_column(uint64_t lanes) {
  lanes |= lanes >> 32;
  return ((lanes | lanes >> 16) >> (threadIdx.x & 15)) & 1;
}

// ---- the rows of a call ------------------------------------------------------------------
// The sequence that a row belongs to, found by all lanes of a wave together: offsets are read 64 at a time.
// Where they decrease anywhere no row belongs to one.
struct RowOf {
  int b, p;   // -1: none; the row's position (negative: it sees nothing)
  int first;  // the sequence's first row
  __device__ __forceinline__ RowOf(const int32_t* ro, const int32_t* lens, int batch, int rows, int row) {
    const int lane = threadIdx.x & 63;
    bool ordered = true;
    int begin = 0, end = 0, len = 0;
    b = -1;
    for (int i0 = 0; i0 < batch; i0 += 64) {  // all that is needed of a sequence in one wait
      const int i = i0 + lane;
      const int at = ro[min(i, batch)], next = ro[min(i + 1, batch)], n = lens[min(i, batch - 1)];
      const uint64_t below = __ballot(i < batch && at <= row);
      ordered = ordered && at <= next;
      if (below) {
        const int f = 63 - __clzll((long long)below);
        b = i0 + f;
        begin = __builtin_amdgcn_readlane(at, f);
        end = __builtin_amdgcn_readlane(next, f);
        len = __builtin_amdgcn_readlane(n, f);
      }
    }
    end = min(end, rows);
    if (__ballot(!ordered) || row >= end) b = -1;
    first = max(begin, 0);
    p = max(len, 0) - (end - row);
  }
};

// ---- host side ----------------------------------------------------------------------
inline int compute_units() {
  static std::atomic<int> known[64];  // calls may come from several threads
  int dev = 0, n = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  if ((n = known[dev].load(std::memory_order_relaxed)) != 0) return n;
  if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) n = 256;
  known[dev].store(n, std::memory_order_relaxed);
  return n;
}

}  // namespace
}  // namespace rstr
