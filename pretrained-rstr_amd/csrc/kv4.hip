// kv4.hip -- the 4-bit paged K/V cache (format: kv4.h): quantising append,
// dequantising read and attention over it.
#include <hip/hip_runtime.h>

#include "../../include/rstr_hip.h"
#include "device_math.h"
#include "kv4.h"

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
  static __device__ __forceinline__ T put(float x) {  // to nearest, ties to even
    uint32_t u = __float_as_uint(x);
    if ((u & 0x7FFFFFFFu) > 0x7F800000u) return (T)((u >> 16) | 0x40u);
    return (T)((u + 0x7FFFu + ((u >> 16) & 1u)) >> 16);
  }
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

// ---- addresses inside a record ----------------------------------------------------
template <int D>
struct Rec {
  static constexpr int NB = D / 32;                 // blocks of a row
  static constexpr int BQ = NB < 4 ? NB : 4;        // K: blocks a lane loads together
  static constexpr int BP = D / 64 < 2 ? D / 64 : 2;  // V: block pairs a lane loads together
  // byte offsets of a K code dword, a V code halfword (its j = 0) and a scale
  static __device__ __forceinline__ int k(int tok, int b, int g) {
    return tok * (D / 2) + (b / BQ) * (16 * BQ) + g * (4 * BQ) + (b % BQ) * 4;
  }
  static __device__ __forceinline__ int v(int tg, int bp, int c) {
    return tg * (2 * D) + (bp / BP) * (128 * BP) + c * (8 * BP) + (bp % BP) * 8;
  }
  static __device__ __forceinline__ int s(int tg, int b) { return (tg * NB + b) * 8; }
  static __device__ __forceinline__ int vbase(int ps) { return ps * (D / 2); }
  static __device__ __forceinline__ int ksbase(int ps) { return ps * D; }
  static __device__ __forceinline__ int vsbase(int ps) { return ps * D + ps * NB * 2; }
};

__device__ __forceinline__ float h2f(uint16_t h) { return (float)__builtin_bit_cast(_Float16, h); }

// ---- append -------------------------------------------------------------------------
// One thread quantises 8 elements; the four threads of a block agree on its
// scale.  Eight threads (64 elements, two blocks) hold the nibbles of eight V
// columns between them and exchange them, so that each writes two halfwords.
//
// x / d is decided exactly: r = x - c * d is exact in fp32 near a half step
// (both are multiples of the smaller operand's last place, and |r| < d), so the
// estimate's nearest integer is corrected where |r| passes d / 2 and a tie goes
// to the even code.
template <int D, class E, bool VEC>
__global__ void __launch_bounds__(256) k_kv4_append(Kv4Layer L, int rows, Rows kr, Rows vr, const int32_t* __restrict__ slots) {
  typedef Rec<D> R;
  constexpr int TPR = D / 8;  // threads a row
  const bool is_v = blockIdx.y != 0;
  const int64_t gid = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int t = (int)(gid % TPR);
  const int64_t rh = gid / TPR;
  const int h = (int)(rh % L.n_kv);
  const int64_t row = rh / L.n_kv;
  const bool live = row < rows;  // lanes behind the last row still take part in the exchanges
  const int slot = live ? slots[row] : -1;
  const Rows src = is_v ? vr : kr;
  float x[8] = {};
  if (live) load8<E, VEC>((const typename E::T*)src.p + row * src.row + h * src.head + t * 8, x);
  // the block's element of greatest magnitude, the first of equals
  float m = 0.0f;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    if (fabsf(x[i]) > fabsf(m)) m = x[i];
    bad |= !(fabsf(x[i]) < INFINITY);
  }
  float o = xor_lane<1>(m);
  m = (fabsf(o) > fabsf(m) || (fabsf(o) == fabsf(m) && (t & 1))) ? o : m;
  o = xor_lane<2>(m);
  m = (fabsf(o) > fabsf(m) || (fabsf(o) == fabsf(m) && (t & 2))) ? o : m;
  const uint64_t any_bad = __ballot(bad);
  bad = (any_bad >> ((threadIdx.x & 63) & ~3)) & 0xF;
  uint16_t db = f2h_bits(__builtin_amdgcn_fmed3f(m * -0.125f, -65504.0f, 65504.0f));
  if ((db & 0x7FFFu) == 0) db = 0;
  if (bad) db = 0x7E00u;
  const float d = h2f(db);
  const float id = d != 0.0f ? 1.0f / d : 0.0f, hd = fabsf(d) * 0.5f;
  int c[8];
#pragma unroll
  for (int i = 0; i < 8; i++) {
    float q = __builtin_rintf(__builtin_amdgcn_fmed3f(x[i] * id, -9.0f, 8.0f));
    const float r = __builtin_fmaf(-q, d, x[i]);
    const float up = (r < 0.0f) == (d < 0.0f) ? 1.0f : -1.0f;
    const bool odd = ((int)q & 1) != 0;
    if (fabsf(r) > hd || (fabsf(r) == hd && odd)) q += up;
    c[i] = d != 0.0f && !bad ? (int)__builtin_amdgcn_fmed3f(q, -8.0f, 7.0f) + 8 : 8;
  }
  const int64_t limit = (int64_t)L.pages * L.page_size;
  const bool put = slot >= 0 && slot < limit;
  const int page = put ? slot / L.page_size : 0, tok = put ? slot % L.page_size : 0;
  uint8_t* rec = L.base + ((int64_t)page * L.n_kv + h) * kv4_record_bytes(D, L.page_size);
  const int b = t >> 2;
  if (!is_v) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) w |= (uint32_t)c[2 * i] << (4 * i) | (uint32_t)c[2 * i + 1] << (16 + 4 * i);
    if (put) *(uint32_t*)(rec + R::k(tok, b, t & 3)) = w;
  } else {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) w |= (uint32_t)c[i] << (4 * i);
    const int par = t & 1, n = (t >> 1) & 3;  // columns 8 * par + i; nibble n of a halfword
    uint32_t h0 = 0, h1 = 0;
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const uint32_t o4 = (uint32_t)__shfl((int)w, ((threadIdx.x & 63) & ~7) + 2 * k + par, 64) >> (8 * n);
      h0 |= (o4 & 0xFu) << (4 * k);
      h1 |= ((o4 >> 4) & 0xFu) << (4 * k);
    }
    if (put) {
      uint8_t* at = rec + R::vbase(L.page_size) + (tok & 3) * 2;
      *(uint16_t*)(at + R::v(tok >> 2, t >> 3, 8 * par + 2 * n)) = (uint16_t)h0;
      *(uint16_t*)(at + R::v(tok >> 2, t >> 3, 8 * par + 2 * n + 1)) = (uint16_t)h1;
    }
  }
  if (put && (t & 3) == 0)
    *(uint16_t*)(rec + (is_v ? R::vsbase(L.page_size) : R::ksbase(L.page_size)) + R::s(tok >> 2, b) + (tok & 3) * 2) = db;
}

// ---- read ---------------------------------------------------------------------------
// One thread gives 8 elements back; d * (c - 8) is exact in fp32 (11 + 4 bits)
// and rounded once to the output's type.
template <int D, class E, bool VEC>
__global__ void __launch_bounds__(256) k_kv4_read(Kv4Layer L, int rows, Rows kr, Rows vr, const int32_t* __restrict__ slots) {
  typedef Rec<D> R;
  constexpr int TPR = D / 8;
  const bool is_v = blockIdx.y != 0;
  const int64_t gid = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int t = (int)(gid % TPR);
  const int64_t rh = gid / TPR;
  const int h = (int)(rh % L.n_kv);
  const int64_t row = rh / L.n_kv;
  if (row >= rows) return;
  const int slot = slots[row];
  float x[8] = {};
  if (slot >= 0 && slot < (int64_t)L.pages * L.page_size) {
    const int page = slot / L.page_size, tok = slot % L.page_size, b = t >> 2;
    const uint8_t* rec = L.base + ((int64_t)page * L.n_kv + h) * kv4_record_bytes(D, L.page_size);
    const int sb = is_v ? R::vsbase(L.page_size) : R::ksbase(L.page_size);
    const float d = h2f(*(const uint16_t*)(rec + sb + R::s(tok >> 2, b) + (tok & 3) * 2));
    if (!is_v) {
      const uint32_t w = *(const uint32_t*)(rec + R::k(tok, b, t & 3));
#pragma unroll
      for (int i = 0; i < 4; i++) {
        x[2 * i] = d * (float)((int)((w >> (4 * i)) & 0xF) - 8);
        x[2 * i + 1] = d * (float)((int)((w >> (16 + 4 * i)) & 0xF) - 8);
      }
    } else {
      const uint8_t* at = rec + R::vbase(L.page_size) + (tok & 3) * 2;
      const int par = t & 1, n = (t >> 1) & 3;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const uint32_t w = *(const uint16_t*)(at + R::v(tok >> 2, t >> 3, 8 * par + i));
        x[i] = d * (float)((int)((w >> (4 * n)) & 0xF) - 8);
      }
    }
  }
  const Rows dst = is_v ? vr : kr;
  store8<E, VEC>((typename E::T*)dst.p + row * dst.row + h * dst.head + t * 8, x);
}

inline bool vec_rows(const Rows& r, int size) {
  return ((uintptr_t)r.p % 16) == 0 && (r.row * size) % 16 == 0 && (r.head * size) % 16 == 0;
}

template <int D, class E>
hipError_t rows_launch(hipStream_t st, bool append, const Kv4Layer& c, int rows, const Rows& k, const Rows& v,
                       const int32_t* slots) {
  const int64_t threads = (int64_t)rows * c.n_kv * (D / 8);
  const dim3 grid((unsigned)((threads + 255) / 256), 2);
  const bool vec = vec_rows(k, sizeof(typename E::T)) && vec_rows(v, sizeof(typename E::T));
  auto f = append ? (vec ? k_kv4_append<D, E, true> : k_kv4_append<D, E, false>)
                  : (vec ? k_kv4_read<D, E, true> : k_kv4_read<D, E, false>);
  hipLaunchKernelGGL(f, grid, dim3(256), 0, st, c, rows, k, v, slots);
  return hipGetLastError();
}
template <class E>
hipError_t rows_dim(hipStream_t st, bool append, const Kv4Layer& c, int rows, const Rows& k, const Rows& v,
                    const int32_t* slots) {
  if (c.hd == 64) return rows_launch<64, E>(st, append, c, rows, k, v, slots);
  if (c.hd == 128) return rows_launch<128, E>(st, append, c, rows, k, v, slots);
  return rows_launch<256, E>(st, append, c, rows, k, v, slots);
}
hipError_t rows_type(hipStream_t st, bool append, const Kv4Layer& c, int dtype, int rows, const Rows& k, const Rows& v,
                     const int32_t* slots) {
  if (rows == 0) return hipSuccess;
  if (dtype == RSTR_F32) return rows_dim<F32>(st, append, c, rows, k, v, slots);
  if (dtype == RSTR_F16) return rows_dim<F16>(st, append, c, rows, k, v, slots);
  return rows_dim<BF16>(st, append, c, rows, k, v, slots);
}

// ---- attention ----------------------------------------------------------------------
// One workgroup per (query row, head): tiles of 256 tokens, one token's score a
// thread, then one dim a thread over the tile's probabilities; running maximum
// and sum in fp32.
template <int D, class E>
__global__ void __launch_bounds__(256) k_kv4_attn_row(Kv4Attn a) {
  typedef Rec<D> R;
  __shared__ float q[D], p[256], red[4], acc2[256];
  const int row = blockIdx.x, hq = blockIdx.y, tid = threadIdx.x;
  const int group = a.n_q / a.c.n_kv, h = hq / group;
  int lo = 0, hi = a.batch;  // the sequence of the row
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (a.row_offsets[mid] <= row) lo = mid; else hi = mid;
  }
  const int b = lo, r0 = a.row_offsets[b], r1 = a.row_offsets[b + 1];
  if (row < r0 || row >= r1) return;
  const int ps = a.c.page_size;
  const int64_t len = min((int64_t)max(a.lengths[b], 0), (int64_t)a.pps * ps);
  const int64_t end = max((int64_t)0, len - (r1 - row) + 1);
  const int64_t beg = a.window > 0 ? max((int64_t)0, end - a.window) : 0;
  if (tid < D) q[tid] = E::get(((const typename E::T*)a.q.p)[row * a.q.row + hq * a.q.head + tid]);
  __syncthreads();
  float m = -INFINITY, l = 0.0f, acc = 0.0f;
  const int dim = tid % D, part = tid / D, parts = 256 / D;
  for (int64_t t0 = beg; t0 < end; t0 += 256) {
    const int64_t t = t0 + tid;
    float s = -INFINITY;
    if (t < end) {
      const int page = a.page_table[(int64_t)b * a.pps + t / ps];
      if (page >= 0 && page < a.c.pages) {
        const uint8_t* rec = a.c.base + ((int64_t)page * a.c.n_kv + h) * kv4_record_bytes(D, ps);
        const int tok = (int)(t % ps);
        s = 0.0f;
        for (int bk = 0; bk < R::NB; bk++) {
          const float d = h2f(*(const uint16_t*)(rec + R::ksbase(ps) + R::s(tok >> 2, bk) + (tok & 3) * 2));
          float sum = 0.0f;
          for (int g = 0; g < 4; g++) {
            const uint32_t w = *(const uint32_t*)(rec + R::k(tok, bk, g));
            for (int i = 0; i < 4; i++) {
              sum = __builtin_fmaf(q[bk * 32 + g * 8 + 2 * i], (float)((int)((w >> (4 * i)) & 0xF) - 8), sum);
              sum = __builtin_fmaf(q[bk * 32 + g * 8 + 2 * i + 1], (float)((int)((w >> (16 + 4 * i)) & 0xF) - 8), sum);
            }
          }
          s = __builtin_fmaf(d, sum, s);
        }
        s *= a.scale;
      }
    }
    float top = wave_max(s);
    if ((tid & 63) == 0) red[tid >> 6] = top;
    __syncthreads();
    top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float mn = fmaxf(m, top);
    const float keep = m == -INFINITY ? 0.0f : dexp(m - mn);
    const float e = s == -INFINITY ? 0.0f : dexp(s - mn);
    m = mn;
    p[tid] = e;
    float sum = wave_tree_sum(e);
    __syncthreads();
    if ((tid & 63) == 0) red[tid >> 6] = sum;
    __syncthreads();
    l = l * keep + (red[0] + red[1] + red[2] + red[3]);
    acc *= keep;
    const int n = (int)min((int64_t)256, end - t0);
    const int bk = dim >> 5, c = dim & 15, nib = (bk & 1) * 2 + ((dim >> 4) & 1);
    for (int i = part; i < n; i += parts) {
      if (p[i] == 0.0f) continue;
      const int64_t tt = t0 + i;
      const int page = a.page_table[(int64_t)b * a.pps + tt / ps], tok = (int)(tt % ps);
      const uint8_t* rec = a.c.base + ((int64_t)page * a.c.n_kv + h) * kv4_record_bytes(D, ps);
      const float d = h2f(*(const uint16_t*)(rec + R::vsbase(ps) + R::s(tok >> 2, bk) + (tok & 3) * 2));
      const uint32_t w = *(const uint16_t*)(rec + R::vbase(ps) + R::v(tok >> 2, bk >> 1, c) + (tok & 3) * 2);
      acc = __builtin_fmaf(p[i], d * (float)((int)((w >> (4 * nib)) & 0xF) - 8), acc);
    }
    __syncthreads();
  }
  acc2[tid] = acc;
  __syncthreads();
  if (tid < D) {
    for (int i = 1; i < parts; i++) acc += acc2[tid + i * D];
    ((typename E::T*)a.out.p)[row * a.out.row + hq * a.out.head + tid] = E::put(l > 0.0f ? acc / l : (l == 0.0f ? 0.0f : l));
  }
}

template <class E>
hipError_t attn_row(hipStream_t st, const Kv4Attn& a) {
  const dim3 grid((unsigned)a.rows, (unsigned)a.n_q);
  if (a.c.hd == 64) hipLaunchKernelGGL((k_kv4_attn_row<64, E>), grid, dim3(256), 0, st, a);
  else if (a.c.hd == 128) hipLaunchKernelGGL((k_kv4_attn_row<128, E>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((k_kv4_attn_row<256, E>), grid, dim3(256), 0, st, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_kv4_append(hipStream_t st, const Kv4Layer& c, int dtype, int rows, const Rows& k, const Rows& v,
                             const int32_t* slots) {
  return rows_type(st, true, c, dtype, rows, k, v, slots);
}
hipError_t launch_kv4_read(hipStream_t st, const Kv4Layer& c, int dtype, int rows, const int32_t* slots, const Rows& k,
                           const Rows& v) {
  return rows_type(st, false, c, dtype, rows, k, v, slots);
}

size_t kv4_attn_workspace(int, int, int, int, int) { return 256; }

hipError_t launch_kv4_attn(hipStream_t st, int dtype, const Kv4Attn& a) {
  if (a.rows == 0 || a.batch == 0) return hipSuccess;
  if (dtype == RSTR_F32) return attn_row<F32>(st, a);
  if (dtype == RSTR_F16) return attn_row<F16>(st, a);
  return attn_row<BF16>(st, a);
}

}  // namespace rstr
