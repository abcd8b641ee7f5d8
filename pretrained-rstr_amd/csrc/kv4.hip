// kv4.hip -- the 4-bit paged K/V cache (format: kv4.h): quantising append,
// dequantising read and attention over it.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "../../include/rstr_hip.h"
#include "attn_line.h"
#include "device_math.h"
#include "kv4.h"
#include "kv4_line.h"

namespace rstr {

namespace {

// ---- addresses inside a record ----------------------------------------------------
template <int D>
struct Rec {
  static constexpr int NB = D / 32;                 // blocks of a row
  static constexpr int BQ = NB < 4 ? NB : 4;        // K: blocks a lane loads together
  static constexpr int BP = D / 64 < 2 ? D / 64 : 2;  // V: block pairs a lane loads together
  // byte offsets of a K code dword, a V code halfword (its j = 0) and a scale
  static __device__ __forceinline__ int k(int tok, int b, int g) {
    return (tok >> 4) * (8 * D) + (b / BQ) * (256 * BQ) + g * (64 * BQ) + (tok & 15) * (4 * BQ) + (b % BQ) * 4;
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

// ---- append and read ------------------------------------------------------------------
// A thread takes 8 elements of four rows: four that may lie in one group of four tokens,
// whose V codes are then written (read) as 8 bytes a column instead of 2, and a
// workgroup four quads of four heads, the 16 tokens that lines of K are made of (lines
// written in parts by several chips' caches cost far more than their bytes).  So that they
// do where a prompt's rows fill consecutive slots, the quads begin where the first slot's
// 16 do.  K: 8 neighbours of a block (blockIdx.y 0); V: columns 2i, 2i + 1 of a block pair,
// that is 2 neighbours at four places, so that a thread holds whole halfwords.
//
// Bound by memory and, for the codes, nearly so by vector instructions: 16411 bf16 rows of 8 heads of 128
// (86 MB) are appended in 22 us, 3.9 TB/s, and read in 17, 5.0.
// Few rows take one row a thread: 128 fp32 rows of 8 heads are then appended in 3.4 us (four
// rows a thread: 5.9) and read in 3.3 (5.1); the 16411 rows above would be 27 and 27.
//
// Codes: x / d is the product with d's reciprocal, corrected once by its residual, and adding
// 1.5 * 2^23 rounds it to the nearest integer, ties to even, and leaves that in the low bits.
// The corrected quotient is x / d rounded to fp32, so it is a half only where x / d is, or
// is nearer to one than fp32 tells.  Quotients of two numbers of 11 bits are not, so for fp16 and
// bf16 rows that is exact; for fp32 rows, where some lane's quotient is a half,
// the codes are decided by r = x - c * d, which is exact there.
//
// The first element of greatest magnitude.  16-bit elements have room below their bits
// for the place and the sign: one integer maximum.  fp32: the larger of maximum and
// -minimum; only where these are equal does the order of the elements matter.
struct Extreme {
  float m;
  int at;
  __device__ __forceinline__ void meet(float om, int oat) {
    const bool other = fabsf(om) > fabsf(m) || (fabsf(om) == fabsf(m) && oat < at);
    m = other ? om : m;
    at = other ? oat : at;
  }
};
__device__ __forceinline__ float max_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ float min_nan(float a, float b) { return __builtin_elementwise_minimum(a, b); }
__device__ __forceinline__ uint32_t dpp_max(uint32_t v, uint32_t o) { return o > v ? o : v; }
// Of a block spread over aligned groups of G lanes, N elements a lane, element i at
// place(i) of the block: the first element of greatest magnitude; `bad` if one is
// a NaN or infinite.
template <class E, int N, int G, class P>
__device__ __forceinline__ float extreme(const float* x, P place, bool& bad) {
  if constexpr (sizeof(typename E::T) == 2) {
    uint32_t k = 0;
#pragma unroll
    for (int i = 0; i < N; i++) {
      const uint32_t u = __float_as_uint(x[i]);
      k = dpp_max(k, __builtin_rotateleft32(u, 1) | (uint32_t)(31 - place(i)) << 1);
    }
    k = dpp_max(k, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)k, 0xB1, 0xF, 0xF, true));
    k = dpp_max(k, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)k, 0x4E, 0xF, 0xF, true));
    if constexpr (G == 8) k = dpp_max(k, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)k, 0x141, 0xF, 0xF, true));
    bad = k >= 0xFF000000u;
    return __uint_as_float(__builtin_rotateright32(k & ~0x3Eu, 1));
  }
  float hi = x[0], lo = x[0];
#pragma unroll
  for (int i = 1; i < N; i++) {
    hi = max_nan(hi, x[i]);
    lo = min_nan(lo, x[i]);
  }
  hi = max_nan(hi, xor_lane<1>(hi));
  lo = min_nan(lo, xor_lane<1>(lo));
  hi = max_nan(hi, xor_lane<2>(hi));
  lo = min_nan(lo, xor_lane<2>(lo));
  if constexpr (G == 8) {
    hi = max_nan(hi, half_mirror_lane(hi));
    lo = min_nan(lo, half_mirror_lane(lo));
  }
  bad = !(hi < INFINITY && lo > -INFINITY);
  float m = hi > -lo ? hi : lo;
  if (__ballot(hi == -lo && hi > 0.0f)) {
    Extreme e{x[0], place(0)};
#pragma unroll
    for (int i = 1; i < N; i++) e.meet(x[i], place(i));
    e.meet(xor_lane<1>(e.m), __builtin_amdgcn_update_dpp(0, e.at, 0xB1, 0xF, 0xF, true));
    e.meet(xor_lane<2>(e.m), __builtin_amdgcn_update_dpp(0, e.at, 0x4E, 0xF, 0xF, true));
    if constexpr (G == 8) e.meet(half_mirror_lane(e.m), __builtin_amdgcn_update_dpp(0, e.at, 0x141, 0xF, 0xF, true));
    if (hi == -lo) m = e.m;
  }
  return m;
}

struct Scale {
  uint16_t bits;
  float d, id;
  __device__ __forceinline__ Scale(float m, bool bad) {
    bits = f2h_bits(__builtin_amdgcn_fmed3f(m * -0.125f, -65504.0f, 65504.0f));
    if ((bits & 0x7FFFu) == 0) bits = 0;
    d = h2f(bits);
    if (bad) bits = 0x7E00u;
    id = bad || d == 0.0f ? 0.0f : __builtin_amdgcn_rcpf(d);
  }
  __device__ __forceinline__ float quotient(float x) const {
    const float t = x * id;
    return __builtin_fmaf(__builtin_fmaf(-t, d, x), id, t);
  }
  static __device__ __forceinline__ uint32_t nearest(float t) {
    return __float_as_uint(__builtin_amdgcn_fmed3f(t + (0x1.8p23f + 8.0f), 0x1.8p23f, 0x1.8p23f + 15.0f)) & 0xFu;
  }
  __device__ __forceinline__ uint32_t exact(float x) const {
    float q = __builtin_rintf(__builtin_amdgcn_fmed3f(x * id, -9.0f, 8.0f));
    const float r = __builtin_fmaf(-q, d, x), up = (r < 0.0f) == (d < 0.0f) ? 1.0f : -1.0f, half = fabsf(d) * 0.5f;
    const bool odd = ((int)q & 1) != 0;
    if (fabsf(r) > half || (fabsf(r) == half && odd)) q += up;
    return (uint32_t)((int)__builtin_amdgcn_fmed3f(q, -8.0f, 7.0f) + 8);
  }
  // N elements' codes, put(i, code) for each; 8, that is 0, where there is no scale.
  template <class E, int N, class F>
  __device__ __forceinline__ void codes(const float* x, bool bad, F put) const {
    float y[N];
    uint32_t c[N];
#pragma unroll
    for (int i = 0; i < N; i++) y[i] = x[i];
    if (__ballot(bad)) {
#pragma unroll
      for (int i = 0; i < N; i++) y[i] = bad ? 0.0f : y[i];
    }
#pragma unroll
    for (int i = 0; i < N; i++) y[i] = quotient(y[i]);
#pragma unroll
    for (int i = 0; i < N; i++) c[i] = nearest(y[i]);
    if constexpr (sizeof(typename E::T) == 4) {
      bool half = false;
#pragma unroll
      for (int i = 0; i < N; i++) half |= __builtin_amdgcn_fractf(y[i]) == 0.5f;
      if (__ballot(half)) {
#pragma unroll
        for (int i = 0; i < N; i++)
          if (!bad && id != 0.0f) c[i] = exact(x[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < N; i++) put(i, c[i]);
  }
};

// N rows from `row` on, their slots (-1: none) and whether these are one group of tokens.
template <int N>
struct Quad {
  int row, slot[N];
  bool group;
  __device__ __forceinline__ Quad(const int32_t* slots, int rows, int quad, int64_t limit) {
    row = quad * N;
    if constexpr (N == 4) {
      const int first = slots[0];
      row -= first > 0 ? first & 15 : 0;
    }
    group = N == 4;
#pragma unroll
    for (int i = 0; i < N; i++) {
      const int r = row + i;
      const int s = r >= 0 && r < rows ? slots[r] : -1;
      slot[i] = s >= 0 && s < limit ? s : -1;
      group = group && slot[i] >= 0 && slot[i] == slot[0] + i;
    }
    group = group && (slot[0] & 3) == 0;
  }
  // the row that is loaded in row i's place: one that is there
  __device__ __forceinline__ int64_t read(int i, int rows) const { return min(max(row + i, 0), rows - 1); }
  __device__ __forceinline__ bool live(int i, int rows) const { return row + i >= 0 && row + i < rows; }
};

// The record and token of a slot.
struct Place {
  uint8_t* rec;
  int tok;
  __device__ __forceinline__ Place(const Kv4Layer& L, int hd, int h, int slot) {
    const uint32_t page = (uint32_t)slot / (uint32_t)L.page_size;
    tok = slot - (int)(page * (uint32_t)L.page_size);
    rec = L.base + ((int64_t)page * L.n_kv + h) * kv4_record_bytes(hd, L.page_size);
  }
};

// Two neighbours, aligned to both where VEC.
template <class E, bool VEC>
__device__ __forceinline__ void load2(const typename E::T* p, float* x) {
  struct __attribute__((aligned(2 * sizeof(typename E::T)))) Pair { typename E::T a, b; };
  if constexpr (VEC) {
    const Pair t = *(const Pair*)p;
    x[0] = E::get(t.a);
    x[1] = E::get(t.b);
  } else {
    x[0] = E::get(p[0]);
    x[1] = E::get(p[1]);
  }
}
template <class E, bool VEC>
__device__ __forceinline__ void store2(typename E::T* p, const float* x) {
  struct __attribute__((aligned(2 * sizeof(typename E::T)))) Pair { typename E::T a, b; };
  if constexpr (VEC) {
    *(Pair*)p = Pair{E::put(x[0]), E::put(x[1])};
  } else {
    p[0] = E::put(x[0]);
    p[1] = E::put(x[1]);
  }
}

template <int D, class E, bool VEC, int N>
__global__ void __launch_bounds__(256) k_kv4_append(Kv4Layer L, int rows, int quads, Rows kr, Rows vr, const int32_t* __restrict__ slots) {
  typedef Rec<D> R;
  typedef typename E::T T;
  constexpr int TPR = D / 8;  // threads a quad and head
  const bool is_v = blockIdx.y != 0;
  const uint32_t gid = blockIdx.x * 256u + threadIdx.x, qh = gid / TPR;
  constexpr uint32_t SIDE = N == 4 ? 4 : 1;  // quads before the next head's
  const uint32_t hq = qh / SIDE, side = hq / (uint32_t)L.n_kv;
  const int t = (int)(gid % TPR), quad = (int)(side * SIDE + qh % SIDE), h = (int)(hq - side * (uint32_t)L.n_kv);
  const int ps = L.page_size;
  // lanes behind the last quad take part in the exchanges
  const Quad<N> Q(slots, quad < quads ? rows : 0, quad, (int64_t)L.pages * ps);
  if (!is_v) {
    float x[N][8];
#pragma unroll
    for (int i = 0; i < N; i++) load8<E, VEC>((const T*)kr.p + Q.read(i, rows) * kr.row + (int64_t)h * kr.head + t * 8, x[i]);
    const int b = t >> 2, g = t & 3;
    uint16_t sc[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
      bool bad;
      const float m = extreme<E, 8, 4>(x[i], [&](int j) { return g * 8 + j; }, bad);
      const Scale s(m, bad);
      sc[i] = s.bits;
      uint32_t w = 0;
      s.template codes<E, 8>(x[i], bad, [&](int j, uint32_t c) { w |= c << (4 * (j >> 1) + 16 * (j & 1)); });
      if (Q.slot[i] >= 0) {
        const Place p(L, D, h, Q.slot[i]);
        *(uint32_t*)(p.rec + R::k(p.tok, b, g)) = w;
        if (!Q.group && g == 0) *(uint16_t*)(p.rec + R::ksbase(ps) + R::s(p.tok >> 2, b) + (p.tok & 3) * 2) = s.bits;
      }
    }
    if constexpr (N == 4)
    if (Q.group && g == 0) {
      const Place p(L, D, h, Q.slot[0]);
      *(u32x2*)(p.rec + R::ksbase(ps) + R::s(p.tok >> 2, b)) = u32x2{sc[0] | (uint32_t)sc[1] << 16, sc[2] | (uint32_t)sc[3] << 16};
    }
    return;
  }
  const int bp = t >> 3, c = (t & 7) * 2;
  float x[N][2][4];  // row, block of the pair, (half, column)
#pragma unroll
  for (int i = 0; i < N; i++)
#pragma unroll
    for (int k = 0; k < 4; k++) {
      load2<E, VEC>((const T*)vr.p + Q.read(i, rows) * vr.row + (int64_t)h * vr.head + bp * 64 + k * 16 + c, &x[i][k >> 1][2 * (k & 1)]);
    }
  uint16_t sc[2][N], cols[2][N];  // block or column, row
#pragma unroll
  for (int i = 0; i < N; i++) {
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int k = 0; k < 2; k++) {
      const float* y = x[i][k];
      bool bad;
      const float m = extreme<E, 4, 8>(y, [&](int j) { return c + (j & 1) + 16 * (j >> 1); }, bad);
      const Scale s(m, bad);
      sc[k][i] = s.bits;
      s.template codes<E, 4>(y, bad, [&](int j, uint32_t c) { w[j & 1] |= c << (8 * k + 4 * (j >> 1)); });
    }
    cols[0][i] = (uint16_t)w[0];
    cols[1][i] = (uint16_t)w[1];
    if (!Q.group && Q.slot[i] >= 0) {
      const Place p(L, D, h, Q.slot[i]);
      uint8_t* at = p.rec + (p.tok & 3) * 2;
#pragma unroll
      for (int k = 0; k < 2; k++) {
        *(uint16_t*)(at + R::vbase(ps) + R::v(p.tok >> 2, bp, c + k)) = cols[k][i];
        if ((t & 7) == 0) *(uint16_t*)(at + R::vsbase(ps) + R::s(p.tok >> 2, 2 * bp + k)) = sc[k][i];
      }
    }
  }
  if constexpr (N == 4)
  if (Q.group) {
    const Place p(L, D, h, Q.slot[0]);
#pragma unroll
    for (int k = 0; k < 2; k++) {
      *(u32x2*)(p.rec + R::vbase(ps) + R::v(p.tok >> 2, bp, c + k)) =
          u32x2{cols[k][0] | (uint32_t)cols[k][1] << 16, cols[k][2] | (uint32_t)cols[k][3] << 16};
      if ((t & 7) == 0)
        *(u32x2*)(p.rec + R::vsbase(ps) + R::s(p.tok >> 2, 2 * bp + k)) =
            u32x2{sc[k][0] | (uint32_t)sc[k][1] << 16, sc[k][2] | (uint32_t)sc[k][3] << 16};
    }
  }
}

// d * (c - 8) is exact in fp32 (11 + 4 bits) and rounded once to the output's type.
template <int D, class E, bool VEC, int N>
__global__ void __launch_bounds__(256) k_kv4_read(Kv4Layer L, int rows, int quads, Rows kr, Rows vr, const int32_t* __restrict__ slots) {
  typedef Rec<D> R;
  typedef typename E::T T;
  constexpr int TPR = D / 8;
  const bool is_v = blockIdx.y != 0;
  const uint32_t gid = blockIdx.x * 256u + threadIdx.x, qh = gid / TPR;
  constexpr uint32_t SIDE = N == 4 ? 4 : 1;  // quads before the next head's
  const uint32_t hq = qh / SIDE, side = hq / (uint32_t)L.n_kv;
  const int t = (int)(gid % TPR), quad = (int)(side * SIDE + qh % SIDE), h = (int)(hq - side * (uint32_t)L.n_kv);
  const int ps = L.page_size;
  if (quad >= quads) return;
  const Quad<N> Q(slots, rows, quad, (int64_t)L.pages * ps);
  if (!is_v) {
    const int b = t >> 2, g = t & 3;
    uint32_t w[N];
    uint16_t sc[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
      w[i] = 0x88888888u;
      sc[i] = 0;
      if (Q.slot[i] >= 0) {
        const Place p(L, D, h, Q.slot[i]);
        w[i] = *(const uint32_t*)(p.rec + R::k(p.tok, b, g));
        sc[i] = *(const uint16_t*)(p.rec + R::ksbase(ps) + R::s(p.tok >> 2, b) + (p.tok & 3) * 2);
      }
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
      if (!Q.live(i, rows)) continue;
      const float d = h2f(sc[i]);
      float x[8];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        x[2 * j] = d * (float)((int)((w[i] >> (4 * j)) & 0xF) - 8);
        x[2 * j + 1] = d * (float)((int)((w[i] >> (16 + 4 * j)) & 0xF) - 8);
      }
      store8<E, VEC>((T*)kr.p + (int64_t)(Q.row + i) * kr.row + (int64_t)h * kr.head + t * 8, x);
    }
    return;
  }
  const int bp = t >> 3, c = (t & 7) * 2;
  uint16_t cols[2][N], sc[2][N];
  bool loaded = false;
  if constexpr (N == 4)
  if (Q.group) {
    loaded = true;
    const Place p(L, D, h, Q.slot[0]);
#pragma unroll
    for (int k = 0; k < 2; k++) {
      const u32x2 a = *(const u32x2*)(p.rec + R::vbase(ps) + R::v(p.tok >> 2, bp, c + k));
      const u32x2 s = *(const u32x2*)(p.rec + R::vsbase(ps) + R::s(p.tok >> 2, 2 * bp + k));
#pragma unroll
      for (int i = 0; i < N; i++) {
        cols[k][i] = (uint16_t)(a[i >> 1] >> (16 * (i & 1)));
        sc[k][i] = (uint16_t)(s[i >> 1] >> (16 * (i & 1)));
      }
    }
  }
  if (!loaded) {
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
      for (int k = 0; k < 2; k++) {
        cols[k][i] = 0x8888;
        sc[k][i] = 0;
        if (Q.slot[i] >= 0) {
          const Place p(L, D, h, Q.slot[i]);
          const uint8_t* at = p.rec + (p.tok & 3) * 2;
          cols[k][i] = *(const uint16_t*)(at + R::vbase(ps) + R::v(p.tok >> 2, bp, c + k));
          sc[k][i] = *(const uint16_t*)(at + R::vsbase(ps) + R::s(p.tok >> 2, 2 * bp + k));
        }
      }
  }
#pragma unroll
  for (int i = 0; i < N; i++) {
    if (!Q.live(i, rows)) continue;
#pragma unroll
    for (int k = 0; k < 4; k++) {  // block k >> 1 of the pair, half k & 1
      const float d = h2f(sc[k >> 1][i]);
      float x[2];
#pragma unroll
      for (int j = 0; j < 2; j++) x[j] = d * (float)((int)((cols[j][i] >> (4 * k)) & 0xF) - 8);
      store2<E, VEC>((T*)vr.p + (int64_t)(Q.row + i) * vr.row + (int64_t)h * vr.head + bp * 64 + k * 16 + c, x);
    }
  }
}

template <int D, class E>
hipError_t rows_launch(hipStream_t st, bool append, const Kv4Layer& c, int rows, const Rows& k, const Rows& v,
                       const int32_t* slots) {
  // a row a thread while that does not fill the chip twice over (measured above); else four, the first quad
  // beginning up to 15 rows before the first row
  const bool few = (int64_t)rows * c.n_kv * (D / 8) * 2 < (int64_t)1 << 19;
  const int quads = few ? rows : (int)(((int64_t)rows + 15 + 15) / 16) * 4;
  const int64_t threads = (int64_t)quads * c.n_kv * (D / 8);
  const dim3 grid((unsigned)((threads + 255) / 256), 2);
  const bool vec = vec_rows(k, sizeof(typename E::T)) && vec_rows(v, sizeof(typename E::T));
#define RSTR_ROWS(N)                                                                            \
  (append ? (vec ? k_kv4_append<D, E, true, N> : k_kv4_append<D, E, false, N>)                  \
          : (vec ? k_kv4_read<D, E, true, N> : k_kv4_read<D, E, false, N>))
  auto f = few ? RSTR_ROWS(1) : RSTR_ROWS(4);
#undef RSTR_ROWS
  hipLaunchKernelGGL(f, grid, dim3(256), 0, st, c, rows, quads, k, v, slots);
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
// One wave works on 16 * NT columns (a query row of one head of the kv head's
// group is a column) of one sequence and kv head, over tiles of 32 tokens:
//
//   S^T = K Q^T     K (codes) is the A operand, Q^T the B operand of 16x16x32 f16
//                   products, one block of 32 dims each: S = sum_b d_b * S_b with
//                   the blocks' scales applied to the fp32 products
//   O^T += V^T P^T  a lane's S^T values are four consecutive tokens of one column,
//                   which is what the B operand P^T wants from that lane, and V codes
//                   are laid out so that its A operand is what a lane loads: neither
//                   LDS nor lane exchanges.  The scales of V differ by (token,
//                   block), so P is multiplied by them, one copy for each block.
//
// Codes are exact in fp16: (w & 0x00F000F0) | 0x54005400 is the pair 64 + c.
// Queries are brought to [0.5, 1) of their row's largest element by a power of
// two and taken as one fp16 term (f16, bf16: no bit of an element above 2^-14 of
// the largest is lost) or two (fp32: 22 bits).  Probabilities p = 2^(s - mref)
// likewise: one term, or two of p * d.  mref follows the running maximum only
// when a score passes it by 2^4, so the exchange between lanes that the
// maximum needs, and the rescaling of O and l, happen a few times a segment; p
// carries a factor 2^10, so small weights keep their bits: fp16's subnormals
// begin 2^24 below the largest.  With two terms, a power of two that follows the largest
// scale of V seen so far, up to 2, brings small products up.  Scales of 2 and more are taken
// with 2^-15 of themselves, and the rest of their part, 2^15 - 1 times as much, is added by products of their
// own, so that scales beside them keep their bits.
//
// The tiles of all (sequence, kv head, column tile) items form one line of units
// that is cut into equal parts, one a wave: the load is even whatever the
// lengths are.  A wave writes the output of an item that lies in its part as a
// whole; else (O, mref, l) of its piece, and k_kv4_merge joins the pieces in
// order.
//
// NT = 1 where no sequence has more than 16 columns: 128 sequences of 128 to 4608 tokens, one fp16 row of 32
// heads each (8 kv heads of 128, 351 MB) take 80 us, 4.4 TB/s, bound by memory (362 MB are read; loads
// alone: 65) and vector instructions (busy 63 % of the time) together; the whole call 88, with NT = 2 137.  Three of 20161
// to 131072 tokens, bf16 (261 MB): 51 us, 5.1 TB/s, memory, and 11 for the merge; 33 of 5 to 8192 with up to six fp32
// rows of 16 heads (157 MB) 52 and 8: vector instructions are busy 58 %, as every weight and its rest need a product each,
// and memory gives 3.4 TB/s, so neither alone is the bound: waves wait to issue a third of the time, for memory a fifth.
// Where a table holds no more than kWhole tiles a wave does an item by itself: one sequence of 37 tokens 8.1 us,
// without the 4 of a merge.  Parts of two tiles at least, where there is little work: 16 windows of 512
// tokens, head dim 256, 15 us (four tiles: 20, one: 14), and 16 sequences of 200 tokens 14 (15, 17).
constexpr int kStart = 6;  // what beginning an item costs, in tiles
// Queries are brought down by no more, so that what brings their scores up again stays finite: the largest are 2^8 then.
constexpr int kLargestPower = 120;

// Terms of a weight; ONCE: p * d is rounded once, from fp32.  bf16 results round to 8
// bits anyway, so there p is rounded to fp16 and multiplied by pairs.
template <class E> struct Terms { static constexpr int n = 1; static constexpr bool ONCE = true; };
template <> struct Terms<F32> { static constexpr int n = 2; static constexpr bool ONCE = true; };
template <> struct Terms<BF16> { static constexpr int n = 1; static constexpr bool ONCE = false; };

// Tiles of a wave's ring: what 160 KB of LDS hold for that many waves.
constexpr int attn_ring(int hd, int nt) { return attn_waves(hd, nt) == 3 && hd == 128 ? 2 : 4; }

template <int N>
__device__ __forceinline__ void load_dwords(const uint8_t* p, uint32_t* o) {
  if constexpr (N == 2) {
    const u32x2 v = *(const u32x2*)p;
    o[0] = v[0]; o[1] = v[1];
  } else {
#pragma unroll
    for (int i = 0; i < N / 4; i++) {
      const u32x4 v = ((const u32x4*)p)[i];
      o[4 * i] = v[0]; o[4 * i + 1] = v[1]; o[4 * i + 2] = v[2]; o[4 * i + 3] = v[3];
    }
  }
}

// Masks and exponents of the code expansion in registers: an instruction that
// selects and merges takes no literals, and with literals it is two.
struct Magic {
  uint32_t lo = 0x000F000Fu, hi = 0x00F000F0u, e1024 = 0x64006400u, e64 = 0x54005400u;
  __device__ __forceinline__ Magic() {
    asm("" : "+s"(lo));
    asm("" : "+s"(hi));
    asm("" : "+v"(e1024));
    asm("" : "+v"(e64));
  }
};
// Pair i of a dword's eight codes c as two fp16, c - 8: 1024 + c (i even) or 64 + c
// (odd) from the bits, less that bias.  (Fewer instructions leave the bias in the
// products, or take the codes as fp16 subnormals, c * 2^-24: both were exact only to 2^-14
// of a block's scale, and no faster.)
__device__ __forceinline__ h2 code_pair(const Magic& m, uint32_t w, int i) {
  const uint32_t x = i < 2 ? w : w >> 8;
  const _Float16 b = (i & 1) ? (_Float16)-72.0f : (_Float16)-1032.0f;
  return __builtin_bit_cast(h2, (i & 1) ? (x & m.hi) | m.e64 : (x & m.lo) | m.e1024) + h2{b, b};
}
__device__ __forceinline__ h8 pack8(h2 a, h2 b, h2 c, h2 d) {
  return h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ __forceinline__ float half_of(uint32_t w, int i) { return (float)__builtin_bit_cast(h2, w)[i]; }

// Codes and scales of a tile's keys or values, by half of 16 tokens.
template <int D>
struct TileRegs {
  static constexpr int NB = D / 32;
  uint32_t c[2][NB], s[2][2 * NB];
};

// The ring of tiles that a wave keeps in LDS (bytes): K codes, V codes, then the
// scales of both, each as its halves of 16 tokens lie in the records.
template <int D>
struct Ring {
  static constexpr int CODES = 16 * D, SCALES = 2 * D, TILE = 2 * CODES + 2 * SCALES;
  static constexpr int LOADS = D == 64 ? 3 : 2 * (D / 64) + 1;  // instructions a tile
};
#define RSTR_LDS(p) ((__attribute__((address_space(3))) void*)(p))
typedef const __attribute__((address_space(4))) int32_t* TablePtr;  // read-only for the kernel: scalar loads

// s_waitcnt vmcnt(N) alone.
template <int N>
__device__ __forceinline__ void wait_loads() {
  __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | ((N >> 4) << 14));
}

template <int D, int NT, int NS, class E>
__global__ void __launch_bounds__(256, attn_waves(D, NT))
    k_kv4_attn(Kv4Attn a, const int32_t* __restrict__ ro, const int32_t* __restrict__ lens, const int32_t* __restrict__ table,
               const uint8_t* __restrict__ base, Pieces pc, int workers, int least, bool whole) {
  typedef Rec<D> R;
  typedef typename E::T T;
  constexpr int NB = D / 32, COLS = 16 * NT, TERMS = Terms<E>::n;
  constexpr bool ONCE = Terms<E>::ONCE;
  const Magic magic;
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int w = uniform(blockIdx.x * 4 + (threadIdx.x >> 6));
  const int group = a.n_q / a.c.n_kv, ps = a.c.page_size;
  const Lines L{ro, lens, a.rows, a.c.n_kv, group, a.window, COLS, (int)min((int64_t)a.pps * ps, (int64_t)0x7FFFFFC0), kStart, whole};

  Line line(L, a.batch, w, workers, least);
  if (w == 0 && !whole) *pc.n_items = line.items();

  typedef Ring<D> G;
  __shared__ __attribute__((aligned(16))) uint8_t rings[4][NS][G::TILE];
  uint8_t(*ring)[G::TILE] = rings[uniform(threadIdx.x >> 6)];
  const int64_t rec = kv4_record_bytes(D, ps);
  // where a lane's pieces lie in a tile of the ring, and where the lane's scales come from
  const uint32_t k_at = lane * (4 * R::BQ), v_at = G::CODES + R::v(g, 0, col), ks_at = 2 * G::CODES + g * (8 * NB), vs_at = ks_at + G::SCALES;
  constexpr int SL = D / 16;  // lanes that load the scales of one half
  const uint32_t sc_off = (lane & (2 * SL) ? R::vsbase(ps) : R::ksbase(ps)) + (lane % SL) * 16;

  while (line.next()) {
    const Seq& s = line.s;
    const int b = line.b, h = line.h, ct = line.ct, at = line.at, n = line.n;
    const bool begins = line.begins, ends = line.ends;
    if (begins && !whole && lane == 0) pc.begun[line.item] = Begun{b, h, ct, w, line.pieces};

    // the columns' rows and what they see
    const int c0 = ct * COLS, p0 = s.len - s.m, held = L.held(s.len);
    const auto end_seen = [&](int r) { return min(max(p0 + r + 1, 0), held); };
    const auto first_seen = [&](int r) { return a.window > 0 ? max(max(p0 + r + 1, 0) - a.window, 0) : 0; };
    const int rf = c0 / group, rl = min(s.m - 1, (c0 + COLS - 1) / group);
    int hi[NT], lo[NT];
    int64_t qrow[NT], qhead[NT];
    bool valid[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) {
      const int cc = c0 + t * 16 + col, r = cc / group;
      valid[t] = r < s.m;
      hi[t] = valid[t] ? end_seen(r) : 0;
      lo[t] = first_seen(r);
      qrow[t] = s.r0 + r;
      qhead[t] = (int64_t)h * group + (cc - r * group);
    }
    const int hi_last = end_seen(rl), hi_first = end_seen(rf);
    const int lo_first = first_seen(rf), lo_last = first_seen(rl);
    int t0 = s.lo + (whole ? 0 : max(at - kStart, 0)), t1 = s.lo + (whole ? s.tiles : max(at + n - kStart, 0));
    t0 = max(t0, lo_first / kTile);
    t1 = min(t1, (hi_last + kTile - 1) / kTile);

    f4 acc[NT][2 * NB];
    float mref[NT], kcol[NT], fs[NT];
    f4 l[NT];      // ONCE: the lane's own part of the sum of p in the first; else the sum, in all four
    int elim[NT];  // two terms: exponents of the V scales below 2 seen so far are no larger; fs = 2^(15 - elim)
    h8 q[NT][TERMS][NB];
#pragma unroll
    for (int t = 0; t < NT; t++) {
#pragma unroll
      for (int i = 0; i < 2 * NB; i++) acc[t][i] = f4{0, 0, 0, 0};
      mref[t] = -FLT_MAX;
      l[t] = f4{0, 0, 0, 0};
      elim[t] = 0;
      fs[t] = __builtin_amdgcn_ldexpf(1.0f, 15 - elim[t]);
    }
    if (t0 < t1) {
      // Tiles come into the ring NS - 1 ahead, straight into LDS; behind the last one, and
      // for a page that is not there, from page 0, so that the count of loads in
      // flight is known.  Page ids are read one tile ahead of their loads.
      const TablePtr row = (TablePtr)(table + (int64_t)b * a.pps);
      const int n_pages = (int)(((int64_t)held + ps - 1) / ps);
      int pg = t0 * kTile / ps, off = t0 * kTile - pg * ps, slot = 0;
      const uint8_t* head = base + (int64_t)h * rec;
      const uint32_t page_bytes = (uint32_t)(a.c.n_kv * rec);
      int id[2], id_off[2];
      const auto look = [&] {
#pragma unroll
        for (int j = 0; j < 2; j++) {
          const int v = row[min(pg, n_pages - 1)];
          id[j] = pg < n_pages ? v : -1;
          id_off[j] = off;
          off += 16;
          if (off == ps) { off = 0; pg++; }
        }
      };
      uint32_t lost = 0;  // halves whose page is not there: two bits a tile, the tile computed lowest
      const auto issue = [&] {
        const uint8_t* r[2];
#pragma unroll
        for (int j = 0; j < 2; j++) {
          const bool ok = (uint32_t)id[j] < (uint32_t)a.c.pages;
          r[j] = head + (uint64_t)(uint32_t)(ok ? id[j] : 0) * page_bytes;
          if (!ok) lost |= 1u << (2 * (NS - 1) + j);
        }
        uint8_t* to = ring[slot];
        slot = slot + 1 == NS ? 0 : slot + 1;
#pragma unroll
        for (int kv = 0; kv < 2; kv++) {
          const uint32_t start = kv ? R::vbase(ps) : 0;
          if constexpr (D == 64) {  // half a wave a half
            const uint8_t* p = lane < 32 ? r[0] + (uint32_t)id_off[0] * (D / 2) : r[1] + (uint32_t)id_off[1] * (D / 2);
            __builtin_amdgcn_global_load_lds((const void*)(p + (start + (lane & 31) * 16)), RSTR_LDS(to + kv * G::CODES), 16, 0, 0);
          } else {
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
              for (int i = 0; i < D / 128; i++)
                __builtin_amdgcn_global_load_lds((const void*)(r[j] + (start + (uint32_t)id_off[j] * (D / 2) + i * 1024 + lane * 16)),
                                                 RSTR_LDS(to + kv * G::CODES + (j * (D / 128) + i) * 1024), 16, 0, 0);
          }
        }
        const bool second = (lane & SL) != 0;
        const uint8_t* p = second ? r[1] + (uint32_t)id_off[1] * SL : r[0] + (uint32_t)id_off[0] * SL;
        if (lane < 4 * SL) __builtin_amdgcn_global_load_lds((const void*)(p + sc_off), RSTR_LDS(to + 2 * G::CODES), 16, 0, 0);
        look();
      };
      // a tile's codes or scales from the ring, by half
      const auto codes = [&](const uint8_t* at, uint32_t (&o)[2][NB]) {
#pragma unroll
        for (int j = 0; j < 2; j++) {
          if constexpr (NB == 8) {
            load_dwords<4>(at + j * 8 * D, o[j]);
          } else {
            load_dwords<NB>(at + j * 8 * D, o[j]);
          }
        }
      };
      const auto scales = [&](const uint8_t* at, uint32_t (&o)[2][2 * NB]) {
#pragma unroll
        for (int j = 0; j < 2; j++) load_dwords<2 * NB>(at + j * D, o[j]);
      };
      int now = 0;  // the ring's tile that is computed
      look();
#pragma unroll
      for (int i = 0; i < NS - 1; i++) {
        lost >>= 2;
        issue();
      }

      const bool vec = vec_rows(a.q, sizeof(T));
#pragma unroll
      for (int t = 0; t < NT; t++) {
        float x[NB][8];
        float big = 0.0f;
#pragma unroll
        for (int bk = 0; bk < NB; bk++) {
          if (valid[t]) {
            const T* src = (const T*)a.q.p + qrow[t] * a.q.row + qhead[t] * a.q.head + bk * 32 + g * 8;
            if (vec) load8<E, true>(src, x[bk]); else load8<E, false>(src, x[bk]);
          } else {
#pragma unroll
            for (int i = 0; i < 8; i++) x[bk][i] = 0.0f;
          }
#pragma unroll
          for (int i = 0; i < 8; i++) big = fmaxf(big, fabsf(x[bk][i]));
        }
        big = xor_max<32>(xor_max<16>(big));
        const int e = min(__builtin_amdgcn_frexp_expf(big), kLargestPower);
        kcol[t] = __builtin_amdgcn_ldexpf(a.scale * 1.4426950408889634f, e);
#pragma unroll
        for (int bk = 0; bk < NB; bk++)
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const float y = __builtin_amdgcn_ldexpf(x[bk][i], -e);
            const _Float16 top = (_Float16)y;
            q[t][0][bk][i] = top;
            if constexpr (TERMS == 2) q[t][1][bk][i] = (_Float16)(y - (float)top);
          }
      }

      const uint32_t one = 0x3C003C00u;
      const h8 ones = __builtin_bit_cast(h8, u32x4{one, one, one, one});

      for (int tile = t0; tile < t1; tile++) {
        // the slot filled next was read a tile ago: those reads have returned
        lost >>= 2;
        issue();
        wait_loads<(NS - 1) * G::LOADS>();
        asm volatile("" ::: "memory");
        const uint8_t* at = ring[now];
        now = now + 1 == NS ? 0 : now + 1;
        TileRegs<D> xk, xv;
        codes(at + k_at, xk.c);
        if constexpr (NB == 8) {
          load_dwords<4>(at + k_at + 1024, xk.c[0] + 4);
          load_dwords<4>(at + k_at + 1024 + 8 * D, xk.c[1] + 4);
        }
        scales(at + ks_at, xk.s);
        const int tok0 = tile * kTile;
        const bool edge = (lost & 3) || tok0 < lo_last || tok0 + kTile > hi_first;
        float sc[NT][8];  // scores over 2^e of their column's queries, before the scale
        {
          h8 kq[2][NB];
#pragma unroll
          for (int j = 0; j < 2; j++)
#pragma unroll
            for (int bk = 0; bk < NB; bk++) {
              const uint32_t w = xk.c[j][bk];
              kq[j][bk] = pack8(code_pair(magic, w, 0), code_pair(magic, w, 1), code_pair(magic, w, 2), code_pair(magic, w, 3));
            }
#pragma unroll
          for (int t = 0; t < NT; t++) {
            f4 d[2][NB];
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
              for (int bk = 0; bk < NB; bk++) {
                d[j][bk] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kq[j][bk], q[t][0][bk], f4{0, 0, 0, 0}, 0, 0, 0);
                if constexpr (TERMS == 2) d[j][bk] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kq[j][bk], q[t][1][bk], d[j][bk], 0, 0, 0);
              }
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
              for (int i = 0; i < 4; i++) {
                float sum = __builtin_fmaf(half_of(xk.s[j][i >> 1], i & 1), d[j][0][i], 0.0f);
#pragma unroll
                for (int bk = 1; bk < NB; bk++) sum = __builtin_fmaf(half_of(xk.s[j][2 * bk + (i >> 1)], i & 1), d[j][bk][i], sum);
                sc[t][4 * j + i] = sum;
              }
          }
        }
        codes(at + v_at, xv.c);
        if constexpr (NB == 8) {
          load_dwords<4>(at + v_at + 256, xv.c[0] + 4);
          load_dwords<4>(at + v_at + 256 + 8 * D, xv.c[1] + 4);
        }
        scales(at + vs_at, xv.s);
        // exponents of 2 against mref: -infinity where a token is not seen
        float e2[NT][8];
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
          for (int i = 0; i < 8; i++) e2[t][i] = __builtin_fmaf(sc[t][i], kcol[t], -mref[t]);
        // the largest exponent of a V scale, from above: of all bits together (exponents
        // to 15 have no bit that 15 has not; 15 where there are larger ones)
        const auto exponent = [](uint32_t o) { return min((int)(((o | (o >> 16)) >> 10) & 31), 15); };
        uint32_t ors = 0;
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
          for (int i = 0; i < 2 * NB; i++) ors |= xv.s[j][i];
        int exps[NT];
        uint32_t see[NT];  // bit i: the lane's token i is seen by its column
#pragma unroll
        for (int t = 0; t < NT; t++) {
          see[t] = 0xFF;
          exps[t] = exponent(ors);
        }
        if (edge) {
#pragma unroll
          for (int t = 0; t < NT; t++) {
            uint32_t m = 0, pairs[4], o = 0;
#pragma unroll
            for (int i = 0; i < 8; i++) {
              const int tok = tok0 + 16 * (i >> 2) + 4 * g + (i & 3);
              const bool ok = tok >= lo[t] && tok < hi[t] && !((lost >> (i >> 2)) & 1);
              m |= ok ? 1u << i : 0u;
              if (!ok) e2[t][i] = -INFINITY;
            }
            see[t] = m;
#pragma unroll
            for (int i = 0; i < 4; i++) {
              pairs[i] = ((m >> (2 * i)) & 1 ? 0xFFFFu : 0) | ((m >> (2 * i + 1)) & 1 ? 0xFFFF0000u : 0);
#pragma unroll
              for (int bk = 0; bk < NB; bk++) {
                // 0 * NaN of a token that is not seen: scales of no token of this column become 0
                if constexpr (NT == 1) xv.s[i >> 1][2 * bk + (i & 1)] &= pairs[i];
                o |= xv.s[i >> 1][2 * bk + (i & 1)] & pairs[i];
              }
            }
            exps[t] = exponent(o);
          }
        }
        // does a score pass what mref allows, or a scale of V what fs does?
        bool grow = false, passed[NT];
#pragma unroll
        for (int t = 0; t < NT; t++) {
          float m = e2[t][0];
#pragma unroll
          for (int i = 1; i < 8; i++) m = fmaxf(m, e2[t][i]);
          passed[t] = m > 14.0f;
          grow |= passed[t] || (TERMS == 2 && exps[t] > elim[t]);
        }
        if (__ballot(grow)) {
#pragma unroll
          for (int t = 0; t < NT; t++) {
            float m = -INFINITY;
#pragma unroll
            for (int i = 0; i < 8; i++)
              if ((see[t] >> i) & 1) m = fmaxf(m, sc[t][i] * kcol[t]);
            m = xor_max<32>(xor_max<16>(m));
            // A column that needs no change has none: it does not depend on its neighbours.  One that does
            // takes differences of rounded scores, which stay below 14 however large the scores are.
            const bool own = of_column(__ballot(passed[t]));
            const float now = own && m - mref[t] > 14.0f ? m - 10.0f : mref[t];
            const float keep = __builtin_amdgcn_exp2f(mref[t] - now);
            mref[t] = now;
            l[t] *= keep;
            float less = keep;
            if constexpr (TERMS == 2) {
              int e = max(exps[t], elim[t]);
              e = max(e, __shfl_xor(e, 16, 64));
              e = max(e, __shfl_xor(e, 32, 64));
              e |= e >> 1;
              e |= e >> 2;
              less = __builtin_amdgcn_ldexpf(keep, elim[t] - e);
              elim[t] = e;
              fs[t] = __builtin_amdgcn_ldexpf(1.0f, 15 - e);
            }
#pragma unroll
            for (int i = 0; i < 2 * NB; i++) acc[t][i] *= less;
#pragma unroll
            for (int i = 0; i < 8; i++)
              if (own) e2[t][i] = (see[t] >> i) & 1 ? sc[t][i] * kcol[t] - mref[t] : -INFINITY;
          }
        }
        // scales of 2 and more (finite), and what makes 2^-15 of them
        const auto large = [](uint32_t d) { return (d & 0x7FFFu) >= 0x4000u && (d & 0x7FFFu) < 0x7C00u; };
        constexpr uint32_t kLess = 15u << 10;
        const bool some_large = __ballot((ors & 0x40004000u) != 0) != 0;
        if (some_large) {
          asm volatile("");  // stays a branch
#pragma unroll
          for (int j = 0; j < 2; j++)
#pragma unroll
            for (int i = 0; i < 2 * NB; i++)
#pragma unroll
              for (int k = 0; k < 2; k++) xv.s[j][i] -= large(xv.s[j][i] >> (16 * k)) ? kLess << (16 * k) : 0u;
        }
#pragma unroll
        for (int t = 0; t < NT; t++) {
          float p[8];
#pragma unroll
          for (int i = 0; i < 8; i++) p[i] = __builtin_amdgcn_exp2f(e2[t][i]);
          h2 ph[2][2];
          if constexpr (ONCE) {
            l[t][0] += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
            if constexpr (TERMS == 2)
#pragma unroll
              for (int i = 0; i < 8; i++) p[i] *= fs[t];
          } else {
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
              for (int i = 0; i < 2; i++) ph[j][i] = h2{(_Float16)p[4 * j + 2 * i], (_Float16)p[4 * j + 2 * i + 1]};
            l[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pack8(ph[0][0], ph[0][1], ph[1][0], ph[1][1]), l[t], 0, 0, 0);
          }
#pragma unroll
          for (int bk = 0; bk < NB; bk++) {
            h8 pd[TERMS];
            if constexpr (ONCE) {
#pragma unroll
              for (int i = 0; i < 8; i++) {
                float y = p[i] * half_of(xv.s[i >> 2][2 * bk + ((i >> 1) & 1)], i & 1);
                if (NT > 1 && edge && !((see[t] >> i) & 1)) y = 0.0f;  // 0 * NaN of a token that is not seen
                // two terms: one product, not one for each term, of which the compiler would round
                // one to fp32 and then fp16 and the other to fp16 at once
                if constexpr (TERMS == 2) asm("" : "+v"(y));
                const _Float16 top = (_Float16)y;
                pd[0][i] = top;
                if constexpr (TERMS == 2) pd[1][i] = (_Float16)(y - (float)top);
              }
            } else {
              h2 y[2][2];
#pragma unroll
              for (int j = 0; j < 2; j++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                  y[j][i] = ph[j][i] * __builtin_bit_cast(h2, xv.s[j][2 * bk + i]);
                  if constexpr (NT > 1) {
                    const uint32_t m = see[t] >> (4 * j + 2 * i);
                    const uint32_t pair = (m & 1 ? 0xFFFFu : 0) | (m & 2 ? 0xFFFF0000u : 0);
                    if (edge) y[j][i] = __builtin_bit_cast(h2, __builtin_bit_cast(uint32_t, y[j][i]) & pair);
                  }
                }
              pd[0] = pack8(y[0][0], y[0][1], y[1][0], y[1][1]);
            }
#pragma unroll
            for (int hh = 0; hh < 2; hh++) {
              const int pr = (bk & 1) * 2 + hh, dw = (bk >> 1) * 2;
              const auto pair = [&](int j, int k) { return code_pair(magic, xv.c[j][dw + k], pr); };
              const h8 vq = pack8(pair(0, 0), pair(0, 1), pair(1, 0), pair(1, 1));
              f4& o = acc[t][2 * bk + hh];
              o = __builtin_amdgcn_mfma_f32_16x16x32_f16(vq, pd[0], o, 0, 0, 0);
              if constexpr (TERMS == 2) o = __builtin_amdgcn_mfma_f32_16x16x32_f16(vq, pd[1], o, 0, 0, 0);
            }
          }
          if (some_large) {  // the rest of their part; scales and codes come from the ring once more, as there are no registers for both
            asm volatile("" ::: "memory");
#pragma unroll
            for (int bk = 0; bk < NB; bk++) {
              h8 pd[TERMS];
#pragma unroll
              for (int i = 0; i < 8; i++) {
                const uint32_t s = *(const uint16_t*)(at + vs_at + (i >> 2) * D + 8 * bk + 2 * (i & 3));
                float y = ONCE ? p[i] : (float)ph[i >> 2][(i >> 1) & 1][i & 1];
                y = large(s) ? y * half_of(s - kLess, 0) : 0.0f;
                if constexpr (TERMS == 2) asm("" : "+v"(y));
                const _Float16 top = (_Float16)y;
                pd[0][i] = top;
                if constexpr (TERMS == 2) pd[1][i] = (_Float16)(y - (float)top);
              }
              const uint8_t* c = at + v_at + (bk < 4 ? 0 : 256) + ((bk >> 1) & 1) * 8;
#pragma unroll
              for (int hh = 0; hh < 2; hh++) {
                const int pr = (bk & 1) * 2 + hh;
                const auto pair = [&](int j, int k) { return code_pair(magic, *(const uint32_t*)(c + j * 8 * D + 4 * k), pr); };
                const h8 vq = pack8(pair(0, 0), pair(0, 1), pair(1, 0), pair(1, 1));
                f4 d = __builtin_amdgcn_mfma_f32_16x16x32_f16(vq, pd[0], f4{0, 0, 0, 0}, 0, 0, 0);
                if constexpr (TERMS == 2) d = __builtin_amdgcn_mfma_f32_16x16x32_f16(vq, pd[1], d, 0, 0, 0);
                acc[t][2 * bk + hh] += 32767.0f * d;
              }
              __builtin_amdgcn_sched_barrier(0);
            }
          }
        }
        __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the slot is free
      }
      wait_loads<0>();  // the next part's loads into the ring come behind these
    }

    // O on the scale of l
#pragma unroll
    for (int t = 0; t < NT; t++)
      if constexpr (TERMS == 2)
#pragma unroll
        for (int i = 0; i < 2 * NB; i++)
#pragma unroll
          for (int j = 0; j < 4; j++) acc[t][i][j] = __builtin_amdgcn_ldexpf(acc[t][i][j], elim[t] - 15);

    const int64_t slot = (begins ? 2 * (int64_t)w + 1 : 2 * (int64_t)w) * COLS;
#pragma unroll
    for (int t = 0; t < NT; t++) {
      const float sum = ONCE ? xor_add<32>(xor_add<16>(l[t][0])) : l[t][0];
      if (!valid[t]) continue;
      if (begins && ends) {
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        T* dst = (T*)a.out.p + qrow[t] * a.out.row + qhead[t] * a.out.head + 4 * g;
        const bool ovec = vec_rows(a.out, sizeof(T));
#pragma unroll
        for (int i = 0; i < 2 * NB; i++) {
          T o[4];
#pragma unroll
          for (int j = 0; j < 4; j++) o[j] = E::put(acc[t][i][j] * inv);
          if (ovec) {
            if constexpr (sizeof(T) == 4) *(u32x4*)(dst + 16 * i) = *(u32x4*)o;
            else *(u32x2*)(dst + 16 * i) = *(u32x2*)o;
          } else {
#pragma unroll
            for (int j = 0; j < 4; j++) dst[16 * i + j] = o[j];
          }
        }
      } else {
        const int64_t c = slot + t * 16 + col;
        if (g == 0) pc.ml[c] = float2{mref[t], sum};
        if (sum == 0.0f) continue;
#pragma unroll
        for (int i = 0; i < 2 * NB; i++) *(f4*)(pc.acc + c * D + 16 * i + 4 * g) = acc[t][i];
      }
    }
  }
}

// ---- attention of prompts ---------------------------------------------------------------
// Many columns, fp16 or bf16, head dim 128: the waves of a workgroup take 32 columns each of
// one sequence and kv head and share the expansion of its tiles.  They write the codes of the
// next 64 tokens into LDS as matrix operands: K as c - 8 (fp16), or with its scale (bf16,
// whose queries and results have 8 bits, K then 11); V with its scale, rounded to fp16, so that
// O += V^T P^T takes P as it is.  A wave of k_kv4_attn spends 150 of its 300 vector instructions a
// tile on the expansion; here it is a quarter of 200.  Parts, pieces and the merge are
// those of k_kv4_attn with a workgroup in the place of a wave.
//
// 512 rows of 32 heads at 4096 tokens (8 kv heads, bf16), and 77 at 77: 81 us, 15 for the merge (the whole call back to back
// 90; k_kv4_attn 107), a third of the matrix rate.  Waits bind it: matrix instructions are busy 16 % of the time, vector
// instructions 35 %.  A step of 64 tokens takes 3.3 us, of which matrix
// instructions are 0.9 and vector instructions 1.7; before its first one a part waits 10 us
// for its sequence, its pages, queries and codes, one after the other.  Four waves a workgroup, two of
// those a CU: 87 us.  One wave of a SIMD expanding while the other multiplies: 84.
//
// Scales of 2^13 and more would pass fp16's range times c - 8: those blocks are expanded with 2^-4 of their
// scale, and the missing 15 / 16 of their part are added by products of their own, so that scales beside them
// keep their bits.  A NaN scale of V is expanded as 0, which
// spares the columns that do not see its token, and written into O of those that do.
constexpr int kPromptStart = 8;  // what beginning an item costs, in tiles

template <int WAVES, class E>
__global__ void __launch_bounds__(64 * WAVES, 2)
    k_kv4_prompt(Kv4Attn a, const int32_t* __restrict__ ro, const int32_t* __restrict__ lens, const int32_t* __restrict__ table,
                 const uint8_t* __restrict__ base, Pieces pc, int workers, int least) {
  constexpr int D = 128, NB = 4, NT = 2, COLS = 32 * WAVES, SUB = WAVES / 4;  // SUB tiles at a time
  constexpr bool SCALED_K = std::is_same<E, BF16>::value;
  typedef Rec<D> R;
  typedef typename E::T T;
  const Magic magic;
  struct Tile {
    h8 k[2][NB][64], v[NB][2][64];
    u32x2 ks[2][4][NB];       // K scales of four tokens: half, token group, block (SCALED_K: where the half has large ones)
    u32x4 vs[2][4][NB / 2];   // V scales: half, token group, two blocks
    uint32_t about[4];        // what each of the four waves that expanded it found
  };
  enum { LARGE_K = 1, LARGE_V = 2, NOT_FINITE = 4, GONE = 8 };
  __shared__ Tile tiles[2][SUB];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
  const int w = blockIdx.x, group = a.n_q / a.c.n_kv, ps = a.c.page_size;
  const Lines L{ro, lens, a.rows, a.c.n_kv, group, a.window, COLS, (int)min((int64_t)a.pps * ps, (int64_t)0x7FFFFFC0), kPromptStart, false};
  Line line(L, a.batch, w, workers, least);
  if (w == 0 && wave == 0) *pc.n_items = line.items();

  const int64_t rec = kv4_record_bytes(D, ps);
  const uint32_t page_bytes = (uint32_t)(a.c.n_kv * rec);
  // a thread's part of a step: 8 bytes of codes of K and of V, of half j of tile `sub`
  const int sub = wave >> 2, j = (wave >> 1) & 1, r = threadIdx.x & 127;
  const int kg = r >> 5, ktok = (r >> 1) & 15, kb = (r & 1) * 2;  // K: eight dims of blocks kb, kb + 1
  const int vt = r >> 5, vc = (r >> 1) & 15, vp = r & 1;          // V: token group, column, block pair

  while (line.next()) {
    const Seq& s = line.s;
    const int h = line.h, c0 = line.ct * COLS, p0 = s.len - s.m, held = L.held(s.len);
    const bool begins = line.begins, ends = line.ends;
    if (begins && threadIdx.x == 0) pc.begun[line.item] = Begun{line.b, h, line.ct, w, line.pieces};
    const auto row_of = [&](int c) { return min(s.m - 1, c / group); };
    const int rf = row_of(c0), rl = row_of(c0 + COLS - 1);
    const int cw = c0 + wave * 16 * NT, wf = row_of(cw), wl = row_of(cw + 16 * NT - 1);  // the wave's rows
    // a column's row and head; found anew where they are needed, as keeping them costs registers of the loop
    struct Column {
      int row, head;
    };
    const auto column = [&](int t) {
      int cc = cw + t * 16 + col;
      asm("" : "+v"(cc));
      const int row = cc / group;
      return Column{row, h * group + (cc - row * group)};
    };
    const auto first_seen = [&](int row) { return a.window > 0 ? max(max(p0 + row + 1, 0) - a.window, 0) : 0; };
    const auto end_seen = [&](int row) { return min(max(p0 + row + 1, 0), held); };
    int hi[NT], lo[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) {
      const int row = column(t).row;
      hi[t] = row < s.m ? end_seen(row) : 0;
      lo[t] = first_seen(row);
    }
    const int t0 = max(s.lo + max(line.at - kPromptStart, 0), first_seen(rf) / kTile);
    const int t1 = min(s.lo + max(line.at + line.n - kPromptStart, 0), (end_seen(rl) + kTile - 1) / kTile);
    const bool any = cw < s.m * group;  // the wave has columns
    const int w_lo = first_seen(wf), w_hi = any ? end_seen(wl) : 0, w_lo_last = first_seen(wl), w_hi_first = end_seen(wf);

    f4 acc[NT][2 * NB], l[NT];
    float mref[NT], kcol[NT];
    h8 q[NT][NB];
#pragma unroll
    for (int t = 0; t < NT; t++) {
#pragma unroll
      for (int i = 0; i < 2 * NB; i++) acc[t][i] = f4{0, 0, 0, 0};
      l[t] = f4{0, 0, 0, 0};
      mref[t] = -FLT_MAX;
      kcol[t] = 0.0f;
    }
    if (t0 < t1) {
      const TablePtr rowp = (TablePtr)(table + (int64_t)line.b * a.pps);
      const int n_pages = (int)(((int64_t)held + ps - 1) / ps);
      const uint8_t* head = base + (int64_t)h * rec;
      // the wave's 16 tokens of a step: page and token in it, and the id, read a step ahead of its use
      int pg, off, id, id_off;
      bool id_there;
      const auto look = [&] {
        id = rowp[min(pg, n_pages - 1)];
        id_there = pg < n_pages;
        id_off = off;
        off += SUB * kTile;
        while (off >= ps) { off -= ps; pg++; }
      };
      const auto start = [&](int step) {
        const int tok = (step + sub) * kTile + 16 * j;
        pg = tok / ps;
        off = tok - pg * ps;
        look();
      };
      // a thread's part, loaded a step ahead of its expansion
      u32x2 kc, vcode;
      uint16_t ks[2];
      u32x4 vs;
      bool there = false;
      const auto fetch = [&] {
        there = id_there && (uint32_t)id < (uint32_t)a.c.pages;
        const uint32_t off0 = (uint32_t)id_off;
        const uint8_t* p = head + (uint64_t)(uint32_t)(there ? id : 0) * page_bytes;
        kc = *(const u32x2*)(p + (off0 * (D / 2) + r * 8));
        vcode = *(const u32x2*)(p + (R::vbase(ps) + off0 * (D / 2) + r * 8));
        const uint32_t so = off0 * (D / 16);
        ks[0] = *(const uint16_t*)(p + (R::ksbase(ps) + so + R::s(ktok >> 2, kb) + (ktok & 3) * 2));
        ks[1] = *(const uint16_t*)(p + (R::ksbase(ps) + so + R::s(ktok >> 2, kb + 1) + (ktok & 3) * 2));
        vs = *(const u32x4*)(p + (R::vsbase(ps) + so + R::s(vt, 2 * vp)));
        look();
      };
      // fp16 scales of 2^13 and more (finite), and what makes a sixteenth of them
      const auto large = [](uint32_t d) { return (d & 0x7FFFu) >= 0x7000u && (d & 0x7FFFu) < 0x7C00u; };
      constexpr uint32_t kSixteenth = 4u << 10;
      // its expansion into buffer i
      const auto expand = [&](int i, int step) {
        Tile& x = tiles[i][sub];
        const int tok = (step + sub) * kTile + 16 * j;  // of the wave's first
        uint16_t kd[2] = {ks[0], ks[1]};
        uint32_t vd[4] = {vs[0], vs[1], vs[2], vs[3]};
        if (!there || tok + 16 > held) {  // scales of no token are 0
#pragma unroll
          for (int n = 0; n < 2; n++) kd[n] = there && tok + ktok < held ? kd[n] : 0;
#pragma unroll
          for (int n = 0; n < 4; n++) {
            const int at = tok + 4 * vt + 2 * (n & 1);
            vd[n] &= there ? (at + 1 < held ? 0xFFFFFFFFu : at < held ? 0xFFFFu : 0u) : 0u;
          }
        }
        if (vc == 0) x.vs[j][vt][vp] = u32x4{vd[0], vd[1], vd[2], vd[3]};
        // the largest scale
        typedef uint16_t us2 __attribute__((ext_vector_type(2)));
        const auto abs2 = [](uint32_t v) { return __builtin_bit_cast(us2, v & 0x7FFF7FFFu); };
        us2 e = __builtin_elementwise_max(__builtin_elementwise_max(abs2(vd[0]), abs2(vd[1])), __builtin_elementwise_max(abs2(vd[2]), abs2(vd[3])));
        if constexpr (SCALED_K) e = __builtin_elementwise_max(e, abs2(kd[0] | (uint32_t)kd[1] << 16));
        uint32_t about = there ? 0 : GONE;
        if (__ballot(max(e[0], e[1]) >= 0x7000)) {  // 2^13 and more, or not finite: hardly ever
          asm volatile("");
          bool large_k = false, large_v = false, odd = false;
#pragma unroll
          for (int n = 0; n < 8; n++) {
            const uint32_t d = vd[n >> 1] >> (16 * (n & 1));
            odd |= (d & 0x7FFFu) >= 0x7C00u;
            if ((d & 0x7FFFu) >= 0x7C00u) vd[n >> 1] &= n & 1 ? 0xFFFFu : 0xFFFF0000u;
            if (large(d)) {
              large_v = true;
              vd[n >> 1] -= kSixteenth << (16 * (n & 1));
            }
          }
          if constexpr (SCALED_K)
#pragma unroll
            for (int n = 0; n < 2; n++) {
              if (kg == 0) ((uint16_t*)&x.ks[j][ktok >> 2][kb + n])[ktok & 3] = kd[n];
              if (large(kd[n])) {
                large_k = true;
                kd[n] -= kSixteenth;
              }
            }
          about |= (__ballot(large_k) ? LARGE_K : 0) | (__ballot(large_v) ? LARGE_V : 0) | (__ballot(odd) ? NOT_FINITE : 0);
        }
        if (lane == 0) x.about[wave & 3] = about;
#pragma unroll
        for (int n = 0; n < 2; n++) {
          h2 p[4];
#pragma unroll
          for (int k = 0; k < 4; k++) {
            p[k] = code_pair(magic, kc[n], k);
            if constexpr (SCALED_K) p[k] *= __builtin_bit_cast(h2, (uint32_t)kd[n] * 0x10001u);
          }
          x.k[j][kb + n][kg * 16 + ktok] = pack8(p[0], p[1], p[2], p[3]);
          if constexpr (!SCALED_K)
            if (kg == 0) ((uint16_t*)&x.ks[j][ktok >> 2][kb + n])[ktok & 3] = kd[n];
        }
#pragma unroll
        for (int n = 0; n < 4; n++) {  // block 2 vp + n / 2, its half n % 2
          const h2 y0 = code_pair(magic, vcode[0], n) * __builtin_bit_cast(h2, vd[2 * (n >> 1)]);
          const h2 y1 = code_pair(magic, vcode[1], n) * __builtin_bit_cast(h2, vd[2 * (n >> 1) + 1]);
          ((u32x2*)&x.v[2 * vp + (n >> 1)][n & 1][vt * 16 + vc])[j] = u32x2{__builtin_bit_cast(uint32_t, y0), __builtin_bit_cast(uint32_t, y1)};
        }
      };

      start(t0);
      fetch();
      const bool vec = vec_rows(a.q, sizeof(T));
#pragma unroll
      for (int t = 0; t < NT; t++) {
        float x[NB][8], big = 0.0f;
        const Column c = column(t);
#pragma unroll
        for (int bk = 0; bk < NB; bk++) {
          if (c.row < s.m) {
            const T* src = (const T*)a.q.p + (int64_t)(s.r0 + c.row) * a.q.row + (int64_t)c.head * a.q.head + bk * 32 + g * 8;
            if (vec) load8<E, true>(src, x[bk]); else load8<E, false>(src, x[bk]);
          } else {
#pragma unroll
            for (int i = 0; i < 8; i++) x[bk][i] = 0.0f;
          }
#pragma unroll
          for (int i = 0; i < 8; i++) big = fmaxf(big, fabsf(x[bk][i]));
        }
        big = xor_max<32>(xor_max<16>(big));
        const int e = min(__builtin_amdgcn_frexp_expf(big), kLargestPower);
        kcol[t] = __builtin_amdgcn_ldexpf(a.scale * 1.4426950408889634f, e);
#pragma unroll
        for (int bk = 0; bk < NB; bk++)
#pragma unroll
          for (int i = 0; i < 8; i++) q[t][bk][i] = (_Float16)__builtin_amdgcn_ldexpf(x[bk][i], -e);
      }
      const uint32_t one = 0x3C003C00u;
      const h8 ones = __builtin_bit_cast(h8, u32x4{one, one, one, one});

      const auto compute = [&](int buf, int step) {
#pragma unroll 1
        for (int i = 0; i < SUB; i++) {
          const Tile& x = tiles[buf][i];
          const int tok0 = (step + i) * kTile;
          if (step + i >= t1 || tok0 >= w_hi || tok0 + kTile <= w_lo) continue;
          const u32x4 about = *(const u32x4*)x.about;
          const uint32_t found = uniform(about[0] | about[1] | about[2] | about[3]);
          const uint32_t lost = uniform((about[0] & GONE) / GONE | (about[2] & GONE) / GONE << 1);
          const bool edge = lost || tok0 < w_lo_last || tok0 + kTile > w_hi_first;
          float sc[NT][8];
          {
            h8 kq[2][NB];
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
              for (int bk = 0; bk < NB; bk++) kq[i][bk] = x.k[i][bk][lane];
            if constexpr (SCALED_K) {
              f4 d[NT][2] = {};
#pragma unroll
              for (int bk = 0; bk < NB; bk++)
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                  for (int t = 0; t < NT; t++) d[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kq[i][bk], q[t][bk], d[t][i], 0, 0, 0);
#pragma unroll
              for (int t = 0; t < NT; t++)
#pragma unroll
                for (int i = 0; i < 8; i++) sc[t][i] = d[t][i >> 2][i & 3];
            } else {
#pragma unroll
              for (int t = 0; t < NT; t++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                  f4 d[NB];
#pragma unroll
                  for (int bk = 0; bk < NB; bk++) d[bk] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kq[i][bk], q[t][bk], f4{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
                  for (int n = 0; n < 4; n++) {
                    float sum = 0.0f;
#pragma unroll
                    for (int bk = 0; bk < NB; bk++) sum = __builtin_fmaf(half_of(x.ks[i][g][bk][n >> 1], n & 1), d[bk][n], sum);
                    sc[t][4 * i + n] = sum;
                  }
                }
            }
          }
          h8 v[NB][2];
#pragma unroll
          for (int bk = 0; bk < NB; bk++)
#pragma unroll
            for (int hh = 0; hh < 2; hh++) v[bk][hh] = x.v[bk][hh][lane];
          asm volatile("" ::: "memory");  // these loads run while the weights are computed
          if (SCALED_K && (found & LARGE_K)) {
            asm volatile("");
#pragma unroll
            for (int bk = 0; bk < NB; bk++)
#pragma unroll
              for (int i = 0; i < 2; i++) {
                if (!(uniform(about[2 * i]) & LARGE_K)) continue;  // no scales were left for the half
                const u32x2 ks = x.ks[i][g][bk];
#pragma unroll
                for (int t = 0; t < NT; t++) {
                  const f4 part = __builtin_amdgcn_mfma_f32_16x16x32_f16(x.k[i][bk][lane], q[t][bk], f4{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
                  for (int n = 0; n < 4; n++)
                    if (large(ks[n >> 1] >> (16 * (n & 1)))) sc[t][4 * i + n] = __builtin_fmaf(15.0f, part[n], sc[t][4 * i + n]);
                }
              }
          }
          uint32_t see[NT];
          float e2[NT][8];
          bool grow = false, passed[NT];
#pragma unroll
          for (int t = 0; t < NT; t++) {
            see[t] = 0xFF;
#pragma unroll
            for (int i = 0; i < 8; i++) e2[t][i] = __builtin_fmaf(sc[t][i], kcol[t], -mref[t]);
          }
          if (edge) {
#pragma unroll
            for (int t = 0; t < NT; t++) {
              see[t] = 0;
#pragma unroll
              for (int i = 0; i < 8; i++) {
                const int tok = tok0 + 16 * (i >> 2) + 4 * g + (i & 3);
                const bool ok = (tok >= lo[t]) & (tok < hi[t]) & !((lost >> (i >> 2)) & 1);
                see[t] |= ok ? 1u << i : 0u;
                if (!ok) e2[t][i] = -INFINITY;
              }
            }
          }
#pragma unroll
          for (int t = 0; t < NT; t++) {
            float m = e2[t][0];
#pragma unroll
            for (int i = 1; i < 8; i++) m = fmaxf(m, e2[t][i]);
            passed[t] = m > 14.0f;
            grow |= passed[t];
          }
          if (__ballot(grow)) {
#pragma unroll
            for (int t = 0; t < NT; t++) {
              asm volatile("" : "+v"(see[t]));  // its bits are looked at here only
              float m = -INFINITY;
#pragma unroll
              for (int i = 0; i < 8; i++)
                if ((see[t] >> i) & 1) m = fmaxf(m, sc[t][i] * kcol[t]);
              m = xor_max<32>(xor_max<16>(m));
              const bool own = of_column(__ballot(passed[t]));  // (as in k_kv4_attn)
              const float now = own && m - mref[t] > 14.0f ? m - 10.0f : mref[t];
              const float keep = __builtin_amdgcn_exp2f(mref[t] - now);
              mref[t] = now;
              l[t] *= keep;
#pragma unroll
              for (int i = 0; i < 2 * NB; i++) acc[t][i] *= keep;
#pragma unroll
              for (int i = 0; i < 8; i++)
                if (own) e2[t][i] = (see[t] >> i) & 1 ? sc[t][i] * kcol[t] - mref[t] : -INFINITY;
            }
          }
          h8 p[NT];
#pragma unroll
          for (int t = 0; t < NT; t++) {
#pragma unroll
            for (int i = 0; i < 8; i++) p[t][i] = (_Float16)__builtin_amdgcn_exp2f(e2[t][i]);
            l[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, p[t], l[t], 0, 0, 0);
          }
#pragma unroll
          for (int bk = 0; bk < NB; bk++)
#pragma unroll
            for (int hh = 0; hh < 2; hh++) {
#pragma unroll
              for (int t = 0; t < NT; t++) acc[t][2 * bk + hh] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[bk][hh], p[t], acc[t][2 * bk + hh], 0, 0, 0);
            }
          if (found & (LARGE_V | NOT_FINITE)) {
            asm volatile("");
            if (found & LARGE_V) {
#pragma unroll
              for (int bk = 0; bk < NB; bk++) {
                h8 pl[NT];
#pragma unroll
                for (int n = 0; n < 8; n++) {
                  const bool here = large(x.vs[n >> 2][g][bk >> 1][2 * (bk & 1) + ((n >> 1) & 1)] >> (16 * (n & 1)));
#pragma unroll
                  for (int t = 0; t < NT; t++) pl[t][n] = here ? p[t][n] : (_Float16)0.0f;
                }
#pragma unroll
                for (int hh = 0; hh < 2; hh++)
#pragma unroll
                  for (int t = 0; t < NT; t++)
                    acc[t][2 * bk + hh] += 15.0f * __builtin_amdgcn_mfma_f32_16x16x32_f16(x.v[bk][hh][lane], pl[t], f4{0, 0, 0, 0}, 0, 0, 0);
              }
            }
            if (found & NOT_FINITE) {  // scales of V that were left out, among the tokens that a column sees
#pragma unroll
              for (int t = 0; t < NT; t++) {
                uint32_t bad = 0;
#pragma unroll
                for (int n = 0; n < 8; n++)
#pragma unroll
                  for (int bk = 0; bk < NB; bk++) {
                    const uint32_t d = x.vs[n >> 2][g][bk >> 1][2 * (bk & 1) + ((n >> 1) & 1)] >> (16 * (n & 1));
                    if ((d & 0x7FFFu) >= 0x7C00u && ((see[t] >> n) & 1)) bad |= 1u << bk;
                  }
                bad |= __shfl_xor(bad, 16, 64);
                bad |= __shfl_xor(bad, 32, 64);
#pragma unroll
                for (int bk = 0; bk < NB; bk++)
                  if ((bad >> bk) & 1) {
                    const float n = __builtin_nanf("");
                    acc[t][2 * bk] = f4{n, n, n, n};
                    acc[t][2 * bk + 1] = f4{n, n, n, n};
                  }
              }
            }
          }
        }
      };
      int buf = 1;
      for (int step = t0 - SUB;;) {
        const int next = step + SUB;
        if (step >= t0) compute(buf, step);
        if (next >= t1) break;
        expand(buf ^ 1, next);
        fetch();  // the step after it, also where there is none
        __syncthreads();
        step = next;
        buf ^= 1;
      }
      __syncthreads();  // the buffers are the next part's
    }
    const int64_t slot = (begins ? 2 * (int64_t)w + 1 : 2 * (int64_t)w) * COLS;
#pragma unroll
    for (int t = 0; t < NT; t++) {
      const float sum = l[t][0];
      const Column at = column(t);
      if (at.row >= s.m) continue;
      if (begins && ends) {
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        T* dst = (T*)a.out.p + (int64_t)(s.r0 + at.row) * a.out.row + (int64_t)at.head * a.out.head + 4 * g;
        const bool ovec = vec_rows(a.out, sizeof(T));
#pragma unroll
        for (int i = 0; i < 2 * NB; i++) {
          T o[4];
#pragma unroll
          for (int k = 0; k < 4; k++) o[k] = E::put(acc[t][i][k] * inv);
          if (ovec) {
            *(u32x2*)(dst + 16 * i) = *(u32x2*)o;
          } else {
#pragma unroll
            for (int k = 0; k < 4; k++) dst[16 * i + k] = o[k];
          }
        }
      } else {
        const int64_t c = slot + wave * 16 * NT + t * 16 + col;
        if (g == 0) pc.ml[c] = float2{mref[t], sum};
        if (sum == 0.0f) continue;
#pragma unroll
        for (int i = 0; i < 2 * NB; i++) *(f4*)(pc.acc + c * D + 16 * i + 4 * g) = acc[t][i];
      }
    }
  }
}

// Joins the pieces of an item that several waves computed, in their order: a workgroup
// an item and `per` columns (more for every gridDim.y), its waves by column and by piece.  It waits for memory
// four times, 4 us at the least; 38 MB of a prompt's pieces take 15.
template <int D, class E>
__global__ void k_kv4_merge(Kv4Attn a, Lines L, Pieces pc, int per) {
  constexpr int V = D / 64;  // dims a lane
  typedef typename E::T T;
  __shared__ float part[16][D];
  __shared__ float pl[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int items = *pc.n_items;
  const Begun it = pc.begun[blockIdx.x];  // (of an item that is not: whatever is there)
  const int n = it.pieces;
  if ((int)blockIdx.x >= items || n == 0) return;
  const int64_t w0 = it.w;
  const int c0 = it.ct * L.cols;
  const int32_t* ro = L.ro + it.b;
  const int r0 = min(max(ro[0], 0), L.rows), m = max(min(max(ro[1], 0), L.rows) - r0, 0);
  const auto slot = [&](int i, int c) { return (i == 0 ? 2 * w0 + 1 : 2 * (w0 + i)) * L.cols + c; };
  const int share = (blockDim.x >> 6) / per, mine = wave % share;  // waves a column
  // The first columns' loads do not wait for the sequence's rows: behind the last one they are joined
  // and not written.
  const int at0 = blockIdx.y * per;
  for (int at = at0; at < L.cols && (at == at0 || (c0 + at) / L.group < m); at += gridDim.y * per) {  // the same for all waves
    const int c = at + wave / share;
    float acc[V] = {}, l = 0.0f;
    {
      float top = -INFINITY;
      for (int i0 = mine; i0 == mine || i0 < n; i0 += 8 * share) {
        float2 x[8];
        float v[8][V];
#pragma unroll
        for (int k = 0; k < 8; k++) {  // all loads before the first use
          const int64_t p = slot(min(i0 + k * share, n - 1), c);
          x[k] = pc.ml[p];
#pragma unroll
          for (int j = 0; j < V; j++) v[k][j] = pc.acc[p * D + lane * V + j];
        }
        if (i0 == mine) {
          for (int i = lane; i < n; i += 64) {
            const float2 y = pc.ml[slot(i, c)];
            if (y.y != 0.0f) top = fmaxf(top, y.x);
          }
          top = wave_max(top);
        }
#pragma unroll
        for (int k = 0; k < 8; k++) {
          const bool some = i0 + k * share < n && x[k].y != 0.0f;
          const float f = some ? __builtin_amdgcn_exp2f(x[k].x - top) : 0.0f;
          l = __builtin_fmaf(f, some ? x[k].y : 0.0f, l);
#pragma unroll
          for (int j = 0; j < V; j++) acc[j] = __builtin_fmaf(f, some ? v[k][j] : 0.0f, acc[j]);
        }
      }
    }
    if (share > 1) {
#pragma unroll
      for (int j = 0; j < V; j++) part[wave][lane * V + j] = acc[j];
      if (lane == 0) pl[wave] = l;
      __syncthreads();
      if (mine == 0)
        for (int k = 1; k < share; k++) {
#pragma unroll
          for (int j = 0; j < V; j++) acc[j] += part[wave + k][lane * V + j];
          l += pl[wave + k];
        }
      __syncthreads();
    }
    const int cc = c0 + c, r = cc / L.group;
    if (r < m && mine == 0) {
      T* dst = (T*)a.out.p + (int64_t)(r0 + r) * a.out.row + ((int64_t)it.h * L.group + cc % L.group) * a.out.head + lane * V;
#pragma unroll
      for (int j = 0; j < V; j++) dst[j] = E::put(l == 0.0f ? 0.0f : acc[j] / l);
    }
  }
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

namespace {

constexpr int kMergeWaves = 4096;
constexpr int kWhole = 4;        // tiles of an item that one wave does, without a merge
constexpr int kLeast = 2;        // tiles a wave takes at least
constexpr int kPromptLeast = 4;  // and a workgroup of k_kv4_prompt

// The parts of the workspace for `items` items, and `workers` workers of `cols` columns.
Pieces pieces_in(void* ws, int64_t items, int64_t workers, int cols) {
  char* p = (char*)ws;
  Pieces pc;
  pc.n_items = (int*)p;
  p += 256;
  pc.begun = (Begun*)p;
  p += align256(sizeof(Begun) * items);
  pc.ml = (float2*)p;
  p += align256(sizeof(float2) * 2 * workers * cols);
  pc.acc = (float*)p;
  return pc;
}

template <int D, class E>
hipError_t merge(hipStream_t st, const Kv4Attn& a, const Pieces& pc, int64_t items, int64_t workers, int cols, int cap, int start) {
  const int group = a.n_q / a.c.n_kv;
  const Lines L{a.row_offsets, a.lengths, a.rows, a.c.n_kv, group, a.window, cols, cap, start, false};
  // Waves a column: more where an item has many pieces, but not where there are columns enough
  // to fill the card (8 items of 256 columns in 16 pieces: 60 -> 35 us with their attention).
  const int64_t columns = std::min<int64_t>(cols, (int64_t)a.max_rows * group);
  const int pieces = (int)(workers / items);
  int share = pieces >= 16 ? 16 : pieces >= 4 ? 4 : 1;
  while (share > 1 && items * columns * share > kMergeWaves) share /= 4;
  const int per = share == 1 ? 4 : 1;
  hipLaunchKernelGGL((k_kv4_merge<D, E>), dim3((unsigned)items, (unsigned)((columns + per - 1) / per)), dim3(share == 16 ? 1024 : 256), 0,
                     st, a, L, pc, per);
  return hipGetLastError();
}

int attn_cap(const Kv4Attn& a) { return (int)std::min<int64_t>((int64_t)a.pps * a.c.page_size, 0x7FFFFFC0); }

template <int D, int NT, class E>
hipError_t attn_tiles(hipStream_t st, const Kv4Attn& a) {
  const int cols = 16 * NT;
  const int cap = attn_cap(a);
  const int64_t tiles = ((int64_t)cap + kTile - 1) / kTile;
  const int64_t items = attn_items(a.n_q, a.c.n_kv, a.batch, a.rows, cols);
  const bool whole = tiles <= kWhole;
  const int64_t most = attn_workers(D, NT, compute_units());
  const int64_t want = whole ? items : (items * (tiles + kStart) + kLeast - 1) / kLeast;
  const int workers = (int)((std::min(most, want) + 3) / 4 * 4), least = whole ? 1 : kLeast;
  const Pieces pc = pieces_in(a.ws, items, workers, cols);
  hipLaunchKernelGGL((k_kv4_attn<D, NT, attn_ring(D, NT), E>), dim3((unsigned)(workers / 4)), dim3(256), 0, st, a, a.row_offsets, a.lengths,
                     a.page_table, a.c.base, pc, workers, least, whole);
  const hipError_t e = hipGetLastError();
  return e != hipSuccess || whole ? e : merge<D, E>(st, a, pc, items, workers, cols, cap, kStart);
}

template <class E>
hipError_t attn_prompt(hipStream_t st, const Kv4Attn& a) {
  constexpr int cols = 32 * kPromptWaves;
  const int cap = attn_cap(a);
  const int64_t tiles = ((int64_t)cap + kTile - 1) / kTile;
  const int64_t items = attn_items(a.n_q, a.c.n_kv, a.batch, a.rows, cols);
  const int64_t most = prompt_workers(compute_units()), want = (items * (tiles + kPromptStart) + kPromptLeast - 1) / kPromptLeast;
  const int workers = (int)std::min(most, want);
  const Pieces pc = pieces_in(a.ws, items, workers, cols);
  hipLaunchKernelGGL((k_kv4_prompt<kPromptWaves, E>), dim3((unsigned)workers), dim3(64 * kPromptWaves), 0, st, a, a.row_offsets, a.lengths,
                     a.page_table, a.c.base, pc, workers, kPromptLeast);
  const hipError_t e = hipGetLastError();
  return e != hipSuccess ? e : merge<128, E>(st, a, pc, items, workers, cols, cap, kPromptStart);
}

// Columns enough for the waves of a workgroup to share a tile's expansion: 64 a sequence, and a table of more
// than 256 tokens.  32 heads, 8 kv heads, bf16, k_kv4_prompt against k_kv4_attn with NT = 2: one sequence of 64 rows
// at 16384 tokens 59 and 70 us, of 512 rows at 2048 61 and 71 (fp16 66 and 81); at the border the other form is the faster
// one for short tables, 16 sequences of 16 rows at 1024 45 and 41.  Not taken: 64 sequences of 8 rows (32 columns
// each) 92 and 62, one of 256 rows and tokens 31 and 27.  (Calls back to back, with their merges.)
bool many_columns(const Kv4Attn& a) {
  const int64_t group = a.n_q / a.c.n_kv;
  return a.max_rows * group >= kManyColumns && a.rows * group >= (int64_t)kManyColumns * a.batch && attn_cap(a) > 256;
}

template <class E>
hipError_t attn_type(hipStream_t st, const Kv4Attn& a) {
  const bool one = (int64_t)a.max_rows * (a.n_q / a.c.n_kv) <= kOneTile;
  if (a.c.hd == 64) return one ? attn_tiles<64, 1, E>(st, a) : attn_tiles<64, 2, E>(st, a);
  if constexpr (sizeof(typename E::T) == 2)
    if (a.c.hd == 128 && many_columns(a)) return attn_prompt<E>(st, a);
  if (a.c.hd == 128) return one ? attn_tiles<128, 1, E>(st, a) : attn_tiles<128, 2, E>(st, a);
  return attn_tiles<256, 1, E>(st, a);
}

}  // namespace

size_t kv4_attn_workspace(int n_q, int n_kv, int hd, int batch, int rows) {
  const int64_t columns = piece_columns(hd, (int64_t)rows * (n_q / n_kv), compute_units());
  return 256 + align256(sizeof(Begun) * attn_items(n_q, n_kv, batch, rows, 16)) + align256(sizeof(float2) * columns) + sizeof(float) * columns * hd;
}

hipError_t launch_kv4_attn(hipStream_t st, int dtype, const Kv4Attn& a) {
  if (a.rows == 0 || a.batch == 0) return hipSuccess;
  if (dtype == RSTR_F32) return attn_type<F32>(st, a);
  if (dtype == RSTR_F16) return attn_type<F16>(st, a);
  return attn_type<BF16>(st, a);
}

}  // namespace rstr
