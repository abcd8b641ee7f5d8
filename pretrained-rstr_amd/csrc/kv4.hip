// kv4.hip -- the 4-bit paged K/V cache (format: kv4.h): quantising append,
// dequantising read and attention over it.
#include <hip/hip_runtime.h>

#include <algorithm>

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

__host__ __device__ inline bool vec_rows(const Rows& r, int size) {
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
// begin 2^24 below the largest.  Scales of V of 2 and more are brought below 2 by a
// power of two that follows the largest one seen (and with two terms, small
// ones are brought up).
//
// The tiles of all (sequence, kv head, column tile) items form one line of units
// that is cut into equal parts, one a wave: the load is even whatever the
// lengths are.  A wave writes the output of an item that lies in its part as a
// whole; else (O, mref, l) of its piece, and k_kv4_merge joins the pieces in
// order.
constexpr int kTile = 32;

template <class E> struct Terms { static constexpr int n = 1; };
template <> struct Terms<F32> { static constexpr int n = 2; };

// The sequences of a call, as every wave sees them.
struct Lines {
  const int32_t *ro, *lens;
  int rows, n_kv, group, window, cols;  // cols: of a column tile
  int64_t cap;                          // tokens that a page table row can hold
  bool whole;                           // one unit an item
};
struct Seq {
  int r0, m, len, lo, tiles, nct;
  int64_t units;
};
__device__ __forceinline__ Seq sequence(const Lines& L, int b) {
  Seq s;
  s.r0 = min(max(L.ro[b], 0), L.rows);
  s.m = max(min(max(L.ro[b + 1], 0), L.rows) - s.r0, 0);
  s.len = (int)min((int64_t)max(L.lens[b], 0), L.cap);
  const int64_t lo = L.window > 0 ? (int64_t)s.len - s.m + 1 - L.window : 0;
  s.lo = lo > 0 ? (int)lo / kTile : 0;  // first tile
  s.tiles = max((int)(((int64_t)s.len + kTile - 1) / kTile) - s.lo, 0);
  s.nct = (int)(((int64_t)s.m * L.group + L.cols - 1) / L.cols);
  s.units = (int64_t)L.n_kv * s.nct * (L.whole ? 1 : s.tiles);
  return s;
}

__device__ __forceinline__ int64_t shfl64(int64_t v, int lane) { return __shfl((long long)v, lane, 64); }
__device__ __forceinline__ int64_t wave_sum_i64(int64_t v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v += __shfl_xor((long long)v, d, 64);
  return v;
}
__device__ __forceinline__ int64_t wave_scan_i64(int64_t v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t o = __shfl_up((long long)v, d, 64);
    if (lane >= d) v += o;
  }
  return v;
}
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uniform64(int64_t v) {
  return (int64_t)((uint64_t)(uint32_t)uniform((int)(v >> 32)) << 32 | (uint32_t)uniform((int)v));
}

// Units a wave takes, of `total` over `workers` waves.
__device__ __forceinline__ int64_t part_of(int64_t total, int workers, int least) {
  const int64_t n = (total + workers - 1) / workers;
  return n > least ? n : least;
}

// Pieces of items that several waves share: two a wave (the end of an item
// that an earlier wave began, the beginning of one that later waves end).
struct Pieces {
  float2* ml;   // [2 * workers][cols] (mref, l)
  float* acc;   // [2 * workers][cols][D]
};

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

// Pair i of a dword's eight codes, minus 8, as two fp16.
__device__ __forceinline__ h2 code_pair(uint32_t w, int i) {
  const uint32_t x = i < 2 ? w : w >> 8;
  if (i & 1) {
    const h2 bias = {(_Float16)-72.0f, (_Float16)-72.0f};
    return __builtin_bit_cast(h2, (x & 0x00F000F0u) | 0x54005400u) + bias;
  }
  const h2 bias = {(_Float16)-1032.0f, (_Float16)-1032.0f};
  return __builtin_bit_cast(h2, (x & 0x000F000Fu) | 0x64006400u) + bias;
}
__device__ __forceinline__ h8 pack8(h2 a, h2 b, h2 c, h2 d) {
  return h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ __forceinline__ float half_of(uint32_t w, int i) { return (float)__builtin_bit_cast(h2, w)[i]; }

template <int D>
struct TileRegs {
  static constexpr int NB = D / 32;
  uint32_t k[2][NB], v[2][NB], ks[2][2 * NB], vs[2][2 * NB];
};

// A wave's walk over the 16-token halves of consecutive tiles: page ids of 64
// table entries at a time, one a lane, and the offset inside the current page.
struct Walk {
  const int32_t* row;
  int pages, n_pages, ps;  // of the cache; of the sequence; tokens a page
  int ids, first, pg, off;
  __device__ __forceinline__ void fill() {
    const int i = first + (threadIdx.x & 63);
    ids = i < n_pages ? row[i] : -1;
    if (ids < 0 || ids >= pages) ids = -1;
  }
  __device__ __forceinline__ void start(int token) {
    pg = token / ps;
    off = token - pg * ps;
    first = pg;
    fill();
  }
  __device__ __forceinline__ int page() const { return __builtin_amdgcn_readlane(ids, pg - first); }
  __device__ __forceinline__ void next() {
    off += 16;
    if (off == ps) {
      off = 0;
      pg++;
      if (pg - first == 64) {
        first = pg;
        fill();
      }
    }
  }
};

template <int D, int NT, class E>
__global__ void __launch_bounds__(256, D == 256 ? 1 : 2)
    k_kv4_attn(Kv4Attn a, const int32_t* __restrict__ ro, const int32_t* __restrict__ lens, const int32_t* __restrict__ table,
               const uint8_t* __restrict__ base, Pieces pc, int64_t* __restrict__ firsts, int workers, int least, bool whole) {
  typedef Rec<D> R;
  typedef typename E::T T;
  constexpr int NB = D / 32, COLS = 16 * NT, TERMS = Terms<E>::n;
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int w = uniform(blockIdx.x * 4 + (threadIdx.x >> 6));
  const int group = a.n_q / a.c.n_kv, ps = a.c.page_size;
  const Lines L{ro, lens, a.rows, a.c.n_kv, group, a.window, COLS, min((int64_t)a.pps * ps, (int64_t)0x7FFFFFC0), whole};

  if (w >= workers) {  // one wave more than workers: the sequences' first units, for the merge
    if (w > workers || whole) return;
    int64_t run = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
      const int64_t n = b0 + lane < a.batch ? sequence(L, b0 + lane).units : 0;
      const int64_t in = wave_scan_i64(n);
      if (b0 + lane < a.batch) firsts[b0 + lane] = run + in - n;
      run += shfl64(in, 63);
    }
    if (lane == 0) firsts[a.batch] = run;
    return;
  }
  int64_t mine = 0;
  for (int b = lane; b < a.batch; b += 64) mine += sequence(L, b).units;
  const int64_t total = uniform64(wave_sum_i64(mine));
  const int64_t part = part_of(total, workers, least);
  int64_t u = (int64_t)w * part;
  const int64_t u_end = min(u + part, total);
  if (u >= u_end) return;
  int b = 0;            // the sequence that unit u lies in, and its first unit
  int64_t first = 0;
  for (int64_t run = 0;; b += 64) {
    const int64_t n = b + lane < a.batch ? sequence(L, b + lane).units : 0;
    const int64_t in = wave_scan_i64(n);
    const uint64_t over = __ballot(run + in > u);
    if (over) {
      const int f = __ffsll((unsigned long long)over) - 1;
      first = uniform64(run + shfl64(in - n, f));
      b = uniform(b + f);
      break;
    }
    run += shfl64(in, 63);
  }

  const int64_t rec = kv4_record_bytes(D, ps);
  const int kl = R::k(col, 0, g), vl = R::vbase(ps) + R::v(g, 0, col), sl = R::s(g, 0);
  const int ksb = R::ksbase(ps) + sl, vsb = R::vsbase(ps) + sl;

  while (u < u_end) {
    const Seq s = sequence(L, b);
    if (u >= first + s.units) {  // behind b: the next sequence that has units
      first += s.units;
      b++;
      for (;; b += 64) {
        const uint64_t some = __ballot(b + lane < a.batch && sequence(L, b + lane).units > 0);
        if (some) {
          b = uniform(b + __ffsll((unsigned long long)some) - 1);
          break;
        }
      }
      continue;
    }
    const int64_t rel = u - first;
    const int per_item = whole ? 1 : s.tiles;
    const int64_t item = rel / per_item;
    const int at = (int)(rel - item * per_item);
    const int h = (int)(item / s.nct), ct = (int)(item - (int64_t)h * s.nct);
    const int n = (int)min((int64_t)(per_item - at), u_end - u);
    const bool begins = at == 0, ends = at + n == per_item;
    u += n;

    // the columns' rows and what they see
    const int c0 = ct * COLS, p0 = s.len - s.m;
    const int rf = c0 / group, rl = min(s.m - 1, (c0 + COLS - 1) / group);
    int hi[NT], lo[NT];
    int64_t qrow[NT], qhead[NT];
    bool valid[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) {
      const int cc = c0 + t * 16 + col, r = cc / group;
      valid[t] = r < s.m;
      hi[t] = valid[t] ? max(p0 + r + 1, 0) : 0;
      lo[t] = a.window > 0 ? max(p0 + r + 1 - a.window, 0) : 0;
      qrow[t] = s.r0 + r;
      qhead[t] = (int64_t)h * group + (cc - r * group);
    }
    const int hi_last = max(p0 + rl + 1, 0), hi_first = max(p0 + rf + 1, 0);
    const int lo_first = a.window > 0 ? max(p0 + rf + 1 - a.window, 0) : 0, lo_last = a.window > 0 ? max(p0 + rl + 1 - a.window, 0) : 0;
    int t0 = s.lo + (whole ? 0 : at), t1 = whole ? s.lo + s.tiles : t0 + n;
    t0 = max(t0, lo_first / kTile);
    t1 = min(t1, (hi_last + kTile - 1) / kTile);

    f4 acc[NT][2 * NB];
    float mref[NT], l[NT], kcol[NT], fs[NT];
    int elim[NT];         // exponents of the V scales seen so far are no larger; fs = 2^(15 - elim)
    bool scaled = false;  // some column's fs is below 1
    h8 q[NT][TERMS][NB];
#pragma unroll
    for (int t = 0; t < NT; t++) {
#pragma unroll
      for (int i = 0; i < 2 * NB; i++) acc[t][i] = f4{0, 0, 0, 0};
      mref[t] = -1e30f;
      l[t] = 0.0f;
      elim[t] = TERMS == 1 ? 15 : 0;
      fs[t] = __builtin_amdgcn_ldexpf(1.0f, 15 - elim[t]);
    }
    if (t0 < t1) {
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
        const int e = __builtin_amdgcn_frexp_expf(big);
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

      Walk walk;
      walk.row = table + (int64_t)b * a.pps;
      walk.pages = a.c.pages;
      walk.n_pages = (int)(((int64_t)s.len + ps - 1) / ps);
      walk.ps = ps;
      walk.start(t0 * kTile);
      int gone = 0;  // halves of the tile just loaded whose page is not there (bits)
      const auto load = [&](TileRegs<D>& x) {
        gone = 0;
#pragma unroll
        for (int j = 0; j < 2; j++) {
          int pg = walk.page();
          if (pg < 0) { gone |= 1 << j; pg = 0; }
          const uint8_t* r = base + ((int64_t)pg * a.c.n_kv + h) * rec;
          const int code = walk.off * (D / 2), scl = walk.off * (D / 16);
          if constexpr (NB == 8) {
            load_dwords<4>(r + (code + kl), x.k[j]);
            load_dwords<4>(r + (code + kl + 16 * R::BQ), x.k[j] + 4);
            load_dwords<4>(r + (code + vl), x.v[j]);
            load_dwords<4>(r + (code + vl + 128 * R::BP), x.v[j] + 4);
          } else {
            load_dwords<NB>(r + (code + kl), x.k[j]);
            load_dwords<NB>(r + (code + vl), x.v[j]);
          }
          load_dwords<2 * NB>(r + (scl + ksb), x.ks[j]);
          load_dwords<2 * NB>(r + (scl + vsb), x.vs[j]);
          walk.next();
        }
      };

      const auto compute = [&](const TileRegs<D>& x, int tile, int lost) {
        const int tok0 = tile * kTile;
        const bool edge = lost || tok0 < lo_last || tok0 + kTile > hi_first;
        h8 kq[2][NB];
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
          for (int bk = 0; bk < NB; bk++)
            kq[j][bk] = pack8(code_pair(x.k[j][bk], 0), code_pair(x.k[j][bk], 1), code_pair(x.k[j][bk], 2), code_pair(x.k[j][bk], 3));
        float sc[NT][8];
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
          for (int j = 0; j < 2; j++) {
            f4 sum = {0, 0, 0, 0};
#pragma unroll
            for (int bk = 0; bk < NB; bk++) {
              const f4 zero = {0, 0, 0, 0};
              f4 d = __builtin_amdgcn_mfma_f32_16x16x32_f16(kq[j][bk], q[t][0][bk], zero, 0, 0, 0);
              if constexpr (TERMS == 2) d = __builtin_amdgcn_mfma_f32_16x16x32_f16(kq[j][bk], q[t][1][bk], d, 0, 0, 0);
#pragma unroll
              for (int i = 0; i < 4; i++) sum[i] = __builtin_fmaf(half_of(x.ks[j][2 * bk + (i >> 1)], i & 1), d[i], sum[i]);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) sc[t][4 * j + i] = sum[i] * kcol[t];
          }
        uint32_t see[NT];  // bit 4j + i: token 16j + 4g + i of the tile is seen
#pragma unroll
        for (int t = 0; t < NT; t++) {
          see[t] = 0xFF;
          if (edge) {
            see[t] = 0;
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
              for (int i = 0; i < 4; i++) {
                const int tok = tok0 + 16 * j + 4 * g + i;
                const bool ok = tok >= lo[t] && tok < hi[t] && !((lost >> j) & 1);
                if (ok) see[t] |= 1u << (4 * j + i);
                else sc[t][4 * j + i] = -INFINITY;
              }
          }
        }
        // does a score pass what mref allows, or a scale of V what 2^a allows?
        bool grow = false;
#pragma unroll
        for (int t = 0; t < NT; t++) {
          float m = sc[t][0];
#pragma unroll
          for (int i = 1; i < 8; i++) m = fmaxf(m, sc[t][i]);
          grow |= m - mref[t] > 14.0f;
        }
        uint32_t ors[2][2];  // of the bits of the scales, by half and token pair
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
          for (int i = 0; i < 2; i++) {
            ors[j][i] = x.vs[j][i];
#pragma unroll
            for (int bk = 1; bk < NB; bk++) ors[j][i] |= x.vs[j][2 * bk + i];
          }
        // the largest exponent, from above: of all bits together (exponents to 15 have no
        // bit that 15 has not), and exactly where that is more than 15
        int exps[NT];
        const uint32_t o = ors[0][0] | ors[0][1] | ors[1][0] | ors[1][1];
        const int all = (int)(((o | (o >> 16)) >> 10) & 31);
        const bool large = __ballot(all > 15) != 0;
#pragma unroll
        for (int t = 0; t < NT; t++) {
          exps[t] = all;
          if (edge) {
            uint32_t k = 0;
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
              for (int i = 0; i < 4; i++)
                if ((see[t] >> (4 * j + i)) & 1) k |= ors[j][i >> 1] >> (16 * (i & 1));
            exps[t] = (int)((k >> 10) & 31);
          }
          if (large) {
            int e = 0;
#pragma unroll
            for (int i = 0; i < 8; i++)
#pragma unroll
              for (int bk = 0; bk < NB; bk++) {
                const int k = (int)((x.vs[i >> 2][2 * bk + ((i >> 1) & 1)] >> (16 * (i & 1) + 10)) & 31);
                if (((see[t] >> i) & 1) && k < 31) e = max(e, k);
              }
            exps[t] = e;
          }
          grow |= exps[t] > elim[t];
        }
        if (__ballot(grow)) {
          bool big = false;
#pragma unroll
          for (int t = 0; t < NT; t++) {
            float m = sc[t][0];
#pragma unroll
            for (int i = 1; i < 8; i++) m = fmaxf(m, sc[t][i]);
            m = xor_max<32>(xor_max<16>(m));
            int e = max(exps[t], elim[t]);
            e = max(e, __shfl_xor(e, 16, 64));
            e = max(e, __shfl_xor(e, 32, 64));
            if (e <= 15) { e |= e >> 1; e |= e >> 2; }
            const float now = fmaxf(mref[t], m - 10.0f);
            const float keep = __builtin_amdgcn_exp2f(mref[t] - now);
            mref[t] = now;
            l[t] *= keep;
            const float less = __builtin_amdgcn_ldexpf(keep, elim[t] - e);
            elim[t] = e;
            fs[t] = __builtin_amdgcn_ldexpf(1.0f, 15 - e);
            big |= e > 15;
#pragma unroll
            for (int i = 0; i < 2 * NB; i++) acc[t][i] *= less;
          }
          scaled = __ballot(big) != 0;
        }
#pragma unroll
        for (int t = 0; t < NT; t++) {
          float p[8];
#pragma unroll
          for (int i = 0; i < 8; i++) {
            p[i] = __builtin_amdgcn_exp2f(sc[t][i] - mref[t]);
            l[t] += p[i];
          }
          h2 ph[2][2];
          if constexpr (TERMS == 1)
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
              for (int i = 0; i < 2; i++) ph[j][i] = h2{(_Float16)p[4 * j + 2 * i], (_Float16)p[4 * j + 2 * i + 1]};
#pragma unroll
          for (int bk = 0; bk < NB; bk++) {
            h8 pd[TERMS];
            if constexpr (TERMS == 1) {
              h2 y[2][2];
#pragma unroll
              for (int j = 0; j < 2; j++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                  h2 d = __builtin_bit_cast(h2, x.vs[j][2 * bk + i]);
                  if (scaled) d *= h2{(_Float16)fs[t], (_Float16)fs[t]};
                  y[j][i] = ph[j][i] * d;
                  if (edge) {  // 0 * NaN of a token that is not seen
                    const uint32_t keep = ((see[t] >> (4 * j + 2 * i)) & 1 ? 0xFFFFu : 0) | ((see[t] >> (4 * j + 2 * i + 1)) & 1 ? 0xFFFF0000u : 0);
                    y[j][i] = __builtin_bit_cast(h2, __builtin_bit_cast(uint32_t, y[j][i]) & keep);
                  }
                }
              pd[0] = pack8(y[0][0], y[0][1], y[1][0], y[1][1]);
            } else {
#pragma unroll
              for (int i = 0; i < 8; i++) {
                float y = p[i] * fs[t] * half_of(x.vs[i >> 2][2 * bk + ((i >> 1) & 1)], i & 1);
                if (edge && !((see[t] >> i) & 1)) y = 0.0f;
                const _Float16 top = (_Float16)y;
                pd[0][i] = top;
                pd[1][i] = (_Float16)(y - (float)top);
              }
            }
#pragma unroll
            for (int hh = 0; hh < 2; hh++) {
              const int pr = (bk & 1) * 2 + hh, dw = (bk >> 1) * 2;
              const h8 vq = pack8(code_pair(x.v[0][dw], pr), code_pair(x.v[0][dw + 1], pr), code_pair(x.v[1][dw], pr), code_pair(x.v[1][dw + 1], pr));
              f4& o = acc[t][2 * bk + hh];
              o = __builtin_amdgcn_mfma_f32_16x16x32_f16(vq, pd[0], o, 0, 0, 0);
              if constexpr (TERMS == 2) o = __builtin_amdgcn_mfma_f32_16x16x32_f16(vq, pd[1], o, 0, 0, 0);
            }
          }
        }
      };

      TileRegs<D> x, y;
      load(x);
      int lost = gone;
      for (int tile = t0;;) {
        int next = 0;
        if (tile + 1 < t1) { load(y); next = gone; }
        compute(x, tile, lost);
        if (++tile >= t1) break;
        if (tile + 1 < t1) { load(x); lost = gone; }
        compute(y, tile, next);
        if (++tile >= t1) break;
      }
    }

    // O on the scale of l
#pragma unroll
    for (int t = 0; t < NT; t++)
      if (TERMS == 2 || scaled)
#pragma unroll
        for (int i = 0; i < 2 * NB; i++)
#pragma unroll
          for (int j = 0; j < 4; j++) acc[t][i][j] = __builtin_amdgcn_ldexpf(acc[t][i][j], elim[t] - 15);

    const int64_t slot = (begins ? 2 * (int64_t)w + 1 : 2 * (int64_t)w) * COLS;
#pragma unroll
    for (int t = 0; t < NT; t++) {
      const float sum = xor_add<32>(xor_add<16>(l[t]));
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

// One workgroup per (query row, head): the pieces of an item that several waves
// computed, joined in their order (a wave takes every n-th piece); zeros for a
// row whose item has no tiles.
template <int D, class E>
__global__ void k_kv4_merge(Kv4Attn a, Lines L, Pieces pc, const int64_t* __restrict__ firsts, int workers, int least) {
  constexpr int V = D / 64;  // dims a lane
  __shared__ float part[16][D];
  __shared__ float pl[16];
  const int row = blockIdx.x, hq = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  int lo = 0, hi = a.batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (L.ro[mid] <= row) lo = mid; else hi = mid;
  }
  const int b = lo;
  const Seq s = sequence(L, b);
  if (row < s.r0 || row >= s.r0 + s.m) return;
  typename E::T* dst = (typename E::T*)a.out.p + (int64_t)row * a.out.row + (int64_t)hq * a.out.head;
  if (s.tiles == 0) {
    for (int i = threadIdx.x; i < D; i += blockDim.x) dst[i] = E::put(0.0f);
    return;
  }
  const int h = hq / L.group, c = (row - s.r0) * L.group + hq % L.group, ct = c / L.cols;
  const int64_t part_units = part_of(firsts[a.batch], workers, least);
  const int64_t u0 = firsts[b] + ((int64_t)h * s.nct + ct) * s.tiles, u1 = u0 + s.tiles - 1;
  const int64_t w0 = u0 / part_units, w1 = u1 / part_units;
  if (w0 == w1) return;  // written as a whole
  const int n = (int)(w1 - w0 + 1), cc = c % L.cols;
  const auto slot = [&](int i) { return (i == 0 ? 2 * w0 + 1 : 2 * (w0 + i)) * L.cols + cc; };
  float m = -INFINITY;
  for (int i = lane; i < n; i += 64) {
    const float2 x = pc.ml[slot(i)];
    if (x.y != 0.0f) m = fmaxf(m, x.x);
  }
  m = wave_max(m);
  float acc[V] = {}, l = 0.0f;
  for (int i = wave; i < n; i += waves) {
    const int64_t k = slot(i);
    const float2 x = pc.ml[k];
    if (x.y == 0.0f) continue;
    const float f = __builtin_amdgcn_exp2f(x.x - m);
    l = __builtin_fmaf(f, x.y, l);
#pragma unroll
    for (int j = 0; j < V; j++) acc[j] = __builtin_fmaf(f, pc.acc[k * D + lane * V + j], acc[j]);
  }
#pragma unroll
  for (int j = 0; j < V; j++) part[wave][lane * V + j] = acc[j];
  if (lane == 0) pl[wave] = l;
  __syncthreads();
  for (int i = threadIdx.x; i < D; i += blockDim.x) {
    float o = 0.0f, sum = 0.0f;
    for (int k = 0; k < waves; k++) {
      o += part[k][i];
      sum += pl[k];
    }
    dst[i] = E::put(sum == 0.0f ? 0.0f : o / sum);
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

int compute_units() {
  static int n[64] = {};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  if (n[dev] == 0 && (hipDeviceGetAttribute(&n[dev], hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n[dev] <= 0)) n[dev] = 256;
  return n[dev];
}

constexpr int kMaxWaves = 2;  // a SIMD, of the attention kernel's
constexpr int kLeast = 4;     // tiles a wave takes at least

inline size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

// Workspace: the sequences' first units, then the pieces of up to `workers` waves.
size_t attn_bytes(int batch, int64_t workers, int cols, int hd) {
  return align256(sizeof(int64_t) * ((size_t)batch + 1)) + align256(sizeof(float2) * 2 * workers * cols) +
         sizeof(float) * 2 * workers * cols * hd;
}

template <int D, int NT, class E>
hipError_t attn_tiles(hipStream_t st, const Kv4Attn& a) {
  const int cols = 16 * NT, group = a.n_q / a.c.n_kv;
  const int64_t cap = std::min<int64_t>((int64_t)a.pps * a.c.page_size, 0x7FFFFFC0);
  const int64_t items = a.c.n_kv * ((int64_t)a.rows * group / cols + std::min(a.batch, a.rows));  // at most
  const int64_t tiles = (cap + kTile - 1) / kTile;
  const bool whole = tiles <= kLeast;
  const int64_t most = (int64_t)compute_units() * 4 * kMaxWaves;
  const int64_t want = whole ? items : (items * tiles + kLeast - 1) / kLeast;
  const int workers = (int)((std::min(most, want) + 3) / 4 * 4), least = whole ? 1 : kLeast;
  char* ws = (char*)a.ws;
  int64_t* firsts = (int64_t*)ws;
  ws += align256(sizeof(int64_t) * ((size_t)a.batch + 1));
  Pieces pc;
  pc.ml = (float2*)ws;
  ws += align256(sizeof(float2) * 2 * workers * cols);
  pc.acc = (float*)ws;
  hipLaunchKernelGGL((k_kv4_attn<D, NT, E>), dim3((unsigned)(workers / 4 + (whole ? 0 : 1))), dim3(256), 0, st, a, a.row_offsets, a.lengths,
                     a.page_table, a.c.base, pc, firsts, workers, least, whole);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || whole) return e;
  const Lines L{a.row_offsets, a.lengths, a.rows, a.c.n_kv, group, a.window, cols, cap, false};
  const int64_t heads = (int64_t)a.rows * a.n_q;
  const int threads = heads <= 1024 ? 1024 : 256;  // few rows have many pieces each
  hipLaunchKernelGGL((k_kv4_merge<D, E>), dim3((unsigned)a.rows, (unsigned)a.n_q), dim3(threads), 0, st, a, L, pc, firsts, workers, least);
  return hipGetLastError();
}

template <class E>
hipError_t attn_type(hipStream_t st, const Kv4Attn& a) {
  const bool one = (int64_t)a.max_rows * (a.n_q / a.c.n_kv) <= 16;
  if (a.c.hd == 64) return one ? attn_tiles<64, 1, E>(st, a) : attn_tiles<64, 2, E>(st, a);
  if (a.c.hd == 128) return one ? attn_tiles<128, 1, E>(st, a) : attn_tiles<128, 2, E>(st, a);
  return attn_tiles<256, 1, E>(st, a);
}

}  // namespace

size_t kv4_attn_workspace(int n_q, int n_kv, int hd, int batch, int rows) {
  (void)n_q;
  (void)n_kv;
  (void)rows;
  return attn_bytes(batch, (int64_t)compute_units() * 4 * kMaxWaves, hd == 256 ? 16 : 32, hd);
}

hipError_t launch_kv4_attn(hipStream_t st, int dtype, const Kv4Attn& a) {
  if (a.rows == 0 || a.batch == 0) return hipSuccess;
  if (dtype == RSTR_F32) return attn_type<F32>(st, a);
  if (dtype == RSTR_F16) return attn_type<F16>(st, a);
  return attn_type<BF16>(st, a);
}

}  // namespace rstr
