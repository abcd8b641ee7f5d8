// pool_rows.hip -- rows of the fp16 page pool: appends with norms of heads and the position rotation on the
// way, the bounds of blocks of keys, and the blocks that a query's scores against these bounds select.
#include <hip/hip_runtime.h>

#include "../../include/rstr_hip.h"
#include "attn_line.h"
#include "device_math.h"
#include "pool_line.h"
#include "pool_ops.h"

namespace rstr {

namespace {

// ---- rotated append -------------------------------------------------------------------
// y = R(p) n(x) for the heads of q and k, y = x for those of v; n(x) = x / sqrt(mean x^2 + eps) * (offset + gain) or x;
// R turns the pairs (i, i + rot/2) by the angle p * f_i.  q goes to its output, k and v as fp16 to their slots.

// sin and cos of p * f in fp32.  The angle is a product in 64 bits (far positions turn many times: fp32 would
// leave an angle of 10^5 off by 4e-3).  With n the nearest multiple of pi/2, r = a - n pi/2 from two parts of
// pi/2 (the first subtraction is exact), and the Taylor series of sin r and cos r for |r| <= pi/4 up to r^13 and
// r^14, whose rests are below 2^-44: rounded to fp32 they are the correctly rounded value but for one case
// in about 2^20.  Good for angles up to 2^32; NaN beyond.
__device__ __forceinline__ void turn(int p, double f, float& c, float& s) {
  const double a = (double)p * f;
  const double n = __builtin_rint(a * 0.63661977236758134);
  double r = __builtin_fma(-n, 1.5707963267948966, a);
  r = __builtin_fma(-n, 6.123233995736766e-17, r);
  const double z = r * r;
  double u = 1.6059043836821613e-10;
  u = __builtin_fma(u, z, -2.5052108385441720e-08);
  u = __builtin_fma(u, z, 2.7557319223985893e-06);
  u = __builtin_fma(u, z, -1.9841269841269841e-04);
  u = __builtin_fma(u, z, 8.3333333333333332e-03);
  u = __builtin_fma(u, z, -1.6666666666666666e-01);
  const double sn = __builtin_fma(u * z, r, r);
  double w = -1.1470745597729725e-11;
  w = __builtin_fma(w, z, 2.0876756987868100e-09);
  w = __builtin_fma(w, z, -2.7557319223985888e-07);
  w = __builtin_fma(w, z, 2.4801587301587302e-05);
  w = __builtin_fma(w, z, -1.3888888888888889e-03);
  w = __builtin_fma(w, z, 4.1666666666666664e-02);
  w = __builtin_fma(w, z, -0.5);
  const double cs = __builtin_fma(w, z, 1.0);
  const bool far = !(__builtin_fabs(a) <= 0x1p32);
  const int quarter = far ? 0 : (int)((int64_t)n & 3);
  const double ss = quarter & 1 ? cs : sn, cc = quarter & 1 ? sn : cs;
  s = far ? __builtin_nanf("") : (float)(quarter & 2 ? -ss : ss);
  c = far ? __builtin_nanf("") : (float)(quarter == 1 || quarter == 2 ? -cc : cc);
}

// Sum over aligned groups of N lanes (4, 8 or 16), in 64 bits.
template <int CTRL>
__device__ __forceinline__ double dpp_f64(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u, CTRL, 0xF, 0xF, true);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(u >> 32), CTRL, 0xF, 0xF, true);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
template <int N>
__device__ __forceinline__ double group_sum(double v) {
  v += dpp_f64<0xB1>(v);
  v += dpp_f64<0x4E>(v);
  if constexpr (N >= 8) v += dpp_f64<0x141>(v);
  if constexpr (N >= 16) v += dpp_f64<0x128>(v);
  return v;
}

// A thread takes 16 elements of a head: eight pairs that turn (or 16 that do not), a workgroup R rows, whose
// angles it works out once for all heads.  Memory bounds it where rows are many: 16 411 rows of 48 heads of 128, bf16, 403 MB in 74 us (5.4 TB/s;
// a copy of 2 GiB reaches 5.0); below some 1000 rows it is one launch and one chain of waits (4.1 to 4.6 us).
template <int D, int R, class E, bool VEC>
__global__ void __launch_bounds__(256) k_rope_append(RopeAppend a) {
  typedef typename E::T T;
  constexpr int TPH = D / 16;  // threads a head
  __shared__ float cs[R][D / 2], sn[R][D / 2];
  const int row0 = blockIdx.x * R, n_rows = min(R, a.rows - row0), half = a.rot >> 1;
  for (int i = threadIdx.x; i < n_rows * half; i += 256) {
    const int r = i / half, j = i - r * half;
    turn(a.positions[row0 + r], a.freqs[j], cs[r][j], sn[r][j]);
  }
  __syncthreads();
  const int n_kv = a.c.n_kv, heads = a.n_q + 2 * n_kv, units = n_rows * heads * TPH;
  const int64_t limit = (int64_t)a.c.pages * a.c.page_size;
  // lanes behind the last unit take part in the exchanges
  for (int u0 = 0; u0 < units; u0 += 256) {
    const int u = u0 + (int)threadIdx.x;
    const bool live = u < units;
    const int uu = live ? u : units - 1, hr = uu / TPH, t = uu - hr * TPH, r = hr / heads, h = hr - r * heads;
    const int row = row0 + r;
    const bool is_q = h < a.n_q, is_v = h >= a.n_q + n_kv;
    const int kh = is_v ? h - a.n_q - n_kv : h - a.n_q;
    const int pairs = is_v ? 0 : a.rot >> 4;  // threads of the head whose elements turn
    const bool turns = t < pairs;
    const int o0 = turns ? 8 * t : is_v ? 16 * t : a.rot + 16 * (t - pairs), o1 = turns ? half + 8 * t : o0 + 8;
    const Rows& src = is_q ? a.q : is_v ? a.v : a.k;
    const T* p = (const T*)src.p + (int64_t)row * src.row + (int64_t)(is_q ? h : kh) * src.head;
    float x[2][8];
    load8<E, VEC>(p + o0, x[0]);
    load8<E, VEC>(p + o1, x[1]);
    const float* gain = is_q ? a.q_gain : is_v ? nullptr : a.k_gain;
    if (a.q_gain || a.k_gain) {  // (all lanes: a head's lanes are neighbours)
      double sum = 0.0;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        sum = __builtin_fma((double)x[0][i], (double)x[0][i], sum);
        sum = __builtin_fma((double)x[1][i], (double)x[1][i], sum);
      }
      sum = group_sum<TPH>(sum);
      if (gain) {
        const double factor = 1.0 / __builtin_sqrt(sum * (1.0 / D) + (double)a.eps);
        // in two factors, the first a power of two: for rows next to fp32's largest and smallest numbers theirs is no normal one
        const float lift = factor > 0x1p126 ? 0x1p64f : factor < 0x1p-126 ? 0x1p-64f : 1.0f;
        const float s = (float)(factor > 0x1p126 ? factor * 0x1p-64 : factor < 0x1p-126 ? factor * 0x1p64 : factor);
#pragma unroll
        for (int i = 0; i < 8; i++) {
          x[0][i] = ((x[0][i] * lift) * s) * (a.gain_offset + gain[o0 + i]);
          x[1][i] = ((x[1][i] * lift) * s) * (a.gain_offset + gain[o1 + i]);
        }
      }
    }
    if (turns) {
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const float c = cs[r][o0 + i], s = sn[r][o0 + i], lo = x[0][i], hi = x[1][i];
        x[0][i] = (lo * c) - (hi * s);
        x[1][i] = (hi * c) + (lo * s);
      }
    }
    if (!live) continue;
    if (is_q) {
      T* out = (T*)a.q_out.p + (int64_t)row * a.q_out.row + (int64_t)h * a.q_out.head;
      store8<E, VEC>(out + o0, x[0]);
      store8<E, VEC>(out + o1, x[1]);
    } else {
      const int slot = a.slots[row];
      if (slot < 0 || slot >= limit) continue;
      _Float16* out = (_Float16*)(is_v ? a.c.v : a.c.k) + ((int64_t)slot * n_kv + kh) * D;
      store8<F16, true>(out + o0, x[0]);
      store8<F16, true>(out + o1, x[1]);
    }
  }
}

template <int D, class E>
hipError_t rope_dim(hipStream_t st, const RopeAppend& a) {
  const int size = sizeof(typename E::T);
  const bool vec = vec_rows(a.k, size) && vec_rows(a.v, size) && (a.n_q == 0 || (vec_rows(a.q, size) && vec_rows(a.q_out, size)));
  // One row a workgroup where its heads fill it (8000 rows of 48 heads of 128, fp32: 70 us, four rows a workgroup 76) or rows are few; where
  // heads are few four (8000 rows of 12 heads of 64: 10.0 us, one row 14.2).
  const bool one = a.rows < 2048 || (int64_t)(a.n_q + 2 * a.c.n_kv) * D / 16 >= 256;
  const unsigned grid = (unsigned)(one ? a.rows : (a.rows + 3) / 4);
  auto f = one ? (vec ? k_rope_append<D, 1, E, true> : k_rope_append<D, 1, E, false>)
               : (vec ? k_rope_append<D, 4, E, true> : k_rope_append<D, 4, E, false>);
  hipLaunchKernelGGL(f, dim3(grid), dim3(256), 0, st, a);
  return hipGetLastError();
}
template <class E>
hipError_t rope_type(hipStream_t st, const RopeAppend& a) {
  if (a.c.hd == 64) return rope_dim<64, E>(st, a);
  if (a.c.hd == 128) return rope_dim<128, E>(st, a);
  return rope_dim<256, E>(st, a);
}

// ---- bounds of blocks --------------------------------------------------------------------
// The least and the greatest element of every channel over a block's tokens (NaN where there is one).  A wave
// takes one block and kv head: the block of a row that is the first of its sequence's new rows there.  A step of single tokens is a launch and
// three dependent loads: 4.8 us for one sequence, 5.4 for 32.
template <int D>
__global__ void __launch_bounds__(256) k_bounds_update(BoundsUpdate a) {
  constexpr int CH = D / 8, TOK = 64 / CH;  // lanes of a token, tokens at a time
  const int lane = threadIdx.x & 63, ps = a.c.page_size, n_kv = a.c.n_kv;
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int row = uniform((int)(unit / n_kv)), h = uniform((int)(unit % n_kv));
  if (row >= a.rows) return;
  const RowOf of(a.row_offsets, a.lengths, a.batch, a.rows, row);
  if (of.b < 0 || of.p < 0) return;
  const int block = of.p / ps, place = of.p - block * ps;
  // the sequence's first row with a position, or the block's first token
  const bool begins = place == 0 || row == of.first || of.p == 0;
  if (!begins || block >= a.pps) return;
  const int page = a.page_table[(int64_t)of.b * a.pps + block];
  if ((uint32_t)page >= (uint32_t)a.c.pages) return;
  const int held = min(ps, max(a.lengths[of.b], 0) - block * ps);
  const int c = lane % CH;
  float lo[8], hi[8];
#pragma unroll
  for (int i = 0; i < 8; i++) lo[i] = INFINITY, hi[i] = -INFINITY;
  const _Float16* base = (const _Float16*)a.c.k + ((int64_t)page * ps * n_kv + h) * D + 8 * c;
  for (int t = lane / CH; t < held; t += TOK) {
    float x[8];
    load8<F16, true>(base + (int64_t)t * n_kv * D, x);
#pragma unroll
    for (int i = 0; i < 8; i++) {
      lo[i] = __builtin_elementwise_minimum(lo[i], x[i]);
      hi[i] = __builtin_elementwise_maximum(hi[i], x[i]);
    }
  }
#pragma unroll
  for (int d = CH; d < 64; d <<= 1)
#pragma unroll
    for (int i = 0; i < 8; i++) {
      lo[i] = __builtin_elementwise_minimum(lo[i], __shfl_xor(lo[i], d, 64));
      hi[i] = __builtin_elementwise_maximum(hi[i], __shfl_xor(hi[i], d, 64));
    }
  _Float16* out = (_Float16*)a.bounds + ((int64_t)page * n_kv + h) * 2 * D + 8 * c;
  if (lane < CH) store8<F16, true>(out, lo);
  else if (lane < 2 * CH) store8<F16, true>(out + D, hi);
}

// ---- selection of blocks -----------------------------------------------------------------
// A row's score of a block is the most that a product of one of the group's queries with a key inside the block's bounds can
// be: s_j = max over the heads g of sum_d max(q_gd lo_jd, q_gd hi_jd).  Sums are in 64 bits, where products of fp16 with
// fp16 or bf16 lose nothing, and only the bound that a query takes enters them: which of two blocks is taken is part of the result, and
// blocks whose bounds are alike where the queries take them are equal.
// 1. k_block_scores: the scores.  2. k_block_pick: the border between what is taken and what is not, and the list in ascending order.

// The blocks that a row's list is chosen from: those from `first` on up to, not with, the last ones.
struct Choice {
  int cur, lo, n;  // the row's own block; candidates [lo, lo + n); n = 0: no choice
  __device__ __forceinline__ Choice(const BlockSelect& a, int p) {
    cur = min(p / a.page_size, a.pps - 1);
    lo = a.first;
    n = cur + 1 <= a.top ? 0 : cur + 1 - a.last - a.first;
  }
};

// Sum over aligned groups of N lanes (8, 16 or 32) of HG values at once: a lane ends with the sum of value lane % HG
// (the first steps halve the values that a lane holds instead of adding all of them).
template <int N, int HG>
__device__ __forceinline__ double scatter_sum(double (&v)[HG]) {
  const int lane = threadIdx.x & 63;
  double x = v[0];
  if constexpr (HG == 4) {
    const bool odd = lane & 1;
    double keep[2], give[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
      keep[i] = odd ? v[2 * i + 1] : v[2 * i];
      give[i] = odd ? v[2 * i] : v[2 * i + 1];
      keep[i] += dpp_f64<0xB1>(give[i]);
    }
    const bool high = lane & 2;
    x = (high ? keep[1] : keep[0]) + dpp_f64<0x4E>(high ? keep[0] : keep[1]);
  } else if constexpr (HG == 2) {
    const bool odd = lane & 1;
    x = (odd ? v[1] : v[0]) + dpp_f64<0xB1>(odd ? v[0] : v[1]);
    x += dpp_f64<0x4E>(x);
  } else {
    x += dpp_f64<0xB1>(x);
    x += dpp_f64<0x4E>(x);
  }
  // within rows of 16 lanes, the lanes of one residue modulo 4 (rotations keep it)
  if constexpr (N == 8) {
    x += __shfl_xor(x, 4, 64);
  } else {
    x += dpp_f64<0x124>(x);
    x += dpp_f64<0x128>(x);
    if constexpr (N == 32) x += __shfl_xor(x, 16, 64);
  }
  return x;
}

// By the definition: where something is not finite.
template <int D, class E>
__device__ double odd_score(const typename E::T* q, int64_t head, int group, const _Float16* bound) {
  double best = -INFINITY;
  for (int g = 0; g < group; g++) {
    double s = 0.0;
#pragma unroll 1
    for (int d = 0; d < D; d++) {
      const double x = (double)E::get(q[g * head + d]) * (double)(float)bound[d], y = (double)E::get(q[g * head + d]) * (double)(float)bound[D + d];
      s += x > y || x != x ? x : y;
    }
    if (s != s) return INFINITY;
    best = s > best ? s : best;
  }
  return best;
}

// A wave scores `per` blocks for one row and kv head, D / 8 lanes a block, HG heads of the group at a time.  With finite numbers
// the larger of q lo and q hi is q hi where q is positive and q lo where it is not: a selection and a multiply-add a product (q (lo + hi) + |q| |hi - lo|, two
// multiply-adds, would leave the rounding of the bound that is not taken in the sum); where a sum is not finite the block is scored by the definition.  Four steps' bounds are in flight.  32 sequences of 2048 to
// 16 384 tokens in pages of 16, 32 heads over 8 of 128, f16: 76 MB of bounds in 33 us, twice what reading them takes; vector instructions are busy
// half of that, with selections, conversions and multiply-adds in 64 bits.  One sequence of 131 071: 34 MB in 15.
template <int D, int HG, class E>
__global__ void __launch_bounds__(256, 4) k_block_scores(BlockSelect a, double* __restrict__ scores, int chunks, int per) {
  typedef typename E::T T;
  constexpr int CH = D / 8, PER = 64 / CH, AHEAD = 4;  // lanes of a block, blocks at a time, steps in flight
  const int lane = threadIdx.x & 63, c = lane % CH;
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t rh = unit / chunks;
  const int chunk = uniform((int)(unit - rh * chunks));
  const int row = uniform((int)(rh / a.n_kv)), h = uniform((int)(rh - (int64_t)row * a.n_kv));
  if (row >= a.rows) return;
  const int group = a.n_q / a.n_kv;
  const T* q0 = (const T*)a.q.p + (int64_t)row * a.q.row + (int64_t)h * group * a.q.head;
  const bool vec = vec_rows(a.q, sizeof(T));
  double q[HG][8];
  const auto queries = [&](int g0) {  // behind the last head: that head again
#pragma unroll
    for (int i = 0; i < HG; i++) {
      const T* p = q0 + (int64_t)min(g0 + i, group - 1) * a.q.head + 8 * c;
      float x[8];
      if (vec) load8<E, true>(p, x); else load8<E, false>(p, x);
#pragma unroll
      for (int k = 0; k < 8; k++) q[i][k] = (double)x[k];
    }
  };
  queries(0);
  const RowOf of(a.row_offsets, a.lengths, a.batch, a.rows, row);
  if (of.b < 0 || of.p < 0) return;
  const Choice ch(a, of.p);
  const int j0 = chunk * per, n = min(per, ch.n - j0);
  if (n <= 0) return;
  double* out = scores + rh * a.ws_blocks + j0;
  const int page = lane < n ? a.page_table[(int64_t)of.b * a.pps + ch.lo + j0 + lane] : -1;
  const int64_t head = (int64_t)2 * D;
  const _Float16* base = (const _Float16*)a.bounds + h * head + 8 * c;
  const auto bound_of = [&](int step) {
    const int id = __shfl(page, min(step * PER + lane / CH, 63), 64);
    return base + (int64_t)((uint32_t)id < (uint32_t)a.pages ? id : 0) * a.n_kv * head;
  };
  uint32_t odds = 0;  // steps whose block has no finite score
  for (int g0 = 0; g0 < group; g0 += HG) {
    if (g0) queries(g0);
    u32x4 lo[AHEAD], hi[AHEAD];
    const auto load = [&](int i, int step) {
      const _Float16* p = bound_of(step);
      lo[i] = *(const u32x4*)p;
      hi[i] = *(const u32x4*)(p + D);
    };
    const auto score = [&](int i, int step) {
      // (bounds that are not in order, as a caller may write them, count as their least and greatest; a NaN stays one)
      h2 least[4], most[4], wide = {0, 0};
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const uint32_t l = lo[i][k], h = hi[i][k];
        least[k] = __builtin_elementwise_minimum(__builtin_bit_cast(h2, l), __builtin_bit_cast(h2, h));
        most[k] = __builtin_elementwise_maximum(__builtin_bit_cast(h2, l), __builtin_bit_cast(h2, h));
        wide = __builtin_elementwise_maximum(wide, most[k] - least[k]);
      }
      double s[HG];
      // an infinity among the bounds that no query takes here may be a NaN by the definition (0 times it)
      s[0] = (double)(((float)wide[0] + (float)wide[1]) * 0.0f);
#pragma unroll
      for (int g = 1; g < HG; g++) s[g] = 0.0;
#pragma unroll
      for (int k = 0; k < 8; k++) {
        const double x = (double)(float)least[k >> 1][k & 1], y = (double)(float)most[k >> 1][k & 1];
#pragma unroll
        for (int g = 0; g < HG; g++) s[g] = __builtin_fma(q[g][k], q[g][k] > 0.0 ? y : x, s[g]);
      }
      double x = scatter_sum<CH, HG>(s);
      int odd = !(__builtin_fabs(x) < INFINITY);
      if constexpr (HG >= 2) {
        odd |= __builtin_amdgcn_update_dpp(0, odd, 0xB1, 0xF, 0xF, true);
        const double o = dpp_f64<0xB1>(x);
        x = o > x ? o : x;
      }
      if constexpr (HG == 4) {
        odd |= __builtin_amdgcn_update_dpp(0, odd, 0x4E, 0xF, 0xF, true);
        const double o = dpp_f64<0x4E>(x);
        x = o > x ? o : x;
      }
      const int j = step * PER + lane / CH, id = __shfl(page, min(j, 63), 64);
      if (c == 0 && j < n) {
        const bool there = (uint32_t)id < (uint32_t)a.pages;
        if (g0) x = out[j] > x ? out[j] : x;
        if (odd) odds |= 1u << step;
        out[j] = there ? x : -INFINITY;
      }
    };
#pragma unroll
    for (int i = 0; i < AHEAD; i++) load(i, i);
#pragma unroll 1
    for (int step = 0; step * PER < n; step += AHEAD)  // (loads behind the last block are of a page that is there)
#pragma unroll
      for (int i = 0; i < AHEAD; i++) {
        score(i, step + i);
        load(i, step + i + AHEAD);
      }
  }
  while (odds) {
    const int step = __ffs(odds) - 1, j = step * PER + lane / CH;
    odds &= odds - 1;
    const int id = a.page_table[(int64_t)of.b * a.pps + ch.lo + j0 + j];
    if ((uint32_t)id < (uint32_t)a.pages) out[j] = odd_score<D, E>(q0, a.q.head, group, base + (int64_t)id * a.n_kv * head);
  }
}

// ---- the list of one row and kv head ----
// Inclusive sum over the workgroup's threads; `tmp` holds one value a wave.
template <int THREADS>
__device__ __forceinline__ int block_sum(int v, int* tmp, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int in = (int)wave_scan_i64(v);
  __syncthreads();
  if (lane == 63) tmp[wave] = in;
  __syncthreads();
  total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; w++) {
    const int x = tmp[w];
    if (w < wave) in += x;
    total += x;
  }
  return in;
}
__device__ __forceinline__ uint64_t order_of(double s) {  // integers of the same order
  const uint64_t u = __builtin_bit_cast(uint64_t, s + 0.0);  // -0 is 0
  return u >> 63 ? ~u : u | 1ull << 63;
}

constexpr int kBuckets = 2048, kFew = 256;

// The n candidates lie in registers, KPT neighbours a thread.  Their scores' range is cut into equal buckets, and what is in the
// bucket that the border falls into is ranked by counting; where that is too much (many alike, or a few far from the rest) the border is found by
// eight bits of the scores' integers at a time.  A chain of barriers: 2.8 us where all blocks are listed, 5 to 6 for up to 1024 blocks,
// 13 for 8192.
template <int THREADS, int KPT>
__global__ void __launch_bounds__(THREADS) k_block_pick(BlockSelect a, const double* __restrict__ scores) {
  constexpr int WAVES = THREADS / 64;
  __shared__ int hist[kBuckets], tmp[WAVES], chosen[2], few_n;
  __shared__ float ends[2][WAVES];
  __shared__ uint64_t few[kFew];
  __shared__ int few_at[kFew];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t rh = blockIdx.x;
  const int row = (int)(rh / a.n_kv);
  // scores, asked for before the row's candidates are known (in the workspace wherever they end)
  const double* from = scores + rh * a.ws_blocks + min(tid * KPT, (int)a.ws_blocks - KPT);
  double s[KPT];
#pragma unroll
  for (int i = 0; i < KPT / 2; i++) ((u32x4*)s)[i] = a.pps > a.top ? ((const u32x4*)from)[i] : u32x4{0, 0, 0, 0};
  const RowOf of(a.row_offsets, a.lengths, a.batch, a.rows, row);
  if (of.b < 0) return;
  int32_t* out = a.blocks + rh * a.top;
  const Choice ch(a, of.p);
  if (of.p < 0 || ch.n == 0) {
    for (int i = tid; i < a.top; i += THREADS) out[i] = of.p >= 0 && i <= ch.cur ? i : -1;
    return;
  }
  const int take = a.top - a.first - a.last;  // of the candidates
  for (int i = tid; i < a.first; i += THREADS) out[i] = i;
  for (int i = tid; i < a.last; i += THREADS) out[a.top - a.last + i] = ch.cur + 1 - a.last + i;
  if (take == 0) return;
  // the range of the finite ones, in fp32 (rounding keeps the order)
  float lo = INFINITY, hi = -INFINITY;
#pragma unroll
  for (int i = 0; i < KPT; i++) {
    const float x = (float)s[i];
    const bool fin = tid * KPT + i < ch.n && fabsf(x) < INFINITY;
    lo = fin ? fminf(lo, x) : lo;
    hi = fin ? fmaxf(hi, x) : hi;
  }
  lo = -wave_max(-lo);
  hi = wave_max(hi);
  if (lane == 0) ends[0][wave] = lo, ends[1][wave] = hi;
  for (int i = tid; i < kBuckets; i += THREADS) hist[i] = 0;
  if (tid == 0) few_n = 0;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WAVES; w++) {
    lo = fminf(lo, ends[0][w]);
    hi = fmaxf(hi, ends[1][w]);
  }
  // a bucket's number does not decrease with the score
  const float per = (float)(kBuckets - 2) / (hi - lo);  // (all alike: infinite or none, and one bucket)
  const auto bucket = [&](double score) {
    const float x = (float)score;
    if (x == INFINITY) return kBuckets - 1;
    if (x == -INFINITY) return 0;
    const float at = (x - lo) * per;
    return at >= 0.0f ? (at < (float)(kBuckets - 3) ? 1 + (int)at : kBuckets - 2) : 1;
  };
  int in[KPT];
#pragma unroll
  for (int i = 0; i < KPT; i++) {
    in[i] = tid * KPT + i < ch.n ? bucket(s[i]) : -1;
    if (in[i] >= 0) atomicAdd(&hist[in[i]], 1);
  }
  __syncthreads();
  // from the highest bucket down: where the count reaches `take`
  constexpr int BPT = kBuckets / THREADS;
  int mine[BPT], sum = 0, total;
#pragma unroll
  for (int i = 0; i < BPT; i++) sum += mine[i] = hist[kBuckets - 1 - tid * BPT - i];
  int run = block_sum<THREADS>(sum, tmp, total) - sum;
#pragma unroll
  for (int i = 0; i < BPT; i++) {
    if (run < take && run + mine[i] >= take) {
      chosen[0] = kBuckets - 1 - tid * BPT - i;
      chosen[1] = take - run;
    }
    run += mine[i];
  }
  __syncthreads();
  const int border_bucket = chosen[0], left = chosen[1], inside = hist[border_bucket];
  // of the border's bucket: keys above `border` are taken, and of those equal to it the first `equal`
  uint64_t border = 0;
  int equal = 0;
  if (inside == left) {
    // all of it: border 0
  } else if (inside <= kFew) {
#pragma unroll
    for (int i = 0; i < KPT; i++)
      if (in[i] == border_bucket) {
        const int at = atomicAdd(&few_n, 1);
        few[at] = order_of(s[i]);
        few_at[at] = tid * KPT + i;
      }
    __syncthreads();
    for (int i = tid; i < inside; i += THREADS) {  // its rank; the one of rank left - 1 is the last that is taken
      const uint64_t k = few[i];
      const int at = few_at[i];
      int above = 0, same_before = 0;
      for (int o = 0; o < inside; o++) {
        above += few[o] > k;
        same_before += few[o] == k && few_at[o] < at;
      }
      if (above + same_before == left - 1) chosen[0] = i, chosen[1] = same_before + 1;
    }
    __syncthreads();
    border = few[chosen[0]];
    equal = chosen[1];
  } else {
    int want = left, shift = 56;
    for (;; shift -= 8) {
      __syncthreads();
      for (int i = tid; i < 256; i += THREADS) hist[i] = 0;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < KPT; i++) {
        const uint64_t k = order_of(s[i]);
        if (in[i] == border_bucket && (shift == 56 || ((k ^ border) >> (shift + 8)) == 0)) atomicAdd(&hist[(k >> shift) & 255], 1);
      }
      __syncthreads();
      const int here = tid < 256 ? hist[255 - tid] : 0;
      const int before = block_sum<THREADS>(here, tmp, total) - here;
      if (before < want && before + here >= want) chosen[0] = 255 - tid, chosen[1] = want - before;
      __syncthreads();
      border |= (uint64_t)chosen[0] << shift;
      want = chosen[1];
      if (shift == 0) break;
    }
    equal = want;
  }
  // the list, in the blocks' order: a thread's candidates are neighbours
  int ties = 0, sure = 0;
  uint32_t tie = 0, taken = 0;
#pragma unroll
  for (int i = 0; i < KPT; i++) {
    bool t = in[i] > border_bucket, e = false;
    if (in[i] == border_bucket) {
      const uint64_t k = order_of(s[i]);
      t = inside == left || k > border;
      e = !t && k == border;
    }
    taken |= t ? 1u << i : 0u;
    tie |= e ? 1u << i : 0u;
    sure += t;
    ties += e;
  }
  int tie_rank = block_sum<THREADS>(ties, tmp, total) - ties;
  const int ties_taken = min(max(equal - tie_rank, 0), ties);
  int at = block_sum<THREADS>(sure + ties_taken, tmp, total) - sure - ties_taken;
#pragma unroll
  for (int i = 0; i < KPT; i++) {
    bool t = (taken >> i) & 1;
    if ((tie >> i) & 1) t = tie_rank++ < equal;
    if (t) out[a.first + at++] = ch.lo + tid * KPT + i;
  }
}

// Any number of candidates: the border by eight bits at a time, from the workspace.
__global__ void __launch_bounds__(1024) k_block_pick_many(BlockSelect a, const double* __restrict__ scores) {
  constexpr int THREADS = 1024;
  __shared__ int hist[256], tmp[THREADS / 64], chosen[2];
  const int tid = threadIdx.x;
  const int64_t rh = blockIdx.x;
  const int row = (int)(rh / a.n_kv);
  const RowOf of(a.row_offsets, a.lengths, a.batch, a.rows, row);
  if (of.b < 0) return;
  int32_t* out = a.blocks + rh * a.top;
  const Choice ch(a, of.p);
  if (of.p < 0 || ch.n == 0) {
    for (int i = tid; i < a.top; i += THREADS) out[i] = of.p >= 0 && i <= ch.cur ? i : -1;
    return;
  }
  const double* s = scores + rh * a.ws_blocks;
  const int take = a.top - a.first - a.last;
  for (int i = tid; i < a.first; i += THREADS) out[i] = i;
  for (int i = tid; i < a.last; i += THREADS) out[a.top - a.last + i] = ch.cur + 1 - a.last + i;
  if (take == 0) return;
  uint64_t border = 0;
  int want = take, total;
  for (int shift = 56; shift >= 0; shift -= 8) {
    __syncthreads();
    for (int i = tid; i < 256; i += THREADS) hist[i] = 0;
    __syncthreads();
    for (int j = tid; j < ch.n; j += THREADS) {
      const uint64_t k = order_of(s[j]);
      if (shift == 56 || ((k ^ border) >> (shift + 8)) == 0) atomicAdd(&hist[(k >> shift) & 255], 1);
    }
    __syncthreads();
    const int here = tid < 256 ? hist[255 - tid] : 0;
    const int before = block_sum<THREADS>(here, tmp, total) - here;
    if (before < want && before + here >= want) chosen[0] = 255 - tid, chosen[1] = want - before;
    __syncthreads();
    border |= (uint64_t)chosen[0] << shift;
    want = chosen[1];
  }
  int at = a.first, ties = 0;
  for (int j0 = 0; j0 < ch.n; j0 += THREADS) {
    const int j = j0 + tid;
    const uint64_t k = j < ch.n ? order_of(s[j]) : 0;
    const bool same = j < ch.n && k == border;
    int all;
    const int rank = ties + block_sum<THREADS>(same, tmp, all) - same;
    ties += all;
    const bool t = j < ch.n && (k > border || (same && rank < want));
    const int place = at + block_sum<THREADS>(t, tmp, all) - t;
    at += all;
    if (t) out[place] = ch.lo + j;
  }
}

template <int D, class E>
hipError_t select_dim(hipStream_t st, const BlockSelect& a) {
  double* scores = (double*)a.ws;
  const int group = a.n_q / a.n_kv;
  const int64_t rh = (int64_t)a.rows * a.n_kv;
  const ScoreCut cut = score_cut(rh, a.pps, compute_units());
  const int64_t units = rh * cut.chunks;
  if (a.pps > a.top) {
    auto f = group == 1 ? k_block_scores<D, 1, E> : group == 2 ? k_block_scores<D, 2, E> : k_block_scores<D, 4, E>;
    hipLaunchKernelGGL(f, dim3((unsigned)((units + 3) / 4)), dim3(256), 0, st, a, scores, cut.chunks, cut.per);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  const dim3 grid((unsigned)rh);
  // The fewest threads and registers that hold the blocks: 1024 threads for tables of up to 1024 blocks 98 us for 90 (128 rows of 8 kv heads, the
  // selection with its attention), 16 blocks a thread for up to 4096 75 for 67 (8 rows of 3750 blocks).
  if (a.pps <= 256 * 4) hipLaunchKernelGGL((k_block_pick<256, 4>), grid, dim3(256), 0, st, a, scores);
  else if (a.pps <= 1024 * 4) hipLaunchKernelGGL((k_block_pick<1024, 4>), grid, dim3(1024), 0, st, a, scores);
  else if (a.pps <= 1024 * 16) hipLaunchKernelGGL((k_block_pick<1024, 16>), grid, dim3(1024), 0, st, a, scores);
  else hipLaunchKernelGGL(k_block_pick_many, grid, dim3(1024), 0, st, a, scores);
  return hipGetLastError();
}
template <class E>
hipError_t select_type(hipStream_t st, const BlockSelect& a) {
  if (a.hd == 64) return select_dim<64, E>(st, a);
  if (a.hd == 128) return select_dim<128, E>(st, a);
  return select_dim<256, E>(st, a);
}

}  // namespace

hipError_t launch_rope_append(hipStream_t st, int dtype, const RopeAppend& a) {
  if (a.rows == 0) return hipSuccess;
  if (dtype == RSTR_F32) return rope_type<F32>(st, a);
  if (dtype == RSTR_F16) return rope_type<F16>(st, a);
  return rope_type<BF16>(st, a);
}

hipError_t launch_bounds_update(hipStream_t st, const BoundsUpdate& a) {
  if (a.rows == 0 || a.batch == 0) return hipSuccess;
  const int64_t units = (int64_t)a.rows * a.c.n_kv;
  const unsigned grid = (unsigned)((units + 3) / 4);
  if (a.c.hd == 64) hipLaunchKernelGGL(k_bounds_update<64>, dim3(grid), dim3(256), 0, st, a);
  else if (a.c.hd == 128) hipLaunchKernelGGL(k_bounds_update<128>, dim3(grid), dim3(256), 0, st, a);
  else hipLaunchKernelGGL(k_bounds_update<256>, dim3(grid), dim3(256), 0, st, a);
  return hipGetLastError();
}

size_t select_workspace(int n_kv, int rows, int blocks) {
  return (size_t)rows * n_kv * select_stride(blocks) * sizeof(double);
}

hipError_t launch_block_select(hipStream_t st, int dtype, const BlockSelect& a) {
  if (a.rows == 0 || a.batch == 0) return hipSuccess;
  if (dtype == RSTR_F32) return select_type<F32>(st, a);
  if (dtype == RSTR_F16) return select_type<F16>(st, a);
  return select_type<BF16>(st, a);
}

}  // namespace rstr
