// pool_rows.hip -- rows of the fp16 page pool: appends with norms of heads and the position rotation on the
// way, the bounds of blocks of keys, and the blocks that a query's scores against these bounds select.
#include <hip/hip_runtime.h>

#include "../../include/rstr_hip.h"
#include "attn_line.h"
#include "device_math.h"
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
// angles it works out once for all heads.
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
        const float s = (float)(1.0 / __builtin_sqrt(sum * (1.0 / D) + (double)a.eps));
#pragma unroll
        for (int i = 0; i < 8; i++) {
          x[0][i] = (x[0][i] * s) * (a.gain_offset + gain[o0 + i]);
          x[1][i] = (x[1][i] * s) * (a.gain_offset + gain[o1 + i]);
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
  const bool few = a.rows < 2048;
  const unsigned grid = (unsigned)(few ? a.rows : (a.rows + 3) / 4);
  auto f = few ? (vec ? k_rope_append<D, 1, E, true> : k_rope_append<D, 1, E, false>)
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
// takes one block and kv head: the block of a row that is the first of its sequence's new rows there.
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
// A row's score of a block is the most that a product of one of the group's queries with a key of the block could
// be: s_j = max over the heads g of sum_d max(q_gd lo_jd, q_gd hi_jd).  Sums are in 64 bits, where products of fp16 with
// fp16 or bf16 lose nothing: which of two blocks is taken is part of the result.
// 1. k_block_scores: the scores, as integers of the same order (a NaN counts as +infinity).
// 2. k_block_pick: the border, found by eight bits of it at a time, and the list in ascending order.

__device__ __forceinline__ uint64_t order_of(double s) {
  if (s != s) s = INFINITY;
  s += 0.0;  // -0 is 0
  const uint64_t u = __builtin_bit_cast(uint64_t, s);
  return u >> 63 ? ~u : u | 1ull << 63;
}

// The blocks that a row's list is chosen from: those from `first` on up to, not with, the last ones.
struct Choice {
  int cur, lo, n;  // the row's own block; candidates [lo, lo + n); n = 0: no choice
  __device__ __forceinline__ Choice(const BlockSelect& a, int p) {
    cur = min(p / a.page_size, a.pps - 1);
    lo = a.first;
    n = cur + 1 <= a.top ? 0 : cur + 1 - a.last - a.first;
  }
};

template <int D, class E>
__global__ void __launch_bounds__(256) k_block_scores(BlockSelect a, uint64_t* __restrict__ keys, int chunks) {
  typedef typename E::T T;
  constexpr int CH = D / 8, PER = 64 / CH;  // lanes of a block, blocks at a time
  const int lane = threadIdx.x & 63, c = lane % CH;
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int chunk = uniform((int)(unit % chunks));
  const int64_t rh = unit / chunks;
  const int row = uniform((int)(rh / a.n_kv)), h = uniform((int)(rh % a.n_kv));
  if (row >= a.rows) return;
  const RowOf of(a.row_offsets, a.lengths, a.batch, a.rows, row);
  if (of.b < 0 || of.p < 0) return;
  const Choice ch(a, of.p);
  const int group = a.n_q / a.n_kv;
  const int j0 = chunk * kScoreBlocks, j1 = min(j0 + kScoreBlocks, ch.n);
  uint64_t* out = keys + rh * a.ws_blocks;
  for (int j = j0 + lane / CH; j - lane / CH < j1; j += PER) {
    const int jj = min(j, j1 - 1);
    const int page = a.page_table[(int64_t)of.b * a.pps + ch.lo + jj];
    const bool there = (uint32_t)page < (uint32_t)a.pages;
    const _Float16* src = (const _Float16*)a.bounds + ((int64_t)(there ? page : 0) * a.n_kv + h) * 2 * D + 8 * c;
    float lo[8], hi[8];
    load8<F16, true>(src, lo);
    load8<F16, true>(src + D, hi);
    double best = -INFINITY;
    bool nan = false;
    for (int g = 0; g < group; g++) {
      float q[8];
      load8<E, false>((const T*)a.q.p + (int64_t)row * a.q.row + (int64_t)(h * group + g) * a.q.head + 8 * c, q);
      double s = 0.0;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const double x = (double)q[i] * (double)lo[i], y = (double)q[i] * (double)hi[i];
        s += x > y || x != x ? x : y;
      }
#pragma unroll
      for (int d = 1; d < CH; d <<= 1) s += __shfl_xor(s, d, 64);
      nan = nan || s != s;
      best = s > best ? s : best;
    }
    if (c == 0 && j < j1) out[j] = order_of(there ? (nan ? INFINITY : best) : -INFINITY);
  }
}

// The list of one row and kv head.
template <int THREADS>
__global__ void __launch_bounds__(THREADS) k_block_pick(BlockSelect a, const uint64_t* __restrict__ keys) {
  __shared__ int hist[256], wsum[THREADS / 64], chosen[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
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
  const uint64_t* key = keys + rh * a.ws_blocks;
  const int take = a.top - a.first - a.last;  // of the candidates
  for (int i = tid; i < a.first; i += THREADS) out[i] = i;
  for (int i = tid; i < a.last; i += THREADS) out[a.top - a.last + i] = ch.cur + 1 - a.last + i;
  if (take == 0) return;
  // the border: keys above it are taken, and of those equal to it the first `left`
  uint64_t border = 0;
  int left = take, shift = 56;
  for (;; shift -= 8) {
    for (int i = tid; i < 256; i += THREADS) hist[i] = 0;
    __syncthreads();
    for (int j = tid; j < ch.n; j += THREADS) {
      const uint64_t k = key[j];
      if (shift == 56 || ((k ^ border) >> (shift + 8)) == 0) atomicAdd(&hist[(k >> shift) & 255], 1);
    }
    __syncthreads();
    if (wave == 0) {  // from the highest digit down: where the count reaches `left`
      int mine[4], sum = 0;
#pragma unroll
      for (int i = 0; i < 4; i++) sum += mine[i] = hist[255 - 4 * lane - i];
      int in = sum;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(in, d, 64);
        if (lane >= d) in += o;
      }
      int run = in - sum;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        if (run < left && run + mine[i] >= left) {
          chosen[0] = 255 - 4 * lane - i;
          chosen[1] = left - run;
        }
        run += mine[i];
      }
    }
    __syncthreads();
    border |= (uint64_t)chosen[0] << shift;
    left = chosen[1];
    const bool all = hist[chosen[0]] == left;  // the whole bucket is taken
    __syncthreads();
    if (shift == 0 || all) break;
  }
  // with the whole bucket taken the low bits of the border are 0 and no key counts as equal to it
  const uint64_t high = border >> shift;
  const bool whole = shift > 0;
  int before = 0, equal = 0;
  for (int j0 = 0; j0 < ch.n; j0 += THREADS) {
    const int j = j0 + tid;
    const uint64_t k = j < ch.n ? key[j] >> shift : 0;
    const bool same = !whole && j < ch.n && k == high;
    const bool above = j < ch.n && (whole ? k >= high : k > high);
    const uint64_t sb = __ballot(same), ab = __ballot(above);
    const uint64_t below = (1ull << lane) - 1;
    if (lane == 0) wsum[wave] = __popcll(ab) << 16 | __popcll(sb);
    __syncthreads();
    int a_before = before, s_before = equal, a_all = 0, s_all = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; w++) {
      if (w < wave) {
        a_before += wsum[w] >> 16;
        s_before += wsum[w] & 0xFFFF;
      }
      a_all += wsum[w] >> 16;
      s_all += wsum[w] & 0xFFFF;
    }
    const int s_rank = s_before + __popcll(sb & below), a_rank = a_before + __popcll(ab & below);
    if (above || (same && s_rank < left)) out[a.first + a_rank + min(s_rank, left)] = ch.lo + j;
    before += a_all;
    equal += s_all;
    __syncthreads();
  }
}

template <int D, class E>
hipError_t select_dim(hipStream_t st, const BlockSelect& a) {
  uint64_t* keys = (uint64_t*)a.ws;
  const int chunks = (a.pps + kScoreBlocks - 1) / kScoreBlocks;
  const int64_t rh = (int64_t)a.rows * a.n_kv, units = rh * chunks;
  if (a.pps > a.top) {
    hipLaunchKernelGGL((k_block_scores<D, E>), dim3((unsigned)((units + 3) / 4)), dim3(256), 0, st, a, keys, chunks);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(k_block_pick<256>, dim3((unsigned)rh), dim3(256), 0, st, a, keys);
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

size_t select_workspace(int n_q, int n_kv, int hd, int rows, int blocks) {
  (void)n_q, (void)hd;
  return (size_t)rows * n_kv * blocks * sizeof(uint64_t);
}

hipError_t launch_block_select(hipStream_t st, int dtype, const BlockSelect& a) {
  if (a.rows == 0 || a.batch == 0) return hipSuccess;
  if (dtype == RSTR_F32) return select_type<F32>(st, a);
  if (dtype == RSTR_F16) return select_type<F16>(st, a);
  return select_type<BF16>(st, a);
}

}  // namespace rstr
