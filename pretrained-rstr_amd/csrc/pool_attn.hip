// pool_attn.hip -- attention of ragged query rows over the fp16 page pool, over all tokens or over the blocks
// that a list names.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "../../include/rstr_hip.h"
#include "attn_line.h"
#include "device_math.h"
#include "pool_line.h"
#include "pool_ops.h"

namespace rstr {

namespace {

// One wave works on 16 * NT columns (a query row of one head of the kv head's group is a column) of one sequence
// and kv head, over tiles of 32 tokens, and needs neither LDS nor a barrier:
//
//   S^T = K Q^T     K is the A operand of 16x16x32 products as it lies in the pages: lane (c, g) loads 16 bytes
//                   of token c at dims 32 s + 8 g.
//   O^T += V^T P^T  a lane's S^T values are tokens 4g .. 4g + 3 of two halves of 16 of one column, which is what
//                   the B operand P^T wants from that lane.  The A operand wants eight tokens of one dim of V where
//                   a page holds eight dims of one token: the lane loads the same dims, 8 c .. 8 c + 7, of its eight
//                   tokens and pairs their halves, one byte permutation an operand register.  Product j so has the
//                   dims 8 c + j as its rows; 16 lanes read a whole row of a token.
//
// Queries are brought to [2^14, 2^15) of their row's largest element by a power of two and taken as one fp16 term
// (f16, bf16: no bit of an element above 2^-28 of the largest is lost) or two (fp32).  Weights are
// p = 2^((S - m) k + 10) with S the raw products, k the scale and that power of two: differences are taken before
// the scale, so scores of any size give finite weights.  m follows the column's maximum when a score passes it by 2^4, so the exchange between
// lanes and the rescaling of O are rare; p is below 2^14, and the factor 2^10 keeps small weights' bits: fp16's
// subnormals begin 2^24 below the largest.  p is one fp16 term (f16, bf16) or two (fp32).  S, m, l and O are fp32.
//
// Memory bounds it: 128 sequences of 128 to 4608 tokens, 32 heads over 8 of 128, f16, read 1.24 GB in 219 us (5.7 TB/s), four of 9000 to
// 131 000 733 MB in 133 (5.5), 33 of 5 to 8192 with 1 to 6 fp32 rows 556 MB in 111 (5.0).  Two waves a SIMD, each with the next tile's K and V in
// registers: three waves spill (335, 200 and 193 us); loads that bypass the caches' order are worth 234 -> 220 in the first.
//
// The tiles of all (sequence, kv head, column tile) items form one line of units that is cut into equal parts, one
// a wave, as in kv4_line.h; with a list of blocks every row and kv head is an item, and all have as many parts.
template <class E> struct Terms { static constexpr int n = 1; };
template <> struct Terms<F32> { static constexpr int n = 2; };

// The first of two fp16 terms of x, short of it by 2^-12 to 2^-10 of x: the rest has the sign of x and is never 0 (but for an x
// near fp16's smallest numbers), so that products of both terms with an infinity are that infinity.  The rest is rounded to 11
// bits: 1.25 * 2^-21 of x.
__device__ __forceinline__ _Float16 first_term(float x) {
  return (_Float16)__builtin_amdgcn_cvt_pkrtz(x * (1.0f - 0x1p-12f), 0.0f)[0];
}

// The second: the rest, rounded; of an infinity that infinity again, as both products have to be it.
__device__ __forceinline__ _Float16 second_term(float x, _Float16 first) {
  return (_Float16)(fabsf(x) < INFINITY ? x - (float)first : x);
}

// The size of a query's element, for the largest that its row is brought to: an infinity has none, it stays one at any power of two.
__device__ __forceinline__ float size_of(float x) { return fabsf(x) < INFINITY ? fabsf(x) : 0.0f; }

// What raw scores of queries that were brought down by 2^e are multiplied with: finite and not 0, so that it leaves the
// difference of two equal scores 0 and that of a score and -infinity -infinity.
__device__ __forceinline__ float score_scale(float scale, int e) {
  return fmaxf(fminf(__builtin_amdgcn_ldexpf(fabsf(scale) * 1.4426950408889634f, e), FLT_MAX), FLT_MIN);
}

// What the parts of an item leave: (m, l, k) and O of each column.
struct PoolPieces {
  int* n_items;
  Begun* begun;  // [items]
  f4* ml;        // [pieces][cols]
  float* acc;    // [pieces][cols][D]
};

// A part of a column tile's work.
struct Part {
  int b, h, r0, m, p0, c0;  // sequence, kv head, first row, rows, position of the first, first column
  int t0, t1;               // tiles
  bool whole;               // of the item: its output is written, not a piece
  int64_t piece;
  const int32_t* list;      // the row's blocks, or null
  int entries;              // pages (blocks) of it
  int blocks;               // of a list: blocks of the table that begin at the row's token or before
};

template <int D>
struct Dims {
  static constexpr int KS = D / 32, JT = D / 16, VW = D / 32;  // products of a score, of a tile of O; dwords of a token a lane
  static constexpr int PIECE = D / 16 < 8 ? D / 16 : 8;        // neighbouring dims a lane loads
  // dim of row r of product j
  static __device__ __forceinline__ constexpr int dim(int j, int r) { return j / PIECE * 128 + PIECE * r + j % PIECE; }
};

// s_waitcnt vmcnt(0) alone: loads into LDS are not waited for by a barrier.
__device__ __forceinline__ void wait_vmem() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0F70);
  asm volatile("" ::: "memory");
}

template <bool STREAM, class V>
__device__ __forceinline__ V load_page(const void* p) {
  if constexpr (STREAM) return __builtin_nontemporal_load((const V*)p);
  else return *(const V*)p;
}

// LW > 0: a list of blocks; LW waves of a workgroup share a row's list and join their parts in LDS.
constexpr int listed_threads(int lw) { return lw > 1 ? 64 * lw : 256; }
template <int D, int NT, class E, int LW>
__global__ void __launch_bounds__(listed_threads(LW), pool_waves(D))
    k_pool_attn(PoolAttn a, const int32_t* __restrict__ ro, const int32_t* __restrict__ lens, const int32_t* __restrict__ table,
                PoolPieces pc, int workers, int least, bool whole, int parts) {
  typedef Dims<D> G;
  typedef typename E::T T;
  constexpr int KS = G::KS, JT = G::JT, VW = G::VW, COLS = 16 * NT, TERMS = Terms<E>::n;
  constexpr bool LISTED = LW > 0, STREAM = NT == 1 && !LISTED;
  __shared__ f4 join_ml[LW > 1 ? LW : 1][LW > 1 ? COLS : 1];
  __shared__ __attribute__((aligned(16))) float join_acc[LW > 1 ? LW : 1][LW > 1 ? COLS : 1][LW > 1 ? D : 4];
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int wave = uniform(threadIdx.x >> 6), w = uniform(blockIdx.x * (LW > 1 ? LW : 4) + wave);
  const int n_kv = a.c.n_kv, group = a.n_q / n_kv, ps = a.c.page_size;
  const int cap = token_cap(a.pps, ps);
  const int64_t row_bytes = (int64_t)n_kv * D * 2;
  const int step_e = kTile / ps, step_off = kTile - step_e * ps;

  const auto work = [&](const Part& s) {
    const auto end_seen = [&](int r) { return min(max(s.p0 + r + 1, 0), cap); };
    const auto first_seen = [&](int r) { return a.window > 0 ? max(max(s.p0 + r + 1, 0) - a.window, 0) : 0; };
    const int rf = min(s.m - 1, s.c0 / group), rl = min(s.m - 1, (s.c0 + COLS - 1) / group);
    int hi[NT], lo[NT];
    int64_t qrow[NT], qhead[NT];
    bool valid[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) {
      const int cc = s.c0 + t * 16 + col, r = cc / group;
      valid[t] = r < s.m;
      hi[t] = valid[t] ? end_seen(r) : 0;
      lo[t] = first_seen(r);
      qrow[t] = s.r0 + r;
      qhead[t] = (int64_t)s.h * group + (cc - r * group);
    }
    const int hi_last = end_seen(rl), hi_first = end_seen(rf), lo_first = first_seen(rf), lo_last = first_seen(rl);
    int t0 = s.t0, t1 = s.t1;
    if constexpr (!LISTED) {
      t0 = max(t0, lo_first / kTile);
      t1 = min(t1, (hi_last + kTile - 1) / kTile);
    }

    f4 acc[NT][JT];
    float mref[NT], l[NT], kcol[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) {
#pragma unroll
      for (int j = 0; j < JT; j++) acc[t][j] = f4{0, 0, 0, 0};
      mref[t] = -FLT_MAX;
      l[t] = kcol[t] = 0.0f;
    }
    if (t0 < t1) {
      // pages of 64 entries from e0 on, one a lane; -1: not there
      const int32_t* row = table + (int64_t)s.b * a.pps;
      int e0 = 0, page = -1, block = 0;
      const auto look = [&](int from) {
        e0 = from;
        const int e = from + lane;
        int id = -1;
        if (LISTED) {
          block = e < s.entries ? s.list[e] : -1;
          if ((uint32_t)block < (uint32_t)s.blocks) id = row[block];  // (later ones hold nothing that the row sees, and their tokens may pass 32 bits)
          else block = 0;
        } else if (e < s.entries) {
          id = row[e];
        }
        page = (uint32_t)id < (uint32_t)a.c.pages ? id : -1;
      };
      // entry and place of the lane's token of each half, and of the tile's first and last token
      Place tok[2], first = place_of((uint32_t)t0 * kTile, ps);
#pragma unroll
      for (int j = 0; j < 2; j++) tok[j] = place_of((uint32_t)t0 * kTile + 16 * j + col, ps);
      look(first.entry);
      int slot_k[2], slot_v[2], tok_v[2];  // slots of the lane's tokens (-1: none), position of its first token of V
      const auto slots = [&](int tile) {
        if (uniform(entries_to_end(first, e0, ps)) >= 64) look(first.entry);
#pragma unroll
        for (int j = 0; j < 2; j++) {
          const int at = (tok[j].entry - e0) & 63, id = __shfl(page, at, 64);
          slot_k[j] = id < 0 ? -1 : id * ps + tok[j].off;
          slot_v[j] = __shfl(slot_k[j], 4 * g, 64);
          if (LISTED) {
            const int position = __shfl(block, at, 64) * ps + tok[j].off;
            tok_v[j] = __shfl(position, 4 * g, 64);
          } else {
            tok_v[j] = tile * kTile + 16 * j + 4 * g;
          }
          forward(tok[j], step_e, step_off, ps);
        }
        forward(first, step_e, step_off, ps);
      };
      const uint8_t* kbase = (const uint8_t*)a.c.k + (int64_t)s.h * D * 2 + 16 * g;
      const uint8_t* vbase = (const uint8_t*)a.c.v + (int64_t)s.h * D * 2 + 2 * G::PIECE * col;
      h8 kr[2][KS];
      uint32_t vr[2][4][VW];
      const auto load_k = [&] {
#pragma unroll
        for (int j = 0; j < 2; j++) {
          const uint8_t* p = kbase + (uint64_t)(uint32_t)max(slot_k[j], 0) * (uint64_t)row_bytes;
#pragma unroll
          for (int i = 0; i < KS; i++) kr[j][i] = __builtin_bit_cast(h8, load_page<STREAM, u32x4>(p + 64 * i));
        }
      };
      const auto load_v = [&] {
#pragma unroll
        for (int j = 0; j < 2; j++) {
          const uint8_t* p = vbase + (uint64_t)(uint32_t)max(slot_v[j], 0) * (uint64_t)row_bytes;
#pragma unroll
          for (int i = 0; i < 4; i++) {
            if constexpr (VW == 2) {
              const u32x2 x = load_page<STREAM, u32x2>(p + i * row_bytes);
              vr[j][i][0] = x[0];
              vr[j][i][1] = x[1];
            } else {
#pragma unroll
              for (int u = 0; u < VW / 4; u++) {
                const u32x4 x = load_page<STREAM, u32x4>(p + i * row_bytes + 256 * u);
#pragma unroll
                for (int k = 0; k < 4; k++) vr[j][i][4 * u + k] = x[k];
              }
            }
          }
        }
      };
      slots(t0);
      load_k();
      load_v();

      h8 q[NT][TERMS][KS];
      const bool vec = vec_rows(a.q, sizeof(T));
#pragma unroll
      for (int t = 0; t < NT; t++) {
        float x[KS][8], big = 0.0f;
#pragma unroll
        for (int s2 = 0; s2 < KS; s2++) {
          if (valid[t]) {
            const T* src = (const T*)a.q.p + qrow[t] * a.q.row + qhead[t] * a.q.head + s2 * 32 + g * 8;
            if (vec) load8<E, true>(src, x[s2]); else load8<E, false>(src, x[s2]);
          } else {
#pragma unroll
            for (int i = 0; i < 8; i++) x[s2][i] = 0.0f;
          }
#pragma unroll
          for (int i = 0; i < 8; i++) big = fmaxf(big, size_of(x[s2][i]));
        }
        big = xor_max<32>(xor_max<16>(big));
        // (a largest of 0 has the exponent 0; the sign of the scale goes into the queries, and a scale of 0 itself: 0 times an infinity is no number)
        const int e = __builtin_amdgcn_frexp_expf(big) - 15;
        kcol[t] = score_scale(a.scale, e);
#pragma unroll
        for (int s2 = 0; s2 < KS; s2++)
#pragma unroll
          for (int i = 0; i < 8; i++) {
            float y = __builtin_amdgcn_ldexpf(x[s2][i], -e);
            y = a.scale < 0.0f ? -y : a.scale == 0.0f ? y * 0.0f : y;
            if constexpr (TERMS == 2) {
              q[t][0][s2][i] = first_term(y);
              q[t][1][s2][i] = second_term(y, q[t][0][s2][i]);
            } else {
              q[t][0][s2][i] = (_Float16)y;
            }
          }
      }

      for (int tile = t0; tile < t1; tile++) {
        const int sv[2] = {slot_v[0], slot_v[1]}, tv[2] = {tok_v[0], tok_v[1]}, sk[2] = {slot_k[0], slot_k[1]};
        float sc[NT][8];
        {
          f4 d[NT][2];
#pragma unroll
          for (int t = 0; t < NT; t++)
#pragma unroll
            for (int j = 0; j < 2; j++) d[t][j] = f4{0, 0, 0, 0};
#pragma unroll
          for (int i = 0; i < KS; i++)
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
              for (int t = 0; t < NT; t++)
#pragma unroll
                for (int u = 0; u < TERMS; u++) d[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kr[j][i], q[t][u][i], d[t][j], 0, 0, 0);
#pragma unroll
          for (int t = 0; t < NT; t++)
#pragma unroll
            for (int i = 0; i < 8; i++) sc[t][i] = d[t][i >> 2][i & 3];
        }
        const bool more = tile + 1 < t1;
        if (more) {
          slots(tile + 1);
          load_k();
        }
        // tokens that are not there, or that not all columns see
        const int tok0 = tile * kTile;
        bool edge;
        if (LISTED) {
          const bool odd = sv[0] < 0 || sv[1] < 0 || max(tv[0], tv[1]) + 4 > hi_first || min(tv[0], tv[1]) < lo_last;
          edge = __ballot(odd) != 0;
        } else {
          edge = tok0 < lo_last || tok0 + kTile > hi_first || __ballot(sv[0] < 0 || sv[1] < 0) != 0;
        }
        uint32_t see[NT];
#pragma unroll
        for (int t = 0; t < NT; t++) see[t] = 0xFF;
        bool redo = false;  // values of V that are no numbers, of tokens that only some columns see
        if (edge) {
#pragma unroll
          for (int t = 0; t < NT; t++) {
            see[t] = 0;
#pragma unroll
            for (int i = 0; i < 8; i++) {
              const int tok = tv[i >> 2] + (i & 3);
              if (sv[i >> 2] >= 0 && tok >= lo[t] && tok < hi[t]) see[t] |= 1u << i;
            }
          }
          // 0 times an infinity or a NaN: V of tokens that no column sees becomes 0
          uint32_t odd = 0;
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const int tok = tv[i >> 2] + (i & 3);
            const bool some = sv[i >> 2] >= 0 && tok >= lo_first && tok < hi_last, all = tok >= lo_last && tok < hi_first;
#pragma unroll
            for (int k = 0; k < VW; k++) {
              uint32_t& x = vr[i >> 2][i & 3][k];
              if (!some) x = 0;
              else if (!all) odd |= ((x & 0x7C00u) == 0x7C00u || (x & 0x7C000000u) == 0x7C000000u) ? 1u : 0u;
            }
          }
          redo = !LISTED && __ballot(odd != 0) != 0;
        }
        float e2[NT][8];
        bool grow = false;
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
          for (int i = 0; i < 8; i++) {
            e2[t][i] = __builtin_fmaf(sc[t][i] - mref[t], kcol[t], 10.0f);
            if (edge && !((see[t] >> i) & 1)) e2[t][i] = -INFINITY;
            grow |= e2[t][i] > 14.0f;
          }
        if (__ballot(grow)) {
#pragma unroll
          for (int t = 0; t < NT; t++) {
            float m = -INFINITY;
            bool passed = false;
#pragma unroll
            for (int i = 0; i < 8; i++) {
              if ((see[t] >> i) & 1) m = fmaxf(m, sc[t][i]);
              passed |= e2[t][i] > 14.0f;
            }
            m = xor_max<32>(xor_max<16>(m));
            // a column that needs no change has none: it does not depend on its neighbours
            const bool own = of_column(__ballot(passed));
            const float now = own ? fmaxf(m, mref[t]) : mref[t];
            const float keep = own ? __builtin_amdgcn_exp2f((mref[t] - now) * kcol[t]) : 1.0f;
            mref[t] = now;
            l[t] *= keep;
#pragma unroll
            for (int j = 0; j < JT; j++) acc[t][j] *= keep;
#pragma unroll
            for (int i = 0; i < 8; i++)
              if (own) e2[t][i] = (see[t] >> i) & 1 ? __builtin_fmaf(sc[t][i] - now, kcol[t], 10.0f) : -INFINITY;
          }
        }
        float p[NT][8];
        h8 ph[NT][TERMS];
#pragma unroll
        for (int t = 0; t < NT; t++) {
#pragma unroll
          for (int i = 0; i < 8; i++) {
            p[t][i] = __builtin_amdgcn_exp2f(e2[t][i]);
            if constexpr (TERMS == 2) {
              ph[t][0][i] = first_term(p[t][i]);
              ph[t][1][i] = (_Float16)(p[t][i] - (float)ph[t][0][i]);
            } else {
              ph[t][0][i] = (_Float16)p[t][i];
            }
          }
          l[t] += ((p[t][0] + p[t][1]) + (p[t][2] + p[t][3])) + ((p[t][4] + p[t][5]) + (p[t][6] + p[t][7]));
        }
        if (!LISTED && redo) {  // their part is added by itself, to the columns that see them
          asm volatile("");
#pragma unroll 1
          for (int n = 0; n < kTile; n++) {
            const int tok = tok0 + n;
            const bool all = tok >= lo_last && tok < hi_first, some = tok >= lo_first && tok < hi_last;
            if (all || !some) continue;
            const int half = n >> 4, i = n & 3;
            const int slot = __shfl(sk[half], n & 15, 64);
            if (slot < 0) continue;
            const _Float16* v = (const _Float16*)a.c.v + ((int64_t)slot * n_kv + s.h) * D;
#pragma unroll
            for (int t = 0; t < NT; t++) {
              float mine = 0.0f;
#pragma unroll
              for (int k = 0; k < 8; k++) mine = k == 4 * half + i ? p[t][k] : mine;
              mine = __shfl(mine, (((n >> 2) & 3) << 4) + col, 64);
              const bool sees = tok >= lo[t] && tok < hi[t];
#pragma unroll
              for (int j = 0; j < JT; j++)
#pragma unroll
                for (int k = 0; k < 4; k++)
                  if (sees) acc[t][j][k] = __builtin_fmaf(mine, (float)v[G::dim(j, 4 * g + k)], acc[t][j][k]);
            }
          }
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const int tok = tv[i >> 2] + (i & 3);
            if (!(tok >= lo_last && tok < hi_first))
#pragma unroll
              for (int k = 0; k < VW; k++) vr[i >> 2][i & 3][k] = 0;
          }
        }
#pragma unroll
        for (int j = 0; j < JT; j++) {
          const uint32_t sel = j & 1 ? 0x07060302u : 0x05040100u;
          u32x4 o;
#pragma unroll
          for (int i = 0; i < 4; i++) o[i] = __builtin_amdgcn_perm(vr[i >> 1][2 * (i & 1) + 1][j >> 1], vr[i >> 1][2 * (i & 1)][j >> 1], sel);
          const h8 v = __builtin_bit_cast(h8, o);
#pragma unroll
          for (int t = 0; t < NT; t++)
#pragma unroll
            for (int u = 0; u < TERMS; u++) acc[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, ph[t][u], acc[t][j], 0, 0, 0);
        }
        if (more) load_v();
      }
    }

    if constexpr (LW > 1) {
      const float sum = xor_add<32>(xor_add<16>(l[0]));
      if (g == 0) join_ml[wave][col] = f4{mref[0], sum, kcol[0], 0.0f};
      if (valid[0] && sum != 0.0f) {
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
          for (int j = 0; j < JT; j += 4)
            *(f4*)&join_acc[wave][col][G::dim(j, 4 * g + i)] = f4{acc[0][j][i], acc[0][j + 1][i], acc[0][j + 2][i], acc[0][j + 3][i]};
      }
      __syncthreads();
      const int columns = min(COLS, group - s.c0);
      for (int at = threadIdx.x; at < columns * (D / 4); at += 64 * LW) {
        const int c = at / (D / 4), d = at % (D / 4) * 4;
        float top = -FLT_MAX, all = 0.0f, k = FLT_MIN;
        f4 ml[LW], o = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < LW; i++) {
          ml[i] = join_ml[i][c];
          if (ml[i][1] != 0.0f) top = fmaxf(top, ml[i][0]), k = ml[i][2];
        }
#pragma unroll
        for (int i = 0; i < LW; i++) {
          if (ml[i][1] == 0.0f) continue;
          const float f = __builtin_amdgcn_exp2f((ml[i][0] - top) * ml[i][2]);
          const f4 x = *(const f4*)&join_acc[i][c][d];
          all = __builtin_fmaf(f, ml[i][1], all);
#pragma unroll
          for (int j = 0; j < 4; j++) o[j] = __builtin_fmaf(f, x[j], o[j]);
        }
        if (s.whole) {
          const float inv = all == 0.0f ? 0.0f : 1.0f / all;
          T* to = (T*)a.out.p + (int64_t)s.r0 * a.out.row + ((int64_t)s.h * group + s.c0 + c) * a.out.head + d;
          T y[4];
#pragma unroll
          for (int j = 0; j < 4; j++) y[j] = E::put(o[j] * inv);
          if (vec_rows(a.out, sizeof(T))) {
            if constexpr (sizeof(T) == 4) *(u32x4*)to = *(u32x4*)y;
            else *(u32x2*)to = *(u32x2*)y;
          } else {
#pragma unroll
            for (int j = 0; j < 4; j++) to[j] = y[j];
          }
        } else {
          const int64_t p = s.piece * COLS + c;
          if (d == 0) pc.ml[p] = f4{top, all, k, 0.0f};
          *(f4*)(pc.acc + p * D + d) = o;
        }
      }
      return;
    }
#pragma unroll
    for (int t = 0; t < NT; t++) {
      const float sum = xor_add<32>(xor_add<16>(l[t]));
      if (!valid[t]) continue;
      if (s.whole) {
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        T* dst = (T*)a.out.p + qrow[t] * a.out.row + qhead[t] * a.out.head;
        const bool ovec = vec_rows(a.out, sizeof(T));
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
          for (int j = 0; j < JT; j += 4) {
            T* to = dst + G::dim(j, 4 * g + i);
            T o[4];
#pragma unroll
            for (int k = 0; k < 4; k++) o[k] = E::put(acc[t][j + k][i] * inv);
            if (ovec) {
              if constexpr (sizeof(T) == 4) *(u32x4*)to = *(u32x4*)o;
              else *(u32x2*)to = *(u32x2*)o;
            } else {
#pragma unroll
              for (int k = 0; k < 4; k++) to[k] = o[k];
            }
          }
      } else {
        const int64_t c = s.piece * COLS + t * 16 + col;
        if (g == 0) pc.ml[c] = f4{mref[t], sum, kcol[t], 0.0f};
        if (sum == 0.0f) continue;
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
          for (int j = 0; j < JT; j += 4) *(f4*)(pc.acc + c * D + G::dim(j, 4 * g + i)) = f4{acc[t][j][i], acc[t][j + 1][i], acc[t][j + 2][i], acc[t][j + 3][i]};
      }
    }
  };

  if constexpr (LISTED) {
    const int ncts = (group + COLS - 1) / COLS;
    // a wave of its own, or a workgroup: its item and part of it
    const int unit = LW > 1 ? (int)blockIdx.x : w, item = unit / parts, part = unit - item * parts;
    const int row = item / (n_kv * ncts), rest = item - row * (n_kv * ncts);
    if (row >= a.rows) return;
    const RowOf of(ro, lens, a.batch, a.rows, row);
    if (of.b < 0) return;
    Part s;
    s.b = of.b;
    s.h = rest / ncts;
    s.c0 = (rest - s.h * ncts) * COLS;
    s.r0 = row;
    s.m = 1;
    s.p0 = of.p;
    s.list = a.blocks + ((int64_t)row * n_kv + s.h) * a.top;
    s.blocks = of.p < 0 ? 0 : min(a.pps, of.p / ps + 1);
    s.entries = min(a.top, s.blocks);
    const int tiles = (int)(((int64_t)s.entries * ps + kTile - 1) / kTile);
    s.t0 = (LW > 1 ? part * LW + wave : part) * least;
    s.t1 = min(s.t0 + least, tiles);
    s.whole = whole;
    s.piece = unit;
    work(s);
  } else {
    const Lines L{ro, lens, a.rows, n_kv, group, a.window, COLS, cap, kStart, whole};
    Line line(L, a.batch, w, workers, least);
    if (w == 0 && !whole) *pc.n_items = line.items();
    while (line.next()) {
      const Seq& x = line.s;
      if (line.begins && !whole && lane == 0) pc.begun[line.item] = Begun{line.b, line.h, line.ct, w, line.pieces};
      Part s;
      s.b = line.b;
      s.h = line.h;
      s.r0 = x.r0;
      s.m = x.m;
      s.p0 = x.len - x.m;
      s.c0 = line.ct * COLS;
      s.t0 = x.lo + (whole ? 0 : max(line.at - kStart, 0));
      s.t1 = x.lo + (whole ? x.tiles : max(line.at + line.n - kStart, 0));
      s.whole = line.begins && line.ends;
      s.piece = piece_place(w, line.begins);
      s.list = nullptr;
      s.entries = (int)(((int64_t)L.held(x.len) + ps - 1) / ps);
      s.blocks = 0;
      work(s);
    }
  }
}

// ---- prompts -----------------------------------------------------------------------------
// Many columns a sequence: the waves of a workgroup take one or two tiles of 16 columns each of one sequence and kv head and
// share its keys and values, which go straight from the pages into LDS, 64 tokens at a time and one step ahead.
// The products are those of k_pool_attn.  K's operand is 16 bytes of a row; the operand of V, eight tokens of one dim, comes from two
// transposing reads of four tokens x 16 dims.  A row of a token is swizzled in LDS by its number, 16 bytes at a time, so that 16 tokens' same
// dims lie in different banks; the loads into LDS write 1 KB in the lanes' order, so a lane asks for the piece that
// belongs to its place.
// 333 and 1000 rows at 333 and 9000 tokens, 32 heads over 8 of 128, bf16: 240 us with the join in calls back to back, 584 TFLOP/s; in launches that stand apart,
// under the profiler, 253 and 13 for the join (four-row waves that load for themselves: 383).  No one part of a step bounds it: of then 250 us it
// took 219 without its exponentials, 204 and 214 without either product, 219 without its loads;
// matrix instructions are busy 25 % of the time, vector instructions 42 %, and the two waves that a SIMD has registers for wait for LDS and for
// each other's step the rest.  A third buffer (256), the two halves of a workgroup half a step apart (293, 270), all operands read ahead
// (283) and two workgroups of four waves (283) gain nothing.  Head dim 64 has half the products to an exponential (vector 53 %, matrix 19 %); 256 one tile of columns a
// wave, so that an operand read from LDS feeds one product (waits 59 %, matrix 21 %).

typedef short sv4 __attribute__((ext_vector_type(4)));
typedef const __attribute__((address_space(4))) int32_t* TablePtr;  // read-only for the kernel: scalar loads
typedef __attribute__((address_space(3))) uint8_t* LdsPtr;
#define RSTR_LDS(p) ((__attribute__((address_space(3))) void*)(p))

__device__ __forceinline__ u32x2 read_transposed(LdsPtr at) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) sv4*)at));
}
template <int D, class E>
__global__ void __launch_bounds__(64 * kShareWaves, kShareWaves / 4)
    k_pool_prompt(PoolAttn a, const int32_t* __restrict__ ro, const int32_t* __restrict__ lens, const int32_t* __restrict__ table, PoolPieces pc,
                  int workers, int least) {
  typedef typename E::T T;
  constexpr int NT = prompt_tiles(D, Terms<E>::n), TERMS = Terms<E>::n, WAVES = kShareWaves, COLS = 16 * NT * WAVES;
  constexpr int ROW = 2 * D, KS = D / 32, JT = D / 16, TB = kStep / 16;  // bytes of a token; products of a score, of O; 16s of tokens
  constexpr int MINE = kStep / WAVES, GROUPS = MINE / 4, LOADS = MINE * ROW / 1024;  // tokens that a wave loads, fours of them, instructions
  constexpr int BUF = kStep * ROW;                             // bytes of K or V of a step
  __shared__ __attribute__((aligned(1024))) uint8_t lds[2][2][BUF];  // buffer, K or V
  __shared__ uint32_t gone_at[2][WAVES], odd_at[2][WAVES];     // fours of tokens whose page is not there; values left out
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
  // neighbours on the line of work share keys and values: they go to the same chip (workgroups are dealt to the
  // eight of them in turn)
  const int w = uniform((int)(workers % 8 == 0 ? (blockIdx.x % 8) * (workers / 8) + blockIdx.x / 8 : blockIdx.x));
  const int n_kv = a.c.n_kv, group = a.n_q / n_kv, ps = a.c.page_size;
  const int cap = token_cap(a.pps, ps);
  const int64_t row_bytes = (int64_t)n_kv * ROW;
  const Lines L{ro, lens, a.rows, n_kv, group, a.window, COLS, cap, kPromptStart, false};
  Line line(L, a.batch, w, workers, least);
  if (w == 0 && wave == 0) *pc.n_items = line.items();

  // places in LDS
  const auto swizzle = [](int token) { return D == 64 ? (token >> 1) & 7 : token & 15; };
  const LdsPtr lds0 = (LdsPtr)RSTR_LDS(&lds[0][0][0]);
  LdsPtr k_at[KS], v_at[JT];
#pragma unroll
  for (int i = 0; i < KS; i++) k_at[i] = lds0 + col * ROW + (((4 * i + g) ^ swizzle(col)) << 4);
#pragma unroll
  for (int j = 0; j < JT; j++) {
    const int token = 4 * g + (col >> 2);
    v_at[j] = lds0 + BUF + token * ROW + (((2 * j + ((col & 3) >> 1)) ^ swizzle(token)) << 4) + (col & 1) * 8;
  }
  // the piece of a token that a lane's load asks for
  const auto piece_of = [&](int n, int& token) {  // instruction n of the wave's
    const int byte = n * 1024 + lane * 16;
    token = byte / ROW;
    return (((byte % ROW) >> 4) ^ swizzle(wave * MINE + token)) << 4;
  };

  while (line.next()) {
    const Seq& s = line.s;
    const int b = line.b, h = line.h, c0 = line.ct * COLS, p0 = s.len - s.m, held = L.held(s.len);
    const bool begins = line.begins, ends = line.ends;
    if (begins && threadIdx.x == 0) pc.begun[line.item] = Begun{b, h, line.ct, w, line.pieces};
    const auto row_of = [&](int c) { return min(s.m - 1, c / group); };
    const auto first_seen = [&](int row) { return a.window > 0 ? max(max(p0 + row + 1, 0) - a.window, 0) : 0; };
    const auto end_seen = [&](int row) { return min(max(p0 + row + 1, 0), cap); };
    const int rf = row_of(c0), rl = row_of(c0 + COLS - 1);
    const int cw = c0 + wave * 16 * NT;
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
    const bool any = cw < s.m * group;
    const int wf = row_of(cw), wl = row_of(cw + 16 * NT - 1);  // the wave's rows
    const int t0 = max(s.lo + max(line.at - kPromptStart, 0), first_seen(rf) / kTile);
    const int t1 = min(s.lo + max(line.at + line.n - kPromptStart, 0), (end_seen(rl) + kTile - 1) / kTile);
    const int part_end = t1 * kTile;
    const int g_lo = first_seen(rf), g_hi = min(end_seen(rl), part_end), g_lo_last = first_seen(rl), g_hi_first = min(end_seen(rf), part_end);
    const int w_lo = first_seen(wf), w_hi = any ? min(end_seen(wl), part_end) : 0, w_lo_last = first_seen(wl), w_hi_first = min(end_seen(wf), part_end);

    f4 acc[NT][JT];
    float mref[NT], l[NT], kcol[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) {
#pragma unroll
      for (int j = 0; j < JT; j++) acc[t][j] = f4{0, 0, 0, 0};
      mref[t] = -FLT_MAX;
      l[t] = kcol[t] = 0.0f;
    }
    if (t0 < t1) {
      const TablePtr rowp = (TablePtr)(table + (int64_t)b * a.pps);
      const int n_pages = (int)(((int64_t)held + ps - 1) / ps);
      const int step_e = kStep / ps, step_off = kStep - step_e * ps;
      // page and place in it of the wave's fours of tokens, and the page's id, read a step ahead of its use
      Place four[GROUPS];
      int id[GROUPS], id_off[GROUPS];
#pragma unroll
      for (int n = 0; n < GROUPS; n++) four[n] = place_of((uint32_t)t0 * kTile + wave * MINE + 4 * n, ps);
      const auto look = [&] {
#pragma unroll
        for (int n = 0; n < GROUPS; n++) {
          const int v = rowp[min(four[n].entry, n_pages - 1)];
          id[n] = four[n].entry < n_pages ? v : -1;
          id_off[n] = four[n].off;
          forward(four[n], step_e, step_off, ps);
        }
      };
      const uint8_t* kbase = (const uint8_t*)a.c.k + (int64_t)h * ROW;
      const uint8_t* vbase = (const uint8_t*)a.c.v + (int64_t)h * ROW;
      const auto issue = [&](int buf) {
        int64_t at[GROUPS];
        uint32_t gone = 0;
#pragma unroll
        for (int n = 0; n < GROUPS; n++) {
          const bool ok = (uint32_t)id[n] < (uint32_t)a.c.pages;
          if (!ok) gone |= 1u << n;
          at[n] = ((int64_t)(ok ? id[n] : 0) * ps + id_off[n]) * row_bytes;
        }
        if (lane == 0) gone_at[buf][wave] = gone, odd_at[buf][wave] = 0;
#pragma unroll
        for (int n = 0; n < LOADS; n++) {
          int token;
          const int piece = piece_of(n, token);
          int64_t from = at[0];
#pragma unroll
          for (int j = 1; j < GROUPS; j++) from = (D == 64 ? token >> 2 : n * 1024 / ROW / 4) == j ? at[j] : from;
          const int64_t byte = from + (int64_t)(token & 3) * row_bytes + piece;
#pragma unroll
          for (int kv = 0; kv < 2; kv++)
            __builtin_amdgcn_global_load_lds((const void*)((kv ? vbase : kbase) + byte), RSTR_LDS(&lds[buf][kv][wave * MINE * ROW + n * 1024]), 16, 0, 0);
        }
        look();
      };
      look();
      issue(0);

      h8 q[NT][TERMS][KS];
      int hi[NT], lo[NT];
      const bool vec = vec_rows(a.q, sizeof(T));
#pragma unroll
      for (int t = 0; t < NT; t++) {
        const Column c = column(t);
        const bool valid = c.row < s.m;
        hi[t] = valid ? min(end_seen(c.row), part_end) : 0;
        lo[t] = first_seen(c.row);
        float x[KS][8], big = 0.0f;
#pragma unroll
        for (int i = 0; i < KS; i++) {
          if (valid) {
            const T* src = (const T*)a.q.p + (int64_t)(s.r0 + c.row) * a.q.row + (int64_t)c.head * a.q.head + i * 32 + g * 8;
            if (vec) load8<E, true>(src, x[i]); else load8<E, false>(src, x[i]);
          } else {
#pragma unroll
            for (int k = 0; k < 8; k++) x[i][k] = 0.0f;
          }
#pragma unroll
          for (int k = 0; k < 8; k++) big = fmaxf(big, size_of(x[i][k]));
        }
        big = xor_max<32>(xor_max<16>(big));
        const int e = __builtin_amdgcn_frexp_expf(big) - 15;
        kcol[t] = score_scale(a.scale, e);
#pragma unroll
        for (int i = 0; i < KS; i++)
#pragma unroll
          for (int k = 0; k < 8; k++) {
            float y = __builtin_amdgcn_ldexpf(x[i][k], -e);
            y = a.scale < 0.0f ? -y : a.scale == 0.0f ? y * 0.0f : y;
            if constexpr (TERMS == 2) {
              q[t][0][i][k] = first_term(y);
              q[t][1][i][k] = second_term(y, q[t][0][i][k]);
            } else {
              q[t][0][i][k] = (_Float16)y;
            }
          }
      }

      // A weight of 0 times an infinity or a NaN: of values whose token some column of the workgroup does not see, those that are no
      // numbers become 0 where they were loaded; odd_at says that there were some of tokens that others see.
      const auto partly = [&](int tok) { return tok >= g_lo && tok < g_hi && !(tok >= g_lo_last && tok < g_hi_first); };
      const auto mend = [&](int buf, int tok0) {
        uint32_t odd = 0;
        const uint32_t gone = gone_at[buf][wave];
#pragma unroll
        for (int n = 0; n < LOADS; n++) {
          const int token = (n * 1024 + lane * 16) / ROW, tok = tok0 + wave * MINE + token;
          const bool there = !((gone >> (token >> 2)) & 1);
          __attribute__((address_space(3))) u32x4* at = (__attribute__((address_space(3))) u32x4*)(lds0 + (buf * 2 + 1) * BUF + wave * MINE * ROW + n * 1024 + lane * 16);
          u32x4 x = *at;
          uint32_t bad = 0;
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const uint32_t halves = ((((x[i] & 0x7C007C00u) + 0x04000400u) >> 15) & 0x10001u) * 0xFFFFu;  // exponents of all ones
            x[i] &= ~halves;
            bad |= halves;
          }
          const bool all = there && tok >= g_lo_last && tok < g_hi_first;
          if (bad != 0 && !all) {
            *at = x;
            if (there && partly(tok)) odd = 1;
          }
        }
        if (__ballot(odd != 0) && lane == 0) odd_at[buf][wave] = 1;
      };

      // one step: tokens [tok0, tok0 + 64) from buffer `buf`; edge: some column does not see some of them
      const auto compute = [&](bool edge, int buf, int tok0) {
        const int base = buf * (2 * BUF);
        f4 sc[NT][TB];
#pragma unroll
        for (int tb = 0; tb < TB; tb++) {
#pragma unroll
          for (int t = 0; t < NT; t++) sc[t][tb] = f4{0, 0, 0, 0};
#pragma unroll
          for (int i = 0; i < KS; i++) {
            const h8 k = __builtin_bit_cast(h8, *(__attribute__((address_space(3))) u32x4*)(k_at[i] + base + tb * 16 * ROW));
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
              for (int u = 0; u < TERMS; u++) sc[t][tb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, q[t][u][i], sc[t][tb], 0, 0, 0);
          }
        }
        if (edge) {
          asm volatile("");  // stays a branch
          // bits of the lane's tokens (bit 4 tb + i is token 16 tb + 4 g + i of the step)
          const auto below = [&](int end) {
            uint32_t o = 0;
#pragma unroll
            for (int tb = 0; tb < TB; tb++) o |= ((1u << min(max(end - tok0 - 16 * tb - 4 * g, 0), 4)) - 1u) << (4 * tb);
            return o;
          };
          uint32_t here = ~0u;
#pragma unroll
          for (int tb = 0; tb < TB; tb++) {
            const int n = 16 * tb + 4 * g;
            if ((gone_at[buf][n / MINE] >> (n % MINE / 4)) & 1) here &= ~(15u << (4 * tb));
          }
#pragma unroll
          for (int t = 0; t < NT; t++) {
            const uint32_t see = below(hi[t]) & ~below(lo[t]) & here;
#pragma unroll
            for (int tb = 0; tb < TB; tb++)
#pragma unroll
              for (int i = 0; i < 4; i++) sc[t][tb][i] = (see >> (4 * tb + i)) & 1 ? sc[t][tb][i] : -INFINITY;
          }
        }
        float m[NT];
        bool passed[NT], grow = false;
#pragma unroll
        for (int t = 0; t < NT; t++) {
          m[t] = -INFINITY;
#pragma unroll
          for (int tb = 0; tb < TB; tb++)
#pragma unroll
            for (int i = 0; i < 4; i++) m[t] = __builtin_elementwise_maximum(m[t], sc[t][tb][i]);  // (a NaN is in the column's sums anyhow)
          passed[t] = __builtin_fmaf(m[t] - mref[t], kcol[t], 10.0f) > 14.0f;
          grow |= passed[t];
        }
        if (__ballot(grow)) {
#pragma unroll
          for (int t = 0; t < NT; t++) {
            // a column that needs no change has none: it does not depend on its neighbours
            const bool own = of_column(__ballot(passed[t]));
            const float top = xor_max<32>(xor_max<16>(m[t])), now = own ? fmaxf(top, mref[t]) : mref[t];
            const float keep = own ? __builtin_amdgcn_exp2f((mref[t] - now) * kcol[t]) : 1.0f;
            mref[t] = now;
            l[t] *= keep;
#pragma unroll
            for (int j = 0; j < JT; j++) acc[t][j] *= keep;
          }
        }
        h8 ph[NT][TB / 2][TERMS];
#pragma unroll
        for (int u = 0; u < TB / 2; u++)
#pragma unroll
          for (int t = 0; t < NT; t++) {
            float p[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
              p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][2 * u + (i >> 2)][i & 3] - mref[t], kcol[t], 10.0f));
              if constexpr (TERMS == 2) {
                ph[t][u][0][i] = first_term(p[i]);
                ph[t][u][1][i] = (_Float16)(p[i] - (float)ph[t][u][0][i]);
              } else {
                ph[t][u][0][i] = (_Float16)p[i];
              }
            }
            if constexpr (TERMS == 2) {
              l[t] += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
            } else {
#pragma unroll
              for (int i = 0; i < 4; i++) l[t] = __builtin_amdgcn_fdot2(h2{ph[t][u][0][2 * i], ph[t][u][0][2 * i + 1]}, h2{(_Float16)1.0f, (_Float16)1.0f}, l[t], false);
            }
#pragma unroll
            for (int x = 0; x < TERMS; x++) asm("" : "+v"(ph[t][u][x]));  // packed from here on, also for what hardly ever needs them singly
          }
#pragma unroll
        for (int u = 0; u < TB / 2; u++)
#pragma unroll
          for (int j = 0; j < JT; j++) {
            u32x4 o;
#pragma unroll
            for (int b2 = 0; b2 < 2; b2++) {
              const u32x2 x = read_transposed(v_at[j] + base + (32 * u + 16 * b2) * ROW);
              o[2 * b2] = x[0];
              o[2 * b2 + 1] = x[1];
            }
            const h8 v = __builtin_bit_cast(h8, o);
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
              for (int x = 0; x < TERMS; x++) acc[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, ph[t][u][x], acc[t][j], 0, 0, 0);
          }
        uint32_t odd = 0;
        if (edge || tok0 < g_lo_last || tok0 + kStep > g_hi_first)  // also where this wave's own columns see all of the step
#pragma unroll
          for (int i = 0; i < WAVES; i++) odd |= odd_at[buf][i];
        if (uniform(odd)) {  // values that mend() left out, for the columns that see them
          const TablePtr pages = (TablePtr)(table + (int64_t)b * a.pps);
#pragma unroll 1
          for (int n = 0; n < kStep; n++) {
            const int tok = tok0 + n;
            if (!uniform(odd_at[buf][n / MINE]) || !partly(tok)) continue;
            const int e = tok / ps, id = pages[e];
            if ((uint32_t)id >= (uint32_t)a.c.pages) continue;
            const uint16_t* v = a.c.v + (((int64_t)id * ps + (tok - e * ps)) * n_kv + h) * D + 4 * g;
            const int reg = 4 * (n >> 4) + (n & 3);
#pragma unroll
            for (int t = 0; t < NT; t++) {
              float mine = 0.0f;
#pragma unroll
              for (int k = 0; k < 4 * TB; k++) {
                float p = (float)ph[t][k >> 3][0][k & 7];
                if constexpr (TERMS == 2) p += (float)ph[t][k >> 3][1][k & 7];
                mine = k == reg ? p : mine;
              }
              mine = __shfl(mine, ((n >> 2) & 3) * 16 + col, 64);
              const bool sees = tok >= lo[t] && tok < hi[t];
#pragma unroll
              for (int j = 0; j < JT; j++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                  const uint16_t x = v[16 * j + i];
                  if (sees && (x & 0x7C00u) == 0x7C00u) acc[t][j][i] = __builtin_fmaf(mine, (float)__builtin_bit_cast(_Float16, x), acc[t][j][i]);
                }
            }
          }
        }
      };

      int buf = 0;
      for (int tok0 = t0 * kTile; tok0 < part_end; tok0 += kStep) {
        wait_vmem();
        if (tok0 < g_lo_last || tok0 + kStep > g_hi_first || uniform(gone_at[buf][wave]) != 0) mend(buf, tok0);
        __syncthreads();  // this step's tokens are there, and the other buffer is free
        if (tok0 + kStep < part_end) issue(buf ^ 1);
        if (tok0 < w_hi && tok0 + kStep > w_lo) {
          uint32_t gone = 0;
#pragma unroll
          for (int i = 0; i < WAVES; i++) gone |= gone_at[buf][i];
          compute(tok0 < w_lo_last || tok0 + kStep > w_hi_first || uniform(gone) != 0, buf, tok0);
        }
        buf ^= 1;
      }
      __syncthreads();  // the buffers are the next part's
    }

    const int64_t piece = piece_place(w, begins) * COLS;
#pragma unroll
    for (int t = 0; t < NT; t++) {
      const float sum = xor_add<32>(xor_add<16>(l[t]));
      const Column at = column(t);
      if (at.row >= s.m) continue;
      if (begins && ends) {
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        T* dst = (T*)a.out.p + (int64_t)(s.r0 + at.row) * a.out.row + (int64_t)at.head * a.out.head + 4 * g;
        const bool ovec = vec_rows(a.out, sizeof(T));
#pragma unroll
        for (int j = 0; j < JT; j++) {
          T o[4];
#pragma unroll
          for (int k = 0; k < 4; k++) o[k] = E::put(acc[t][j][k] * inv);
          if (ovec) {
            if constexpr (sizeof(T) == 4) *(u32x4*)(dst + 16 * j) = *(u32x4*)o;
            else *(u32x2*)(dst + 16 * j) = *(u32x2*)o;
          } else {
#pragma unroll
            for (int k = 0; k < 4; k++) dst[16 * j + k] = o[k];
          }
        }
      } else {
        const int64_t c = piece + (wave * NT + t) * 16 + col;
        if (g == 0) pc.ml[c] = f4{mref[t], sum, kcol[t], 0.0f};
        if (sum == 0.0f) continue;
#pragma unroll
        for (int j = 0; j < JT; j++) *(f4*)(pc.acc + c * D + 16 * j + 4 * g) = acc[t][j];
      }
    }
  }
}

// An item whose pieces are joined: where they are, and where the result goes.
template <bool LISTED>
struct Joined {
  int n, c0, r0, m, h;
  int64_t first, rest;  // the first piece, and what the ones behind it are counted from
  __device__ bool find(const PoolAttn& a, const Lines& L, const PoolPieces& pc, int item, int parts) {
    if constexpr (LISTED) {
      const int ncts = (L.group + L.cols - 1) / L.cols, row = item / (L.n_kv * ncts), hc = item - row * (L.n_kv * ncts);
      const RowOf of(L.ro, L.lens, a.batch, a.rows, row);
      if (of.b < 0) return false;
      n = parts;
      h = hc / ncts;
      c0 = (hc - h * ncts) * L.cols;
      r0 = row;
      m = 1;
      first = rest = (int64_t)item * parts;
    } else {
      const int items = *pc.n_items;
      const Begun it = pc.begun[item];  // (of an item that is not: whatever is there)
      n = it.pieces;
      if (item >= items || n == 0) return false;
      h = it.h;
      c0 = it.ct * L.cols;
      const int32_t* ro = L.ro + it.b;
      r0 = min(max(ro[0], 0), L.rows);
      m = max(min(max(ro[1], 0), L.rows) - r0, 0);
      first = piece_place(it.w, true);
      rest = piece_place(it.w, false);
    }
    return true;
  }
  __device__ int64_t slot(const Lines& L, int i, int c) const { return (i == 0 ? first : LISTED ? rest + i : rest + 2 * i) * L.cols + c; }
  __device__ int64_t out_at(const PoolAttn& a, const Lines& L, int c) const {
    const int cc = c0 + c, r = cc / L.group;
    return (int64_t)(r0 + r) * a.out.row + ((int64_t)h * L.group + (cc - r * L.group)) * a.out.head;
  }
};

// Joins the pieces of an item, in their order: a workgroup a column (more where a sequence has more rows than the call said), its waves by piece.
template <int D, class E, bool LISTED>
__global__ void k_pool_merge(PoolAttn a, Lines L, PoolPieces pc, int parts) {
  constexpr int V = D / 64;  // dims a lane
  typedef typename E::T T;
  __shared__ float part[16][D];
  __shared__ float pl[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, share = blockDim.x >> 6;
  Joined<LISTED> it;
  if (!it.find(a, L, pc, blockIdx.x, parts)) return;
  for (int c = blockIdx.y; c < L.cols && (it.c0 + c) / L.group < it.m; c += gridDim.y) {  // the same for all waves
    float acc[V] = {}, l = 0.0f, top = -FLT_MAX;
    for (int i = lane; i < it.n; i += 64) {
      const f4 y = pc.ml[it.slot(L, i, c)];
      if (y[1] != 0.0f) top = fmaxf(top, y[0]);
    }
    top = wave_max(top);
    for (int i0 = wave; i0 < it.n; i0 += 8 * share) {
      f4 x[8];
      float v[8][V];
#pragma unroll
      for (int k = 0; k < 8; k++) {  // all loads before the first use
        const int64_t p = it.slot(L, min(i0 + k * share, it.n - 1), c);
        x[k] = pc.ml[p];
#pragma unroll
        for (int j = 0; j < V; j++) v[k][j] = pc.acc[p * D + lane * V + j];
      }
#pragma unroll
      for (int k = 0; k < 8; k++) {
        const bool some = i0 + k * share < it.n && x[k][1] != 0.0f;
        const float f = some ? __builtin_amdgcn_exp2f((x[k][0] - top) * x[k][2]) : 0.0f;
        l = __builtin_fmaf(f, some ? x[k][1] : 0.0f, l);
#pragma unroll
        for (int j = 0; j < V; j++) acc[j] = __builtin_fmaf(f, some ? v[k][j] : 0.0f, acc[j]);
      }
    }
    __syncthreads();  // the column before has been read
#pragma unroll
    for (int j = 0; j < V; j++) part[wave][lane * V + j] = acc[j];
    if (lane == 0) pl[wave] = l;
    __syncthreads();
    if (wave != 0) continue;
    for (int k = 1; k < share; k++) {
#pragma unroll
      for (int j = 0; j < V; j++) acc[j] += part[k][lane * V + j];
      l += pl[k];
    }
    T* dst = (T*)a.out.p + it.out_at(a, L, c) + lane * V;
#pragma unroll
    for (int j = 0; j < V; j++) dst[j] = E::put(l == 0.0f ? 0.0f : acc[j] / l);
  }
}

// The same where items have few pieces or there are columns enough: D / 4 lanes a column, four dims each, pieces one after the other.
// Nothing waits for the greatest reference of all pieces: sums that are there are scaled as it grows.  1333 rows of 32 heads, bf16, 55 MB
// of pieces: 11.6 us (a wave a column as above 32 us).
template <int D, class E, bool LISTED>
__global__ void __launch_bounds__(256) k_pool_join(PoolAttn a, Lines L, PoolPieces pc, int parts) {
  constexpr int LANES = D / 4, PER = 256 / LANES, AT_ONCE = 4;  // lanes a column, columns at a time, pieces at a time
  typedef typename E::T T;
  Joined<LISTED> it;
  if (!it.find(a, L, pc, blockIdx.x, parts)) return;
  const int d = threadIdx.x % LANES * 4;
  const bool ovec = vec_rows(a.out, sizeof(T));
  for (int c = blockIdx.y * PER + threadIdx.x / LANES; c < L.cols && (it.c0 + c) / L.group < it.m; c += gridDim.y * PER) {
    f4 acc = f4{0, 0, 0, 0};
    float l = 0.0f, top = -FLT_MAX;
    for (int i0 = 0; i0 < it.n; i0 += AT_ONCE) {
      f4 x[AT_ONCE], v[AT_ONCE];
#pragma unroll
      for (int k = 0; k < AT_ONCE; k++) {
        x[k] = v[k] = f4{0, 0, 0, 0};
        if (i0 + k < it.n) {
          const int64_t p = it.slot(L, i0 + k, c);
          x[k] = pc.ml[p];
          v[k] = *(const f4*)(pc.acc + p * D + d);
        }
      }
      float now = top, scale = 0.0f;
#pragma unroll
      for (int k = 0; k < AT_ONCE; k++)
        if (x[k][1] != 0.0f) now = fmaxf(now, x[k][0]), scale = x[k][2];  // (a column's scale is the same in all)
      const float keep = __builtin_amdgcn_exp2f((top - now) * scale);
      top = now;
      l *= keep;
      acc *= keep;
#pragma unroll
      for (int k = 0; k < AT_ONCE; k++) {
        const bool some = x[k][1] != 0.0f;
        const float f = some ? __builtin_amdgcn_exp2f((x[k][0] - top) * x[k][2]) : 0.0f;
        l = __builtin_fmaf(f, some ? x[k][1] : 0.0f, l);
#pragma unroll
        for (int j = 0; j < 4; j++) acc[j] = __builtin_fmaf(f, some ? v[k][j] : 0.0f, acc[j]);
      }
    }
    T* dst = (T*)a.out.p + it.out_at(a, L, c) + d;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    T o[4];
#pragma unroll
    for (int j = 0; j < 4; j++) o[j] = E::put(acc[j] * inv);
    if (ovec) {
      if constexpr (sizeof(T) == 4) *(u32x4*)dst = *(u32x4*)o;
      else *(u32x2*)dst = *(u32x2*)o;
    } else {
#pragma unroll
      for (int j = 0; j < 4; j++) dst[j] = o[j];
    }
  }
}

// ---- launches ------------------------------------------------------------------------
constexpr int kMergeWaves = 4096;
PoolPieces pool_pieces(void* ws, int64_t items, int64_t columns, int hd) {
  const PoolRoom r = pool_room(sizeof(Begun), items, columns, hd);
  char* p = (char*)ws;
  return PoolPieces{(int*)p, (Begun*)(p + r.begun), (f4*)(p + r.ml), (float*)(p + r.acc)};
}

template <int D, class E, bool LISTED>
hipError_t merge(hipStream_t st, const PoolAttn& a, const PoolPieces& pc, int64_t items, int64_t pieces, int cols, int parts) {
  const int group = a.n_q / a.c.n_kv;
  const int cap = token_cap(a.pps, a.c.page_size);
  const Lines L{a.row_offsets, a.lengths, a.rows, a.c.n_kv, group, a.window, cols, cap, kStart, false};
  // Waves a column: more where an item has many pieces, but not where there are columns enough to fill the card.
  const int64_t columns = std::min<int64_t>(cols, LISTED ? group : (int64_t)a.max_rows * group);
  const int each = (int)(pieces / items);
  int share = each >= 16 ? 16 : each >= 4 ? 4 : 1;
  while (share > 1 && items * columns * share > kMergeWaves) share /= 4;
  constexpr int per = 1024 / D;
  if (share == 1) hipLaunchKernelGGL((k_pool_join<D, E, LISTED>), dim3((unsigned)items, (unsigned)((columns + per - 1) / per)), dim3(256), 0, st, a, L, pc, parts);
  else hipLaunchKernelGGL((k_pool_merge<D, E, LISTED>), dim3((unsigned)items, (unsigned)columns), dim3(64 * share), 0, st, a, L, pc, parts);
  return hipGetLastError();
}

template <int D, int NT, class E>
hipError_t attn_tiles(hipStream_t st, const PoolAttn& a, const PoolForm& f) {
  const PoolPieces pc = pool_pieces(a.ws, f.items, 2 * f.workers * f.cols, D);
  hipLaunchKernelGGL((k_pool_attn<D, NT, E, 0>), dim3((unsigned)(f.workers / 4)), dim3(256), 0, st, a, a.row_offsets, a.lengths, a.page_table,
                     pc, (int)f.workers, f.whole ? 1 : kLeast, f.whole, 0);
  const hipError_t e = hipGetLastError();
  return e != hipSuccess || f.whole ? e : merge<D, E, false>(st, a, pc, f.items, f.workers, f.cols, 0);
}

template <int D, class E>
hipError_t attn_prompt(hipStream_t st, const PoolAttn& a, const PoolForm& f) {
  const PoolPieces pc = pool_pieces(a.ws, f.items, 2 * f.workers * f.cols, D);
  hipLaunchKernelGGL((k_pool_prompt<D, E>), dim3((unsigned)f.workers), dim3(64 * kShareWaves), 0, st, a, a.row_offsets, a.lengths, a.page_table, pc,
                     (int)f.workers, kPromptLeast);
  const hipError_t e = hipGetLastError();
  return e != hipSuccess ? e : merge<D, E, false>(st, a, pc, f.items, f.workers, f.cols, 0);
}

template <int D, class E>
hipError_t attn_listed(hipStream_t st, const PoolAttn& a) {
  const Cut c = listed_cut(a.n_q, a.c.n_kv, D, a.rows, a.top, a.pps, a.c.page_size, compute_units());
  const PoolPieces pc = pool_pieces(a.ws, 0, c.items * c.parts * 16, D);
  auto f = c.waves > 1 ? k_pool_attn<D, 1, E, listed_waves(D)> : k_pool_attn<D, 1, E, 1>;
  hipLaunchKernelGGL(f, dim3((unsigned)c.groups()), dim3(64 * (c.waves > 1 ? c.waves : 4)), 0, st, a, a.row_offsets, a.lengths, a.page_table,
                     pc, (int)c.groups(), c.tiles, c.parts == 1, c.parts);
  const hipError_t e = hipGetLastError();
  return e != hipSuccess || c.parts == 1 ? e : merge<D, E, true>(st, a, pc, c.items, c.items * c.parts, 16, c.parts);
}

template <int D, class E>
hipError_t attn_dim(hipStream_t st, const PoolAttn& a) {
  if (a.blocks) return attn_listed<D, E>(st, a);
  const PoolForm f = pool_form(D, Terms<E>::n, a.n_q, a.c.n_kv, a.batch, a.rows, a.max_rows, token_cap(a.pps, a.c.page_size), compute_units());
  if (f.prompt) return attn_prompt<D, E>(st, a, f);
  if constexpr (D != 256 && Terms<E>::n == 1)
    if (f.nt == 2) return attn_tiles<D, 2, E>(st, a, f);
  return attn_tiles<D, 1, E>(st, a, f);
}

template <class E>
hipError_t attn_type(hipStream_t st, const PoolAttn& a) {
  if (a.c.hd == 64) return attn_dim<64, E>(st, a);
  if (a.c.hd == 128) return attn_dim<128, E>(st, a);
  return attn_dim<256, E>(st, a);
}

}  // namespace

size_t pool_attn_workspace(int n_q, int n_kv, int hd, int batch, int rows) {
  return pool_attn_room(sizeof(Begun), n_q, n_kv, hd, batch, rows, compute_units());
}

hipError_t launch_pool_attn(hipStream_t st, int dtype, const PoolAttn& a) {
  if (a.rows == 0 || a.batch == 0) return hipSuccess;
  if (dtype == RSTR_F32) return attn_type<F32>(st, a);
  if (dtype == RSTR_F16) return attn_type<F16>(st, a);
  return attn_type<BF16>(st, a);
}

}  // namespace rstr
