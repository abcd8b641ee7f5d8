// kv4.h -- launch interface of the 4-bit paged K/V cache: append, read and
// attention, and of the serving-step operators (step maps, draft verification).
//
// Cache format.  32 consecutive elements of a head's row are one block: an
// fp16 scale d and 32 codes c of 4 bits; an element stands for d * (c - 8).
// d = fp16(-m / 8) for the element m of greatest magnitude (the first of
// equals), at most 65504 in magnitude; c = clamp(rne(x / d) + 8, 0, 15), 8 where d is 0.  A
// block that holds a NaN or an infinity has d = NaN.
//
// One record of kv4_record_bytes per (page, kv head), at
// layer base + (page * n_kv + head) * record, holds ps tokens (ps % 16 == 0):
//   K codes   dword (token, block b, g = k/8 of the block): eight codes.  Code
//             2i is nibble i, code 2i+1 nibble 4+i, so (w >> 4i) & 0x000F000F
//             is a pair of neighbours.  Order [token / 16][b / BQ][g][token % 16][b % BQ],
//             BQ = min(D/32, 4): a matrix operand of 16 tokens x 128 dims is 1 KB, 16
//             bytes a lane in the lanes' order.
//   V codes   halfword (token group tg = token/4, block pair bp, c = k%16, j =
//             token%4): nibbles of dims c and 16+c of block 2bp, then of block
//             2bp+1.  Order [tg][bp / BP][c][bp % BP][j], BP = min(D/64, 2): four
//             tokens' codes of one column are neighbours, which is the order
//             in which the score product leaves its probabilities in a lane.
//   K scales, V scales   fp16 [tg][block][j].
// Everything a lane loads in one instruction is consecutive, and a tile's loads
// cover whole records; records are multiples of 128 bytes.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace rstr {

// One layer of a cache.
struct Kv4Layer {
  uint8_t* base;
  int n_kv, hd, page_size, pages;
};
__host__ __device__ inline int64_t kv4_record_bytes(int hd, int page_size) { return (int64_t)page_size * hd * 9 / 8; }
inline bool kv4_head_dim(int hd) { return hd == 64 || hd == 128 || hd == 256; }

// Rows [rows][heads][hd] of a device array: element type (RSTR_F32, RSTR_F16,
// RSTR_BF16) and strides in elements; hd is contiguous.
struct Rows {
  void* p;
  int64_t row, head;
};

hipError_t launch_kv4_append(hipStream_t st, const Kv4Layer& c, int dtype, int rows, const Rows& k, const Rows& v,
                             const int32_t* slots);
hipError_t launch_kv4_read(hipStream_t st, const Kv4Layer& c, int dtype, int rows, const int32_t* slots, const Rows& k,
                           const Rows& v);

struct Kv4Attn {
  Kv4Layer c;
  int n_q, batch, rows, max_rows, window, pps;
  float scale;
  Rows q, out;
  const int32_t *row_offsets, *page_table, *lengths;
  void* ws;
};
// Bytes of workspace that every call of up to `rows` query rows and `batch`
// sequences can need.
size_t kv4_attn_workspace(int n_q, int n_kv, int hd, int batch, int rows);
hipError_t launch_kv4_attn(hipStream_t st, int dtype, const Kv4Attn& a);

struct StepMaps {
  int page_size, batch, pps, rows, n_free;
  const int32_t *lengths, *counts, *starts, *free_pages;
  int32_t *page_table, *new_lengths, *row_offsets, *positions, *slots, *taken;
};
hipError_t launch_step_maps(hipStream_t st, const StepMaps& m);

struct Verify {
  int batch, rows, vocab;
  const void* logits;
  int64_t logits_row;
  const int32_t *row_offsets, *drafts;
  const float* probs;
  int64_t probs_row;
  const float *temperature, *u_accept, *u_sample;
  int32_t *accepted, *tokens;
  void* ws;
};
size_t verify_workspace(int batch, int rows, int vocab);
hipError_t launch_verify(hipStream_t st, int dtype, const Verify& v);

}  // namespace rstr
