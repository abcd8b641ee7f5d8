// device_args.h -- what the C entries of the operators on device arrays share: the stream of a call, and the checks of arrays that the host can see.
#pragma once
#include <hip/hip_runtime.h>

#include <string>

#include "kv4.h"
#include "session.h"

namespace rstr {
namespace {

inline hipStream_t on_stream(rstr_session* s, void* stream) {
  return stream == RSTR_SESSION_STREAM ? s->stream : (hipStream_t)stream;
}

inline int elem_size(int dtype) { return dtype == RSTR_F32 ? 4 : dtype == RSTR_F16 || dtype == RSTR_BF16 ? 2 : 0; }

inline bool aligned(const void* p, size_t n) { return ((uintptr_t)p % n) == 0; }

// One past the last byte that `rows` rows of `heads` heads reach.
inline uintptr_t rows_end(const Rows& r, int64_t rows, int64_t heads, int64_t hd, int size) {
  return (uintptr_t)r.p + (uintptr_t)(((rows - 1) * r.row + (heads - 1) * r.head + hd) * size);
}

// Strides of a written array: no two of its rows may share an element.
inline bool apart(const Rows& r, int64_t rows, int64_t heads, int64_t hd) {
  const bool heads_in = (heads == 1 || r.head >= hd) && (rows == 1 || r.row >= (heads - 1) * r.head + hd);
  const bool rows_in = (rows == 1 || r.row >= hd) && (heads == 1 || r.head >= (rows - 1) * r.row + hd);
  return heads_in || rows_in;
}

inline bool ranges_meet(uintptr_t a0, uintptr_t a1, uintptr_t b0, uintptr_t b1) { return a0 < b1 && b0 < a1; }
inline bool ranges_meet(const void* a, size_t an, const void* b, size_t bn) {
  return ranges_meet((uintptr_t)a, (uintptr_t)a + an, (uintptr_t)b, (uintptr_t)b + bn);
}

// Do two arrays of one shape share an element?  Where their ranges meet they do not if, on the same
// strides, one lies in the gaps of the other: between its rows or its heads.
inline bool share(const Rows& a, const Rows& b, int64_t rows, int64_t heads, int64_t hd, int size) {
  if (!ranges_meet((uintptr_t)a.p, rows_end(a, rows, heads, hd, size), (uintptr_t)b.p, rows_end(b, rows, heads, hd, size))) return false;
  const uintptr_t bytes = a.p < b.p ? (uintptr_t)b.p - (uintptr_t)a.p : (uintptr_t)a.p - (uintptr_t)b.p;
  if (a.row != b.row || a.head != b.head || bytes % size) return true;
  const int64_t d = (int64_t)(bytes / size);
  const auto between = [&](int64_t stride, int64_t span) { return stride > 0 && d % stride >= span && d % stride + span <= stride; };
  return !(between(a.row, (heads - 1) * a.head + hd) || between(a.head, (rows - 1) * a.row + hd) ||
           (a.head > 0 && a.row % a.head == 0 && between(a.head, hd)) || (a.row > 0 && a.head % a.row == 0 && between(a.row, hd)));
}

inline int check_rows(rstr_session* s, const char* what, const Rows& r, int size) {
  if (!r.p) return fail(s, RSTR_E_INVALID, std::string("null ") + what + " rows");
  if (!aligned(r.p, size)) return fail(s, RSTR_E_INVALID, std::string(what) + " rows are not aligned to their elements");
  if (r.row < 0 || r.head < 0) return fail(s, RSTR_E_INVALID, std::string(what) + " strides must not be negative");
  return RSTR_OK;
}

inline int check_ints(rstr_session* s, const char* what, const int32_t* p) {
  if (!p) return fail(s, RSTR_E_INVALID, std::string("null ") + what);
  if (!aligned(p, 4)) return fail(s, RSTR_E_INVALID, std::string(what) + " not aligned to its elements");
  return RSTR_OK;
}

constexpr int64_t kGridGroups = 1 << 24;  // workgroups of 256 threads that a grid cannot hold any more

#define TRY(expr)                \
  do {                           \
    const int rc_ = (expr);      \
    if (rc_ != RSTR_OK) return rc_; \
  } while (0)

}  // namespace
}  // namespace rstr
