// What the sources of the expert_* targets share: types of 16 and 32 bits, pieces of 16 bytes at any element, and the
// checks of a call.  Everything computes in 32 bits; a result is rounded once, to nearest even, when it is stored.
#pragma once

#include "common.h"

namespace bpl {

using half_t = _Float16;
using bfloat_t = __bf16;

constexpr uint32_t kMostExperts = 1024;
constexpr uint32_t kMostPerToken = 64;  // one pair of a token to a lane

template <typename T>
struct Piece {
  static constexpr uint32_t kElems = 16 / sizeof(T);
  typedef T type __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
};

// Elements col .. col + kElems - 1 of a row of `width`, zero beyond its end.  (The row may begin at any element: loads of
// 16 bytes need no alignment here, and nothing beyond the row is touched.)  WHOLE: the row is known to end with a piece, so
// that there is no other way to take.  ONCE: what is read once, and is to take no room in the caches from what is not.
template <typename T, bool WHOLE = false, bool ONCE = false>
__device__ __forceinline__ typename Piece<T>::type load_piece(const T *__restrict__ row, uint32_t col, uint32_t width) {
  typename Piece<T>::type v;
  if (WHOLE || col + Piece<T>::kElems <= width) {
    const auto *const from = reinterpret_cast<const typename Piece<T>::type *>(row + col);
    v = ONCE ? __builtin_nontemporal_load(from) : *from;
  } else {
#pragma unroll
    for (uint32_t j = 0; j < Piece<T>::kElems; ++j) v[j] = col + j < width ? row[col + j] : static_cast<T>(0.f);
  }
  return v;
}

// PAST: past the caches, for results larger than they are (kept there, they only push out what is read again).
template <typename T, bool WHOLE = false, bool PAST = false>
__device__ __forceinline__ void store_piece(T *__restrict__ row, uint32_t col, uint32_t width, typename Piece<T>::type v) {
  if (WHOLE || col + Piece<T>::kElems <= width) {
    auto *const to = reinterpret_cast<typename Piece<T>::type *>(row + col);
    if (PAST)
      __builtin_nontemporal_store(v, to);
    else
      *to = v;
  } else {
#pragma unroll
    for (uint32_t j = 0; j < Piece<T>::kElems; ++j)
      if (col + j < width) row[col + j] = v[j];
  }
}

inline bool expert_limits(const char *target, const bpl_expert_descriptor &d) {
  constexpr uint64_t kMost = 0x7fffffffu;
  if (d.experts < 1 || d.experts > kMostExperts) {
    set_error("%s: 1 to %u experts, got %u", target, kMostExperts, d.experts);
    return false;
  }
  if (d.per_token > kMostPerToken) {
    set_error("%s: at most %u experts a token, got %u", target, kMostPerToken, d.per_token);
    return false;
  }
  if (d.tokens > kMost || d.rows > kMost || d.width > kMost || d.out > kMost ||
      static_cast<uint64_t>(d.tokens) * d.per_token > kMost) {
    set_error("%s: tokens * k, rows and widths are at most 2^31 - 1", target);
    return false;
  }
  return true;
}

// One definition for each of the three element types: NAME_float, NAME_half, NAME_bfloat16 call FN<type>.
#define BPL_EXPERT_DEFINE(NAME, FN)                                                                     \
  BPL_TARGET(NAME##_float) { FN<float>(#NAME "_float", static_cast<hipStream_t>(stream), buffers, opaque, opaque_len); } \
  BPL_TARGET(NAME##_half) { FN<bpl::half_t>(#NAME "_half", static_cast<hipStream_t>(stream), buffers, opaque, opaque_len); } \
  BPL_TARGET(NAME##_bfloat16) { FN<bpl::bfloat_t>(#NAME "_bfloat16", static_cast<hipStream_t>(stream), buffers, opaque, opaque_len); }

}  // namespace bpl
