// Rows of scores: element types, loads of any alignment, and the argument checks that the entry points share.
#pragma once
#include <string.h>

#include <algorithm>

#include "sky_common.h"

namespace sky {

// A 16-byte piece of a row.  Rows begin wherever their stride puts them, so that a piece need not be aligned to more than an
// element: global memory takes such vector loads and stores as they are (an access more where a piece straddles two lines).
template <typename T>
struct Piece {
  static constexpr int N = 16 / (int)sizeof(T);
  T e[N];
};
// (As words: of elements the compiler makes four loads.)
template <typename T>
__device__ __forceinline__ Piece<T> load_piece(const T* p) {
  uint4 w;
  __builtin_memcpy(&w, p, 16);
  return __builtin_bit_cast(Piece<T>, w);
}
template <typename T>
__device__ __forceinline__ void store_piece(T* p, const Piece<T>& v) {
  const uint4 w = __builtin_bit_cast(uint4, v);
  __builtin_memcpy(p, &w, 16);
}

// NaN and -inf are -inf (not there), +inf is the largest number, -0 is 0: what is left compares as the order of a row asks.
__device__ __forceinline__ float plain_score(float x) {
  x = x >= -3.402823466e38f ? x : -__builtin_inff();
  return fminf(x, 3.402823466e38f) + 0.0f;
}
// A whole number that ascends with the score.
__device__ __forceinline__ uint32_t score_key(float x) {
  const uint32_t b = __float_as_uint(x);
  return b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float key_score(uint32_t k) { return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xFFFFFFFFu)); }

inline size_t dtype_size(int dtype) { return dtype == SKY_F32 ? 4 : dtype == SKY_F16 || dtype == SKY_BF16 ? 2 : 0; }

// A matrix argument: its stride is filled in, and refused where rows would overlap or elements be split.
inline int check_rows(const char* who, const char* name, const void* p, int dtype, uint32_t rows, uint32_t columns, uint64_t* stride) {
  const size_t size = dtype_size(dtype);
  if (!size) return fail(SKY_ERR_ARG, std::string(who) + ": dtype is none of SKY_F32, SKY_F16, SKY_BF16");
  if (rows > 0x7FFFFFFFu || columns > 0x7FFFFFFFu) return fail(SKY_ERR_LIMIT, std::string(who) + ": more than 2^31 - 1 rows or columns");
  if (!*stride) *stride = columns;
  if (*stride < columns) return fail(SKY_ERR_ARG, std::string(who) + ": the stride of " + name + " is smaller than a row");
  if (rows && columns && !p) return fail(SKY_ERR_ARG, std::string(who) + ": " + name + " is null");
  if ((uintptr_t)p % size) return fail(SKY_ERR_ARG, std::string(who) + ": " + name + " is not aligned to its elements");
  if (rows && *stride > (1ull << 46) / rows) return fail(SKY_ERR_LIMIT, std::string(who) + ": " + name + " is too large");
  return SKY_OK;
}
inline int check_aligned(const char* who, const char* name, const void* p, size_t size) {
  if ((uintptr_t)p % size) return fail(SKY_ERR_ARG, std::string(who) + ": " + name + " is not aligned to its elements");
  return SKY_OK;
}
inline int check_launch() {
  SKY_HIP(hipGetLastError());
  return SKY_OK;
}

}  // namespace sky
