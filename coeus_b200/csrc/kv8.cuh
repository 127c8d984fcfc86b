// A paged cache in 8 bits.  A page holds 64 tokens; of one page and head the keys are
// [dh / 64][token][64] codes and the values [dh][token] codes, so both are rows of 64 bytes: a block
// of 64 dh contiguous bytes that one bulk copy moves and whose rows warps read without bank conflicts,
// with the token axis of the values innermost, as the second product wants its operand.
// The value of a code is code * 2^e with one e per page, head and side (held as the fp32 number 2^e):
// scaling by powers of two is exact, so a code is the value rounded once, and a page whose scale has to
// grow for a new token only shifts the codes it holds.
#pragma once
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include "common.cuh"
#include "ptx.cuh"

namespace cb {

int sm_count();

constexpr int KV8_PAGE = 64;
enum : int { KV8_INT8 = 0, KV8_E4M3 = 1 };

struct Kv8Cache {
  uint8_t* k;              // [pages, heads, dh / 64, 64, 64]
  uint8_t* v;              // [pages, heads, dh, 64]
  float* k_scale;          // [pages, heads]
  float* v_scale;
  const int* page_table;   // [entries, max_pages]
  int max_pages, num_pages, heads;
};

// Smallest e >= -126 with amax <= largest code * 2^e, from the bits of a finite fp32 amax.
template <int KIND>
__device__ __forceinline__ int kv8_exponent(float amax) {
  if (amax == 0.f) return -126;
  int x;
  const float f = frexpf(amax, &x);          // amax = f 2^x, 1/2 <= f < 1
  // 127 = (127/128) 2^7 and 448 = (7/8) 2^9
  const int e = KIND == KV8_INT8 ? x - 7 + (f > 127.f / 128.f) : x - 9 + (f > 0.875f);
  return max(e, -126);
}
__device__ __forceinline__ float pow2(int e) {       // -126 <= e <= 127
  return __int_as_float((e + 127) << 23);
}

// The page of a position, or -1 (recorded in the status word) where the table has none.
__device__ __forceinline__ int kv8_page(const Kv8Cache& c, int entry, int lp, int* status, int where) {
  int page = -1;
  if (lp >= 0 && lp < c.max_pages) page = c.page_table[static_cast<size_t>(entry) * c.max_pages + lp];
  if (page < 0 || page >= c.num_pages) {
    record_status(status, ST_BOUNDS, where);
    page = -1;
  }
  return page;
}

// The rows of entry e: row0[e] .. row0[e + 1] - 1.  False where they are more than `most`, run backwards or leave the
// tensors' `rows`; nothing is subtracted before that is known.
__device__ __forceinline__ bool kv8_rows_of(const int* row0, int e, int rows, int most, int& first, int& n) {
  first = row0[e];
  const int end = row0[e + 1];
  n = 0;
  if (first < 0 || end < first || end > rows || end - first > most) return false;
  n = end - first;
  return true;
}

}  // namespace cb
