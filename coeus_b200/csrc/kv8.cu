// Appending keys and values to the 8-bit cache, and reading them back (kv8.cuh has the layout).
//
// write   one CTA per entry, page that its new rows touch, head and side (keys or values).  The largest
//         new magnitude is a maximum of bits (so that NaN and infinities win), the exponent follows from
//         it, is not below that of a page that holds earlier tokens, and where it grows by d the earlier
//         codes become round(code 2^-d).  Two bytes in, one out per number: 16384 tokens of 8 heads of 128
//         in 24 us, 0.64 of the copy rate (100 MB), 54 % of the issue slots in conversions and the transposition of
//         the values.  One token per entry: a warp each, 4.6 us for 64 entries of 16 heads of 64, all latency.
// read    the same split; one byte in, two out; 20 us for the same tokens, 0.77 of the copy rate.
#include "kv8.cuh"

namespace cb {

constexpr int KV8_THREADS = 128;

struct Kv8Rows {           // entry e owns rows row0[e] .. row0[e + 1] - 1 (null: row e), the first at pos0[e]
  const int* row0;
  const int* pos0;
  int rows, most;          // rows of the tensors; the host's bound on the rows of an entry
  int pieces;              // pages that an entry may touch
};

// Rows of entry e that lie in the piece-th page from its first on: false if there are none.
struct Kv8Piece {
  int page, lo, hi, row;   // tokens lo .. hi - 1 of the page; the row of token lo
};
__device__ __forceinline__ bool kv8_piece(const Kv8Cache& c, const Kv8Rows& r, int e, int piece, int* status,
                                          Kv8Piece& out) {
  int first = e, n = 1;
  const int pos0 = r.pos0[e];
  const bool ok = r.row0 == nullptr || kv8_rows_of(r.row0, e, r.rows, r.most, first, n);
  if (ok && n == 0) return false;
  if (!ok || pos0 < 0 || pos0 > 0x7fffffff - n - KV8_PAGE) {
    record_status(status, ST_BOUNDS, e);
    return false;
  }
  const int lp = pos0 / KV8_PAGE + piece, base = lp * KV8_PAGE;
  if (base >= pos0 + n) return false;
  out.lo = max(0, pos0 - base);
  out.hi = min(KV8_PAGE, pos0 + n - base);
  out.row = first + base + out.lo - pos0;
  out.page = kv8_page(c, e, lp, status, e);
  return out.page >= 0;
}

// Bits of the largest magnitude of two bf16 numbers, each in its half; NaN is above infinity, that above all else.
__device__ __forceinline__ uint32_t top2(uint32_t a, uint32_t b) { return __vmaxu2(a & 0x7fff7fffu, b & 0x7fff7fffu); }
__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// Four values, already divided by the scale, to codes in the order of the bytes; |y| is at most the largest code.
template <int KIND>
__device__ __forceinline__ uint32_t codes4(float y0, float y1, float y2, float y3) {
  if constexpr (KIND == KV8_INT8) {
    // 1.5 2^23 + y rounds y to a whole number (ties to even), whose low byte is the code
    const float h = 12582912.f;
    const uint32_t a = __byte_perm(__float_as_uint(y0 + h), __float_as_uint(y1 + h), 0x0040);
    const uint32_t b = __byte_perm(__float_as_uint(y2 + h), __float_as_uint(y3 + h), 0x0040);
    return __byte_perm(a, b, 0x5410);
  } else {
    const uint32_t a = __nv_cvt_float2_to_fp8x2(make_float2(y0, y1), __NV_SATFINITE, __NV_E4M3);
    const uint32_t b = __nv_cvt_float2_to_fp8x2(make_float2(y2, y3), __NV_SATFINITE, __NV_E4M3);
    return a | b << 16;
  }
}
template <int KIND>
__device__ __forceinline__ void values4(uint32_t w, float* v) {
  if constexpr (KIND == KV8_INT8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = static_cast<float>(static_cast<int8_t>(w >> (8 * i)));
  } else {
    const float2 a = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w & 0xffffu), __NV_E4M3)));
    const float2 b = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w >> 16), __NV_E4M3)));
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
  }
}
// Four codes under a scale that is 2^d times as large; f = 2^-d.
template <int KIND>
__device__ __forceinline__ uint32_t shift4(uint32_t w, float f) {
  float v[4];
  values4<KIND>(w, v);
  return codes4<KIND>(v[0] * f, v[1] * f, v[2] * f, v[3] * f);
}

// What the block's new scale is and what its earlier codes are multiplied by.
struct Rescale {
  bool bad;                // not finite: the scale is NaN, new codes are 0
  float scale, mul, shift; // new scale, its reciprocal, the factor of the earlier codes (1: none)
};
template <int KIND>
__device__ __forceinline__ Rescale rescale(uint32_t top, float before, bool kept) {
  Rescale r;
  r.bad = top >= 0x7f80u || (kept && before != before);
  r.shift = 1.f;
  int ex = r.bad ? 0 : kv8_exponent<KIND>(__uint_as_float(top << 16));
  if (kept && !r.bad) {
    const int was = (__float_as_int(before) >> 23) - 127;
    if (ex > was) r.shift = ldexpf(1.f, was - ex);
    ex = max(ex, was);
  }
  r.scale = r.bad ? __int_as_float(0x7fffffff) : pow2(ex);
  r.mul = r.bad ? 0.f : ldexpf(1.f, -ex);
  return r;
}
// The codes of tokens 0 .. lo - 1 under the new scale, by `threads` threads.
template <int KIND, int DH>
__device__ __forceinline__ void shift_block(uint8_t* block, int side, int lo, float f, int tid, int threads) {
  uint32_t* w = reinterpret_cast<uint32_t*>(block);
  if (side == 0) {         // rows of a token in every half
    for (int i = tid; i < DH / 64 * lo * 16; i += threads) {
      uint32_t* q = w + i / (lo * 16) * (KV8_PAGE * 16) + i % (lo * 16);
      *q = shift4<KIND>(*q, f);
    }
  } else {                 // the first lo bytes of every channel's row
    const int n = (lo + 3) / 4;
    for (int i = tid; i < DH * n; i += threads) {
      uint32_t* q = w + i / n * 16 + i % n;
      const int left = lo - i % n * 4;
      const uint32_t mask = left >= 4 ? 0xffffffffu : (1u << (8 * left)) - 1u;
      *q = (*q & ~mask) | (shift4<KIND>(*q, f) & mask);
    }
  }
}

template <int KIND, int DH>
__global__ void __launch_bounds__(KV8_THREADS)
kv8_write_kernel(const __nv_bfloat16* __restrict__ k, const __nv_bfloat16* __restrict__ v, int ldk, int ldv,
                 const Kv8Cache c, const Kv8Rows r, int* status) {
  constexpr int VEC = DH / 8;                           // 16-byte vectors of a row
  constexpr int PER = KV8_PAGE * VEC / KV8_THREADS;     // of a thread
  constexpr int HALVES = DH / 64;
  __shared__ uint32_t s_max[KV8_THREADS / 32];
  __shared__ uint32_t tile[DH][17];                     // values: codes by channel, four tokens a word
  const int side = blockIdx.x & 1;
  int b = blockIdx.x >> 1;
  const int h = b % c.heads;
  b /= c.heads;
  const int piece = b % r.pieces, e = b / r.pieces;
  Kv8Piece p;
  if (!kv8_piece(c, r, e, piece, status, p)) return;
  const int n = p.hi - p.lo, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const __nv_bfloat16* src = (side ? v : k) + h * DH;
  const size_t ld = side ? ldv : ldk;
  // Keys: 16-byte vectors of a row.  Values: a warp has 16 tokens (by their place in the page), a lane two channels of
  // each half, so that four tokens of a channel are a word.
  uint4 x[PER];
  uint32_t y[HALVES][16], top = 0;
  if (side == 0) {
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int i = threadIdx.x + u * KV8_THREADS, t = i / VEC;
      x[u] = make_uint4(0u, 0u, 0u, 0u);
      if (t < n) x[u] = __ldg(reinterpret_cast<const uint4*>(src + (p.row + t) * ld) + i % VEC);
    }
#pragma unroll
    for (int u = 0; u < PER; ++u) top = __vmaxu2(top, __vmaxu2(top2(x[u].x, x[u].y), top2(x[u].z, x[u].w)));
  } else {
#pragma unroll
    for (int z = 0; z < HALVES; ++z)
#pragma unroll
      for (int t = 0; t < 16; ++t) {
        const int tt = warp * 16 + t - p.lo;
        y[z][t] = 0u;
        if (tt >= 0 && tt < n) y[z][t] = __ldg(reinterpret_cast<const uint32_t*>(src + (p.row + tt) * ld + z * 64) + lane);
      }
#pragma unroll
    for (int z = 0; z < HALVES; ++z)
#pragma unroll
      for (int t = 0; t < 16; t += 2) top = __vmaxu2(top, top2(y[z][t], y[z][t + 1]));
  }
  top = __reduce_max_sync(0xffffffffu, max(top & 0xffffu, top >> 16));
  if (lane == 0) s_max[warp] = top;
  const size_t cell = static_cast<size_t>(p.page) * c.heads + h;
  float* scale = (side ? c.v_scale : c.k_scale) + cell;
  const float before = p.lo > 0 ? *scale : 0.f;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < KV8_THREADS / 32; ++w) top = max(top, s_max[w]);
  const Rescale q = rescale<KIND>(top, before, p.lo > 0);
  uint8_t* block = (side ? c.v : c.k) + cell * (KV8_PAGE * DH);
  if (q.shift != 1.f) {
    shift_block<KIND, DH>(block, side, p.lo, q.shift, threadIdx.x, KV8_THREADS);
    __syncthreads();                                    // words of values at the border are written again below
  }
  if (threadIdx.x == 0) *scale = q.scale;
  if (side == 0) {
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int i = threadIdx.x + u * KV8_THREADS, t = i / VEC, d = i % VEC * 8;
      if (t >= n) continue;
      const uint32_t* w = reinterpret_cast<const uint32_t*>(&x[u]);
      uint2 o = make_uint2(codes4<KIND>(bf16_lo(w[0]) * q.mul, bf16_hi(w[0]) * q.mul, bf16_lo(w[1]) * q.mul, bf16_hi(w[1]) * q.mul),
                           codes4<KIND>(bf16_lo(w[2]) * q.mul, bf16_hi(w[2]) * q.mul, bf16_lo(w[3]) * q.mul, bf16_hi(w[3]) * q.mul));
      if (q.bad) o = make_uint2(0u, 0u);
      *reinterpret_cast<uint2*>(block + (d / 64 * KV8_PAGE + p.lo + t) * 64 + d % 64) = o;
    }
    return;
  }
#pragma unroll
  for (int z = 0; z < HALVES; ++z)
#pragma unroll
    for (int t = 0; t < 16; t += 4) {
      uint32_t a = codes4<KIND>(bf16_lo(y[z][t]) * q.mul, bf16_lo(y[z][t + 1]) * q.mul, bf16_lo(y[z][t + 2]) * q.mul, bf16_lo(y[z][t + 3]) * q.mul);
      uint32_t d = codes4<KIND>(bf16_hi(y[z][t]) * q.mul, bf16_hi(y[z][t + 1]) * q.mul, bf16_hi(y[z][t + 2]) * q.mul, bf16_hi(y[z][t + 3]) * q.mul);
      if (q.bad) a = d = 0u;
      tile[z * 64 + 2 * lane][warp * 4 + t / 4] = a;
      tile[z * 64 + 2 * lane + 1][warp * 4 + t / 4] = d;
    }
  __syncthreads();
  for (int i = threadIdx.x; i < DH * 4; i += KV8_THREADS) {       // 16 tokens of a channel
    const int d = i >> 2, t0 = (i & 3) * 16;
    if (t0 + 16 <= p.lo || t0 >= p.hi) continue;
    uint32_t* dst = reinterpret_cast<uint32_t*>(block + d * KV8_PAGE + t0);
    const uint32_t* w = &tile[d][(i & 3) * 4];
    if (t0 >= p.lo && t0 + 16 <= p.hi) {
      *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
      continue;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int t = t0 + 4 * j;
      if (t >= p.lo && t + 4 <= p.hi) dst[j] = w[j];
      else
#pragma unroll
        for (int z = 0; z < 4; ++z)
          if (t + z >= p.lo && t + z < p.hi) reinterpret_cast<uint8_t*>(dst + j)[z] = static_cast<uint8_t>(w[j] >> (8 * z));
    }
  }
}

// One new token per entry: a warp per entry, head and side.
template <int KIND, int DH>
__global__ void __launch_bounds__(KV8_THREADS)
kv8_write_token_kernel(const __nv_bfloat16* __restrict__ k, const __nv_bfloat16* __restrict__ v, int ldk, int ldv,
                       const Kv8Cache c, const Kv8Rows r, int n, int* status) {
  const int lane = threadIdx.x & 31, side = (threadIdx.x >> 5) & 1;
  const int b = blockIdx.x * (KV8_THREADS / 64) + (threadIdx.x >> 6), h = b % c.heads, e = b / c.heads;
  Kv8Piece p;
  if (e >= n || !kv8_piece(c, r, e, 0, status, p)) return;
  constexpr int W = DH / 64;                            // words of a lane
  const uint32_t* src = reinterpret_cast<const uint32_t*>((side ? v : k) + static_cast<size_t>(p.row) * (side ? ldv : ldk) + h * DH) + lane * W;
  uint32_t x[W], top;
  if constexpr (W == 2) {
    const uint2 t = __ldg(reinterpret_cast<const uint2*>(src));
    x[0] = t.x;
    x[1] = t.y;
    top = top2(x[0], x[1]);
  } else {
    x[0] = __ldg(src);
    top = top2(x[0], x[0]);
  }
  const size_t cell = static_cast<size_t>(p.page) * c.heads + h;
  float* scale = (side ? c.v_scale : c.k_scale) + cell;
  const float before = p.lo > 0 ? *scale : 0.f;
  top = __reduce_max_sync(0xffffffffu, max(top & 0xffffu, top >> 16));
  const Rescale q = rescale<KIND>(top, before, p.lo > 0);
  uint8_t* block = (side ? c.v : c.k) + cell * (KV8_PAGE * DH);
  if (q.shift != 1.f) shift_block<KIND, DH>(block, side, p.lo, q.shift, lane, 32);
  __syncwarp();
  if (lane == 0) *scale = q.scale;
  uint32_t o = codes4<KIND>(bf16_lo(x[0]) * q.mul, bf16_hi(x[0]) * q.mul, W == 2 ? bf16_lo(x[W - 1]) * q.mul : 0.f, W == 2 ? bf16_hi(x[W - 1]) * q.mul : 0.f);
  if (q.bad) o = 0u;
  const int d = lane * 2 * W;
  if (side == 0) {
    uint8_t* dst = block + (d / 64 * KV8_PAGE + p.lo) * 64 + d % 64;
    if constexpr (W == 2) *reinterpret_cast<uint32_t*>(dst) = o;
    else *reinterpret_cast<uint16_t*>(dst) = static_cast<uint16_t>(o);
  } else {
#pragma unroll
    for (int i = 0; i < 2 * W; ++i) block[(d + i) * KV8_PAGE + p.lo] = static_cast<uint8_t>(o >> (8 * i));
  }
}

template <int KIND, int DH>
__global__ void __launch_bounds__(KV8_THREADS)
kv8_read_kernel(const Kv8Cache c, const Kv8Rows r, __nv_bfloat16* __restrict__ k, __nv_bfloat16* __restrict__ v,
                int ld, int* status) {
  constexpr int VEC = DH / 8;
  __shared__ uint32_t tile[DH][17];
  const int side = blockIdx.x & 1;
  int b = blockIdx.x >> 1;
  const int h = b % c.heads;
  b /= c.heads;
  const int piece = b % r.pieces, e = b / r.pieces;
  Kv8Piece p;
  if (!kv8_piece(c, r, e, piece, status, p)) return;
  const int n = p.hi - p.lo;
  const size_t cell = static_cast<size_t>(p.page) * c.heads + h;
  const float f = (side ? c.v_scale : c.k_scale)[cell];
  const uint8_t* block = (side ? c.v : c.k) + cell * (KV8_PAGE * DH);
  __nv_bfloat16* dst = (side ? v : k) + static_cast<size_t>(p.row) * ld + h * DH;
  if (side == 0) {
#pragma unroll 4
    for (int i = threadIdx.x; i < n * VEC; i += KV8_THREADS) {
      const int t = i / VEC, d = i % VEC * 8;
      const uint2 w = __ldg(reinterpret_cast<const uint2*>(block + (d / 64 * KV8_PAGE + p.lo + t) * 64 + d % 64));
      float x[8];
      values4<KIND>(w.x, x);
      values4<KIND>(w.y, x + 4);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] *= f;
      store8(dst + static_cast<size_t>(t) * ld + d, x);
    }
    return;
  }
#pragma unroll
  for (int u = 0; u < DH * 4 / KV8_THREADS; ++u) {
    const int i = threadIdx.x + u * KV8_THREADS, d = i >> 2, t0 = (i & 3) * 16;
    if (t0 + 16 <= p.lo || t0 >= p.hi) continue;
    const uint4 w = __ldg(reinterpret_cast<const uint4*>(block + d * KV8_PAGE + t0));
    uint32_t* q = &tile[d][(i & 3) * 4];
    q[0] = w.x; q[1] = w.y; q[2] = w.z; q[3] = w.w;
  }
  __syncthreads();
  // a warp has four tokens of two channels a lane at a time
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int t = (p.lo & ~3) + 4 * warp; t < p.hi; t += 4 * (KV8_THREADS / 32))
#pragma unroll
    for (int z = 0; z < DH / 64; ++z) {
      float x[2][4];
      values4<KIND>(tile[z * 64 + 2 * lane][t >> 2], x[0]);
      values4<KIND>(tile[z * 64 + 2 * lane + 1][t >> 2], x[1]);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (t + j >= p.lo && t + j < p.hi)
          *reinterpret_cast<__nv_bfloat162*>(dst + static_cast<size_t>(t + j - p.lo) * ld + z * 64 + 2 * lane) =
              __floats2bfloat162_rn(x[0][j] * f, x[1][j] * f);
    }
}

}  // namespace cb

using namespace cb;

static int fill_rows(Kv8Rows& r, const int* row0, const int* pos0, int rows, int most) {
  if (most < 1 || rows < 1) return -1;
  r.row0 = row0; r.pos0 = pos0; r.rows = rows; r.most = most;
  r.pieces = (most + KV8_PAGE - 2) / KV8_PAGE + 1;
  return 0;
}

extern "C" int cb_kv8_write(const void* k, const void* v, int ldk, int ldv, void* k_cache, void* v_cache,
                            float* k_scale, float* v_scale, const int* page_table, int max_pages, int num_pages,
                            int heads, int dh, int kind, const int* row0, const int* pos0, int n, int rows,
                            int most, int* status, void* stream) {
  const Kv8Cache c{static_cast<uint8_t*>(k_cache), static_cast<uint8_t*>(v_cache), k_scale, v_scale, page_table,
                   max_pages, num_pages, heads};
  Kv8Rows r;
  if (fill_rows(r, row0, pos0, rows, most) != 0 || n < 1 || heads < 1) return -1;
  if ((dh != 64 && dh != 128) || (kind != KV8_INT8 && kind != KV8_E4M3)) return -2;
  const long long blocks = 2ll * n * r.pieces * heads;
  if (blocks > 0x7fffffffll) return -4;
  auto* K = static_cast<const __nv_bfloat16*>(k);
  auto* V = static_cast<const __nv_bfloat16*>(v);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
#define CB_WRITE(KIND_, DH_)                                                                                        \
  do {                                                                                                              \
    if (most == 1)                                                                                                  \
      kv8_write_token_kernel<KIND_, DH_><<<static_cast<unsigned>((1ll * n * heads + 1) / 2), KV8_THREADS, 0, st>>>( \
          K, V, ldk, ldv, c, r, n, status);                                                                         \
    else                                                                                                            \
      kv8_write_kernel<KIND_, DH_><<<static_cast<unsigned>(blocks), KV8_THREADS, 0, st>>>(K, V, ldk, ldv, c, r, status); \
  } while (0)
  if (kind == KV8_INT8) {
    if (dh == 64) CB_WRITE(KV8_INT8, 64); else CB_WRITE(KV8_INT8, 128);
  } else {
    if (dh == 64) CB_WRITE(KV8_E4M3, 64); else CB_WRITE(KV8_E4M3, 128);
  }
#undef CB_WRITE
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

extern "C" int cb_kv8_read(const void* k_cache, const void* v_cache, const float* k_scale, const float* v_scale,
                           const int* page_table, int max_pages, int num_pages, int heads, int dh, int kind,
                           const int* row0, const int* pos0, int n, int rows, int most, void* k, void* v, int ld,
                           int* status, void* stream) {
  const Kv8Cache c{static_cast<uint8_t*>(const_cast<void*>(k_cache)), static_cast<uint8_t*>(const_cast<void*>(v_cache)),
                   const_cast<float*>(k_scale), const_cast<float*>(v_scale), page_table, max_pages, num_pages, heads};
  Kv8Rows r;
  if (fill_rows(r, row0, pos0, rows, most) != 0 || n < 1 || heads < 1) return -1;
  if ((dh != 64 && dh != 128) || (kind != KV8_INT8 && kind != KV8_E4M3)) return -2;
  const long long blocks = 2ll * n * r.pieces * heads;
  if (blocks > 0x7fffffffll) return -4;
  auto* K = static_cast<__nv_bfloat16*>(k);
  auto* V = static_cast<__nv_bfloat16*>(v);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
#define CB_READ(KIND_, DH_) \
  kv8_read_kernel<KIND_, DH_><<<static_cast<unsigned>(blocks), KV8_THREADS, 0, st>>>(c, r, K, V, ld, status)
  if (kind == KV8_INT8) {
    if (dh == 64) CB_READ(KV8_INT8, 64); else CB_READ(KV8_INT8, 128);
  } else {
    if (dh == 64) CB_READ(KV8_E4M3, 64); else CB_READ(KV8_E4M3, 128);
  }
#undef CB_READ
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}
