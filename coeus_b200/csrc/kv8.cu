// Appending keys and values to the 8-bit cache, and reading them back (kv8.cuh has the layout).
//
// write   one CTA per entry, page that its new rows touch, head and side (keys or values).  The largest
//         new magnitude is a maximum of bits (so that NaN and infinities win), the exponent follows from
//         it, is not below that of a page that holds earlier tokens, and where it grows by d the earlier
//         codes become round(code 2^-d).  Bound by memory: two bytes in, one out per number.
// read    the same split; one byte in, two out.
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
  const int first = r.row0 != nullptr ? r.row0[e] : e;
  int n = r.row0 != nullptr ? r.row0[e + 1] - first : 1;
  const int pos0 = r.pos0[e];
  if (n <= 0) return false;
  if (n > r.most || first < 0 || first + n > r.rows || pos0 < 0) {
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

template <int KIND, int DH>
__global__ void __launch_bounds__(KV8_THREADS)
kv8_write_kernel(const __nv_bfloat16* __restrict__ k, const __nv_bfloat16* __restrict__ v, int ldk, int ldv,
                 const Kv8Cache c, const Kv8Rows r, int* status) {
  constexpr int VEC = DH / 8;                           // 16-byte vectors of a row
  constexpr int PER = KV8_PAGE * VEC / KV8_THREADS;     // of a thread
  __shared__ uint32_t s_max[KV8_THREADS / 32];
  const int side = blockIdx.x & 1;
  int b = blockIdx.x >> 1;
  const int h = b % c.heads;
  b /= c.heads;
  const int piece = b % r.pieces, e = b / r.pieces;
  Kv8Piece p;
  if (!kv8_piece(c, r, e, piece, status, p)) return;
  const __nv_bfloat16* src = (side ? v : k) + h * DH;
  const int ld = side ? ldv : ldk;
  uint4 x[PER];
  uint32_t top = 0;
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const int i = threadIdx.x + u * KV8_THREADS, t = i / VEC;
    x[u] = make_uint4(0u, 0u, 0u, 0u);
    if (t < p.hi - p.lo) x[u] = __ldg(reinterpret_cast<const uint4*>(src + static_cast<size_t>(p.row + t) * ld) + i % VEC);
    top = __vmaxu2(top, __vmaxu2(__vmaxu2(x[u].x & 0x7fff7fffu, x[u].y & 0x7fff7fffu),
                                 __vmaxu2(x[u].z & 0x7fff7fffu, x[u].w & 0x7fff7fffu)));
  }
  top = max(top & 0xffffu, top >> 16);
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = top;
  const size_t cell = static_cast<size_t>(p.page) * c.heads + h;
  float* scale = (side ? c.v_scale : c.k_scale) + cell;
  const float before = p.lo > 0 ? *scale : 0.f;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < KV8_THREADS / 32; ++w) top = max(top, s_max[w]);
  const bool bad = top >= 0x7f80u || before != before;
  int ex = bad ? 0 : kv8_exponent<KIND>(__uint_as_float(top << 16));
  uint8_t* block = (side ? c.v : c.k) + cell * (KV8_PAGE * DH);
  if (p.lo > 0 && !bad) {
    const int was = (__float_as_int(before) >> 23) - 127;
    if (ex > was) {
      const float f = ldexpf(1.f, was - ex);
      for (int i = threadIdx.x; i < p.lo * DH; i += KV8_THREADS) {
        const int t = i % p.lo, d = i / p.lo;
        uint8_t* q = block + (side ? d * KV8_PAGE + t : (d / 64 * KV8_PAGE + t) * 64 + d % 64);
        *q = kv8_code<KIND>(kv8_value<KIND>(*q) * f);
      }
    }
    ex = max(ex, was);
  }
  if (threadIdx.x == 0) *scale = bad ? __int_as_float(0x7fffffff) : pow2(ex);
  const float f = bad ? 0.f : ldexpf(1.f, -ex);
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const int i = threadIdx.x + u * KV8_THREADS, t = i / VEC, d = i % VEC * 8;
    if (t >= p.hi - p.lo) continue;
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&x[u]);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float y = __uint_as_float(j & 1 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16) * f;
      const int tt = p.lo + t, dd = d + j;
      block[side ? dd * KV8_PAGE + tt : (dd / 64 * KV8_PAGE + tt) * 64 + dd % 64] = kv8_code<KIND>(y);
    }
  }
}

template <int KIND, int DH>
__global__ void __launch_bounds__(KV8_THREADS)
kv8_read_kernel(const Kv8Cache c, const Kv8Rows r, __nv_bfloat16* __restrict__ k, __nv_bfloat16* __restrict__ v,
                int ld, int* status) {
  const int side = blockIdx.x & 1;
  int b = blockIdx.x >> 1;
  const int h = b % c.heads;
  b /= c.heads;
  const int piece = b % r.pieces, e = b / r.pieces;
  Kv8Piece p;
  if (!kv8_piece(c, r, e, piece, status, p)) return;
  const size_t cell = static_cast<size_t>(p.page) * c.heads + h;
  const float f = (side ? c.v_scale : c.k_scale)[cell];
  const uint8_t* block = (side ? c.v : c.k) + cell * (KV8_PAGE * DH);
  __nv_bfloat16* dst = (side ? v : k) + h * DH;
  for (int i = threadIdx.x; i < (p.hi - p.lo) * DH; i += KV8_THREADS) {
    const int t = i / DH, d = i % DH, tt = p.lo + t;
    const uint8_t q = block[side ? d * KV8_PAGE + tt : (d / 64 * KV8_PAGE + tt) * 64 + d % 64];
    dst[static_cast<size_t>(p.row + t) * ld + d] = __float2bfloat16(kv8_value<KIND>(q) * f);
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
#define CB_WRITE(KIND_, DH_) \
  kv8_write_kernel<KIND_, DH_><<<static_cast<unsigned>(blocks), KV8_THREADS, 0, st>>>(K, V, ldk, ldv, c, r, status)
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
