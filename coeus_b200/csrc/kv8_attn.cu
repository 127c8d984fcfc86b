// Attention over the 8-bit cache (kv8.cuh has the layout).  Row i of entry e (r rows, context n) sits
// at position n - r + i of its sequence and sees the positions up to that one; query head h reads
// key/value head h / (heads / kv_heads).  A row that sees nothing gets zeros.
//
//   o = sum_t w_t v_t / sum_t w_t,  w_t = exp(scale q . k_t - max),  k_t = code 2^ek, v_t = code 2^ev
//
// One CTA per row and head; its warps take the pages in turn and are merged at the end.
#include "kv8.cuh"

namespace cb {

struct Kv8Attn {
  Kv8Cache c;
  const __nv_bfloat16* q;  // [rows, ldq]
  __nv_bfloat16* out;      // [rows, ldo]
  int ldq, ldo, heads;
  const int* ctx;          // [entries]
  const int* row0;         // [entries + 1] or null: entry e has row e alone
  int rows, most;
  float scale_log2;
  int* status;
};

constexpr int KA_WARPS = 4;

template <int KIND, int DH>
__global__ void __launch_bounds__(KA_WARPS * 32) kv8_attn_kernel(const Kv8Attn a) {
  __shared__ float sq[DH], sw[KA_WARPS][KV8_PAGE], sm[KA_WARPS], sl[KA_WARPS], so[KA_WARPS][DH];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int b = blockIdx.x;
  const int h = b % a.heads;
  b /= a.heads;
  const int i = b % a.most, e = b / a.most;
  const int first = a.row0 != nullptr ? a.row0[e] : e;
  const int n = a.row0 != nullptr ? a.row0[e + 1] - first : 1;
  if (i >= n) return;
  if (n > a.most || first < 0 || first + n > a.rows) {
    record_status(a.status, ST_BOUNDS, e);
    return;
  }
  const int seen = a.ctx[e] - n + i + 1;
  const int hk = h / (a.heads / a.c.heads);
  for (int d = threadIdx.x; d < DH; d += KA_WARPS * 32)
    sq[d] = __bfloat162float(a.q[static_cast<size_t>(first + i) * a.ldq + h * DH + d]) * a.scale_log2;
  __syncthreads();
  float m = -INFINITY, l = 0.f, o[DH / 32];
#pragma unroll
  for (int x = 0; x < DH / 32; ++x) o[x] = 0.f;
  for (int p = warp; p * KV8_PAGE < seen; p += KA_WARPS) {
    const int page = kv8_page(a.c, e, p, a.status, e);
    if (page < 0) continue;
    const size_t cell = static_cast<size_t>(page) * a.c.heads + hk;
    const uint8_t* kb = a.c.k + cell * (KV8_PAGE * DH);
    const uint8_t* vb = a.c.v + cell * (KV8_PAGE * DH);
    const float ks = a.c.k_scale[cell], vs = a.c.v_scale[cell];
    float s[2], mx = -INFINITY;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int t = lane + 32 * x;
      float dot = 0.f;
      for (int d = 0; d < DH; ++d) dot += sq[d] * kv8_value<KIND>(kb[(d / 64 * KV8_PAGE + t) * 64 + d % 64]);
      s[x] = p * KV8_PAGE + t < seen ? dot * ks : -INFINITY;
      mx = fmaxf(mx, s[x]);
    }
    const float mn = fmaxf(m, warp_max(mx)), c = exp2f(m - mn);
    m = mn;
    l *= c;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const float w = exp2f(s[x] - mn);
      l += w;
      sw[warp][lane + 32 * x] = w;
    }
    __syncwarp();
    const int nt = min(KV8_PAGE, seen - p * KV8_PAGE);
#pragma unroll
    for (int x = 0; x < DH / 32; ++x) {
      float acc = 0.f;
      for (int t = 0; t < nt; ++t) acc += sw[warp][t] * kv8_value<KIND>(vb[(lane + 32 * x) * KV8_PAGE + t]);
      o[x] = o[x] * c + acc * vs;
    }
    __syncwarp();
  }
  l = warp_sum(l);
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
#pragma unroll
  for (int x = 0; x < DH / 32; ++x) so[warp][lane + 32 * x] = o[x];
  __syncthreads();
  float gm = -INFINITY, gl = 0.f;
  for (int w = 0; w < KA_WARPS; ++w) gm = fmaxf(gm, sm[w]);
  for (int w = 0; w < KA_WARPS; ++w) gl += sl[w] == 0.f ? 0.f : sl[w] * exp2f(sm[w] - gm);   // NaN stays
  for (int d = threadIdx.x; d < DH; d += KA_WARPS * 32) {
    float v = 0.f;
    for (int w = 0; w < KA_WARPS; ++w) v += sm[w] == -INFINITY ? 0.f : so[w][d] * exp2f(sm[w] - gm);
    a.out[static_cast<size_t>(first + i) * a.ldo + h * DH + d] = __float2bfloat16(seen > 0 ? v / gl : 0.f);
  }
}

}  // namespace cb

using namespace cb;

extern "C" int cb_kv8_attn(const void* q, int ldq, const void* k_cache, const void* v_cache, const float* k_scale,
                           const float* v_scale, const int* page_table, int max_pages, int num_pages, int kv_heads,
                           int dh, int kind, const int* ctx, const int* row0, int n, int rows, int most, int heads,
                           float scale, void* out, int ldo, int* status, void* stream) {
  if (n < 1 || rows < 1 || most < 1 || kv_heads < 1 || heads < 1 || heads % kv_heads != 0) return -1;
  if ((dh != 64 && dh != 128) || (kind != KV8_INT8 && kind != KV8_E4M3)) return -2;
  Kv8Attn a;
  a.c = Kv8Cache{static_cast<uint8_t*>(const_cast<void*>(k_cache)), static_cast<uint8_t*>(const_cast<void*>(v_cache)),
                 const_cast<float*>(k_scale), const_cast<float*>(v_scale), page_table, max_pages, num_pages, kv_heads};
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.out = static_cast<__nv_bfloat16*>(out);
  a.ldq = ldq; a.ldo = ldo; a.heads = heads; a.ctx = ctx; a.row0 = row0; a.rows = rows; a.most = most;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.status = status;
  const long long blocks = 1ll * n * most * heads;
  if (blocks > 0x7fffffffll) return -4;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
#define CB_ATTN(KIND_, DH_) \
  kv8_attn_kernel<KIND_, DH_><<<static_cast<unsigned>(blocks), KA_WARPS * 32, 0, st>>>(a)
  if (kind == KV8_INT8) {
    if (dh == 64) CB_ATTN(KV8_INT8, 64); else CB_ATTN(KV8_INT8, 128);
  } else {
    if (dh == 64) CB_ATTN(KV8_E4M3, 64); else CB_ATTN(KV8_E4M3, 128);
  }
#undef CB_ATTN
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}
