// What the two attention kernels of the 8-bit cache share: arguments, the plan of the work, the conversion of
// codes, the merge of tiles that lie in more than one CTA.
#pragma once
#include "kv8.cuh"

namespace cb {

constexpr int KA_ENTRIES = 256;                   // of one launch
constexpr float KA_LOG2E = 1.4426950408889634f;

struct Kv8Desc {           // the tile that a CTA's run of units starts in
  int lo, hi, share, units;
  int entry, head, tile, pad;
};

struct Kv8Attn {
  Kv8Cache c;
  const __nv_bfloat16* q;  // [rows, ldq]
  __nv_bfloat16* out;      // [rows, ldo]
  int ldq, ldo, group;     // query heads per key/value head
  const int* ctx;          // [entries]
  const int* row0;         // [entries + 1] or null: entry e has row first + e alone
  int first, n, rows, most;
  float scale_log2;
  float* part_o;           // [CTAs, 2, tile rows, dh]
  float* part_ml;          // [CTAs, 2, tile rows, 2]
  Kv8Desc* desc;           // [CTAs]
  int* status;
};

// Four codes to two pairs of fp16.
template <int KIND>
__device__ __forceinline__ void kv8_half4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (KIND == KV8_INT8) {
    const uint32_t x = w ^ 0x80808080u;                       // code + 128
    lo = __byte_perm(x, 0x64646464u, 0x4140);                 // 1024 + that
    hi = __byte_perm(x, 0x64646464u, 0x4342);
    const __half2 off = __half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));      // 1152
    const __half2 p = __hsub2(*reinterpret_cast<__half2*>(&lo), off), q = __hsub2(*reinterpret_cast<__half2*>(&hi), off);
    lo = *reinterpret_cast<const uint32_t*>(&p);
    hi = *reinterpret_cast<const uint32_t*>(&q);
  } else {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
  }
}
__device__ __forceinline__ uint32_t half2_bits(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// Wait for a phase, with a limit; the clock is asked only after many tries have failed.
__device__ __forceinline__ bool wait_phase(uint64_t* bar, uint32_t parity, volatile uint32_t* abort_flag) {
  const uint32_t at = smem_u32(bar);
  uint64_t began = 0;
  for (uint32_t n = 1;; ++n) {
    if (mbar_try_wait(at, parity)) return true;
    if (n % 256u == 0u) {
      if (*abort_flag) return false;
      const uint64_t now = globaltimer_ns();
      if (began == 0) began = now;
      else if (now - began > CB_WAIT_LIMIT_NS) {
        *abort_flag = 1u;
        return false;
      }
    }
  }
}

// What one part of a softmax counts against the whole: its maximum m and sum l, the largest maximum.
// A part without keys has m = -inf and l = 0; one whose scores are NaN has l = NaN, which stays.
__device__ __forceinline__ float part_weight(float m, float l, float gm) {
  if (m == -INFINITY) return l == 0.f ? 0.f : 1.f;
  return fast_exp2(m - gm);
}

// Entry of a launch: rows and context as they are used; -1 rows if something is out of range.
struct Kv8Entry {
  int first, rows, ctx;
};
__device__ __forceinline__ Kv8Entry kv8_entry(const Kv8Attn& a, int e) {
  Kv8Entry x;
  x.first = a.row0 != nullptr ? a.row0[e] : a.first + e;
  x.rows = a.row0 != nullptr ? a.row0[e + 1] - x.first : 1;
  x.ctx = max(0, a.ctx[e]);
  if (x.rows <= 0) x.rows = 0;
  else if (x.rows > a.most || x.first < 0 || x.first + x.rows > a.rows) x.rows = -1;
  return x;
}


// The launch's plan, made by one warp: units before every entry (prefix, in shared memory) and in all.  A tile of
// `tile` rows counts as many units as its sequence has pages, and `extra`.
__device__ __forceinline__ Kv8Entry kv8_used(const Kv8Attn& a, int e) {          // rows 0: nothing to do
  Kv8Entry x = kv8_entry(a, e);
  x.rows = max(x.rows, 0);
  x.ctx = min(x.ctx, a.c.max_pages * KV8_PAGE);
  return x;
}
__device__ __forceinline__ int kv8_plan(const Kv8Attn& a, int tile, int extra, int* prefix, int lane) {
  int units = 0;
  if (lane == 0) prefix[0] = 0;
#pragma unroll 4
  for (int e0 = 0; e0 < a.n; e0 += 32) {
    const int e = e0 + lane;
    int s = 0;
    if (e < a.n) {
      const Kv8Entry x = kv8_used(a, e);
      if (blockIdx.x == 0 && (kv8_entry(a, e).rows < 0 || a.ctx[e] > a.c.max_pages * KV8_PAGE)) record_status(a.status, ST_BOUNDS, e);
      if (x.ctx > 0) s = (x.rows * a.group + tile - 1) / tile * ((x.ctx + KV8_PAGE - 1) / KV8_PAGE + extra) * a.c.heads;
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += t;
    }
    if (e < a.n) prefix[e + 1] = units + s;
    units += __shfl_sync(0xffffffffu, s, 31);
  }
  __syncwarp();
  return units;
}
struct Kv8Where {          // a unit's tile
  int e, hk, tile, pages;
  int lo;                  // its first unit
  Kv8Entry x;
};
__device__ __forceinline__ Kv8Where kv8_locate(const Kv8Attn& a, int tile, int extra, const int* prefix, int u) {
  int lo = 0, hi = a.n;                                         // prefix[lo] <= u < prefix[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (prefix[mid] <= u) lo = mid;
    else hi = mid;
  }
  Kv8Where w;
  w.e = lo;
  w.x = kv8_used(a, lo);
  w.pages = (w.x.ctx + KV8_PAGE - 1) / KV8_PAGE;
  const int tiles = (w.x.rows * a.group + tile - 1) / tile, t = (u - prefix[lo]) / (w.pages + extra);
  w.hk = t / tiles;
  w.tile = t % tiles;
  w.lo = prefix[lo] + t * (w.pages + extra);
  return w;
}
__device__ __forceinline__ void kv8_describe(const Kv8Attn& a, int tile, int extra, const int* prefix, int u0, int n_units, int share, int units) {
  Kv8Desc d{u0, u0, share, units, 0, 0, 0, 0};
  if (n_units > 0) {
    const Kv8Where w = kv8_locate(a, tile, extra, prefix, u0);
    d.lo = w.lo;
    d.hi = w.lo + w.pages;
    d.entry = w.e;
    d.head = w.hk;
    d.tile = w.tile;
  }
  a.desc[blockIdx.x] = d;
}
// Rows of entries without keys are zero.
template <int DH>
__device__ __forceinline__ void kv8_zero_rows(const Kv8Attn& a, int tid, int threads) {
  for (int e = blockIdx.x; e < a.n; e += gridDim.x) {
    const Kv8Entry x = kv8_used(a, e);
    if (x.ctx == 0)
      for (int r = 0; r < x.rows; ++r)
        for (int i = tid; i < a.group * a.c.heads * DH; i += threads) a.out[static_cast<size_t>(x.first + r) * a.ldo + i] = __float2bfloat16(0.f);
  }
}
// Tiles that lie in more than one CTA: the CTA behind the tile's first boundary has its block here.  The warps take the
// parts in turn.
constexpr int KM_WARPS = 16;
template <int DH, int TILE>
__global__ void __launch_bounds__(32 * KM_WARPS) kv8_attn_merge_kernel(const __grid_constant__ Kv8Attn a) {
  constexpr int QR = 8, PER = DH / 32;                           // rows of a block: the blockIdx.y-th eight of the tile
  __shared__ float s_max[KM_WARPS], s_sum[KM_WARPS];
  __shared__ float s_o[KM_WARPS][DH];
  asm volatile("griddepcontrol.wait;" ::: "memory");             // the parts are complete
  const int b = blockIdx.x + 1;
  const Kv8Desc d = a.desc[b];
  const long long at = static_cast<long long>(d.share) * b;
  // starts here, ends before, or has begun before the last boundary
  if (at >= d.units || d.lo >= at || d.hi <= at || d.lo < at - d.share) return;
  const int parts = static_cast<int>((d.hi - at + d.share - 1) / d.share) + 1;
  const size_t s0 = static_cast<size_t>(b - 1) * 2 + (d.lo == at - d.share ? 0 : 1);
  auto slot = [&](int i) { return i == 0 ? s0 : static_cast<size_t>(b - 1 + i) * 2; };
  const Kv8Entry x = kv8_entry(a, d.entry);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int base = d.tile * TILE + blockIdx.y * QR, n_rows = min(QR, x.rows * a.group - base);
  if (n_rows <= 0) return;
  const int ctx = min(x.ctx, a.c.max_pages * KV8_PAGE);
  // warp w has row w mod n_rows, and of its parts every subs-th from w / n_rows on
  const int r = warp % n_rows, sub = warp / n_rows, subs = KM_WARPS / n_rows;
  const int mine = sub < subs && sub < parts ? (parts - sub + subs - 1) / subs : 0;
  auto ml = [&](int i) { return *reinterpret_cast<const float2*>(a.part_ml + (slot(sub + subs * i) * TILE + blockIdx.y * QR + r) * 2); };
  float gm = -INFINITY, gl = 0.f, o[PER];
  for (int i = lane; i < mine; i += 32) gm = fmaxf(gm, ml(i).x);
  gm = warp_max(gm);
  if (lane == 0) s_max[warp] = gm;
#pragma unroll
  for (int y = 0; y < PER; ++y) o[y] = 0.f;
  __syncthreads();
  for (int w = r; w < subs * n_rows; w += n_rows) gm = fmaxf(gm, s_max[w]);
  for (int i0 = 0; i0 < mine; i0 += 32) {
    float k = 0.f;
    if (i0 + lane < mine) {
      const float2 v = ml(i0 + lane);
      k = part_weight(v.x, v.y, gm);
      if (k != 0.f) gl += k * v.y;
    }
    const int n = min(32, mine - i0);
#pragma unroll 8
    for (int i = 0; i < n; ++i) {
      const float ki = __shfl_sync(0xffffffffu, k, i);
      const float* src = a.part_o + (slot(sub + subs * (i0 + i)) * TILE + blockIdx.y * QR + r) * DH + lane * PER;
#pragma unroll
      for (int y = 0; y < PER; ++y) o[y] = fmaf(ki, src[y], o[y]);
    }
  }
  gl = warp_sum(gl);
  if (lane == 0) s_sum[warp] = gl;
#pragma unroll
  for (int y = 0; y < PER; ++y) s_o[warp][lane * PER + y] = o[y];
  __syncthreads();
  for (int e = threadIdx.x; e < n_rows * DH; e += 32 * KM_WARPS) {
    const int er = e / DH, ch = e % DH, rr = base + er;
    float v = 0.f, sum = 0.f;
    for (int w = er; w < subs * n_rows; w += n_rows) {
      v += s_o[w][ch];
      sum += s_sum[w];
    }
    const bool any = ctx - x.rows + rr / a.group + 1 > 0;
    a.out[static_cast<size_t>(x.first + rr / a.group) * a.ldo + (d.head * a.group + rr % a.group) * DH + ch] =
        __float2bfloat16(any ? v / sum : 0.f);
  }
}


// Behind the kernel whose parts it merges, launched while that one runs: it waits for that one's end itself.
template <int DH, int TILE>
static int launch_kv8_merge(const Kv8Attn& a, int ctas, cudaStream_t st) {
  if (ctas < 2) return 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas - 1, TILE / 8);
  cfg.blockDim = 32 * KM_WARPS;
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kv8_attn_merge_kernel<DH, TILE>, a) == cudaSuccess ? 0 : -3;
}

}  // namespace cb
