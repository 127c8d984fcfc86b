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
  x.first = a.first + e;
  x.rows = 1;
  x.ctx = max(0, a.ctx[e]);
  if (a.row0 != nullptr && !kv8_rows_of(a.row0, e, a.rows, a.most, x.first, x.rows)) x.rows = -1;
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
// Behind the kernel whose parts it merges, launched while that one runs: it waits for that one's end itself.
inline int launch_kv8_merge(void (*kernel)(Kv8Attn), dim3 grid, int threads, const Kv8Attn& a, int ctas, cudaStream_t st) {
  if (ctas < 2) return 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = threads;
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, a) == cudaSuccess ? 0 : -3;
}

}  // namespace cb
