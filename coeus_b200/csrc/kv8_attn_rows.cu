// Attention over the 8-bit cache for many query rows per sequence (kv8_attn.cu has the mathematics and the
// kernel for few): tiles of 128 rows (rows and heads that share a key/value head) on the fifth-generation
// tensor cores, a page of 64 keys at a time.
//
//   warps 4 - 7   turn the page's codes into fp16 operands in shared memory (exactly; 128-byte swizzle), the next page
//                 on its way in registers, and the tile's queries before its first page
//   warp 8        issues S = Q K^T (one accumulator of two), warp 9 O += P V: one thread for both needed about 1500 cycles
//                 a page to issue them, more than they take
//   warps 0 - 3   a row per thread: weights from S, written back as fp16 in tensor memory, where the second product
//                 reads them; the running maximum, the sum, and at the end the tile's rows
//
// The scale 2^ev of a page's values goes into the weights: with z = s + ev (s the score in units of log2) and m a
// running maximum of z, the weights are P = 2^(z - m).  The denominator has a maximum of its own, md of s alone, and
// sums 2^(m - ev - md) P = 2^(s - md): o = 2^(m - md) sum P code / sum 2^(s - md).  So pages of any scales add up in one
// accumulator, and a page without values, whose ev says nothing, counts for the denominator alone.  m and md are whole
// numbers, only raised when they are exceeded by more than KB_LAG, and the sums so far are multiplied then.  Where a
// page's scale is far below that of the sums (KB_NEAR) but its scores are not, m is lowered to md + ev: its values may
// be all that some channels have.  A page of a tile is 2 x 64 x 128 dh multiply-adds and 8192 exponentials; what bounds
// it is the chain of score product, softmax and value product, two tiles an SM in turn.  Four sequences of 8192 with 512
// rows each, 32 heads over 8 of 128: 443 us and 18 for the merge, 0.35 of the bf16 rate.  Four of 2000 to 8200 with 301
// to 700 rows: 348 us in all (377 with the maxima raised for every page), 469 with one CTA an SM and one issuing thread;
// 200 with nothing but the products and the barriers.  Keys and values handed over separately: 360.
#include "kv8_attn.cuh"

namespace cb {

constexpr int KB_ROWS = 128;                      // of a tile
constexpr int KB_EXTRA = 2;                       // what a tile costs beside its pages, in pages
constexpr int KB_SHARE = 4;                       // pages a CTA takes at least
constexpr int KB_THREADS = 320;
constexpr int KB_STAGES = 2;
constexpr int KB_PLACES = 2;                      // CTAs that share an SM: the waits of one are the other's time
// Weights are held times 2^KB_SHIFT and are at most 2^(KB_SHIFT + KB_LAG) < 65504; fp16 keeps their digits down to 2^-23
// of the row's largest, and 2^-34 is lost.
constexpr float KB_SHIFT = 10.f, KB_LAG = 4.f;
constexpr float KB_LOST = 36.f;                   // weights up to 2^(KB_SHIFT - KB_LOST) are zero in fp16
// Scales that lie under those of the sums by this much lower m, and by how much at most in all: 2^20 keys, weights of 2^14
// and codes of 2^9 leave fp32 that room.
constexpr float KB_NEAR = 8.f, KB_DEEP = 70.f;
constexpr float KB_NONE = -1e30f;                 // maxima of rows that have seen nothing
constexpr uint32_t KB_O = 0, KB_S = 128, KB_COLS = 256;                  // columns of tensor memory; weights lie on their scores

template <int DH>
struct RowsSmem {
  static constexpr int PANEL_K = KV8_PAGE * 128;                 // 64 channels of 64 keys, fp16
  static constexpr int HALVES = DH / 64;
  static constexpr int V = HALVES * PANEL_K, STAGE = V + DH * 128;      // keys, then values [channel][64 keys]
  static constexpr int Q = HALVES * KB_ROWS * 128;
  static constexpr int BYTES = 1024 + Q + KB_STAGES * STAGE + 4 * KB_ROWS * 4 + KB_STAGES * 16 + (KA_ENTRIES + 1) * 4 + 256;
};

// 16 codes to 16 numbers of fp16 in two vectors.
template <int KIND>
__device__ __forceinline__ void half16(const uint4& w, uint4& a, uint4& b) {
  kv8_half4<KIND>(w.x, a.x, a.y);
  kv8_half4<KIND>(w.y, a.z, a.w);
  kv8_half4<KIND>(w.z, b.x, b.y);
  kv8_half4<KIND>(w.w, b.z, b.w);
}
__device__ __forceinline__ constexpr uint32_t idesc_f16(int m, int n) {
  return umma_idesc_bf16(m, n, 0, 0) & ~((7u << 7) | (7u << 10));        // both operands fp16
}

template <int KIND, int DH>
__global__ void __launch_bounds__(KB_THREADS, KB_PLACES) kv8_rows_kernel(const __grid_constant__ Kv8Attn a) {
  using S = RowsSmem<DH>;
  constexpr int HALVES = S::HALVES;
  extern __shared__ __align__(16) unsigned char raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  unsigned char* sq = smem;                                      // [HALVES][128 rows][128 bytes]
  unsigned char* stage = sq + S::Q;                              // [KB_STAGES][STAGE]
  float* sf = reinterpret_cast<float*>(stage + KB_STAGES * S::STAGE);      // [4 tiles][128]: score per product
  float4* meta = reinterpret_cast<float4*>(sf + 4 * KB_ROWS);    // [KB_STAGES]: scales of the page, whether there is one
  uint64_t* bars = reinterpret_cast<uint64_t*>(meta + KB_STAGES);
  uint64_t *full = bars, *empty = full + KB_STAGES, *s_full = empty + KB_STAGES, *p_full = s_full + 2, *o_done = p_full + 2;
  uint64_t *q_full = o_done + 2, *q_free = q_full + 1;
  int* prefix = reinterpret_cast<int*>(q_free + 1);              // [KA_ENTRIES + 1]
  __shared__ volatile uint32_t abort_flag;
  __shared__ uint32_t tmem_slot;
  __shared__ int s_units;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, nkv = a.c.heads;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (warp == 8) {
    tmem_alloc(smem_u32(&tmem_slot), KB_COLS);
    tmem_relinquish();
  } else if (warp == 0) {
    const int n = kv8_plan(a, KB_ROWS, KB_EXTRA, prefix, lane);
    if (lane == 0) s_units = n;
  }
  if (tid == 64) {
    abort_flag = 0u;
    for (int i = 0; i < KB_STAGES; ++i) {
      mbar_init(smem_u32(full + i), 128);
      mbar_init(smem_u32(empty + i), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(s_full + i), 1);
      mbar_init(smem_u32(p_full + i), 128);
      mbar_init(smem_u32(o_done + i), 1);
    }
    mbar_init(smem_u32(q_full), 128);
    mbar_init(smem_u32(q_free), 1);
    mbar_fence_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const int units = s_units, share = max((units - 1) / static_cast<int>(gridDim.x) + 1, KB_SHARE);
  const int u0 = static_cast<int>(min(static_cast<long long>(units), static_cast<long long>(share) * blockIdx.x));
  const int u1 = min(units - u0, share) + u0;
  if (tid == 0) kv8_describe(a, KB_ROWS, KB_EXTRA, prefix, u0, u1 - u0, share, units);
  kv8_zero_rows<DH>(a, tid, KB_THREADS);

  // A tile's pages here: p0 .. p1 - 1 (none for its extra units, or if no row of it sees that far).
  struct Piece {
    Kv8Where w;
    int p0, p1;
    bool any, whole, begins;           // there are pages at all; all of the tile is here; it is the CTA's first tile
  };
  auto piece_at = [&](int u) {
    Piece t;
    t.w = kv8_locate(a, KB_ROWS, KB_EXTRA, prefix, u);
    t.p0 = u - t.w.lo;
    const int end = min(t.w.pages, u1 - t.w.lo), last = min(t.w.x.rows - 1, (t.w.tile * KB_ROWS + KB_ROWS - 1) / a.group);
    const int all_seen = t.w.x.ctx - t.w.x.rows + last + 1;
    t.any = t.p0 < end;
    t.p1 = min(end, (max(all_seen, 0) + KV8_PAGE - 1) / KV8_PAGE);
    t.whole = t.w.lo >= u0 && t.w.lo + t.w.pages <= u1;
    t.begins = t.w.lo <= u0;
    return t;
  };
  auto next_tile = [&](const Piece& t) { return t.w.lo + t.w.pages + KB_EXTRA; };
  bool dead = false;
  auto wait = [&](uint64_t* bar, int n) {                        // the n-th phase (from 0)
    if (dead) return;
    if (!wait_phase(bar, n & 1, &abort_flag)) {
      dead = true;
      record_status(a.status, ST_WAIT_TIMEOUT, blockIdx.x);
    }
  };

  if (warp >= 4 && warp < 8) {
    // ---- operands
    const int t0 = tid - 128;
    int gi = 0, tiles = 0;                                       // pages and tiles so far
    constexpr int VECS = DH / 32;                                // 16-byte vectors of codes of a thread, keys and values each
    for (int u = u0; u < u1;) {
      const Piece t = piece_at(u);
      u = next_tile(t);
      if (!t.any || t.p0 >= t.p1) continue;
      const int* table = a.c.page_table + static_cast<size_t>(t.w.e) * a.c.max_pages;
      auto page_of = [&](int p) { return p < t.p1 ? __ldg(table + p) : 0; };
      uint4 kc[VECS], vc[VECS];
      float ks = 0.f, vs = 0.f;
      const uint4 *kn, *vn;                                      // the next page's codes
      size_t cell_n = 0;
      int ok_n = 0;
      auto aim = [&](int page) {
        ok_n = page >= 0 && page < a.c.num_pages;
        if (!ok_n) {
          if (t0 == 0) record_status(a.status, ST_BOUNDS, t.w.e);
          page = 0;
        }
        cell_n = static_cast<size_t>(page) * nkv + t.w.hk;
        kn = reinterpret_cast<const uint4*>(a.c.k + cell_n * (KV8_PAGE * DH)) + t0;
        vn = reinterpret_cast<const uint4*>(a.c.v + cell_n * (KV8_PAGE * DH)) + t0;
      };
      aim(page_of(t.p0));
      int ok = ok_n;
#pragma unroll
      for (int i = 0; i < VECS; ++i) {
        kc[i] = __ldg(kn + 128 * i);
        vc[i] = __ldg(vn + 128 * i);
      }
      ks = __ldg(a.c.k_scale + cell_n);
      vs = __ldg(a.c.v_scale + cell_n);
      int page = page_of(t.p0 + 1);
      // the tile's queries: a row per thread, divided by the binade of its largest number
      if (tiles > 0) wait(q_free, tiles - 1);
      {
        const int r = t.w.tile * KB_ROWS + t0;
        const bool in = r < t.w.x.rows * a.group;
        const uint4* src = reinterpret_cast<const uint4*>(a.q + (in ? static_cast<size_t>(t.w.x.first + r / a.group) * a.ldq + (t.w.hk * a.group + r % a.group) * DH : 0));
        float top = 0.f;
        if (in)
#pragma unroll 4
          for (int i = 0; i < DH / 8; ++i) {
            const uint4 x = __ldg(src + i);
            const uint32_t* v = reinterpret_cast<const uint32_t*>(&x);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float2 b = unpack_bf16x2(v[j]);
              top = fmaxf(top, fmaxf(fabsf(b.x), fabsf(b.y)));
            }
          }
        const int k = top > 0.f && top < INFINITY ? max(min((__float_as_int(top) >> 23) - 127, 126), -126) : 0;
        const float down = pow2(-k);
        sf[(tiles & 3) * KB_ROWS + t0] = pow2(k) * a.scale_log2;
#pragma unroll 4
        for (int i = 0; i < DH / 8; ++i) {
          uint4 x = make_uint4(0u, 0u, 0u, 0u);
          if (in) {
            x = __ldg(src + i);
            uint32_t* v = reinterpret_cast<uint32_t*>(&x);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float2 b = unpack_bf16x2(v[j]);
              v[j] = half2_bits(b.x * down, b.y * down);
            }
          }
          *reinterpret_cast<uint4*>(sq + (i / 8 * KB_ROWS + t0) * 128 + ((i & 7) ^ (t0 & 7)) * 16) = x;
        }
      }
      fence_proxy_async_smem();
      mbar_arrive(smem_u32(q_full));
      ++tiles;
      const int last = min(t.w.x.rows - 1, (t.w.tile * KB_ROWS + KB_ROWS - 1) / a.group);
      const int all_seen = t.w.x.ctx - t.w.x.rows + last + 1;
      for (int p = t.p0; p < t.p1; ++p, ++gi) {
        const int st = gi % KB_STAGES;
        if (gi >= KB_STAGES) wait(empty + st, gi / KB_STAGES - 1);
        unsigned char* kd = stage + st * S::STAGE;
        const int left = all_seen - p * KV8_PAGE;                // tokens of the page that any row sees
        if (t0 == 0) meta[st] = make_float4(ks, vs, ok ? 1.f : 0.f, 0.f);
        const bool more = p + 1 < t.p1;
        if (more) {
          aim(page);
          page = page_of(p + 2);
          ok = ok_n;
          ks = __ldg(a.c.k_scale + cell_n);
          vs = __ldg(a.c.v_scale + cell_n);
        }
        if (left < KV8_PAGE) {
          // codes of values that no row sees may be anything (not a number even): zero times them is not zero
#pragma unroll
          for (int i = 0; i < VECS; ++i) {
            uint32_t* w = reinterpret_cast<uint32_t*>(&vc[i]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int over = left - 16 * (t0 & 3) - 4 * j;
              w[j] &= over >= 4 ? 0xffffffffu : over <= 0 ? 0u : (1u << (8 * over)) - 1u;
            }
          }
        }
        // row x >> 2 of the operand, 16 codes x & 3 of it; the next page's are asked for as soon as these are used
        unsigned char* const d0 = kd + (t0 >> 2) * 128;
        const int c0 = ((2 * (t0 & 3)) ^ (t0 >> 2 & 7)) * 16, c1 = c0 ^ 16;    // 32 rows on the swizzle is the same
#pragma unroll
        for (int i = 0; i < VECS; ++i) {
          uint4 lo, hi;
          half16<KIND>(kc[i], lo, hi);
          if (more) kc[i] = __ldg(kn + 128 * i);
          *reinterpret_cast<uint4*>(d0 + i * 4096 + c0) = lo;
          *reinterpret_cast<uint4*>(d0 + i * 4096 + c1) = hi;
          half16<KIND>(vc[i], lo, hi);
          if (more) vc[i] = __ldg(vn + 128 * i);
          *reinterpret_cast<uint4*>(d0 + S::V + i * 4096 + c0) = lo;
          *reinterpret_cast<uint4*>(d0 + S::V + i * 4096 + c1) = hi;
        }
        fence_proxy_async_smem();
        mbar_arrive(smem_u32(full + st));
      }
    }
  } else if (warp == 8) {
    // ---- scores: the warp goes through the loop together (its addresses then are uniform registers, which the
    // instruction wants) and one thread of it issues
    constexpr uint32_t id_s = idesc_f16(KB_ROWS, KV8_PAGE);
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    const uint64_t dq = umma_desc_sw128(smem_u32(sq), 16, 1024), dk = umma_desc_sw128(smem_u32(stage), 16, 1024);
    int gi = 0, tiles = 0;
    for (int u = u0; u < u1 && !dead;) {
      const Piece t = piece_at(u);
      u = next_tile(t);
      if (!t.any || t.p0 >= t.p1) continue;
      wait(q_full, tiles++);
      for (int n = t.p1 - t.p0; n > 0; --n, ++gi) {
        const int st = gi % KB_STAGES;
        wait(full + st, gi / KB_STAGES);
        if (gi >= 2) wait(o_done + (gi & 1), (gi >> 1) - 1);     // the weights that were here have been used
        if (__any_sync(0xffffffffu, dead)) {
          dead = true;
          break;
        }
        tc_fence_after();
        const uint64_t dks = dk + static_cast<uint64_t>(st * (S::STAGE >> 4));
        const uint32_t d = tm + KB_S + (gi & 1) * KV8_PAGE;
        if (elect_one()) {
#pragma unroll
          for (int h = 0; h < HALVES; ++h)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              umma_bf16_ss(d, dq + static_cast<uint64_t>((h * KB_ROWS * 128 + k * 32) >> 4),
                           dks + static_cast<uint64_t>((h * S::PANEL_K + k * 32) >> 4), id_s, h + k > 0 ? 1u : 0u);
          umma_commit(smem_u32(s_full + (gi & 1)));
          if (n == 1) umma_commit(smem_u32(q_free));
        }
        __syncwarp();
      }
    }
  } else if (warp == 9) {
    // ---- weighted values
    constexpr uint32_t id_o = idesc_f16(KB_ROWS, DH);
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    const uint64_t dv = umma_desc_sw128(smem_u32(stage + S::V), 16, 1024);
    int gi = 0;
    for (int u = u0; u < u1 && !dead;) {
      const Piece t = piece_at(u);
      u = next_tile(t);
      if (!t.any) continue;
      for (int p = t.p0; p < t.p1; ++p, ++gi) {
        wait(p_full + (gi & 1), gi >> 1);
        if (__any_sync(0xffffffffu, dead)) {
          dead = true;
          break;
        }
        tc_fence_after();
        const int st = gi % KB_STAGES;
        const uint64_t dvs = dv + static_cast<uint64_t>(st * (S::STAGE >> 4));
        const uint32_t pa = tm + KB_S + (gi & 1) * KV8_PAGE;
        const uint32_t more = p > t.p0 ? 1u : 0u;
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < 4; ++k) umma_bf16_ts(tm + KB_O, pa + k * 8, dvs + static_cast<uint64_t>((k * 32) >> 4), id_o, k > 0 ? 1u : more);
          umma_commit(smem_u32(o_done + (gi & 1)));
          umma_commit(smem_u32(empty + st));
        }
        __syncwarp();
      }
    }
  } else {
    // ---- weights: a row per thread
    const uint32_t mine = tmem + (static_cast<uint32_t>(warp * 32) << 16);
    int gi = 0, tiles = 0;
    for (int u = u0; u < u1;) {
      const Piece t = piece_at(u);
      u = next_tile(t);
      if (!t.any) continue;
      const int rows = t.w.x.rows, ctx = t.w.x.ctx, total = rows * a.group, rr = t.w.tile * KB_ROWS + tid;
      const int seen = ctx - rows + min(rr, total - 1) / a.group + 1;
      const int least_seen = ctx - rows + t.w.tile * KB_ROWS / a.group + 1;
      float m = KB_NONE, md = KB_NONE, l = 0.f, f = 0.f;         // maxima of z and s, sum of 2^(s - md)
      float m_top = KB_NONE;                                     // the largest m so far
      for (int p = t.p0; p < t.p1; ++p, ++gi) {
        const int st = gi % KB_STAGES, base = p * KV8_PAGE;
        wait(full + st, gi / KB_STAGES);
        wait(s_full + (gi & 1), gi >> 1);
        if (dead) break;
        tc_fence_after();
        if (p == t.p0) f = sf[(tiles & 3) * KB_ROWS + tid];
        const float4 mt = meta[st];
        const uint32_t sa = mine + KB_S + (gi & 1) * KV8_PAGE;
        const float ev = mt.y == mt.y ? static_cast<float>((__float_as_int(mt.y) >> 23) - 127) : 0.f;
        const float fk = f * mt.x, ef = mt.y == mt.y ? ev : mt.y;
        const bool whole = base + KV8_PAGE <= least_seen && mt.z != 0.f;
        const int n_seen = mt.z != 0.f ? seen - base : 0;        // keys of the page that the row sees
        // The row's scores twice, 32 at a time (two CTAs leave a thread 96 registers): for the maximum, then for the weights.
        float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float s[32];
          tmem_ld_32x32b_x32(sa + 32 * h, reinterpret_cast<uint32_t*>(s));
          tmem_ld_wait();
          if (!whole) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (32 * h + i >= n_seen) s[i] = -INFINITY;
          }
#pragma unroll
          for (int i = 0; i < 32; i += 8)
#pragma unroll
            for (int j = 0; j < 4; ++j) top[j] = max3(top[j], s[i + j], s[i + 4 + j]);
        }
        const float smax = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * fk, z = smax + ef;      // NaN: no maximum
        float scale_gap = m - md - ev;                           // of the sums over the page
        const bool over = z > m + KB_LAG || smax > md + KB_LAG, under = scale_gap > KB_NEAR && mt.y > 1.17549435e-38f;
        if (__any_sync(0xffffffffu, over || under)) {
          if (smax > md + KB_LAG) {
            const float mdn = ceilf(smax);
            l *= fast_exp2(md - mdn);
            md = mdn;
          }
          const bool lower = under && z + KB_LOST > md + ev && m_top - m < KB_DEEP;
          const float mn = z > m + KB_LAG ? ceilf(z) : lower ? fmaxf(fmaxf(md + ev, ceilf(z)), m_top - KB_DEEP) : m;
          m_top = fmaxf(m_top, mn);
          const float c = mn == m ? 1.f : fast_exp2(m - mn);     // exact
          m = mn;
          scale_gap = m - md - ev;
          if (p > t.p0 && __any_sync(0xffffffffu, c != 1.f)) {   // the sums so far: the last product is over
            wait(o_done + ((gi - 1) & 1), (gi - 1) >> 1);
            tc_fence_after();
#pragma unroll
            for (int i = 0; i < DH; i += 32) {
              uint32_t o[32];
              tmem_ld_32x32b_x32(mine + KB_O + i, o);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * c);
              tmem_st_32x32b_x16(mine + KB_O + i, o);
              tmem_st_32x32b_x16(mine + KB_O + i + 16, o + 16);
            }
            tmem_st_wait();
          }
        }
        // Weights below what fp16 holds (m so far above z) are for the denominator only, and formed for it.
        const bool lost = z + KB_LOST < m || mt.y == 0.f;
        const float sub = KB_SHIFT + (lost ? -md : ef - m);
        const float unit = fast_exp2((lost ? 0.f : scale_gap) - KB_SHIFT);
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float s[32];
          tmem_ld_32x32b_x32(sa + 32 * h, reinterpret_cast<uint32_t*>(s));
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            fma2(s[i], s[i + 1], s[i], s[i + 1], fk, fk, sub, sub);
            s[i] = fast_exp2(s[i]);
            s[i + 1] = fast_exp2(s[i + 1]);
          }
          if (!whole) {                                          // whatever the scales are
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (32 * h + i >= n_seen) s[i] = 0.f;
          }
          uint32_t w[16];
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            add2(sum[0], sum[1], sum[0], sum[1], s[i], s[i + 1]);
            add2(sum[2], sum[3], sum[2], sum[3], s[i + 2], s[i + 3]);
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) w[i] = lost ? 0u : half2_bits(s[2 * i], s[2 * i + 1]);
          tmem_st_32x32b_x16(sa + 16 * h, w);                    // on scores that have been read
        }
        if (n_seen > 0) l = fmaf((sum[0] + sum[1]) + (sum[2] + sum[3]), unit, l);
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(smem_u32(p_full + (gi & 1)));
      }
      if (dead) break;
      // ---- the tile's rows, or this CTA's part of them
      const size_t slot = static_cast<size_t>(blockIdx.x) * 2 + (t.begins ? 0 : 1);
      const bool summed = t.p0 < t.p1;
      if (summed) {
        ++tiles;
        wait(o_done + ((gi - 1) & 1), (gi - 1) >> 1);
        if (dead) break;
        tc_fence_after();
      }
      // 2^(m - md) in two factors, so that none leaves fp32's range before the product does
      constexpr float down = 1.f / (1 << static_cast<int>(KB_SHIFT));
      const float up = md > KB_NONE ? fast_exp2(0.5f * (m - md)) : 1.f, inv = seen > 0 && summed ? up / l : 0.f;
      auto part = [&](uint32_t x) { return __uint_as_float(x) * down * up * up; };
      __nv_bfloat16* dst = a.out + static_cast<size_t>(t.w.x.first + rr / a.group) * a.ldo + (t.w.hk * a.group + rr % a.group) * DH;
#pragma unroll
      for (int i = 0; i < DH; i += 32) {
        uint32_t o[32];
        if (summed) {
          tmem_ld_32x32b_x32(mine + KB_O + i, o);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) o[j] = 0u;
        }
        if (rr < total) {
          if (t.whole) {
#pragma unroll
            for (int j = 0; j < 32; j += 8) {
              float v[8];
#pragma unroll
              for (int x = 0; x < 8; ++x) v[x] = seen > 0 ? __uint_as_float(o[j + x]) * down * up * inv : 0.f;
              store8(dst + i + j, v);
            }
          } else {
#pragma unroll
            for (int j = 0; j < 32; j += 4)
              *reinterpret_cast<uint4*>(a.part_o + (slot * KB_ROWS + tid) * DH + i + j) = 
                  make_uint4(__float_as_uint(part(o[j])), __float_as_uint(part(o[j + 1])),
                             __float_as_uint(part(o[j + 2])), __float_as_uint(part(o[j + 3])));
          }
        }
      }
      if (!t.whole && rr < total) *reinterpret_cast<float2*>(a.part_ml + (slot * KB_ROWS + tid) * 2) = make_float2(md > KB_NONE ? md : -INFINITY, l);
      tc_fence_before();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, KB_COLS);
  }
}

// Tiles that lie in more than one CTA, as in kv8_attn.cuh, for tiles of many rows and few parts: a warp a row.
template <int DH>
__global__ void __launch_bounds__(256) kv8_rows_merge_kernel(const __grid_constant__ Kv8Attn a) {
  constexpr int PER = DH / 32;
  asm volatile("griddepcontrol.wait;" ::: "memory");             // the parts are complete
  const int b = blockIdx.x + 1;
  const Kv8Desc d = a.desc[b];
  const long long at = static_cast<long long>(d.share) * b;
  if (at >= d.units || d.lo >= at || d.hi <= at || d.lo < at - d.share) return;
  const int parts = static_cast<int>((d.hi - at + d.share - 1) / d.share) + 1;
  const Kv8Entry x = kv8_entry(a, d.entry);
  const int r = blockIdx.y * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31, rr = d.tile * KB_ROWS + r;
  if (rr >= x.rows * a.group) return;
  const size_t s0 = static_cast<size_t>(b - 1) * 2 + (d.lo == at - d.share ? 0 : 1);
  auto slot = [&](int i) { return (i == 0 ? s0 : static_cast<size_t>(b - 1 + i) * 2) * KB_ROWS + r; };
  float gm = -INFINITY, gl = 0.f, o[PER];
  for (int i = lane; i < parts; i += 32) gm = fmaxf(gm, a.part_ml[slot(i) * 2]);
  gm = warp_max(gm);
#pragma unroll
  for (int y = 0; y < PER; ++y) o[y] = 0.f;
#pragma unroll 2
  for (int i = 0; i < parts; ++i) {
    const float2 v = *reinterpret_cast<const float2*>(a.part_ml + slot(i) * 2);
    const float k = part_weight(v.x, v.y, gm);
    const float* src = a.part_o + slot(i) * DH + lane * PER;
    if (k != 0.f) gl += k * v.y;
#pragma unroll
    for (int y = 0; y < PER; ++y) o[y] = fmaf(k, src[y], o[y]);
  }
  const int ctx = min(x.ctx, a.c.max_pages * KV8_PAGE);
  const float inv = ctx - x.rows + rr / a.group + 1 > 0 ? 1.f / gl : 0.f;
  __nv_bfloat162* dst = reinterpret_cast<__nv_bfloat162*>(
      a.out + static_cast<size_t>(x.first + rr / a.group) * a.ldo + (d.head * a.group + rr % a.group) * DH + lane * PER);
#pragma unroll
  for (int y = 0; y < PER; y += 2) dst[y / 2] = __floats2bfloat162_rn(o[y] * inv, o[y + 1] * inv);
}

static_assert(RowsSmem<128>::BYTES <= 113 * 1024 && KB_PLACES * KB_COLS <= 512, "two CTAs per SM");

template <int KIND, int DH>
static int launch_rows(const Kv8Attn& a, int ctas, cudaStream_t st) {
  using S = RowsSmem<DH>;
  static bool set[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return -4;
  // at least a third of an SM's shared memory, so that no more CTAs share it than its tensor memory has columns for
  const int bytes = S::BYTES > 80 * 1024 ? S::BYTES : 80 * 1024;
  if (dev >= 64 || !set[dev]) {
    if (cudaFuncSetAttribute(kv8_rows_kernel<KIND, DH>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
      return -4;
    if (dev < 64) set[dev] = true;
  }
  kv8_rows_kernel<KIND, DH><<<ctas, KB_THREADS, bytes, st>>>(a);
  const int rc = launch_kv8_merge(kv8_rows_merge_kernel<DH>, dim3(ctas - 1, KB_ROWS / 8), 256, a, ctas, st);
  if (rc != 0) return rc;
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}
int launch_kv8_rows(const Kv8Attn& a, int kind, int dh, int ctas, cudaStream_t st) {
  if (kind == KV8_INT8) return dh == 64 ? launch_rows<KV8_INT8, 64>(a, ctas, st) : launch_rows<KV8_INT8, 128>(a, ctas, st);
  return dh == 64 ? launch_rows<KV8_E4M3, 64>(a, ctas, st) : launch_rows<KV8_E4M3, 128>(a, ctas, st);
}
int kv8_rows_tile() { return KB_ROWS; }
int kv8_rows_places() { return KB_PLACES; }
int kv8_rows_share() { return KB_SHARE; }
int kv8_rows_extra() { return KB_EXTRA; }

}  // namespace cb
