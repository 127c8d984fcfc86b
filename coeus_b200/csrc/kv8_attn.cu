// Attention over the 8-bit cache (kv8.cuh has the layout).  Row i of entry e (r rows, context n) sits
// at position n - r + i of its sequence and sees the positions up to that one; query head h reads
// key/value head h / (heads / kv_heads).  A row that sees nothing gets zeros.
//
//   o = sum_t w_t v_t / sum_t w_t,  w_t = exp(scale q . k_t - max),  k_t = code 2^ek, v_t = code 2^ev
//
// The cache has to be streamed once, two bytes of it per key and channel, and everything else has to
// hide behind that.  Work is cut into units of one page of one key/value head for one tile of eight query rows
// (rows and heads that share the head).  A CTA is one warp that takes an equal run of units, whatever the lengths of
// the sequences, and keeps its next pages coming with bulk copies (a page's keys and values are 64 dh bytes each); as
// many CTAs as shared memory holds share an SM (dh 128: six) and know nothing of each other.  Warps of one CTA that
// took the pages of a tile in turn and merged their parts waited for one another (64 sequences of 1000 to 8200, 32
// heads over 8 of 128: 175 to 255 us, so 124).  64 sequences of 4096 with these heads: 101 us and 12 for the merge, 0.81 of
// the copy rate; 64 of 2048 with 16 heads of 64: 57 and 16, 0.72; one of 131072: 50 and 17, 0.82.  What it waits for is
// latency (36 % of the issue slots are used): the steps of a page follow one another and there are no more warps.
//
// Both products are transposed, S^T = K Q^T and O^T = V^T P^T (mma m16n8k16 in fp16, fp32 sums), so that
// the cached side is the operand of 16 rows and the few query rows are the eight columns.  Which
// token or channel a row or column of a fragment stands for is free as long as both operands agree, and
// is chosen so that every fragment of the cached side is consecutive bytes of a lane:
//   keys     lane (g, c) holds channels 16c .. 16c + 15 of a 64-channel half; one of its four words per k-step
//   tokens   row r of the eight of (step s, half u) is token 16 (r / 2) + 4 s + 2 u + r % 2, so that after
//            the transposition of the weights (movmatrix) lane (g, c) has tokens 16c + 4s .. + 3: the
//            word s of its 16 bytes of a row of values
// Codes become fp16 exactly: int8 by setting the biased byte into the mantissa of 1024 and subtracting, e4m3
// by its conversion.  Queries are fp16 after division by a power of two per row.  Weights enter the second product
// as fp16 times 2^12, against the largest of their page: smaller than 2^-26 of it they start to lose bits, and less than
// 2^-36 of it is lost in all.  What a page's largest weight is against the row's, and the page's 2^ev, are applied in fp32 to
// the sums of the page, so that a page of little weight keeps its part however large its values are.
#include "kv8_attn.cuh"

namespace cb {

constexpr int KA_ROWS = 8;                        // query rows of a tile
constexpr int KA_SHARE = 2;                       // units a CTA takes at least
constexpr int KA_EXTRA = 1;                       // what a tile costs beside its pages, in units
// Rows and heads of an entry that share a key/value head: up to KA_NARROW this kernel's tiles are the faster ones, above
// KA_WIDE the wide ones.  In between a tile of eight more costs 2.6 ns a page here (dh 128, the device full) and nothing
// there, where a page costs 5.7 ns and the call some 18 us more: wide when the tiles over two, times the pages, are more
// than KA_WORK.  24 sequences of 500 to 4100 tokens, 8 heads, 24 / 32 / 48 / 64 rows: 82 / 100 / 137 / 172 us here, 80 / 82 /
// 84 / 88 there; one sequence of 8000: 35 / 37 / 37 / 47 and 45 / 45 / 47 / 47, and
// with 96 and 192 rows 51 / 84 and 51 / 53.
constexpr int KA_NARROW = 24, KA_WIDE = 64, KA_WORK = 7000;
constexpr int KA_BLOCK = 16;                      // units that are planned at a time
constexpr int KA_RING = 4;                        // copies in a warp's ring: the keys and values of two pages
constexpr int KA_PLACES = 6, KA_PLACES64 = 11;    // CTAs that share an SM, by its shared memory: dh 128, 64
constexpr float KA_SHIFT = 12.f;                  // weights are held times 2^12 against their page's largest

__device__ __forceinline__ void mma_f16(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, "
      "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// kv8_attn_rows.cu
int launch_kv8_rows(const Kv8Attn& a, int kind, int dh, int ctas, cudaStream_t st);
int kv8_rows_tile();
int kv8_rows_share();
int kv8_rows_extra();
int kv8_rows_places();

// A unit as it is planned: a page of a tile, and the tile's share of the CTA's units (counted from 0).
struct Kv8Unit {
  int flags;               // UNIT_*
  int page, p;             // page of the cache, of the sequence
  int first, rows, ctx;    // the entry's
  int head, tile;
  float ks, vs;
};
// a page (and not a tile's extra); with keys that count; the tile's first page here; its last; all of the tile is here;
// it is the CTA's first tile
enum : int { UNIT_PAGE = 1, UNIT_LIVE = 2, UNIT_BEGIN = 4, UNIT_LAST = 8, UNIT_WHOLE = 16, UNIT_FIRST = 32 };

template <int DH>
struct Kv8Smem {
  static constexpr int SLOT = KV8_PAGE * DH;                    // bytes of a page's keys, or of its values
  static constexpr int BYTES = KA_RING * (SLOT + 8) + (KA_ENTRIES + 1) * 4 + 2 * KA_BLOCK * static_cast<int>(sizeof(Kv8Unit)) + 32;
};

template <int KIND, int DH>
__global__ void __launch_bounds__(32) kv8_attn_kernel(const __grid_constant__ Kv8Attn a) {
  using S = Kv8Smem<DH>;
  constexpr int QR = KA_ROWS, RING = KA_RING, AHEAD = RING / 2;                 // pages ahead of the one that is computed
  extern __shared__ __align__(128) unsigned char smem[];
  unsigned char* ring = smem;                                                   // [RING][SLOT]
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + RING * S::SLOT);          // [RING]: the copy is there
  int* prefix = reinterpret_cast<int*>(full + RING);                            // [KA_ENTRIES + 1]: units before every entry
  Kv8Unit* book = reinterpret_cast<Kv8Unit*>((reinterpret_cast<uintptr_t>(prefix + KA_ENTRIES + 1) + 15) & ~uintptr_t(15));  // [2][KA_BLOCK]
  __shared__ volatile uint32_t abort_flag;
  const int lane = threadIdx.x, nkv = a.c.heads;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // ---- the plan: units before every entry
  if (lane == 0) {
    abort_flag = 0u;
    for (int i = 0; i < RING; ++i) mbar_init(smem_u32(full + i), 1);
    mbar_fence_init();
  }
  const int units = kv8_plan(a, QR, KA_EXTRA, prefix, lane);
  const int share = max((units - 1) / static_cast<int>(gridDim.x) + 1, KA_SHARE);
  const int u0 = static_cast<int>(min(static_cast<long long>(units), static_cast<long long>(share) * blockIdx.x));
  const int u1 = min(units - u0, share) + u0, n_units = u1 - u0;

  if (lane == 0) kv8_describe(a, QR, KA_EXTRA, prefix, u0, n_units, share, units);
  kv8_zero_rows<DH>(a, lane, 32);

  const int g = lane >> 2, c = lane & 3;
  // Units are planned KA_BLOCK at a time, one a lane, while those before them run: what the page table and the scales
  // take to answer is hidden.
  Kv8Unit x;
  auto plan_page = [&](int block) {                             // place of the lane's unit, its page asked for
    const int j = block * KA_BLOCK + lane;
    x.flags = 0;
    if (j >= n_units || lane >= KA_BLOCK) return;
    const Kv8Where w = kv8_locate(a, QR, KA_EXTRA, prefix, u0 + j);
    x.p = u0 + j - w.lo;
    if (x.p >= w.pages) return;
    x.flags = UNIT_PAGE;
    x.first = w.x.first;
    x.rows = w.x.rows;
    x.ctx = w.x.ctx;
    x.head = w.hk;
    x.tile = w.tile;
    if (x.p == 0 || j == 0) x.flags |= UNIT_BEGIN;
    if (x.p == w.pages - 1 || j == n_units - 1) x.flags |= UNIT_LAST;
    if (w.lo >= u0 && w.lo + w.pages <= u1) x.flags |= UNIT_WHOLE;
    if (w.lo <= u0) x.flags |= UNIT_FIRST;
    // a page behind what the last row of the tile sees is not read
    const int last = min(w.x.rows - 1, (w.tile * QR + QR - 1) / a.group);
    if (x.p * KV8_PAGE < w.x.ctx - w.x.rows + last + 1) {
      x.flags |= UNIT_LIVE;
      x.page = a.c.page_table[static_cast<size_t>(w.e) * a.c.max_pages + x.p];
    }
  };
  auto plan_check = [&]() {                                     // the page is known
    if ((x.flags & UNIT_LIVE) && (x.page < 0 || x.page >= a.c.num_pages)) {
      record_status(a.status, ST_BOUNDS, x.first);
      x.flags &= ~UNIT_LIVE;
    }
  };
  auto plan_scale = [&]() {                                     // its scales are asked for
    if (!(x.flags & UNIT_LIVE)) return;
    const size_t cell = static_cast<size_t>(x.page) * nkv + x.head;
    x.ks = a.c.k_scale[cell];
    x.vs = a.c.v_scale[cell];
  };
  auto plan_done = [&](int block) {
    if (lane < KA_BLOCK) book[(block & 1) * KA_BLOCK + lane] = x;
    __syncwarp();
  };
  auto unit_at = [&](int i) -> const Kv8Unit& { return book[i % (2 * KA_BLOCK)]; };
  int asked = 0, done = 0;                                      // pages copied, computed
  bool dead = false;
  auto ask = [&](int i) {                                       // the copies of unit i
    const Kv8Unit& y = unit_at(i);
    if (!(y.flags & UNIT_LIVE)) return;
    if (lane == 0) {
      const size_t at = (static_cast<size_t>(y.page) * nkv + y.head) * S::SLOT;
      const int k = 2 * asked % RING, v = k + 1;
      mbar_arrive_expect_tx(smem_u32(full + k), S::SLOT);
      bulk_load_g2s(smem_u32(ring + k * S::SLOT), a.c.k + at, S::SLOT, smem_u32(full + k));
      mbar_arrive_expect_tx(smem_u32(full + v), S::SLOT);
      bulk_load_g2s(smem_u32(ring + v * S::SLOT), a.c.v + at, S::SLOT, smem_u32(full + v));
    }
    ++asked;
  };
  auto failed = [&]() {
    dead = true;
    if (lane == 0) record_status(a.status, ST_WAIT_TIMEOUT, blockIdx.x);
  };
  plan_page(0);
  plan_check();
  plan_done(0);
  for (int i = 0; i < min(AHEAD, n_units); ++i) ask(i);          // the first copies do not wait for the scales
  plan_scale();
  plan_done(0);
  uint32_t qf[DH / 64][4][2];
  float f[2], o[DH / 16][4], m[2], l[2];                         // columns 2c and 2c + 1; f: score per product
  int seen[2], least_seen = 0, all_seen = 0;
  for (int i = 0; i < n_units; ++i) {
    if ((i / KA_BLOCK + 1) * KA_BLOCK < n_units) {
      if (i % KA_BLOCK == 0) plan_page(i / KA_BLOCK + 1);
      else if (i % KA_BLOCK == 5) { plan_check(); plan_scale(); }
      else if (i % KA_BLOCK == 10) plan_done(i / KA_BLOCK + 1);
    }
    const Kv8Unit un = unit_at(i);
    if (un.flags & UNIT_PAGE) {
    const bool live = un.flags & UNIT_LIVE;
    const int sk = 2 * done % RING, sv = sk + 1;
    const uint32_t phase = 2 * done / RING & 1;
    const float ks = un.ks, vs = un.vs;
    const int rows = un.rows, ctx = un.ctx, first = un.first;
    const int total = rows * a.group;                            // rows of all tiles of this head
    if (un.flags & UNIT_BEGIN) {
      // ---- a new tile: its queries; lane (g, c) has row g, channels 16c .. of every half
      const int r = un.tile * QR + g;
      uint4 x[DH / 64][2];
      float top = 0.f;
#pragma unroll
      for (int h = 0; h < DH / 64; ++h)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          x[h][y] = make_uint4(0u, 0u, 0u, 0u);
          if (r < total) {
            const __nv_bfloat16* src = a.q + static_cast<size_t>(first + r / a.group) * a.ldq +
                                       (un.head * a.group + r % a.group) * DH + h * 64 + c * 16 + y * 8;
            x[h][y] = __ldg(reinterpret_cast<const uint4*>(src));
          }
        }
#pragma unroll
      for (int h = 0; h < DH / 64; ++h)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const uint32_t* v = reinterpret_cast<const uint32_t*>(&x[h][y]);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 b = unpack_bf16x2(v[i]);
            top = fmaxf(top, fmaxf(fabsf(b.x), fabsf(b.y)));
          }
        }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // 2^k is the binade of the row's largest number; a row of zeros or infinities stays as it is
      const int k = top > 0.f && top < INFINITY ? max(min((__float_as_int(top) >> 23) - 127, 126), -126) : 0;
      const float down = pow2(-k), up = pow2(k) * a.scale_log2;
#pragma unroll
      for (int h = 0; h < DH / 64; ++h)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const uint32_t* v = reinterpret_cast<const uint32_t*>(&x[h][y]);
#pragma unroll
          for (int i = 0; i < 4; ++i) {                          // channels 16c + 8y + 2i, + 1
            const float2 b = unpack_bf16x2(v[i]);
            qf[h][2 * y + i / 2][i % 2] = half2_bits(b.x * down, b.y * down);
          }
        }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        f[i] = __shfl_sync(0xffffffffu, up, (2 * c + i) * 4);
        seen[i] = ctx - rows + min(un.tile * QR + 2 * c + i, total - 1) / a.group + 1;
        m[i] = -INFINITY;
        l[i] = 0.f;
      }
      least_seen = ctx - rows + (un.tile * QR) / a.group + 1;
      all_seen = ctx - rows + min(rows - 1, (un.tile * QR + QR - 1) / a.group) + 1;
#pragma unroll
      for (int i = 0; i < DH / 16; ++i)
#pragma unroll
        for (int x2 = 0; x2 < 4; ++x2) o[i][x2] = 0.f;
    }
    if (live && !dead && !wait_phase(full + sk, phase, &abort_flag)) failed();
    const int base = un.p * KV8_PAGE, key0 = base + 16 * (g >> 1) + (g & 1);
    const bool whole = base + KV8_PAGE <= least_seen;            // every row sees every key
    float s[4][4];
    if (live) {
      // the four steps' sums are independent: their products go round, so that none waits for its own last one
      const uint4* row = reinterpret_cast<const uint4*>(ring + sk * S::SLOT + (16 * (g >> 1) + (g & 1)) * 64 + c * 16);
#pragma unroll
      for (int y = 0; y < 4; ++y)
#pragma unroll
        for (int x = 0; x < 4; ++x) s[y][x] = 0.f;
#pragma unroll
      for (int h = 0; h < DH / 64; ++h) {
        uint4 k0[4], k1[4];
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          k0[y] = row[y * 16 + h * 256];
          k1[y] = row[y * 16 + h * 256 + 8];
        }
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            uint32_t fa[4];
            kv8_half4<KIND>(reinterpret_cast<const uint32_t*>(&k0[y])[x], fa[0], fa[2]);
            kv8_half4<KIND>(reinterpret_cast<const uint32_t*>(&k1[y])[x], fa[1], fa[3]);
            mma_f16(s[y], fa, qf[h][x][0], qf[h][x][1]);
          }
      }
    }
    uint32_t pf[4][2];
    float keep[2], scale_v[2];
    if (live) {
      if (!whole) {
#pragma unroll
        for (int y = 0; y < 4; ++y)
#pragma unroll
          for (int x = 0; x < 4; ++x)
            if (key0 + 4 * y + 2 * (x >> 1) >= seen[x & 1]) s[y][x] = -INFINITY;
      }
      float sub[2], fk[2], part[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float mx = max3(fmaxf(s[0][i], s[0][2 + i]), fmaxf(s[1][i], s[1][2 + i]), max3(s[2][i], s[2][2 + i], fmaxf(s[3][i], s[3][2 + i])));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        fk[i] = f[i] * ks;
        const bool sees = base < seen[i];                        // a row that sees none of it takes none, NaN neither
        const float mp = sees ? mx * fk[i] : -INFINITY, mn = fmaxf(m[i], mp);
        const float base_m = mn == -INFINITY ? 0.f : mn;
        keep[i] = fast_exp2(m[i] - base_m);
        m[i] = mn;
        sub[i] = KA_SHIFT - (mp == -INFINITY ? 0.f : mp);
        part[i] = fast_exp2(mp - base_m - KA_SHIFT);
        scale_v[i] = sees ? vs * part[i] : 0.f;
      }
#pragma unroll
      for (int y = 0; y < 4; ++y)
#pragma unroll
        for (int x = 0; x < 4; ++x) s[y][x] = fast_exp2(fmaf(s[y][x], fk[x & 1], sub[x & 1]));
      if (!whole) {                                              // whatever the scale of the keys is
#pragma unroll
        for (int y = 0; y < 4; ++y)
#pragma unroll
          for (int x = 0; x < 4; ++x)
            if (key0 + 4 * y + 2 * (x >> 1) >= seen[x & 1]) s[y][x] = 0.f;
      }
      // the columns' sums of the rounded weights: a product with ones
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
      const uint32_t ones[4] = {0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u};
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        pf[y][0] = transpose8(half2_bits(s[y][0], s[y][1]));
        pf[y][1] = transpose8(half2_bits(s[y][2], s[y][3]));
        mma_f16(sum, ones, pf[y][0], pf[y][1]);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) l[i] = fmaf(l[i], keep[i], sum[i] * part[i]);
    }
    if (live && !dead && !wait_phase(full + sv, phase, &abort_flag)) failed();
    if (live) {
      if (!whole) {
        // codes of values behind what any row sees may be anything (not a number even): zero times them is not zero
        const int left = all_seen - base;
#pragma unroll 1
        for (int i = lane; i < DH * 16; i += 32) {
          const int over = left - (i & 15) * 4;                  // word i & 15 of a row has four tokens
          if (over < 4) reinterpret_cast<uint32_t*>(ring + sv * S::SLOT)[i] &= over <= 0 ? 0u : (1u << (8 * over)) - 1u;
        }
        fence_proxy_async_smem();
        __syncwarp();
      }
      if (__any_sync(0xffffffffu, keep[0] != 1.f || keep[1] != 1.f)) {       // a maximum has grown (or is NaN)
#pragma unroll
        for (int d = 0; d < DH / 16; ++d)
#pragma unroll
          for (int x = 0; x < 4; ++x) o[d][x] *= keep[x & 1];
      }
      const unsigned char* vb = ring + sv * S::SLOT + g * 64 + c * 16;
      // four rows of results at a time, for the same reason
#pragma unroll
      for (int d0 = 0; d0 < DH / 16; d0 += 4) {
        uint4 v0[4], v1[4];
        float op[4][4];
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          v0[d] = *reinterpret_cast<const uint4*>(vb + (d0 + d) * 1024);
          v1[d] = *reinterpret_cast<const uint4*>(vb + (d0 + d) * 1024 + 512);
#pragma unroll
          for (int x = 0; x < 4; ++x) op[d][x] = 0.f;
        }
#pragma unroll
        for (int y = 0; y < 4; ++y)
#pragma unroll
          for (int d = 0; d < 4; ++d) {
            uint32_t fa[4];
            kv8_half4<KIND>(reinterpret_cast<const uint32_t*>(&v0[d])[y], fa[0], fa[2]);
            kv8_half4<KIND>(reinterpret_cast<const uint32_t*>(&v1[d])[y], fa[1], fa[3]);
            mma_f16(op[d], fa, pf[y][0], pf[y][1]);
          }
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
          for (int x = 0; x < 4; ++x) o[d0 + d][x] = fmaf(op[d][x], scale_v[x & 1], o[d0 + d][x]);
      }
    }
    __syncwarp();
    done += live;
    if (un.flags & UNIT_LAST) {
      // ---- the tile's last page here: its result, or its part of it
      const size_t slot = static_cast<size_t>(blockIdx.x) * 2 + (un.flags & UNIT_FIRST ? 0 : 1);
#pragma unroll
      for (int i2 = 0; i2 < 2; ++i2) {
        const int r = 2 * c + i2, rr = un.tile * QR + r;
        if (rr >= total) continue;
        if (un.flags & UNIT_WHOLE) {
          const float inv = ctx - rows + rr / a.group + 1 > 0 ? 1.f / l[i2] : 0.f;
          __nv_bfloat16* dst = a.out + static_cast<size_t>(first + rr / a.group) * a.ldo + (un.head * a.group + rr % a.group) * DH + g;
#pragma unroll
          for (int d = 0; d < DH / 16; ++d) {
            dst[d * 16] = __float2bfloat16(o[d][i2] * inv);
            dst[d * 16 + 8] = __float2bfloat16(o[d][2 + i2] * inv);
          }
        } else {
          float* dst = a.part_o + (slot * QR + r) * DH + g;
#pragma unroll
          for (int d = 0; d < DH / 16; ++d) {
            dst[d * 16] = o[d][i2];
            dst[d * 16 + 8] = o[d][2 + i2];
          }
          if (g == 0) *reinterpret_cast<float2*>(a.part_ml + (slot * QR + r) * 2) = make_float2(m[i2], l[i2]);
        }
      }
    }
    }
    if (i + AHEAD < n_units) ask(i + AHEAD);
  }
}

// Tiles that lie in more than one CTA: the CTA behind the tile's first boundary has its block here.  The warps take the
// parts in turn.
constexpr int KM_WARPS = 16;
template <int DH>
__global__ void __launch_bounds__(32 * KM_WARPS) kv8_attn_merge_kernel(const __grid_constant__ Kv8Attn a) {
  constexpr int QR = KA_ROWS, PER = DH / 32;
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
  const int base = d.tile * QR, n_rows = min(QR, x.rows * a.group - base);
  const int ctx = min(x.ctx, a.c.max_pages * KV8_PAGE);
  // warp w has row w mod n_rows, and of its parts every subs-th from w / n_rows on
  const int r = warp % n_rows, sub = warp / n_rows, subs = KM_WARPS / n_rows;
  const int mine = sub < subs && sub < parts ? (parts - sub + subs - 1) / subs : 0;
  auto ml = [&](int i) { return *reinterpret_cast<const float2*>(a.part_ml + (slot(sub + subs * i) * QR + r) * 2); };
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
      const float* src = a.part_o + (slot(sub + subs * (i0 + i)) * QR + r) * DH + lane * PER;
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

template <int KIND, int DH>
static int launch_attn(const Kv8Attn& a, int ctas, cudaStream_t st) {
  using S = Kv8Smem<DH>;
  static bool set[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return -4;
  if (dev >= 64 || !set[dev]) {
    if (cudaFuncSetAttribute(kv8_attn_kernel<KIND, DH>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::BYTES) != cudaSuccess)
      return -4;
    if (dev < 64) set[dev] = true;
  }
  kv8_attn_kernel<KIND, DH><<<ctas, 32, S::BYTES, st>>>(a);
  const int rc = launch_kv8_merge(kv8_attn_merge_kernel<DH>, dim3(ctas - 1), 32 * KM_WARPS, a, ctas, st);
  if (rc != 0) return rc;
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

// How a call is cut: the tile (eight rows, or the wide one of kv8_attn_rows.cu), the units of an entry at most,
// entries of a launch, CTAs of a launch (one for every place on the device, where there is work).
struct AttnShape {
  bool wide;
  int tile, each, ctas;
  long long units;
  AttnShape(int n, int rows, int most, int group, int max_pages, int kv_heads, int dh) {
    if (most > rows) most = rows;                              // a row counts at most once
    const long long shared = 1ll * most * group, pages = 1ll * n * kv_heads * max_pages;
    wide = shared > KA_WIDE || (shared > KA_NARROW && ((shared + 7) / 8 - 2) * pages > KA_WORK);
    tile = wide ? kv8_rows_tile() : KA_ROWS;
    units = (1ll * most * group + tile - 1) / tile * (max_pages + (wide ? kv8_rows_extra() : KA_EXTRA)) * kv_heads;
    const long long fit = units > 0 ? 0x7fffffffll / units : 0;
    each = static_cast<int>(fit < n ? fit : n);
    if (each > KA_ENTRIES) each = KA_ENTRIES;
    const int share = wide ? kv8_rows_share() : KA_SHARE;
    const long long places = static_cast<long long>(wide ? kv8_rows_places() : dh == 64 ? KA_PLACES64 : KA_PLACES) * sm_count();
    const long long work = (each * units + share - 1) / share;
    ctas = static_cast<int>(work < places ? work : places);
  }
};

}  // namespace cb

using namespace cb;

// Bytes of scratch of one call.
extern "C" int64_t cb_kv8_attn_scratch(int n, int rows, int most, int group, int max_pages, int kv_heads, int dh) {
  const AttnShape s(n, rows, most, group, max_pages, kv_heads, dh);
  return s.ctas * static_cast<int64_t>(2 * s.tile * (dh + 2) * 4 + sizeof(Kv8Desc)) + 256;
}

extern "C" int cb_kv8_attn(const void* q, int ldq, const void* k_cache, const void* v_cache, const float* k_scale,
                           const float* v_scale, const int* page_table, int max_pages, int num_pages, int kv_heads,
                           int dh, int kind, const int* ctx, const int* row0, int n, int rows, int most, int heads,
                           float scale, void* out, int ldo, void* scratch, int* status, void* stream) {
  if (n < 1 || rows < 1 || most < 1 || kv_heads < 1 || heads < 1 || heads % kv_heads != 0) return -1;
  if ((dh != 64 && dh != 128) || (kind != KV8_INT8 && kind != KV8_E4M3)) return -2;
  const int group = heads / kv_heads;
  const AttnShape s(n, rows, most, group, max_pages, kv_heads, dh);
  if (1ll * max_pages * KV8_PAGE > 0x7fffffffll || s.each < 1) return -5;
  const int each = s.each, ctas = s.ctas;
  Kv8Attn a;
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.out = static_cast<__nv_bfloat16*>(out);
  a.ldq = ldq; a.ldo = ldo; a.group = group; a.rows = rows; a.most = most < rows ? most : rows;
  a.scale_log2 = scale * KA_LOG2E;
  a.desc = static_cast<Kv8Desc*>(scratch);
  a.part_o = reinterpret_cast<float*>(static_cast<char*>(scratch) + (ctas * sizeof(Kv8Desc) + 255) / 256 * 256);
  a.part_ml = a.part_o + static_cast<size_t>(ctas) * 2 * s.tile * dh;
  a.status = status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  for (int e0 = 0; e0 < n; e0 += each) {
    a.c = Kv8Cache{static_cast<uint8_t*>(const_cast<void*>(k_cache)), static_cast<uint8_t*>(const_cast<void*>(v_cache)),
                   const_cast<float*>(k_scale), const_cast<float*>(v_scale),
                   page_table + static_cast<size_t>(e0) * max_pages, max_pages, num_pages, kv_heads};
    a.ctx = ctx + e0;
    a.row0 = row0 != nullptr ? row0 + e0 : nullptr;
    a.first = e0;
    a.n = n - e0 < each ? n - e0 : each;
    int rc;
    if (s.wide) rc = launch_kv8_rows(a, kind, dh, ctas, st);
    else if (kind == KV8_INT8) rc = dh == 64 ? launch_attn<KV8_INT8, 64>(a, ctas, st) : launch_attn<KV8_INT8, 128>(a, ctas, st);
    else rc = dh == 64 ? launch_attn<KV8_E4M3, 64>(a, ctas, st) : launch_attn<KV8_E4M3, 128>(a, ctas, st);
    if (rc != 0) return rc;
  }
  return 0;
}
