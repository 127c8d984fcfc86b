// A beam search's step: the K best continuations of the K beams of every request, and the beams'
// pages moved to where their new parents' are.
//
// Selection.  Continuation t of beam j is worth score_j + logit_jt - logsumexp(logit_j); a beam that has
// ended continues with the end token alone, at its own score.  Taken are the K largest, equal ones by
// the lowest j V + t.  The values are formed in fp64: they differ between beams by less than fp32 resolves.
// 32 requests of 8 beams, 6 of them going on, of 100008 fp32 logits (77 MB): 17.4 us for the pass (0.67 of the copy rate;
// 18.1 for rows of 100003, read one by one), 23 for the choice, which is a chain of reductions of one CTA per request and
// does not get shorter with fewer bytes; 8 of 8 beams in bf16 (51 MB): 21 and 25, bound by the exponentials.
//   pass   one read of the logits: maximum and sum of exponentials of every block of BLK of a row.
//   pick   one CTA per request.  The K best continuations lie in the K blocks whose best ones are
//          the best (equal ones by the lowest place): each of those holds one that precedes whatever lies in
//          another block.  So the blocks' maxima choose K blocks, and only those are read again.
//
// Pages.  A request's beams share the pages of what they have in common.  With n tokens stored the next
// one goes to page n / 64: full pages are taken over from the parent by number; of the beams whose parents
// hold the same page of n mod 64 tokens (children of one parent, or of parents that have not parted yet) the first keeps
// it, the others get a free page of the request's pool and a copy.  A page is free when no new row of the request holds
// it, so nothing is counted from step to step.
#include "common.cuh"
#include "ptx.cuh"

namespace cb {

constexpr int BEAM_MAX = 32;           // beams of a request
constexpr int BLK = 512;               // logits of a block (ops/beam.py sizes the scratch by it)
constexpr int PICK_THREADS = 512;
constexpr int PICK_PER = 4;            // blocks that a thread keeps the values of
constexpr int PICK_CAP = 1024;         // continuations compared at once; at least BEAM_MAX for every warp

// Block k of a row has logits k BLK - skew .. (k + 1) BLK - skew - 1, as far as there are any.  Where all rows begin alike
// against multiples of 16 bytes, `skew` is by how many logits they do, so that they are read in vectors all the same.
// Where they do not, it is 0 and logits are read one by one: were the rows cut each by its own address, rows with the
// same logits would have sums that differ by a rounding, and beams that tie would not.
__device__ __forceinline__ float beam_logit(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float beam_logit(const float* p) { return *p; }
// 16 bytes of logits; `lo` and `hi` cut off what is not the row's.
template <typename T>
__device__ __forceinline__ void beam_vector(const T* row, int t, int V, float* x) {
  constexpr int N = 16 / sizeof(T);
  if (t >= 0 && t + N <= V) {
    const uint4 w = __ldg(reinterpret_cast<const uint4*>(row + t));
    if constexpr (N == 8) {
      const uint32_t* v = reinterpret_cast<const uint32_t*>(&w);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 b = unpack_bf16x2(v[i]);
        x[2 * i] = b.x;
        x[2 * i + 1] = b.y;
      }
    } else {
      x[0] = __uint_as_float(w.x); x[1] = __uint_as_float(w.y); x[2] = __uint_as_float(w.z); x[3] = __uint_as_float(w.w);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = t + i >= 0 && t + i < V ? beam_logit(row + t + i) : -INFINITY;
  }
}

constexpr int PASS_WARPS = 4;
template <typename T, bool VECTORS>
__global__ void __launch_bounds__(32 * PASS_WARPS) beam_pass_kernel(const T* __restrict__ logits, int64_t ld, int V, int nblk,
                                                                    int skew, const float* __restrict__ scores,
                                                                    const uint8_t* __restrict__ done, float2* __restrict__ part) {
  constexpr int N = 16 / sizeof(T), PER = BLK / 32;              // logits of a vector, of a lane
  const int row = blockIdx.y, blk = blockIdx.x * PASS_WARPS + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (blk >= nblk || done[row] || scores[row] == -INFINITY) return;
  const T* x = logits + row * ld;
  const int t0 = blk * BLK - skew;
  float v[PER];
  if constexpr (VECTORS) {
#pragma unroll
    for (int i = 0; i < PER / N; ++i) beam_vector(x, t0 + (i * 32 + lane) * N, V, v + i * N);
  } else {
    x += t0 + lane;
    if (t0 + BLK <= V) {
#pragma unroll
      for (int i = 0; i < PER; ++i) v[i] = beam_logit(x + i * 32);
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i) v[i] = t0 + i * 32 + lane < V ? beam_logit(x + i * 32) : -INFINITY;
    }
  }
  float m = v[0], s = 0.f;
#pragma unroll
  for (int i = 1; i < PER; ++i) m = fmaxf(m, v[i]);
  m = warp_max(m);
  const float base = m == -INFINITY ? 0.f : m;                   // nothing but -inf: the sum is 0
#pragma unroll
  for (int i = 0; i < PER; ++i) s += expf(v[i] - base);          // NaN and +inf make it NaN
  s = warp_sum(s);
  if (lane == 0) part[static_cast<size_t>(row) * nblk + blk] = make_float2(m, s);
}

struct Best {              // a continuation or a block: larger value first, then the lower place
  int64_t v;               // key of the value
  uint32_t at;             // at most 32 beams of 2^26 logits
};
// Values as whole numbers in the same order (-0 below +0, which the sums here never give): comparing these takes a
// tenth of what fp64 comparisons do, and the selection is little else.
__device__ __forceinline__ int64_t value_key(double v) {
  const int64_t b = __double_as_longlong(v + 0.0);
  return b ^ ((b >> 63) & 0x7fffffffffffffffll);
}
__device__ __forceinline__ double key_value(int64_t k) { return __longlong_as_double(k ^ ((k >> 63) & 0x7fffffffffffffffll)); }
__device__ __forceinline__ bool better(int64_t v, uint32_t at, const Best& b) { return v > b.v || (v == b.v && at < b.at); }
__device__ __forceinline__ Best block_best(Best b, Best* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const int64_t v = __shfl_xor_sync(0xffffffffu, b.v, o);
    const uint32_t at = __shfl_xor_sync(0xffffffffu, b.at, o);
    if (better(v, at, b)) b = Best{v, at};
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = b;
  __syncthreads();
  b = red[0];
  for (int w = 1; w < PICK_THREADS / 32; ++w)
    if (better(red[w].v, red[w].at, b)) b = red[w];
  return b;
}

template <typename T>
__global__ void __launch_bounds__(PICK_THREADS)
beam_pick_kernel(const T* __restrict__ logits, int64_t ld, int V, int nblk, int skew, int K, const float* __restrict__ scores,
                 const uint8_t* __restrict__ done, int eos, const float2* __restrict__ part,
                 float* __restrict__ out_score, int64_t* __restrict__ out_parent, int64_t* __restrict__ out_token,
                 uint8_t* __restrict__ out_done) {
  __shared__ Best red[PICK_THREADS / 32];
  enum : int { DEAD, LIVE, ENDED };
  __shared__ double s_lse[BEAM_MAX], s_score[BEAM_MAX];
  __shared__ int s_state[BEAM_MAX];
  __shared__ int s_blk[BEAM_MAX];
  __shared__ int64_t c_v[PICK_CAP];
  __shared__ uint32_t c_at[PICK_CAP];
  __shared__ int64_t s_least;
  __shared__ int s_n;
  const int item = blockIdx.x, row0 = item * K;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t NEG = value_key(-INFINITY), TOP = 0x7fffffffffffffffll;
  constexpr uint32_t NONE = 0xffffffffu;
  for (int j = warp; j < K; j += PICK_THREADS / 32) {
    const float2* p = part + static_cast<size_t>(row0 + j) * nblk;
    // scores and states once, in shared memory: what follows asks for them all the time
    const float score = scores[row0 + j];
    const int state = done[row0 + j] ? ENDED : score != -INFINITY ? LIVE : DEAD;
    double lse = -INFINITY;
    if (state == LIVE) {
      // in fp64 but for the factors of the blocks: their errors (2 units of fp32 each) average out like those of the
      // logits' own exponentials
      float m = -INFINITY;
#pragma unroll 4
      for (int i = lane; i < nblk; i += 32) m = fmaxf(m, p[i].x);
      m = warp_max(m);
      double s = 0.0;
#pragma unroll 1
      for (int i = lane; i < nblk; i += 32) {
        const float2 q = p[i];
        s += q.x == -INFINITY && q.y == 0.f ? 0.0 : static_cast<double>(q.y) * static_cast<double>(expf(q.x - m));
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      lse = static_cast<double>(m) + log(s);
    }
    if (lane == 0) {
      s_lse[j] = lse;
      s_score[j] = static_cast<double>(score);
      s_state[j] = state;
    }
  }
  if (threadIdx.x == 0) s_n = 0;
  __syncthreads();
  // the value of a logit of beam j; what is not a number is no continuation
  auto value = [&](int j, float x) {
    const double v = s_score[j] + (static_cast<double>(x) - s_lse[j]);
    return v == v ? value_key(v) : NEG;
  };
  // the K best blocks (an ended beam is one block): each warp the K best of its share, one after the other without the
  // other warps, then every one of these counts those before it
  auto block_value = [&](int i, float x) {                       // x: the block's maximum
    const int j = i / nblk;
    if (s_state[j] == LIVE) return value(j, x);
    return s_state[j] == ENDED && i == j * nblk && eos >= 0 && s_score[j] == s_score[j] ? value_key(s_score[j]) : NEG;
  };
  const float2* row_part = part + static_cast<size_t>(row0) * nblk;
  {
    int64_t mine[PICK_PER];                                      // a thread keeps its first ones
    float top[PICK_PER];
#pragma unroll
    for (int u = 0; u < PICK_PER; ++u) {
      const int i = threadIdx.x + u * PICK_THREADS;
      top[u] = i < K * nblk && s_state[i / nblk] == LIVE ? row_part[i].x : 0.f;
    }
#pragma unroll
    for (int u = 0; u < PICK_PER; ++u) {
      const int i = threadIdx.x + u * PICK_THREADS;
      mine[u] = i < K * nblk ? block_value(i, top[u]) : NEG;
    }
    Best last{TOP, NONE};
    for (int n = 0; n < K; ++n) {
      Best b{NEG, NONE};
      auto look = [&](int64_t v, uint32_t i) {
        if (v > NEG && better(v, i, b) && !better(v, i, last) && i != last.at) b = Best{v, i};
      };
#pragma unroll
      for (int u = 0; u < PICK_PER; ++u) look(mine[u], threadIdx.x + u * PICK_THREADS);
      for (int i = threadIdx.x + PICK_PER * PICK_THREADS; i < K * nblk; i += PICK_THREADS)
        look(block_value(i, s_state[i / nblk] == LIVE ? row_part[i].x : 0.f), i);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const int64_t v = __shfl_xor_sync(0xffffffffu, b.v, o);
        const uint32_t at = __shfl_xor_sync(0xffffffffu, b.at, o);
        if (better(v, at, b)) b = Best{v, at};
      }
      if (lane == 0) {
        c_v[warp * K + n] = b.v;
        c_at[warp * K + n] = b.at;
      }
      last = b;
      if (!(b.v > NEG)) last.v = NEG;                            // no more: so will be the others
    }
  }
  if (threadIdx.x < K) s_blk[threadIdx.x] = -1;
  __syncthreads();
  const int warp_best = PICK_THREADS / 32 * K;
  for (int i = threadIdx.x; i < warp_best; i += PICK_THREADS) {
    const Best me{c_v[i], c_at[i]};
    if (!(me.v > NEG)) continue;
    int rank = 0;
#pragma unroll 8
    for (int o = 0; o < warp_best; ++o) rank += better(c_v[o], c_at[o], me);
    if (rank < K) {
      s_blk[rank] = static_cast<int>(me.at);
      if (rank == K - 1) s_least = me.v;
    }
  }
  __syncthreads();
  int found = 0;
  while (found < K && s_blk[found] >= 0) ++found;
  const int64_t least = found == K ? s_least : NEG;
  // every continuation of those blocks that is not below the last block's best: a warp a block
  auto each = [&](int64_t floor, auto&& f) {
    for (int n = warp; n < found; n += PICK_THREADS / 32) {
      const int j = s_blk[n] / nblk, k = s_blk[n] % nblk;
      if (s_state[j] == ENDED) {
        if (lane == 0) f(value_key(s_score[j]), static_cast<uint32_t>(j) * V + eos);
        continue;
      }
      const T* x = logits + (row0 + j) * ld;
      const int t0 = k * BLK - skew + lane;
      x += t0;
      float v[BLK / 32];
#pragma unroll
      for (int i = 0; i < BLK / 32; ++i) v[i] = t0 + 32 * i >= 0 && t0 + 32 * i < V ? beam_logit(x + 32 * i) : -INFINITY;
      // few of them count: the others are told by their logit alone
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < BLK / 32; ++i) top = fmaxf(top, v[i]);
      if (value(j, top) < floor) continue;
#pragma unroll 1
      for (int i = 0; i < BLK / 32; ++i) {
        const int t = t0 + 32 * i;
        if (t >= 0 && t < V) f(value(j, beam_logit(x + 32 * i)), static_cast<uint32_t>(j) * V + t);
      }
    }
  };
  __syncthreads();                       // the list is used again
  each(least, [&](int64_t v, uint32_t at) {
    if (v >= least && v > NEG) {
      const int n = atomicAdd(&s_n, 1);
      if (n < PICK_CAP) {
        c_v[n] = v;
        c_at[n] = at;
      }
    }
  });
  __syncthreads();
  const int n = s_n;
  auto put = [&](int place, int64_t v, uint32_t at) {
    const int j = static_cast<int>(at / static_cast<uint32_t>(V)), t = static_cast<int>(at - static_cast<uint32_t>(j) * V);
    out_score[row0 + place] = static_cast<float>(key_value(v));
    out_parent[row0 + place] = j;
    out_token[row0 + place] = t;
    out_done[row0 + place] = s_state[j] == ENDED || t == eos;
  };
  int filled;
  if (n <= PICK_CAP) {
    // a continuation's place is the number of those before it
    for (int i = threadIdx.x; i < n; i += PICK_THREADS) {
      int rank = 0;
      const Best me{c_v[i], c_at[i]};
      for (int o = 0; o < n; ++o) rank += better(c_v[o], c_at[o], me);
      if (rank < K) put(rank, me.v, me.at);
    }
    filled = min(n, K);
  } else {
    // more equal ones than that: one after the other
    Best prev{TOP, NONE};
    for (filled = 0; filled < K; ++filled) {
      Best b{NEG, NONE};
      each(NEG, [&](int64_t v, uint32_t at) {
        if (v > NEG && better(v, at, b) && !better(v, at, prev) && at != prev.at) b = Best{v, at};
      });
      b = block_best(b, red);
      if (!(b.v > NEG)) break;
      if (threadIdx.x == 0) put(filled, b.v, b.at);
      prev = b;
    }
  }
  for (int i = filled + threadIdx.x; i < K; i += PICK_THREADS) {      // places left: dead beams
    out_score[row0 + i] = -INFINITY;
    out_parent[row0 + i] = i;
    out_token[row0 + i] = max(eos, 0);
    out_done[row0 + i] = 1;
  }
}

// ------------------------------------------------------------------------------------ pages
constexpr int BEAM_PAGE = 64;
constexpr int PAGES_SMEM = 200 * 1024;           // of the bitmap, at most (ops/beam.py refuses larger caches)

// One CTA per request.  used: one bit per page of the cache, in shared memory.
__global__ void __launch_bounds__(256) beam_pages_kernel(const int* __restrict__ table, int width, int K,
                                                         const int64_t* __restrict__ parent,
                                                         const int* __restrict__ length, const int* __restrict__ pool,
                                                         int pool_n, int num_pages, int* __restrict__ out,
                                                         int* __restrict__ src, int* __restrict__ dst, int* status) {
  extern __shared__ uint32_t used[];
  __shared__ int s_parent[BEAM_MAX], s_tail[BEAM_MAX], s_keeps[BEAM_MAX], s_free[BEAM_MAX], s_turn[BEAM_MAX];
  const int item = blockIdx.x, row0 = item * K;
  const int len = length[item], lp = len / BEAM_PAGE;
  const bool partial = len % BEAM_PAGE != 0;
  if (len < 0 || lp >= width) {                       // no place for the next token
    for (int i = threadIdx.x; i < K * width; i += blockDim.x) out[static_cast<size_t>(row0) * width + i] = table[static_cast<size_t>(row0) * width + i];
    for (int j = threadIdx.x; j < K; j += blockDim.x) src[row0 + j] = dst[row0 + j] = -1;
    if (threadIdx.x == 0) record_status(status, ST_BOUNDS, item);
    return;
  }
  for (int i = threadIdx.x; i < (num_pages + 31) / 32; i += blockDim.x) used[i] = 0u;
  if (threadIdx.x < K) {
    int64_t p = parent[row0 + threadIdx.x];
    if (p < 0 || p >= K) {
      record_status(status, ST_BOUNDS, item);
      p = threadIdx.x;
    }
    s_parent[threadIdx.x] = static_cast<int>(p);
    s_tail[threadIdx.x] = table[static_cast<size_t>(row0 + p) * width + lp];
  }
  __syncthreads();
  if (threadIdx.x < K) {
    bool keeps = partial;
    for (int j = 0; j < threadIdx.x; ++j) keeps = keeps && s_tail[j] != s_tail[threadIdx.x];
    s_keeps[threadIdx.x] = keeps;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    int n = 0;
    for (int j = 0; j < K; ++j) {
      s_turn[j] = n;
      n += !s_keeps[j];
      s_free[j] = -1;
    }
  }
  auto mark = [&](int page) {
    if (page >= 0 && page < num_pages) atomicOr(&used[page / 32], 1u << (page % 32));
  };
  for (int i = threadIdx.x; i < K * width; i += blockDim.x) {
    const int j = i / width, c = i % width;
    const size_t at = static_cast<size_t>(row0 + j) * width + c;
    const int theirs = table[static_cast<size_t>(row0 + s_parent[j]) * width + c];
    if (c < lp || (c == lp && s_keeps[j])) {
      out[at] = theirs;
      mark(theirs);
    } else if (c > lp) {
      out[at] = table[at];
    }
  }
  __syncthreads();
  if (threadIdx.x < 32) {                              // the first K free pages, in the pool's order
    int n = 0;
    for (int i0 = 0; i0 < pool_n && n < K; i0 += 32) {
      const int i = i0 + threadIdx.x;
      const int page = i < pool_n ? pool[static_cast<size_t>(item) * pool_n + i] : -1;
      bool ok = page >= 0 && page < num_pages && !(used[page / 32] >> (page % 32) & 1u);
      // a page that the pool names twice is one page
      const uint32_t same = __match_any_sync(0xffffffffu, ok ? page : -1 - static_cast<int>(threadIdx.x));
      ok = ok && (same & ((1u << threadIdx.x) - 1u)) == 0;
      __syncwarp();
      if (ok) mark(page);
      __syncwarp();
      const uint32_t all = __ballot_sync(0xffffffffu, ok);
      const int place = n + __popc(all & ((1u << threadIdx.x) - 1u));
      if (ok && place < K) s_free[place] = page;
      n += __popc(all);
    }
  }
  __syncthreads();
  if (threadIdx.x < K) {
    const int j = threadIdx.x;
    int s = -1, d = -1;
    if (!s_keeps[j]) {
      d = s_free[s_turn[j]];
      out[static_cast<size_t>(row0 + j) * width + lp] = d;
      if (partial) s = s_tail[j];
      if (d < 0) record_status(status, ST_BOUNDS, item);       // the pool is too small
    }
    const bool copy = s >= 0 && s < num_pages && d >= 0;
    src[row0 + j] = copy ? s : -1;
    dst[row0 + j] = copy ? d : -1;
  }
}

constexpr int COPY_MAX = 192;          // tensors of one launch
struct CopyArgs {
  void* base[COPY_MAX];
  int bytes[COPY_MAX];                 // of a page, a multiple of 4
};
__global__ void __launch_bounds__(256) beam_copy_kernel(const __grid_constant__ CopyArgs a, const int* __restrict__ src,
                                                        const int* __restrict__ dst, int num_pages, int* status) {
  const int s = src[blockIdx.x], d = dst[blockIdx.x];
  if (s < 0 || d < 0 || s == d) return;
  if (s >= num_pages || d >= num_pages) {
    if (threadIdx.x == 0) record_status(status, ST_BOUNDS, blockIdx.x);
    return;
  }
  const size_t bytes = a.bytes[blockIdx.y];
  const char* from = static_cast<const char*>(a.base[blockIdx.y]) + s * bytes;
  char* to = static_cast<char*>(a.base[blockIdx.y]) + d * bytes;
  const size_t first = blockIdx.z * static_cast<size_t>(blockDim.x) + threadIdx.x, step = gridDim.z * static_cast<size_t>(blockDim.x);
  if (((reinterpret_cast<uintptr_t>(a.base[blockIdx.y]) | bytes) & 15) == 0) {
    const size_t n = bytes / 16;
    size_t i = first;
    for (; i + 3 * step < n; i += 4 * step) {            // four loads on their way
      uint4 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = __ldg(reinterpret_cast<const uint4*>(from) + i + u * step);
#pragma unroll
      for (int u = 0; u < 4; ++u) reinterpret_cast<uint4*>(to)[i + u * step] = v[u];
    }
    for (; i < n; i += step) reinterpret_cast<uint4*>(to)[i] = __ldg(reinterpret_cast<const uint4*>(from) + i);
  } else {
    for (size_t i = first; i < bytes / 4; i += step) reinterpret_cast<uint32_t*>(to)[i] = __ldg(reinterpret_cast<const uint32_t*>(from) + i);
  }
}

}  // namespace cb

using namespace cb;

// part: float2 [B K, ceil((V + 7) / BLK)] scratch
extern "C" int cb_beam_select(const void* logits, int64_t ld, int f32, int B, int K, int V, const float* scores,
                              const void* done, int eos, void* part, float* out_score, int64_t* out_parent,
                              int64_t* out_token, void* out_done, void* stream) {
  if (B < 1 || K < 1 || K > BEAM_MAX || V < 1 || eos >= V) return -1;
  const int nblk = (V + 7 + BLK - 1) / BLK;                       // a row may begin up to seven logits into its first block
  if (1ll * B * K > 65535) return -2;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 grid((nblk + PASS_WARPS - 1) / PASS_WARPS, B * K);
  auto* P = static_cast<float2*>(part);
  auto* D = static_cast<const uint8_t*>(done);
  auto* OD = static_cast<uint8_t*>(out_done);
  auto go = [&](auto* x) {
    using T = std::remove_const_t<std::remove_pointer_t<decltype(x)>>;
    const bool alike = ld * static_cast<int64_t>(sizeof(T)) % 16 == 0;
    const int skew = alike ? static_cast<int>(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T)) : 0;
    if (alike) beam_pass_kernel<T, true><<<grid, 32 * PASS_WARPS, 0, st>>>(x, ld, V, nblk, skew, scores, D, P);
    else beam_pass_kernel<T, false><<<grid, 32 * PASS_WARPS, 0, st>>>(x, ld, V, nblk, skew, scores, D, P);
    beam_pick_kernel<T><<<B, PICK_THREADS, 0, st>>>(x, ld, V, nblk, skew, K, scores, D, eos, P, out_score, out_parent, out_token, OD);
  };
  if (f32) go(static_cast<const float*>(logits));
  else go(static_cast<const __nv_bfloat16*>(logits));
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

extern "C" int cb_beam_pages(const int* table, int width, int B, int K, const int64_t* parent, const int* length,
                             const int* pool, int pool_n, int num_pages, int* out, int* src, int* dst, int* status,
                             void* stream) {
  if (B < 1 || K < 1 || K > BEAM_MAX || width < 1 || pool_n < 0 || num_pages < 1) return -1;
  const int bytes = (num_pages + 31) / 32 * 4;
  if (bytes > PAGES_SMEM) return -2;
  // always the same limit: one that went by the call would be lowered under another thread's launch
  if (bytes > 40 * 1024 &&
      cudaFuncSetAttribute(beam_pages_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, PAGES_SMEM) != cudaSuccess)
    return -4;
  beam_pages_kernel<<<B, 256, bytes, static_cast<cudaStream_t>(stream)>>>(table, width, K, parent, length, pool, pool_n,
                                                                          num_pages, out, src, dst, status);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

// Copies page src[i] to page dst[i] (-1: none) in every tensor; base and bytes are host arrays.
extern "C" int cb_beam_copy(void* const* base, const int* bytes, int tensors, const int* src, const int* dst, int n,
                            int num_pages, int* status, void* stream) {
  if (n < 1 || tensors < 1) return -1;
  for (int t0 = 0; t0 < tensors; t0 += COPY_MAX) {
    CopyArgs a;
    const int nt = tensors - t0 < COPY_MAX ? tensors - t0 : COPY_MAX;
    int most = 0;
    for (int t = 0; t < nt; ++t) {
      a.base[t] = base[t0 + t];
      a.bytes[t] = bytes[t0 + t];
      if (a.bytes[t] < 4 || a.bytes[t] % 4 != 0) return -2;
      most = a.bytes[t] > most ? a.bytes[t] : most;
    }
    const int parts = static_cast<int>((most + 16383ll) / 16384);
    const dim3 grid(n, nt, parts < 65535 ? parts : 65535);
    beam_copy_kernel<<<grid, 256, 0, static_cast<cudaStream_t>(stream)>>>(a, src, dst, num_pages, status);
  }
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}
