// One step of beam search: selection over beams and vocabulary, and the
// reordering of the paged cache's state.
//
// scan_kernel streams the logits: each beam's row is cut into a few segments,
// one wave of blocks over the GPU; a thread only keeps a running maximum and sum
// of exponentials (8 instructions a logit). The segment's `beams` best lie with
// the `beams` threads of the largest maxima, and are not below the smallest of
// these: only those threads' logits are looked at again (from L2).
// select_kernel joins the segments of an item's beams: log sums, totals and the
// `beams` best proposals. With a cache, reorder_kernel then writes the
// children's page tables and copies the partly filled last pages, all layers
// in one launch.
//
// Measured: 32 x 1 beam x 50257 fp16 logits 10 us a call (two launches, 3 MB:
// latency, part of it the order of the threads' maxima and the second look at
// the logits, which one beam does not need); 16 x 8 beams x 131072 fp32 logits and 24 layers of tails 59 us: the
// scan 20 (60 MB; one wave of blocks with 3 or 4 per SM), the selection 7, the
// copies 31 (226 MB moved, part of it within L2).
//
// The order of proposals is (total descending, beam, logit descending, token).
// A beam's proposals are its largest logits, so cutting each segment's list at
// `beams` entries by (logit descending, token) loses none of the best.
#include <algorithm>

#include "decode.h"

namespace wgx {

namespace {

constexpr int BM_THREADS = 256;
constexpr int BM_WARPS = BM_THREADS / 32;
constexpr int BM_ITEMS = 16;                    // logits per thread and tile
constexpr int BM_TILE = BM_THREADS * BM_ITEMS;  // tokens per tile
constexpr int BM_LIST = 1024;                   // logits of a segment ranked by counting
constexpr int BM_CAND = 1024;                   // proposals ranked by counting
constexpr int BM_BLOCKS_PER_SM = 4;             // of scan_kernel (64 registers a thread)
constexpr int BM_SEL_THREADS = 256;
constexpr int BM_HELD = 4;                      // entries a thread of select_kernel holds
constexpr int BM_COPY_THREADS = 256;
constexpr int BM_UNITS = 4;  // units of K and of V a thread has in flight

struct BeamArgs {
  wgx_beam_search_args a;
  int64_t capacity;
  int tiles;        // of a row
  int segments;     // blocks per row
  float2 *seg_ms;   // [row][segment] (max, sum of exp(x - max))
  float *top_x;     // [row][segment][beams] logits, best first
  int32_t *top_t;   // their tokens; -1: none
  int vec;          // cache rows move in 16-byte units
  uint32_t *err;
};

// Numbers in ascending order as unsigned integers.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u ^ (u >> 31 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t k) {
  return __uint_as_float(k ^ (k >> 31 ? 0x80000000u : 0xffffffffu));
}

// The lanes' keys in descending order (bitonic), each with its tag.
__device__ __forceinline__ void warp_sort(uint64_t &x, int &tag) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int k = 2; k <= 32; k *= 2)
#pragma unroll
    for (int j = k / 2; j; j /= 2) {
      const uint64_t y = __shfl_xor_sync(~0u, x, j);
      const int t = __shfl_xor_sync(~0u, tag, j);
      const bool larger = ((lane & k) == 0) == ((lane & j) == 0);
      // (equal keys: threads without tokens; either order will do, but both
      // lanes must agree)
      if (larger ? y > x : y < x) {
        x = y;
        tag = t;
      }
    }
}
__device__ __forceinline__ float warp_sort(float x) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int k = 2; k <= 32; k *= 2)
#pragma unroll
    for (int j = k / 2; j; j /= 2) {
      const float y = __shfl_xor_sync(~0u, x, j);
      x = ((lane & k) == 0) == ((lane & j) == 0) ? fmaxf(x, y) : fminf(x, y);
    }
  return x;
}

// Key of a logit: larger logits first, equal ones by token. No two are equal.
__device__ __forceinline__ uint64_t key_of(float x, int token) {
  return uint64_t(ordered(x)) << 32 | uint32_t(~uint32_t(token));
}

// VEC: every beam's logits start on a 16-byte boundary; otherwise (odd
// vocabularies) tokens are loaded one by one. One mapping of tokens to threads
// for all beams, so that equal logits give equal sums: beams that tie stay
// tied.
template <typename T, bool VEC>
__global__ void __launch_bounds__(BM_THREADS, BM_BLOCKS_PER_SM) scan_kernel(const __grid_constant__ BeamArgs p) {
  constexpr int EPV = VEC ? 16 / int(sizeof(T)) : 1, VECS = BM_ITEMS / EPV;
  __shared__ float red_max[BM_WARPS], red_sum[BM_WARPS];
  __shared__ uint64_t tops[BM_THREADS];       // the warps' sorted thread maxima
  __shared__ uint16_t top_tid[BM_THREADS], hit[WGX_MAX_BEAMS];
  __shared__ uint64_t bound, best[BM_WARPS];
  __shared__ uint64_t list[BM_LIST];
  __shared__ uint32_t n_list;
  const wgx_beam_search_args &a = p.a;
  const int row = blockIdx.y, seg = blockIdx.x, tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  wait_for_prior_kernel();
  let_dependents_launch();
  const bool done = a.finished[row];
  const int K = a.beams;
  const T *x = static_cast<const T *>(a.logits) + int64_t(row / K) * a.logits_batch_stride +
               int64_t(row % K) * a.logits_beam_stride;
  const int tile0 = int(int64_t(p.tiles) * seg / p.segments);
  const int tile1 = int(int64_t(p.tiles) * (seg + 1) / p.segments);
  if (tid == 0) n_list = 0;

  // ---- unit i of thread t of a tile is its EPV tokens from
  // (i * BM_THREADS + t) * EPV on; -infinity behind the end
  union Raw {
    uint4 u[VEC ? VECS : 1];
    T e[BM_ITEMS];
    __device__ Raw() {}
  };
  auto load = [&](int tile, Raw &r) {
    const int t0 = tile * BM_TILE, cnt = a.vocab - t0;
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int o = (i * BM_THREADS + tid) * EPV;
      if (VEC && o + EPV <= cnt) {
        r.u[VEC ? i : 0] = *reinterpret_cast<const uint4 *>(x + t0 + o);
      } else {
#pragma unroll
        for (int j = 0; j < EPV; ++j) r.e[i * EPV + j] = o + j < cnt ? x[t0 + o + j] : T(-INFINITY);
      }
    }
  };
  // NaN counts as -infinity (fmaxf takes its other operand)
  auto value = [](T e) { return fmaxf(float(e), -INFINITY); };
  constexpr float kLog2e = 1.4426950408889634f;
  float m = -INFINITY, sum = 0.f;  // of this thread
  int top_tile = tile0;            // the first tile with its maximum
  Raw next;
  load(tile0, next);   // (beside the load of `done`)
  if (done) return;    // proposes eos: its logits are not needed
#pragma unroll 1
  for (int tile = tile0; tile < tile1; ++tile) {
    float v[BM_ITEMS];
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < BM_ITEMS; ++i) {
      v[i] = value(next.e[i]);
      mx = fmaxf(mx, v[i]);
    }
    if (tile + 1 < tile1) load(tile + 1, next);
    if (mx > m) {
      sum *= exp2_approx((m - mx) * kLog2e);
      m = mx;
      top_tile = tile;
    }
    const float mu = m == -INFINITY ? 0.f : m;
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int i = 0; i < BM_ITEMS; i += 2) {
      s0 += exp2_approx((v[i] - mu) * kLog2e);  // (the difference is exact near the maximum)
      s1 += exp2_approx((v[i + 1] - mu) * kLog2e);
    }
    sum += s0 + s1;
  }
  // ---- this thread's largest key: the first token with its maximum
  uint64_t top = 0;
  {
    if (top_tile != tile1 - 1) load(top_tile, next);  // (the last one is still here)
    const int t0 = top_tile * BM_TILE;
#pragma unroll
    for (int i = BM_ITEMS - 1; i >= 0; --i) {
      const int t = t0 + (i / EPV * BM_THREADS + tid) * EPV + i % EPV;
      if (value(next.e[i]) == m && t < a.vocab) top = key_of(m, t);
    }
  }
  const float wm = warp_max(m);
  const float wmu = wm == -INFINITY ? 0.f : wm;
  const float ws = warp_sum(sum * exp2_approx((m - wmu) * kLog2e));
  if (lane == 0) red_max[warp] = wm, red_sum[warp] = ws;
  // ---- the K threads with the largest keys: they are among the K first of
  // their warps
  int who = tid;
  warp_sort(top, who);
  tops[tid] = top;
  top_tid[tid] = uint16_t(who);
  if (tid == 0) bound = 0;
  __syncthreads();
  const int64_t out = int64_t(row) * p.segments + seg;
  if (tid == 0) {
    float M = red_max[0], all = 0.f;
    for (int w = 1; w < BM_WARPS; ++w) M = fmaxf(M, red_max[w]);
    const float mu = M == -INFINITY ? 0.f : M;
    for (int w = 0; w < BM_WARPS; ++w) all += red_sum[w] * exp2_approx((red_max[w] - mu) * kLog2e);
    p.seg_ms[out] = make_float2(M, all);
  }
  if (tid < BM_WARPS * K) {
    const int w = tid / K, e = tid % K;
    const uint64_t k = tops[w * 32 + e];
    int r = 0;
    for (int o = 0; o < BM_WARPS; ++o)
      for (int j = 0; j < K; ++j) r += tops[o * 32 + j] > k;
    if (k && r < K) {  // (0: a thread without tokens)
      hit[r] = top_tid[w * 32 + e];
      if (r == K - 1) bound = k;
    }
  }
  const int hits = min(K, __syncthreads_count(top != 0));
  // ---- their logits that are not below the bound
  const int units = (tile1 - tile0) * VECS, all = hits * units;
  const uint64_t tau = bound;
  auto each = [&](auto &&f) {
    for (int q = tid; q < all; q += BM_THREADS) {
      const int r = q / units, u = q - r * units, tile = tile0 + u / VECS;
      const int t = tile * BM_TILE + (u % VECS * BM_THREADS + hit[r]) * EPV;
      if (VEC && t + EPV <= a.vocab) {
        const uint4 raw = *reinterpret_cast<const uint4 *>(x + t);
        const T *e = reinterpret_cast<const T *>(&raw);
#pragma unroll
        for (int j = 0; j < EPV; ++j) f(key_of(value(e[j]), t + j));
      } else {
        for (int j = 0; j < EPV; ++j)
          if (t + j < a.vocab) f(key_of(value(x[t + j]), t + j));
      }
    }
  };
  each([&](uint64_t k) {
    if (k >= tau) {
      const uint32_t at = atomicAdd(&n_list, 1u);
      if (at < BM_LIST) list[at] = k;
    }
  });
  __syncthreads();
  const int n = int(n_list), want = min(n, K);
  auto emit = [&](int r, uint64_t k) {
    p.top_x[out * K + r] = unordered(uint32_t(k >> 32));
    p.top_t[out * K + r] = int(~uint32_t(k));
  };
  if (tid >= want && tid < K) p.top_t[out * K + tid] = -1;
  if (n <= BM_LIST) {
    for (int i = tid; i < n; i += BM_THREADS) {
      const uint64_t k = list[i];
      int r = 0;
      for (int j = 0; j < n; ++j) r += list[j] > k;
      if (r < K) emit(r, k);
    }
  } else {
    // a few threads hold very many of the largest logits: one maximum after
    // another
    uint64_t below = ~uint64_t(0);
    for (int r = 0; r < want; ++r) {
      uint64_t k = 0;
      each([&](uint64_t y) {
        if (y < below && y > k) k = y;
      });
#pragma unroll
      for (int d = 16; d; d /= 2) {
        const uint64_t y = __shfl_xor_sync(~0u, k, d);
        if (y > k) k = y;
      }
      if (lane == 0) best[warp] = k;
      __syncthreads();
      k = best[0];
#pragma unroll
      for (int w = 1; w < BM_WARPS; ++w)
        if (best[w] > k) k = best[w];
      __syncthreads();
      if (tid == 0) emit(r, k);
      below = k;
    }
  }
}

struct Proposal {
  float total, logit;
  int beam, token;
};
__device__ __forceinline__ bool before(const Proposal &x, const Proposal &y) {
  if (x.total != y.total) return x.total > y.total;
  if (x.beam != y.beam) return x.beam < y.beam;
  if (x.logit != y.logit) return x.logit > y.logit;
  return x.token < y.token;
}

// One block per item.
__global__ void __launch_bounds__(BM_SEL_THREADS) select_kernel(const __grid_constant__ BeamArgs p) {
  const wgx_beam_search_args &a = p.a;
  __shared__ float row_max[WGX_MAX_BEAMS], row_log[WGX_MAX_BEAMS], row_score[WGX_MAX_BEAMS];
  __shared__ uint8_t row_done[WGX_MAX_BEAMS];
  __shared__ float tops[BM_SEL_THREADS], bound;
  __shared__ Proposal cand[BM_CAND];
  __shared__ Proposal best[BM_SEL_THREADS / 32];
  __shared__ uint32_t n_cand;
  const int b = blockIdx.x, W = a.beams, tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int list = p.segments * W, all = W * list;
  wait_for_prior_kernel();
  let_dependents_launch();
  if (tid == 0) n_cand = 0;
  // entry i % list of beam i / list, i = tid + j * threads: the first BM_HELD of
  // a thread are loaded now, beside the segments' sums
  float held_x[BM_HELD];
  int held_t[BM_HELD];
  const int64_t first = int64_t(b) * all;
#pragma unroll
  for (int j = 0; j < BM_HELD; ++j) {
    const int i = tid + j * BM_SEL_THREADS;
    held_t[j] = i < all ? p.top_t[first + i] : -1;
    held_x[j] = i < all ? p.top_x[first + i] : 0.f;
  }
  for (int w = warp; w < W; w += BM_SEL_THREADS / 32) {
    const int row = b * W + w;
    const bool done = a.finished[row] != 0;
    const float score = a.scores[row];
    const float2 *ms = p.seg_ms + int64_t(row) * p.segments;
    // (a finished beam's sums were not written: they are read, not used)
    const float2 mine = lane < p.segments ? ms[lane] : make_float2(-INFINITY, 0.f);
    float m = mine.x, s = 0.f;
    if (!done) {
      for (int c = lane + 32; c < p.segments; c += 32) m = fmaxf(m, ms[c].x);
      m = warp_max(m);
      const float mu = m == -INFINITY ? 0.f : m;
      s = mine.y * __expf(mine.x - mu);
      for (int c = lane + 32; c < p.segments; c += 32) s += ms[c].y * __expf(ms[c].x - mu);
      s = warp_sum(s);
    }
    if (lane == 0) {
      row_max[w] = m;
      row_log[w] = logf(s);
      row_score[w] = score;
      row_done[w] = done;
    }
  }
  __syncthreads();
  // proposal of entry i; false: none
  auto propose = [&](int i, float x, int t, Proposal &q) {
    const int w = i / list;
    q.beam = w;
    if (row_done[w]) {
      q.token = a.eos;
      q.logit = 0.f;
      q.total = row_score[w];
      if (i != w * list) return false;
    } else {
      q.token = t;
      if (t < 0) return false;
      q.logit = x;
      q.total = row_score[w] + ((x - row_max[w]) - row_log[w]);
    }
    if (q.total != q.total) q.total = -INFINITY;
    return true;
  };
  Proposal held[BM_HELD];  // beam -1: none
#pragma unroll
  for (int j = 0; j < BM_HELD; ++j) {
    const int i = tid + j * BM_SEL_THREADS;
    if (i >= all || !propose(i, held_x[j], held_t[j], held[j])) held[j].beam = -1;
  }
  // f(proposal) for this thread's proposals
  auto each = [&](auto &&f) {
#pragma unroll
    for (int j = 0; j < BM_HELD; ++j)
      if (held[j].beam >= 0) f(held[j]);
    for (int i = tid + BM_HELD * BM_SEL_THREADS; i < all; i += BM_SEL_THREADS) {
      Proposal q;
      if (propose(i, p.top_x[first + i], p.top_t[first + i], q)) f(q);
    }
  };
  // ---- threshold: at least W proposals are not below the W-th largest of the
  // threads' maxima, which are among the W first of their warps; those that
  // pass are ranked by counting. (One beam: one maximum, below.)
  if (W > 1) {
    float most = -INFINITY;
    each([&](const Proposal &q) { most = fmaxf(most, q.total); });
    most = warp_sort(most);
    tops[tid] = most;
    if (tid == 0) bound = -INFINITY;
    __syncthreads();
    if (lane < W) {
      int r = 0;
      for (int o = 0; o < BM_SEL_THREADS / 32; ++o)
        for (int j = 0; j < W; ++j) {
          const float y = tops[o * 32 + j];
          r += y > most || (y == most && o * 32 + j < tid);
        }
      if (r == W - 1) bound = most;
    }
    __syncthreads();
    const float tau = bound;
    each([&](const Proposal &q) {
      if (q.total >= tau) {
        const uint32_t at = atomicAdd(&n_cand, 1u);
        if (at < BM_CAND) cand[at] = q;
      }
    });
    __syncthreads();
  }
  auto emit = [&](int r, const Proposal &q) {
    const int64_t at = int64_t(b) * W + r;
    a.scores_out[at] = q.total;
    a.parents[at] = q.beam;
    a.tokens[at] = q.token;
    a.finished_out[at] = row_done[q.beam] || q.token == a.eos;
  };
  const int n = int(n_cand);
  if (W > 1 && n <= BM_CAND) {
    for (int i = tid; i < n; i += BM_SEL_THREADS) {
      const Proposal q = cand[i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += before(cand[j], q);
      if (rank < W) emit(rank, q);
    }
  } else {
    // one beam, or many equal totals: one maximum after another
    Proposal last{INFINITY, 0.f, -1, -1};
    for (int r = 0; r < W; ++r) {
      Proposal k{-INFINITY, -INFINITY, 0x7fffffff, 0x7fffffff};
      each([&](const Proposal &q) {
        if ((r == 0 || before(last, q)) && before(q, k)) k = q;
      });
#pragma unroll
      for (int d = 16; d; d /= 2) {
        Proposal y;
        y.total = __shfl_xor_sync(~0u, k.total, d);
        y.logit = __shfl_xor_sync(~0u, k.logit, d);
        y.beam = __shfl_xor_sync(~0u, k.beam, d);
        y.token = __shfl_xor_sync(~0u, k.token, d);
        if (before(y, k)) k = y;
      }
      if (lane == 0) best[warp] = k;
      __syncthreads();
      k = best[0];
#pragma unroll
      for (int w = 1; w < BM_SEL_THREADS / 32; ++w)
        if (before(best[w], k)) k = best[w];
      __syncthreads();
      if (tid == 0) emit(r, k);
      last = k;
    }
  }
}

// Block (sequence, piece): the child's table and counters (piece 0), and a
// share of its copied page: units U (16 bytes, or one element; STEP elements)
// of K and V over (layer, head, slot), BM_UNITS at a time.
template <typename U, int STEP>
__global__ void __launch_bounds__(BM_COPY_THREADS) reorder_kernel(const __grid_constant__ BeamArgs p) {
  const wgx_beam_search_args &a = p.a;
  const wgx_kv_cache &c = a.cache;
  const int child = blockIdx.y, tid = threadIdx.x;
  const int spare = a.spare[child];
  wait_for_prior_kernel();
  let_dependents_launch();
  const int from = child / a.beams * a.beams + a.parents[child];
  const int len = a.lengths[from];
  // (a length the table cannot have is handed on as it is, with nothing copied)
  const int used = valid_length(len, p.capacity, p.err) ? len : 0;
  const int full = used / c.page_size, tail = used - full * c.page_size;
  const int32_t *src_table = c.page_table + int64_t(from) * c.table_stride;
  if (blockIdx.x == 0) {
    int32_t *dst = a.page_table_out + int64_t(child) * c.table_width;
    for (int i = tid; i < c.table_width; i += BM_COPY_THREADS)
      dst[i] = tail && i == full ? spare : src_table[i];
    if (tid == 0) a.lengths_out[child] = len;
  }
  if (!tail) return;
  const int old = src_table[full];
  if (old < 0 || old >= c.pages || spare < 0 || spare >= c.pages) {
    if (tid == 0 && blockIdx.x == 0) atomicOr(p.err, kErrCache);
    return;
  }
  const uint32_t units = uint32_t(c.head_dim / STEP), heads = uint32_t(c.kv_heads);
  const uint32_t row = uint32_t(tail) * units;  // units of a (layer, head)
  const U *ks = static_cast<const U *>(c.k) + int64_t(old) * c.k_page_stride / STEP;
  const U *vs = static_cast<const U *>(c.v) + int64_t(old) * c.v_page_stride / STEP;
  U *kd = static_cast<U *>(c.k) + int64_t(spare) * c.k_page_stride / STEP;
  U *vd = static_cast<U *>(c.v) + int64_t(spare) * c.v_page_stride / STEP;
  // a (layer, head) of the page per turn of this block's share
  const uint32_t planes = uint32_t(c.layers) * heads;
  const uint32_t per = row < BM_COPY_THREADS * BM_UNITS ? BM_COPY_THREADS * BM_UNITS / row : 1;  // planes a turn
  for (uint32_t p0 = blockIdx.x * per; p0 < planes; p0 += gridDim.x * per) {
    const uint32_t n = min(per, planes - p0) * row;
    for (uint32_t i0 = tid; i0 < n; i0 += BM_COPY_THREADS * BM_UNITS) {
      U x[BM_UNITS], y[BM_UNITS];
      int64_t ko[BM_UNITS], vo[BM_UNITS];
#pragma unroll
      for (int e = 0; e < BM_UNITS; ++e) {
        const uint32_t i = i0 + e * BM_COPY_THREADS;
        ko[e] = -1;
        if (i >= n) continue;
        const uint32_t pl = i / row, in = i - pl * row, t = in / units, u = in - t * units;
        const uint32_t layer = (p0 + pl) / heads, h = (p0 + pl) - layer * heads;
        ko[e] = (int64_t(layer) * c.k_layer_stride + int64_t(h) * c.k_head_stride + int64_t(t) * c.k_slot_stride) / STEP + u;
        vo[e] = (int64_t(layer) * c.v_layer_stride + int64_t(h) * c.v_head_stride + int64_t(t) * c.v_slot_stride) / STEP + u;
        x[e] = ks[ko[e]];
        y[e] = vs[vo[e]];
      }
#pragma unroll
      for (int e = 0; e < BM_UNITS; ++e) {
        if (ko[e] < 0) continue;
        kd[ko[e]] = x[e];
        vd[vo[e]] = y[e];
      }
    }
  }
}

uint64_t layout(const wgx_beam_search_args &a, BeamArgs *p) {
  const uint64_t rows = uint64_t(a.batch) * a.beams;
  const int tiles = (a.vocab + BM_TILE - 1) / BM_TILE;
  // segments: one wave of blocks over the GPU
  const int segments = int(std::min<uint64_t>(
      uint64_t(tiles), std::max<uint64_t>(1, uint64_t(device_sm_count()) * BM_BLOCKS_PER_SM / rows)));
  const uint64_t lists = rows * segments;
  uint8_t *base = static_cast<uint8_t *>(a.scratch);
  uint64_t off = 0;
  auto take = [&](uint64_t bytes) {
    uint8_t *at = base + off;
    off += align256(bytes);
    return at;
  };
  uint8_t *ms = take(lists * 8), *x = take(lists * a.beams * 4), *t = take(lists * a.beams * 4);
  if (p) {
    p->tiles = tiles;
    p->segments = segments;
    p->seg_ms = reinterpret_cast<float2 *>(ms);
    p->top_x = reinterpret_cast<float *>(x);
    p->top_t = reinterpret_cast<int32_t *>(t);
  }
  return off;
}

}  // namespace

uint64_t beam_search_scratch_bytes(const wgx_beam_search_args &a) { return layout(a, nullptr); }

void launch_beam_search_step(const wgx_beam_search_args &a, cudaStream_t stream) {
  BeamArgs p{};
  p.a = a;
  const uint64_t need = layout(a, &p);
  if (a.scratch_bytes < need || (reinterpret_cast<uintptr_t>(a.scratch) & 255))
    fail("beam_search_step: scratch of " + std::to_string(need) + " bytes, 256-byte aligned, needed");
  const wgx_kv_cache &c = a.cache;
  p.capacity = c.k ? cache_capacity(c) : 0;
  p.vec = c.k && cache_rows_16b(c);
  p.err = device_error_word(current_device());
  const unsigned rows = unsigned(a.batch) * unsigned(a.beams);
  const dim3 grid(unsigned(p.segments), rows);
  const int th = timer_begin("scan_kernel", stream);
  const int ls = dtype_size(a.dtype);
  const bool vec = ((a.logits_batch_stride * ls) | (a.logits_beam_stride * ls) |
                    int64_t(reinterpret_cast<uintptr_t>(a.logits))) % 16 == 0;
  launch_dependent(a.dtype == WGX_FLOAT16 ? (vec ? scan_kernel<__half, true> : scan_kernel<__half, false>)
                                          : (vec ? scan_kernel<float, true> : scan_kernel<float, false>),
                   grid, BM_THREADS, 0, stream, "beam_search_step launch", p);
  timer_end(th, stream);
  launch_dependent(select_kernel, dim3(unsigned(a.batch)), BM_SEL_THREADS, 0, stream,
                   "beam_search_step selection launch", p);
  if (!c.k) return;
  const int es = dtype_size(c.dtype);
  const uint64_t units = uint64_t(c.layers) * c.kv_heads * c.page_size *
                         uint64_t(p.vec ? c.head_dim * es / 16 : c.head_dim);
  // one turn of BM_UNITS units a thread, at most sixteen blocks per SM
  const uint64_t want = (units + BM_COPY_THREADS * BM_UNITS - 1) / (BM_COPY_THREADS * BM_UNITS);
  const uint64_t most = std::max<uint64_t>(1, uint64_t(device_sm_count()) * 16 / rows);
  const dim3 cgrid(unsigned(std::min(want, most)), rows);
  launch_dependent(p.vec ? (es == 2 ? reorder_kernel<uint4, 8> : reorder_kernel<uint4, 4>)
                         : (es == 2 ? reorder_kernel<uint16_t, 1> : reorder_kernel<uint32_t, 1>),
                   cgrid, BM_COPY_THREADS, 0, stream, "beam_search_step reorder launch", p);
}

}  // namespace wgx
