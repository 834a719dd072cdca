// One step of beam search: selection over beams and vocabulary, and the
// reordering of the paged cache's state.
//
// chunk_kernel reads the logits once: a block takes CHUNK tokens of one beam
// into registers, forms their maximum and sum of exponentials and their
// `beams` largest logits (a threshold from the lanes' maxima leaves a few
// candidates, which are ranked by counting). select_kernel joins the chunks of
// an item's beams: log sums, totals and the `beams` best proposals. With a
// cache, reorder_kernel then writes the children's page tables and copies the
// partly filled last pages, all layers in one launch.
//
// The order of proposals is (total descending, beam, logit descending, token).
// A beam's proposals are its largest logits, so cutting each chunk's list at
// `beams` entries by (logit descending, token) loses none of the best.
#include <algorithm>

#include "decode.h"

namespace wgx {

namespace {

constexpr int BM_THREADS = 256;
constexpr int BM_WARPS = BM_THREADS / 32;
constexpr int BM_ITEMS = 32;                     // logits per thread
constexpr int BM_CHUNK = BM_THREADS * BM_ITEMS;  // tokens per block
constexpr int BM_CAND = 1024;                    // candidates ranked by counting
constexpr int BM_SEL_THREADS = 256;
constexpr int BM_COPY_THREADS = 256;

struct BeamArgs {
  wgx_beam_search_args a;
  int64_t capacity;
  int chunks;       // blocks per beam
  float2 *chunk_ms; // [row][chunk] (max, sum of exp(x - max))
  float *top_x;     // [row][chunk][beams] logits, best first
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

__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
  for (int d = 16; d; d /= 2) x = fmaxf(x, __shfl_xor_sync(~0u, x, d));
  return x;
}
__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int d = 16; d; d /= 2) x += __shfl_xor_sync(~0u, x, d);
  return x;
}
// The lanes' values in descending order (bitonic).
__device__ __forceinline__ float warp_sort(float x) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int k = 2; k <= 32; k *= 2)
#pragma unroll
    for (int j = k / 2; j; j /= 2) {
      const float y = __shfl_xor_sync(~0u, x, j);
      const bool up = ((lane & k) == 0) == ((lane & j) == 0);
      x = up ? fmaxf(x, y) : fminf(x, y);
    }
  return x;
}

// VEC: every beam's logits start on a 16-byte boundary; otherwise (odd
// vocabularies) tokens are loaded one by one. One mapping of tokens to threads
// for all beams, so that equal logits give equal sums: beams that tie stay
// tied.
template <typename T, bool VEC>
__global__ void __launch_bounds__(BM_THREADS) chunk_kernel(const __grid_constant__ BeamArgs p) {
  constexpr int EPV = VEC ? 16 / int(sizeof(T)) : 1, VECS = BM_ITEMS / EPV;
  __shared__ float red_max[BM_WARPS], red_sum[BM_WARPS], own_k[BM_WARPS], low_k[BM_WARPS];
  __shared__ uint64_t cand[BM_CAND];
  __shared__ uint32_t n_cand;
  __shared__ uint64_t best[BM_WARPS];
  const wgx_beam_search_args &a = p.a;
  const int row = blockIdx.y, chunk = blockIdx.x, tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  if (a.finished[row]) return;  // proposes eos: its logits are not needed
  const int K = a.beams, t0 = chunk * BM_CHUNK, cnt = min(BM_CHUNK, a.vocab - t0);
  const T *x = static_cast<const T *>(a.logits) + int64_t(row / K) * a.logits_batch_stride +
               int64_t(row % K) * a.logits_beam_stride + t0;
  if (tid == 0) n_cand = 0;
  // ---- the chunk into registers: item i of thread t is token
  // (i / EPV * BM_THREADS + t) * EPV + i % EPV; -infinity behind the end and
  // for NaN
  float v[BM_ITEMS];
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    const int o = (i * BM_THREADS + tid) * EPV;
    if (VEC && o + EPV <= cnt) {
      const uint4 u = __ldcs(reinterpret_cast<const uint4 *>(x + o));
      const T *e = reinterpret_cast<const T *>(&u);
#pragma unroll
      for (int j = 0; j < EPV; ++j) v[i * EPV + j] = float(e[j]);
    } else {
#pragma unroll
      for (int j = 0; j < EPV; ++j) v[i * EPV + j] = o + j < cnt ? float(x[o + j]) : -INFINITY;
    }
  }
  float mx = -INFINITY;
#pragma unroll
  for (int i = 0; i < BM_ITEMS; ++i) {
    if (v[i] != v[i]) v[i] = -INFINITY;
    mx = fmaxf(mx, v[i]);
  }
  // ---- maximum and sum; thresholds: at least `K` logits of the chunk are not
  // below (i) any one warp's K-th largest lane maximum, (ii) the smallest of
  // the warps' ceil(K / BM_WARPS)-th largest
  const float sorted = warp_sort(mx);
  const float wm = __shfl_sync(~0u, sorted, 0);
  const float wk = __shfl_sync(~0u, sorted, K - 1);
  const float wl = __shfl_sync(~0u, sorted, (K + BM_WARPS - 1) / BM_WARPS - 1);
  if (lane == 0) red_max[warp] = wm, own_k[warp] = wk, low_k[warp] = wl;
  __syncthreads();
  float m = red_max[0], high = own_k[0], low = low_k[0];
#pragma unroll
  for (int w = 1; w < BM_WARPS; ++w) {
    m = fmaxf(m, red_max[w]);
    high = fmaxf(high, own_k[w]);
    low = fminf(low, low_k[w]);
  }
  const float tau = fmaxf(high, low);
  const float mu = m == -INFINITY ? 0.f : m;
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < BM_ITEMS; ++i) s += __expf(v[i] - mu);
  s = warp_sum(s);
  if (lane == 0) red_sum[warp] = s;
  // ---- candidates: key = (logit, lower token first)
  auto key_of = [&](float f, int o) { return uint64_t(ordered(f)) << 32 | uint32_t(~uint32_t(o)); };
  auto offer = [&](float f, int o) {
    if (f >= tau && o < cnt) {
      const uint32_t at = atomicAdd(&n_cand, 1u);
      if (at < BM_CAND) cand[at] = key_of(f, o);
    }
  };
#pragma unroll
  for (int i = 0; i < BM_ITEMS; ++i)
    offer(v[i], (i / EPV * BM_THREADS + tid) * EPV + i % EPV);
  __syncthreads();
  const int64_t out = int64_t(row) * p.chunks + chunk;
  if (tid == 0) {
    float sum = 0.f;
    for (int w = 0; w < BM_WARPS; ++w) sum += red_sum[w];
    p.chunk_ms[out] = make_float2(m, sum);
  }
  const int want = min(K, cnt), n = int(n_cand);
  auto emit = [&](int at, uint64_t key) {
    p.top_x[out * K + at] = unordered(uint32_t(key >> 32));
    p.top_t[out * K + at] = t0 + int(~uint32_t(key));
  };
  if (tid >= want && tid < K) p.top_t[out * K + tid] = -1;
  if (n <= BM_CAND) {
    for (int i = tid; i < n; i += BM_THREADS) {
      const uint64_t k = cand[i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += cand[j] > k;
      if (rank < want) emit(rank, k);
    }
  } else {
    // many equal logits at the threshold: one maximum after another
    uint64_t below = ~uint64_t(0);
    for (int r = 0; r < want; ++r) {
      uint64_t k = 0;
#pragma unroll
      for (int i = 0; i < BM_ITEMS; ++i) {
        const int o = (i / EPV * BM_THREADS + tid) * EPV + i % EPV;
        const uint64_t q = key_of(v[i], o);
        if (o < cnt && q < below && q > k) k = q;
      }
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
  __shared__ float red[BM_SEL_THREADS / 32];
  __shared__ Proposal cand[BM_CAND];
  __shared__ Proposal best[BM_SEL_THREADS / 32];
  __shared__ uint32_t n_cand;
  const int b = blockIdx.x, W = a.beams, tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int list = p.chunks * W, all = W * list;
  if (tid == 0) n_cand = 0;
  for (int w = warp; w < W; w += BM_SEL_THREADS / 32) {
    const int row = b * W + w;
    const bool done = a.finished[row] != 0;
    float m = -INFINITY, s = 0.f;
    if (!done) {
      for (int c = lane; c < p.chunks; c += 32) m = fmaxf(m, p.chunk_ms[int64_t(row) * p.chunks + c].x);
      m = warp_max(m);
      const float mu = m == -INFINITY ? 0.f : m;
      for (int c = lane; c < p.chunks; c += 32) {
        const float2 ms = p.chunk_ms[int64_t(row) * p.chunks + c];
        s += ms.y * __expf(ms.x - mu);
      }
      s = warp_sum(s);
    }
    if (lane == 0) {
      row_max[w] = m;
      row_log[w] = logf(s);
      row_score[w] = a.scores[row];
      row_done[w] = done;
    }
  }
  __syncthreads();
  // candidate i: entry i % list of beam i / list; false: none
  auto get = [&](int i, Proposal &q) {
    const int w = i / list, e = i - w * list;
    q.beam = w;
    if (row_done[w]) {
      q.token = a.eos;
      q.logit = 0.f;
      q.total = row_score[w];
      if (e) return false;
    } else {
      const int64_t at = int64_t(b * W + w) * list + e;
      q.token = p.top_t[at];
      if (q.token < 0) return false;
      q.logit = p.top_x[at];
      q.total = row_score[w] + ((q.logit - row_max[w]) - row_log[w]);
    }
    if (q.total != q.total) q.total = -INFINITY;
    return true;
  };
  // ---- threshold: at least W proposals are not below the W-th entry of any
  // one chunk's list
  float tau = -INFINITY;
  for (int i = W - 1 + tid * W; i < all; i += BM_SEL_THREADS * W) {
    Proposal q;
    if (get(i, q)) tau = fmaxf(tau, q.total);
  }
  tau = warp_max(tau);
  if (lane == 0) red[warp] = tau;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < BM_SEL_THREADS / 32; ++w) tau = fmaxf(tau, red[w]);
  for (int i = tid; i < all; i += BM_SEL_THREADS) {
    Proposal q;
    if (get(i, q) && q.total >= tau) {
      const uint32_t at = atomicAdd(&n_cand, 1u);
      if (at < BM_CAND) cand[at] = q;
    }
  }
  __syncthreads();
  auto emit = [&](int r, const Proposal &q) {
    const int64_t at = int64_t(b) * W + r;
    a.scores_out[at] = q.total;
    a.parents[at] = q.beam;
    a.tokens[at] = q.token;
    a.finished_out[at] = row_done[q.beam] || q.token == a.eos;
  };
  const int n = int(n_cand);
  if (n <= BM_CAND) {
    for (int i = tid; i < n; i += BM_SEL_THREADS) {
      const Proposal q = cand[i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += before(cand[j], q);
      if (rank < W) emit(rank, q);
    }
  } else {
    // many equal totals (a single list's threshold can leave more): one
    // maximum after another
    Proposal last{INFINITY, 0.f, -1, -1};
    for (int r = 0; r < W; ++r) {
      Proposal k{-INFINITY, -INFINITY, 0x7fffffff, 0x7fffffff};
      for (int i = tid; i < all; i += BM_SEL_THREADS) {
        Proposal q;
        if (get(i, q) && (r == 0 || before(last, q)) && before(q, k)) k = q;
      }
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
// share of its copied page: units of 16 bytes (or elements) of K and V over
// (layer, head, slot).
template <typename U, bool VEC>
__global__ void __launch_bounds__(BM_COPY_THREADS) reorder_kernel(const __grid_constant__ BeamArgs p) {
  const wgx_beam_search_args &a = p.a;
  const wgx_kv_cache &c = a.cache;
  const int child = blockIdx.y, tid = threadIdx.x;
  const int from = child / a.beams * a.beams + a.parents[child];
  const int len = slots_in_use(a.lengths, from, p.capacity, p.err);
  const int full = len / c.page_size, tail = len - full * c.page_size;
  const int32_t *src_table = c.page_table + int64_t(from) * c.table_stride;
  const int spare = a.spare[child];
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
  const int es = c.dtype == WGX_FLOAT16 ? 2 : 4;
  const int units = VEC ? c.head_dim * es / 16 : c.head_dim;
  const int64_t step = VEC ? 16 / es : 1;
  const uint64_t all = uint64_t(c.layers) * c.kv_heads * tail * units;
  U *k = static_cast<U *>(c.k), *v = static_cast<U *>(c.v);
  for (uint64_t i = uint64_t(blockIdx.x) * BM_COPY_THREADS + tid; i < all;
       i += uint64_t(gridDim.x) * BM_COPY_THREADS) {
    const int u = int(i % units);
    uint64_t r = i / units;
    const int t = int(r % tail);
    r /= tail;
    const int h = int(r % c.kv_heads), layer = int(r / c.kv_heads);
    const int64_t ko = int64_t(layer) * c.k_layer_stride + int64_t(h) * c.k_head_stride + int64_t(t) * c.k_slot_stride;
    const int64_t vo = int64_t(layer) * c.v_layer_stride + int64_t(h) * c.v_head_stride + int64_t(t) * c.v_slot_stride;
    const U x = k[(ko + int64_t(old) * c.k_page_stride) / step + u];
    const U y = v[(vo + int64_t(old) * c.v_page_stride) / step + u];
    k[(ko + int64_t(spare) * c.k_page_stride) / step + u] = x;
    v[(vo + int64_t(spare) * c.v_page_stride) / step + u] = y;
  }
}

uint64_t align256(uint64_t x) { return (x + 255) / 256 * 256; }

uint64_t layout(const wgx_beam_search_args &a, BeamArgs *p) {
  const uint64_t rows = uint64_t(a.batch) * a.beams;
  const int chunks = (a.vocab + BM_CHUNK - 1) / BM_CHUNK;
  const uint64_t lists = rows * chunks;
  uint8_t *base = static_cast<uint8_t *>(a.scratch);
  uint64_t off = 0;
  auto take = [&](uint64_t bytes) {
    uint8_t *at = base + off;
    off += align256(bytes);
    return at;
  };
  uint8_t *ms = take(lists * 8), *x = take(lists * a.beams * 4), *t = take(lists * a.beams * 4);
  if (p) {
    p->chunks = chunks;
    p->chunk_ms = reinterpret_cast<float2 *>(ms);
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
  const dim3 grid(unsigned(p.chunks), rows);
  const int th = timer_begin("chunk_kernel", stream);
  const int ls = dtype_size(a.dtype);
  const bool vec = ((a.logits_batch_stride * ls) | (a.logits_beam_stride * ls) |
                    int64_t(reinterpret_cast<uintptr_t>(a.logits))) % 16 == 0;
  if (a.dtype == WGX_FLOAT16) {
    if (vec) chunk_kernel<__half, true><<<grid, BM_THREADS, 0, stream>>>(p);
    else chunk_kernel<__half, false><<<grid, BM_THREADS, 0, stream>>>(p);
  } else {
    if (vec) chunk_kernel<float, true><<<grid, BM_THREADS, 0, stream>>>(p);
    else chunk_kernel<float, false><<<grid, BM_THREADS, 0, stream>>>(p);
  }
  check_cuda(cudaGetLastError(), "beam_search_step launch");
  timer_end(th, stream);
  select_kernel<<<unsigned(a.batch), BM_SEL_THREADS, 0, stream>>>(p);
  check_cuda(cudaGetLastError(), "beam_search_step selection launch");
  if (!c.k) return;
  const int es = dtype_size(c.dtype);
  const uint64_t units = uint64_t(c.layers) * c.kv_heads * c.page_size *
                         uint64_t(p.vec ? c.head_dim * es / 16 : c.head_dim);
  // about eight units per thread, at most sixteen blocks per SM
  const uint64_t want = (units + BM_COPY_THREADS * 8 - 1) / (BM_COPY_THREADS * 8);
  const uint64_t most = std::max<uint64_t>(1, uint64_t(device_sm_count()) * 16 / rows);
  const dim3 cgrid(unsigned(std::max<uint64_t>(1, std::min(want, most))), rows);
  if (p.vec)
    reorder_kernel<uint4, true><<<cgrid, BM_COPY_THREADS, 0, stream>>>(p);
  else if (es == 2)
    reorder_kernel<uint16_t, false><<<cgrid, BM_COPY_THREADS, 0, stream>>>(p);
  else
    reorder_kernel<uint32_t, false><<<cgrid, BM_COPY_THREADS, 0, stream>>>(p);
  check_cuda(cudaGetLastError(), "beam_search_step reorder launch");
}

}  // namespace wgx
