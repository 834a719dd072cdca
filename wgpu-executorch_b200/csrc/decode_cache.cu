// Upkeep of a paged K/V cache: appending new tokens' rows and evicting slots
// by accumulated attention weight. Both only move bytes; the floor is each
// moved row read and written once.
#include <cooperative_groups.h>

#include <algorithm>
#include <mutex>

#include "decode.h"

namespace cg = cooperative_groups;

namespace wgx {

namespace {

// ------------------------------------------------------------------ append
constexpr int AP_THREADS = 256;

struct AppendArgs {
  wgx_kv_append_args a;
  int64_t capacity;
  int fused;  // one block per sequence: it writes the counters itself
  uint32_t *err;
};

// The counters of sequence b, after its rows (lengths_out may be lengths).
__device__ __forceinline__ void advance(const wgx_kv_append_args &a, int b, int len, bool fits) {
  a.lengths_out[b] = len + (fits ? a.tokens : 0);
  if (a.seen_out) a.seen_out[b] = a.seen[b] + (fits ? a.tokens : 0);
}

// VEC: rows in 16-byte units; otherwise element by element. Thread: one unit
// of K and of V; consecutive threads take consecutive units of a row.
template <typename U, bool VEC>
__global__ void __launch_bounds__(AP_THREADS) append_kernel(const __grid_constant__ AppendArgs p) {
  const wgx_kv_append_args &a = p.a;
  const wgx_kv_cache &c = a.cache;
  const int b = blockIdx.y;
  const int len = slots_in_use(a.lengths, b, p.capacity, p.err);
  const bool fits = int64_t(len) + a.tokens <= p.capacity;
  if (!fits && threadIdx.x == 0 && blockIdx.x == 0) atomicOr(p.err, kErrCache);
  const int es = c.dtype == WGX_FLOAT16 ? 2 : 4;
  const uint32_t units = uint32_t(VEC ? c.head_dim * es / 16 : c.head_dim);
  const int64_t step = VEC ? 16 / es : 1;  // elements per unit
  const uint64_t all = uint64_t(a.tokens) * c.kv_heads * units;
  if (fits) {
    const U *k = static_cast<const U *>(a.k), *v = static_cast<const U *>(a.v);
    U *kc = static_cast<U *>(c.k), *vc = static_cast<U *>(c.v);
    for (uint64_t i = uint64_t(blockIdx.x) * AP_THREADS + threadIdx.x; i < all;
         i += uint64_t(gridDim.x) * AP_THREADS) {
      const uint32_t row = uint32_t(i / units), u = uint32_t(i % units);
      const int t = int(row / uint32_t(c.kv_heads)), h = int(row % uint32_t(c.kv_heads));
      const int slot = len + t, pi = slot / c.page_size, in = slot - pi * c.page_size;
      const int page = c.page_table[int64_t(b) * c.table_stride + pi];
      if (page < 0 || page >= c.pages) {
        atomicOr(p.err, kErrCache);
        continue;
      }
      const int64_t ks = int64_t(b) * a.k_batch_stride + int64_t(t) * a.k_token_stride +
                         int64_t(h) * a.k_head_stride;
      const int64_t vs = int64_t(b) * a.v_batch_stride + int64_t(t) * a.v_token_stride +
                         int64_t(h) * a.v_head_stride;
      const int64_t kd = int64_t(page) * c.k_page_stride + int64_t(h) * c.k_head_stride +
                         int64_t(in) * c.k_slot_stride;
      const int64_t vd = int64_t(page) * c.v_page_stride + int64_t(h) * c.v_head_stride +
                         int64_t(in) * c.v_slot_stride;
      const U x = k[ks / step + u], y = v[vs / step + u];
      kc[kd / step + u] = x;
      vc[vd / step + u] = y;
      if (u == 0 && slot < a.slots) {
        const int64_t at = (int64_t(b) * c.kv_heads + h) * a.slots + slot;
        if (a.weights) a.weights[at] = 0.f;
        if (a.positions) a.positions[at] = a.seen[b] + t;
      }
    }
  }
  if (p.fused) {
    __syncthreads();
    if (threadIdx.x == 0) advance(a, b, len, fits);
  }
}

__global__ void advance_kernel(const __grid_constant__ AppendArgs p) {
  const int b = blockIdx.x * blockDim.x + threadIdx.x;
  if (b >= p.a.cache.batch) return;
  const int len = slots_in_use(p.a.lengths, b, p.capacity, p.err);
  advance(p.a, b, len, int64_t(len) + p.a.tokens <= p.capacity);
}

// ------------------------------------------------------------------- evict
// A cluster of CTAs per (sequence, K/V head). The budget-th largest key is
// found by radix selection (8 bits a pass, histograms summed over the cluster
// through distributed shared memory) on keys held in shared memory: weights
// and positions are read once. Survivors behind the budget then move into the
// holes before it, both listed in slot order.
constexpr int EV_THREADS = 512;
constexpr int EV_MAX_CLUSTER = 8;
constexpr int EV_MAX_CHUNK = 36864;  // slots per CTA: 6 bytes of shared memory each
constexpr uint32_t kProtected = 0xffffffffu;

struct EvictArgs {
  wgx_cache_evict_args a;
  int64_t capacity;
  int chunk;     // slots per CTA
  int vec;       // rows move in 16-byte units
  int counters;  // this kernel writes lengths_out (it is not lengths)
  uint32_t *err;
};

// Larger keys stay. Weights as ordered integers; NaN lowest.
__device__ __forceinline__ uint32_t evict_key(float w, int pos, int recent_from, int sinks) {
  if (pos >= recent_from || pos < sinks) return kProtected;
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(w + 0.f);  // -0 as +0
  return u ^ (u >> 31 ? 0xffffffffu : 0x80000000u);
}

// Exclusive sum over the block's threads, and the total.
__device__ __forceinline__ uint32_t block_scan(uint32_t x, uint32_t *warp_sum, uint32_t *total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t s = x;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const uint32_t y = __shfl_up_sync(~0u, s, d);
    if (lane >= d) s += y;
  }
  __syncthreads();
  if (lane == 31) warp_sum[warp] = s;
  __syncthreads();
  uint32_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < EV_THREADS / 32; ++w) {
    const uint32_t v = warp_sum[w];
    before += w < warp ? v : 0;
    all += v;
  }
  *total = all;
  return before + s - x;
}

__global__ void __launch_bounds__(EV_THREADS) evict_kernel(const __grid_constant__ EvictArgs p) {
  extern __shared__ __align__(16) uint8_t ev_smem[];
  uint32_t *keys = reinterpret_cast<uint32_t *>(ev_smem);
  uint16_t *list = reinterpret_cast<uint16_t *>(ev_smem + size_t(p.chunk) * 4);
  __shared__ uint32_t hist[4][256];
  __shared__ uint32_t warp_sum[EV_THREADS / 32];
  __shared__ uint32_t counts[3];     // ties, holes, movers of this CTA
  __shared__ uint32_t pick[2];       // digit, keys above it
  __shared__ uint32_t hole_end[EV_MAX_CLUSTER], mover_end[EV_MAX_CLUSTER];
  cg::cluster_group cluster = cg::this_cluster();
  const int S = int(cluster.num_blocks()), rank = int(cluster.block_rank());
  const wgx_cache_evict_args &a = p.a;
  const wgx_kv_cache &c = a.cache;
  const int tid = threadIdx.x, row = int(blockIdx.x) / S;
  const int b = row / c.kv_heads, h = row % c.kv_heads, C = a.budget;
  const int len = slots_in_use(a.lengths, b, p.capacity, p.err);
  const int n = int(min(int64_t(len), a.slots));
  const int64_t at = int64_t(row) * a.slots;
  if (p.counters && h == 0 && rank == 0 && tid == 0) a.lengths_out[b] = min(len, C);
  if (n <= C) {  // the same for the whole cluster
    for (int i = rank * EV_THREADS + tid; i < n; i += S * EV_THREADS) {
      if (a.weights_out != a.weights) a.weights_out[at + i] = a.weights[at + i];
      if (a.positions_out != a.positions) a.positions_out[at + i] = a.positions[at + i];
    }
    return;
  }
  const int per = (n + S - 1) / S, s0 = min(rank * per, n), s1 = min(s0 + per, n), cnt = s1 - s0;
  const int recent_from = a.seen[b] - a.recent;

  for (int i = tid; i < 4 * 256; i += EV_THREADS) (&hist[0][0])[i] = 0;
  for (int i = tid; i < cnt; i += EV_THREADS) {
    const float w = a.weights[at + s0 + i];
    const int pos = a.positions[at + s0 + i];
    keys[i] = evict_key(w, pos, recent_from, a.sinks);
    if (s0 + i < C) {  // holes among these are overwritten below
      if (a.weights_out != a.weights) a.weights_out[at + s0 + i] = w;
      if (a.positions_out != a.positions) a.positions_out[at + s0 + i] = pos;
    }
  }
  __syncthreads();

  // ---- the C-th largest key: `found` digit by digit, `left` of the keys that
  // equal it so far still to be taken
  uint32_t found = 0, left = uint32_t(C);
  for (int pass = 0; pass < 4; ++pass) {
    const int shift = 24 - 8 * pass;
    const int rounds = (cnt + EV_THREADS - 1) / EV_THREADS;
    for (int r = 0; r < rounds; ++r) {
      const int i = r * EV_THREADS + tid;
      const bool in = i < cnt && (pass == 0 || (keys[i] >> (shift + 8)) == (found >> (shift + 8)));
      // equal digits of a warp are counted together: weights share exponents
      const uint32_t digit = in ? (keys[i] >> shift) & 255u : 256u;
      const uint32_t peers = __match_any_sync(~0u, digit);
      if (in && (tid & 31) == __ffs(int(peers)) - 1)
        atomicAdd(&hist[pass][digit], uint32_t(__popc(peers)));
    }
    cluster.sync();
    uint32_t mine = 0;
    if (tid < 256)  // thread t: digit 255 - t, so that larger digits come first
      for (int r = 0; r < S; ++r) mine += cluster.map_shared_rank(&hist[pass][0], r)[255 - tid];
    uint32_t total;
    const uint32_t above = block_scan(mine, warp_sum, &total);
    if (tid < 256 && above < left && above + mine >= left) {
      pick[0] = uint32_t(255 - tid);
      pick[1] = above;
    }
    __syncthreads();
    found |= pick[0] << shift;
    left -= pick[1];
    __syncthreads();
  }

  // ---- survivors: keys above `found`, and the first `left` (by slot) of
  // those equal to it. A thread takes `q` consecutive slots (odd: no bank
  // conflicts between threads).
  const int q = ((cnt + EV_THREADS - 1) / EV_THREADS) | 1;
  const int i0 = min(tid * q, cnt), i1 = min(i0 + q, cnt);
  uint32_t ties = 0, total;
  for (int i = i0; i < i1; ++i) ties += keys[i] == found;
  uint32_t tie_rank = block_scan(ties, warp_sum, &total);
  if (tid == 0) counts[0] = total;
  cluster.sync();
  for (int r = 0; r < rank; ++r) tie_rank += cluster.map_shared_rank(&counts[0], r)[0];
  const int split = max(0, min(C - s0, cnt));  // local slots before the budget
  uint32_t hm = 0;  // holes (low half) and movers (high half); chunks are below 2^16 slots
  {
    uint32_t tr = tie_rank;
    for (int i = i0; i < i1; ++i) {
      const uint32_t k = keys[i];
      const bool keep = k > found || (k == found && tr++ < left);
      hm += keep == (i < split) ? 0u : (i < split ? 1u : 0x10000u);
    }
  }
  uint32_t at_list = block_scan(hm, warp_sum, &total);
  if (tid == 0) {
    counts[1] = total & 0xffffu;
    counts[2] = total >> 16;
  }
  // holes from the front of the list, movers behind the place of slot C
  for (int i = i0; i < i1; ++i) {
    const uint32_t k = keys[i];
    const bool keep = k > found || (k == found && tie_rank++ < left);
    if (i < split) {
      if (!keep) list[at_list++ & 0xffffu] = uint16_t(i);
    } else if (keep) {
      list[split + (at_list >> 16)] = uint16_t(i);
      at_list += 0x10000u;
    }
  }
  cluster.sync();
  if (tid == 0) {
    uint32_t hs = 0, ms = 0;
    for (int r = 0; r < S; ++r) {
      const uint32_t *o = cluster.map_shared_rank(&counts[0], r);
      hole_end[r] = hs += o[1];
      mover_end[r] = ms += o[2];
    }
  }
  __syncthreads();

  // ---- moves: pair j = (j-th hole, j-th mover); a warp resolves 32 pairs,
  // one per lane, and copies them with all lanes
  const int lane = tid & 31, warps = S * (EV_THREADS / 32);
  const int moves = int(min(hole_end[S - 1], mover_end[S - 1]));
  const int es = c.dtype == WGX_FLOAT16 ? 2 : 4;
  for (int j0 = (rank * (EV_THREADS / 32) + (tid >> 5)) * 32; j0 < moves; j0 += warps * 32) {
    const int j = j0 + lane;
    int64_t kd = -1, ks = 0, vd = 0, vs = 0;  // byte offsets
    if (j < moves) {
      int r = 0;
      while (uint32_t(j) >= hole_end[r]) ++r;
      const int dst = r * per + cluster.map_shared_rank(list, r)[j - (r ? hole_end[r - 1] : 0)];
      r = 0;
      while (uint32_t(j) >= mover_end[r]) ++r;
      const int rsplit = max(0, min(C - r * per, min(per, n - r * per)));
      const int src =
          r * per + cluster.map_shared_rank(list, r)[rsplit + (j - (r ? mover_end[r - 1] : 0))];
      a.weights_out[at + dst] = a.weights[at + src];
      a.positions_out[at + dst] = a.positions[at + src];
      const int dp = dst / c.page_size, sp = src / c.page_size;
      const int dpage = c.page_table[int64_t(b) * c.table_stride + dp];
      const int spage = c.page_table[int64_t(b) * c.table_stride + sp];
      if (dpage >= 0 && dpage < c.pages && spage >= 0 && spage < c.pages) {
        kd = (int64_t(dpage) * c.k_page_stride + int64_t(h) * c.k_head_stride +
              int64_t(dst - dp * c.page_size) * c.k_slot_stride) * es;
        ks = (int64_t(spage) * c.k_page_stride + int64_t(h) * c.k_head_stride +
              int64_t(src - sp * c.page_size) * c.k_slot_stride) * es;
        vd = (int64_t(dpage) * c.v_page_stride + int64_t(h) * c.v_head_stride +
              int64_t(dst - dp * c.page_size) * c.v_slot_stride) * es;
        vs = (int64_t(spage) * c.v_page_stride + int64_t(h) * c.v_head_stride +
              int64_t(src - sp * c.page_size) * c.v_slot_stride) * es;
      } else {
        atomicOr(p.err, kErrCache);
      }
    }
    uint8_t *kb = static_cast<uint8_t *>(c.k), *vb = static_cast<uint8_t *>(c.v);
    const int pairs = min(32, moves - j0);
    for (int x = 0; x < pairs; ++x) {
      const int64_t xkd = __shfl_sync(~0u, kd, x), xks = __shfl_sync(~0u, ks, x);
      const int64_t xvd = __shfl_sync(~0u, vd, x), xvs = __shfl_sync(~0u, vs, x);
      if (xkd < 0) continue;
      if (p.vec) {
        const int units = c.head_dim * es / 16;
        for (int i = lane; i < 2 * units; i += 32) {
          const bool isv = i >= units;
          const int o = (isv ? i - units : i) * 16;
          const uint8_t *src = isv ? vb + xvs + o : kb + xks + o;
          *reinterpret_cast<uint4 *>(isv ? vb + xvd + o : kb + xkd + o) =
              *reinterpret_cast<const uint4 *>(src);
        }
      } else if (es == 2) {
        for (int i = lane; i < c.head_dim; i += 32) {
          reinterpret_cast<uint16_t *>(kb + xkd)[i] = reinterpret_cast<const uint16_t *>(kb + xks)[i];
          reinterpret_cast<uint16_t *>(vb + xvd)[i] = reinterpret_cast<const uint16_t *>(vb + xvs)[i];
        }
      } else {
        for (int i = lane; i < c.head_dim; i += 32) {
          reinterpret_cast<uint32_t *>(kb + xkd)[i] = reinterpret_cast<const uint32_t *>(kb + xks)[i];
          reinterpret_cast<uint32_t *>(vb + xvd)[i] = reinterpret_cast<const uint32_t *>(vb + xvs)[i];
        }
      }
    }
  }
  cluster.sync();  // a CTA's lists are read by the others until here
}

__global__ void evict_lengths_kernel(const __grid_constant__ EvictArgs p) {
  const int b = blockIdx.x * blockDim.x + threadIdx.x;
  if (b >= p.a.cache.batch) return;
  p.a.lengths_out[b] = min(slots_in_use(p.a.lengths, b, p.capacity, p.err), p.a.budget);
}

}  // namespace

void launch_kv_append(const wgx_kv_append_args &a, cudaStream_t stream) {
  AppendArgs p{};
  const wgx_kv_cache &c = a.cache;
  p.a = a;
  p.capacity = cache_capacity(c);
  p.err = device_error_word(current_device());
  const int es = dtype_size(c.dtype);
  bool vec = cache_rows_16b(c);
  const int64_t strides[] = {a.k_batch_stride, a.k_token_stride, a.k_head_stride,
                             a.v_batch_stride, a.v_token_stride, a.v_head_stride};
  for (int64_t s : strides) vec = vec && (s * es) % 16 == 0;
  vec = vec && ((reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v)) & 15) == 0;
  const uint64_t units = uint64_t(a.tokens) * c.kv_heads * (vec ? c.head_dim * es / 16 : c.head_dim);
  // enough blocks to fill the GPU; a sequence's few rows stay in one block,
  // which then writes the counters too
  const uint64_t want = (units + AP_THREADS - 1) / AP_THREADS;
  const uint64_t most = std::max<uint64_t>(1, uint64_t(device_sm_count()) * 16 / uint64_t(c.batch));
  const unsigned gx = want <= 4 ? 1u : unsigned(std::min(want, most));
  p.fused = gx == 1;
  const dim3 grid(gx, unsigned(c.batch));
  const int th = timer_begin("append_kernel", stream);
  if (vec)
    append_kernel<uint4, true><<<grid, AP_THREADS, 0, stream>>>(p);
  else if (es == 2)
    append_kernel<uint16_t, false><<<grid, AP_THREADS, 0, stream>>>(p);
  else
    append_kernel<uint32_t, false><<<grid, AP_THREADS, 0, stream>>>(p);
  check_cuda(cudaGetLastError(), "kv_append launch");
  timer_end(th, stream);
  if (!p.fused) {
    advance_kernel<<<unsigned(c.batch + 127) / 128, 128, 0, stream>>>(p);
    check_cuda(cudaGetLastError(), "kv_append counters launch");
  }
}

void launch_cache_evict(const wgx_cache_evict_args &a, cudaStream_t stream) {
  EvictArgs p{};
  const wgx_kv_cache &c = a.cache;
  p.a = a;
  p.capacity = cache_capacity(c);
  const int64_t slots = std::min(p.capacity, a.slots);
  const int64_t rows = int64_t(c.batch) * c.kv_heads;
  int S = 1;
  while (S < EV_MAX_CLUSTER &&
         (slots > int64_t(S) * EV_MAX_CHUNK || (rows * S < device_sm_count() && slots > int64_t(S) * 2048)))
    S *= 2;
  if (slots > int64_t(S) * EV_MAX_CHUNK)
    fail("cache_evict: more than " + std::to_string(EV_MAX_CLUSTER * EV_MAX_CHUNK) +
         " slots per sequence are not supported");
  p.chunk = int(((slots + S - 1) / S + 7) / 8 * 8);
  p.vec = cache_rows_16b(c);
  p.counters = a.lengths_out != a.lengths;
  const int dev = current_device();
  p.err = device_error_word(dev);
  {
    static std::mutex mu;
    static bool set[64] = {};
    std::lock_guard<std::mutex> lock(mu);
    if (dev >= 64 || !set[dev]) {
      check_cuda(cudaFuncSetAttribute(evict_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      EV_MAX_CHUNK * 6),
                 "cache_evict smem attr");
      if (dev < 64) set[dev] = true;
    }
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(rows * S));
  cfg.blockDim = dim3(EV_THREADS);
  cfg.dynamicSmemBytes = size_t(p.chunk) * 6;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = unsigned(S);
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const int th = timer_begin("evict_kernel", stream);
  check_cuda(cudaLaunchKernelEx(&cfg, evict_kernel, p), "cache_evict launch");
  timer_end(th, stream);
  if (!p.counters) {
    evict_lengths_kernel<<<unsigned(c.batch + 127) / 128, 128, 0, stream>>>(p);
    check_cuda(cudaGetLastError(), "cache_evict counters launch");
  }
}

}  // namespace wgx
