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
constexpr int AP_UNITS = 4;  // units of K and of V a thread has in flight

struct AppendArgs {
  wgx_kv_append_args a;
  int64_t capacity;
  int block_tokens;
  int vec;       // rows move in 16-byte units
  int counters;  // this kernel writes the counters (their outputs are not its inputs, or one
                 // block per sequence)
  uint32_t *err;
};

// Whether the new tokens of a sequence of `len` slots are written. A length that
// the table cannot have (a negative one too) is no place to write behind.
__device__ __forceinline__ bool fits_behind(const wgx_kv_append_args &a, int len, int64_t capacity) {
  return len >= 0 && int64_t(len) + a.tokens <= capacity;
}
// The counters of sequence b (lengths_out may be lengths).
__device__ __forceinline__ void advance(const wgx_kv_append_args &a, int b, int len, int seen, bool fits) {
  a.lengths_out[b] = len + (fits ? a.tokens : 0);
  if (a.seen_out) a.seen_out[b] = seen + (fits ? a.tokens : 0);
}

// U: the unit that is moved (16 bytes of a row, or one element); STEP elements
// each. A thread keeps its unit of a token's rows (head and place in the row) and
// walks over the block's tokens, AP_UNITS of them at a time; threads side by
// side take units side by side, of several tokens where one has few. Bound by
// the bytes: 8 prompts of 2048 tokens (134 MB moved) take 23.2 us, 0.90 of the
// measured copy rate; with index arithmetic per unit it was 26.3, with plain
// stores instead of streaming ones 24.6, at two units in flight 25.1.
template <typename U, int STEP>
__global__ void __launch_bounds__(AP_THREADS, 3) append_kernel(const __grid_constant__ AppendArgs p) {
  const wgx_kv_append_args &a = p.a;
  const wgx_kv_cache &c = a.cache;
  const int b = blockIdx.y;
  const int units = c.head_dim / STEP, all = c.kv_heads * units;  // of a row, of a token
  const int per = max(1, AP_THREADS / all);                       // tokens side by side
  const int sub = int(threadIdx.x) / all, first = sub < per ? int(threadIdx.x) - sub * all : all;  // (or idle)
  wait_for_prior_kernel();
  let_dependents_launch();
  const int len = a.lengths[b];
  const int seen = a.seen ? a.seen[b] : 0;
  const bool fits = fits_behind(a, len, p.capacity);
  if (!fits && threadIdx.x == 0 && blockIdx.x == 0) atomicOr(p.err, kErrCache);
  const int t0 = int(blockIdx.x) * p.block_tokens, t1 = min(t0 + p.block_tokens, a.tokens);
  if (fits) {
    const int32_t *table = c.page_table + int64_t(b) * c.table_stride;
    const int64_t kt = a.k_token_stride / STEP, vt = a.v_token_stride / STEP;
    const int64_t kp = c.k_page_stride / STEP, vp = c.v_page_stride / STEP;
    const int64_t kl = c.k_slot_stride / STEP, vl = c.v_slot_stride / STEP;
    for (int w = first; w < all; w += AP_THREADS) {
      const int h = w / units, u = w - h * units;
      const U *k = static_cast<const U *>(a.k) + (int64_t(b) * a.k_batch_stride + int64_t(h) * a.k_head_stride) / STEP + u;
      const U *v = static_cast<const U *>(a.v) + (int64_t(b) * a.v_batch_stride + int64_t(h) * a.v_head_stride) / STEP + u;
      U *kc = static_cast<U *>(c.k) + int64_t(h) * c.k_head_stride / STEP + u;
      U *vc = static_cast<U *>(c.v) + int64_t(h) * c.v_head_stride / STEP + u;
      const bool counts = u == 0 && (a.weights || a.positions);
      for (int t = t0 + sub; t < t1; t += per * AP_UNITS) {
        U x[AP_UNITS], y[AP_UNITS];
        int page[AP_UNITS], in[AP_UNITS];
#pragma unroll
        for (int e = 0; e < AP_UNITS; ++e) {
          const int tt = t + e * per;
          page[e] = -1;
          if (tt >= t1) continue;
          const uint32_t at = uint32_t(len + tt), pi = at / uint32_t(c.page_size);
          in[e] = int(at - pi * uint32_t(c.page_size));
          page[e] = table[pi];
          x[e] = __ldcs(k + tt * kt);
          y[e] = __ldcs(v + tt * vt);
          if (uint32_t(page[e]) >= uint32_t(c.pages)) {
            atomicOr(p.err, kErrCache);
            page[e] = -1;
          }
          if (counts) {
            const int64_t to = (int64_t(b) * c.kv_heads + h) * a.slots + at;
            if (a.weights) a.weights[to] = 0.f;
            if (a.positions) a.positions[to] = seen + tt;
          }
        }
#pragma unroll
        for (int e = 0; e < AP_UNITS; ++e) {
          if (page[e] < 0) continue;
          __stcs(kc + page[e] * kp + in[e] * kl, x[e]);
          __stcs(vc + page[e] * vp + in[e] * vl, y[e]);
        }
      }
    }
  }
  if (p.counters && blockIdx.x == 0) {
    __syncthreads();
    if (threadIdx.x == 0) advance(a, b, len, seen, fits);
  }
}

__global__ void advance_kernel(const __grid_constant__ AppendArgs p) {
  const int b = blockIdx.x * blockDim.x + threadIdx.x;
  if (b >= p.a.cache.batch) return;
  const int len = p.a.lengths[b];
  advance(p.a, b, len, p.a.seen ? p.a.seen[b] : 0, fits_behind(p.a, len, p.capacity));
}

// ------------------------------------------------------------------- evict
// A cluster of CTAs per (sequence, K/V head). The order of slots is that of the
// numbers (weight key << 32 | complement of the slot), all distinct; the
// budget-th largest is found by radix selection, 11 bits a pass (histograms in
// shared memory, summed over the cluster through distributed shared memory),
// until the class it lies in is wholly taken or small enough (128) to be
// ranked by counting: one or two passes unless weights tie (ranking 512 took
// 8 us, a pass takes 2.5). Keys are held in
// shared memory, weights and positions are read once. Survivors behind the
// budget then move into the holes before it, both listed in slot order.
// Measured: 128 rows of 1040-1056 slots to 1024 (fp16, 128 channels) 7.4 us a
// call, all of it latency (lengths, weights, one pass, lists, few moves); 64 rows
// of 9000-16384 slots to 2048, clusters of 4: 39 us, of which the moves are 21
// (115 MB at 5.5 TB/s) and the selection, which moves little, 15.
constexpr int EV_THREADS = 512;
constexpr int EV_MAX_CLUSTER = 8;
constexpr int EV_MAX_CHUNK = 32768;  // slots per CTA: 6 bytes of shared memory each
static_assert(kEvictMaxSlots == int64_t(EV_MAX_CLUSTER) * EV_MAX_CHUNK, "the checks' limit");
constexpr int EV_BINS = 2048, EV_BITS = 11;
constexpr int EV_CLASS = 128;        // slots of a class that are ranked by counting
static_assert(EV_CLASS <= EV_THREADS, "one thread ranks one member");
constexpr int EV_FLIGHT = 4;         // rows a warp has in flight
constexpr uint32_t kProtected = 0xffffffffu;

struct EvictArgs {
  wgx_cache_evict_args a;
  int64_t capacity;
  int chunk;     // slots per CTA
  int vec;       // rows move in 16-byte units
  int quads;     // weights and positions move four slots at a time
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

__global__ void __launch_bounds__(EV_THREADS, 2) evict_kernel(const __grid_constant__ EvictArgs p) {
  extern __shared__ __align__(16) uint8_t ev_smem[];
  uint32_t *keys = reinterpret_cast<uint32_t *>(ev_smem);
  uint16_t *list = reinterpret_cast<uint16_t *>(ev_smem + size_t(p.chunk) * 4);
  // three histograms in turn: while one is read by other CTAs the next is
  // filled and the one after it cleared
  __shared__ __align__(16) uint32_t hist[3][EV_BINS];
  __shared__ uint64_t members[EV_CLASS], all_members[EV_CLASS];
  __shared__ uint64_t last_kept;     // the budget-th largest number
  __shared__ uint32_t warp_sum[EV_THREADS / 32];
  __shared__ uint32_t counts[3];     // class members, holes, movers of this CTA
  __shared__ uint32_t pick[3];       // bin, numbers above it, numbers in it
  __shared__ uint32_t hole_end[EV_MAX_CLUSTER], mover_end[EV_MAX_CLUSTER];
  cg::cluster_group cluster = cg::this_cluster();
  const int S = int(cluster.num_blocks()), rank = int(cluster.block_rank());
  const wgx_cache_evict_args &a = p.a;
  const wgx_kv_cache &c = a.cache;
  const int tid = threadIdx.x, row = int(blockIdx.x) / S;
  const int b = row / c.kv_heads, h = row % c.kv_heads, C = a.budget;
  for (int i = tid; i < 3 * EV_BINS; i += EV_THREADS) (&hist[0][0])[i] = 0;
  if (tid == 0) counts[0] = 0;
  wait_for_prior_kernel();
  let_dependents_launch();
  const int len = a.lengths[b];
  const bool valid = valid_length(len, p.capacity, p.err);
  const int recent_from = a.seen[b] - a.recent;
  const int n = valid ? len : 0;  // (a.slots >= capacity)
  const int64_t at = int64_t(row) * a.slots;
  if (p.counters && h == 0 && rank == 0 && tid == 0) a.lengths_out[b] = valid ? min(len, C) : len;
  if (n <= C) {  // the same for the whole cluster
    for (int i = rank * EV_THREADS + tid; i < n; i += S * EV_THREADS) {
      if (a.weights_out != a.weights) a.weights_out[at + i] = a.weights[at + i];
      if (a.positions_out != a.positions) a.positions_out[at + i] = a.positions[at + i];
    }
    return;
  }
  const int per = ((n + S - 1) / S + 3) & ~3, s0 = min(rank * per, n), s1 = min(s0 + per, n), cnt = s1 - s0;
  // one CTA alone needs no cluster barrier and reads its own shared memory
  auto sync_all = [&]() {
    if (S == 1) __syncthreads();
    else cluster.sync();
  };
  auto of = [&](auto *mine, int r) { return S == 1 ? mine : cluster.map_shared_rank(mine, r); };

  const bool w_apart = a.weights_out != a.weights, p_apart = a.positions_out != a.positions;
  int done = 0;
  if (p.quads) {
    done = cnt & ~3;
#pragma unroll 2
    for (int i = 4 * tid; i < done; i += 4 * EV_THREADS) {
      const float4 w = *reinterpret_cast<const float4 *>(a.weights + at + s0 + i);
      const int4 pos = *reinterpret_cast<const int4 *>(a.positions + at + s0 + i);
      *reinterpret_cast<uint4 *>(keys + i) =
          make_uint4(evict_key(w.x, pos.x, recent_from, a.sinks), evict_key(w.y, pos.y, recent_from, a.sinks),
                     evict_key(w.z, pos.z, recent_from, a.sinks), evict_key(w.w, pos.w, recent_from, a.sinks));
      if (s0 + i + 4 <= C) {  // holes among these are overwritten below
        if (w_apart) *reinterpret_cast<float4 *>(a.weights_out + at + s0 + i) = w;
        if (p_apart) *reinterpret_cast<int4 *>(a.positions_out + at + s0 + i) = pos;
      } else {
        for (int e = 0; e < 4 && s0 + i + e < C; ++e) {
          a.weights_out[at + s0 + i + e] = e == 0 ? w.x : e == 1 ? w.y : w.z;
          a.positions_out[at + s0 + i + e] = e == 0 ? pos.x : e == 1 ? pos.y : pos.z;
        }
      }
    }
  }
#pragma unroll 4
  for (int i = done + tid; i < cnt; i += EV_THREADS) {
    const float w = a.weights[at + s0 + i];
    const int pos = a.positions[at + s0 + i];
    keys[i] = evict_key(w, pos, recent_from, a.sinks);
    if (s0 + i < C) {
      if (w_apart) a.weights_out[at + s0 + i] = w;
      if (p_apart) a.positions_out[at + s0 + i] = pos;
    }
  }
  __syncthreads();
  auto number = [&](int i) { return uint64_t(keys[i]) << 32 | uint32_t(~uint32_t(s0 + i)); };

  // ---- the C-th largest number: its leading bits are those of `found`, and
  // `left` of the numbers with these bits are still to be taken
  uint64_t found = 0;
  uint32_t left = uint32_t(C);
  int shift = 64;  // bits not yet looked at
  for (int pass = 0;; ++pass) {
    const int bits = min(EV_BITS, shift);
    const int low = shift - bits;
    uint32_t *mine = hist[pass % 3];
    for (int i = tid; i < cnt; i += EV_THREADS) {
      const uint64_t x = number(i);
      if (shift == 64 || (x >> shift) == (found >> shift))
        atomicAdd(&mine[uint32_t(x >> low) & (EV_BINS - 1)], 1u);
    }
    if (pass) {  // (the first three are clear)
      uint32_t *next = hist[(pass + 1) % 3];
      for (int i = tid; i < EV_BINS; i += EV_THREADS) next[i] = 0;
    }
    sync_all();
    // thread t: the four bins from 4 * (511 - t), largest first
    uint4 q = make_uint4(0, 0, 0, 0);
    const int bin = EV_BINS - 4 * (tid + 1);
    for (int r = 0; r < S; ++r) {
      const uint4 y = *reinterpret_cast<const uint4 *>(of(mine, r) + bin);
      q.x += y.x;
      q.y += y.y;
      q.z += y.z;
      q.w += y.w;
    }
    uint32_t total;
    uint32_t above = block_scan(q.x + q.y + q.z + q.w, warp_sum, &total);
    const uint32_t v[4] = {q.w, q.z, q.y, q.x};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (above < left && above + v[j] >= left) {
        pick[0] = uint32_t(bin + 3 - j);
        pick[1] = above;
        pick[2] = v[j];
      }
      above += v[j];
    }
    __syncthreads();
    shift = low;
    found |= uint64_t(pick[0]) << shift;
    left -= pick[1];
    const uint32_t members_all = pick[2];
    if (members_all == left) break;  // wholly taken (always so with no bits left)
    if (members_all <= EV_CLASS) {
      for (int i = tid; i < cnt; i += EV_THREADS) {
        const uint64_t x = number(i);
        if ((x >> shift) == (found >> shift)) members[atomicAdd(&counts[0], 1u)] = x;
      }
      sync_all();
      // every CTA ranks them all: thread i counts the members larger than i
      uint32_t base = 0;
      for (int r = 0; r < S; ++r) {
        const uint32_t m = *of(&counts[0], r);
        if (uint32_t(tid) < m) all_members[base + tid] = of(members, r)[tid];
        base += m;
      }
      __syncthreads();
      if (uint32_t(tid) < members_all) {
        const uint64_t x = all_members[tid];
        uint32_t larger = 0;
#pragma unroll 8
        for (uint32_t j = 0; j < members_all; ++j) larger += all_members[j] > x;
        if (larger == left - 1) last_kept = x;
      }
      __syncthreads();
      found = last_kept;
      break;
    }
    __syncthreads();  // pick is written again
  }

  // ---- holes and movers. A thread takes `q` consecutive slots (odd: no bank
  // conflicts between threads).
  const int q = ((cnt + EV_THREADS - 1) / EV_THREADS) | 1;
  const int i0 = min(tid * q, cnt), i1 = min(i0 + q, cnt);
  const int split = max(0, min(C - s0, cnt));  // local slots before the budget
  uint32_t hm = 0, total;  // holes (low half) and movers (high half); chunks are below 2^16 slots
  for (int i = i0; i < i1; ++i)
    if ((number(i) >= found) != (i < split)) hm += i < split ? 1u : 0x10000u;
  uint32_t at_list = block_scan(hm, warp_sum, &total);
  if (tid == 0) {
    counts[1] = total & 0xffffu;
    counts[2] = total >> 16;
  }
  // holes from the front of the list, movers behind the place of slot C
  for (int i = i0; i < i1; ++i) {
    if ((number(i) >= found) == (i < split)) continue;
    if (i < split) {
      list[at_list++ & 0xffffu] = uint16_t(i);
    } else {
      list[split + (at_list >> 16)] = uint16_t(i);
      at_list += 0x10000u;
    }
  }
  sync_all();
  if (tid == 0) {
    uint32_t hs = 0, ms = 0;
    for (int r = 0; r < S; ++r) {
      const uint32_t *o = of(&counts[0], r);
      hole_end[r] = hs += o[1];
      mover_end[r] = ms += o[2];
    }
  }
  __syncthreads();

  // ---- moves: pair j = (j-th hole, j-th mover). A warp resolves up to 32
  // pairs, one per lane, and copies them with all lanes; few pairs are spread
  // over all warps
  const int lane = tid & 31, warps = S * (EV_THREADS / 32);
  const int moves = int(min(hole_end[S - 1], mover_end[S - 1]));
  const int batch = min(32, (moves + warps - 1) / warps);
  const int es = c.dtype == WGX_FLOAT16 ? 2 : 4;
  for (int j0 = (rank * (EV_THREADS / 32) + (tid >> 5)) * batch; j0 < moves; j0 += warps * batch) {
    const int j = j0 + lane;
    int64_t kd = -1, ks = -1, vd = 0, vs = 0;  // byte offsets; -1: no pair
    if (lane < batch && j < moves) {
      int r = 0;
      while (uint32_t(j) >= hole_end[r]) ++r;
      const int dst = r * per + of(list, r)[j - (r ? hole_end[r - 1] : 0)];
      r = 0;
      while (uint32_t(j) >= mover_end[r]) ++r;
      const int rsplit = max(0, min(C - r * per, min(per, n - r * per)));
      const int src =
          r * per + of(list, r)[rsplit + (j - (r ? mover_end[r - 1] : 0))];
      const int dp = dst / c.page_size, sp = src / c.page_size;
      const int dpage = c.page_table[int64_t(b) * c.table_stride + dp];
      const int spage = c.page_table[int64_t(b) * c.table_stride + sp];
      if (dpage >= 0 && dpage < c.pages && spage >= 0 && spage < c.pages) {
        // (a slot's weight and position move with its row only)
        a.weights_out[at + dst] = a.weights[at + src];
        a.positions_out[at + dst] = a.positions[at + src];
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
    const int pairs = min(batch, moves - j0);
    if (p.vec) {
      // a unit of EV_FLIGHT rows at a time: loads first, then stores
      const int units = c.head_dim * es / 16;
      for (int x0 = 0; x0 < pairs; x0 += EV_FLIGHT) {
        for (int i0 = 0; i0 < 2 * units; i0 += 32) {
          const int i = i0 + lane;
          const bool isv = i >= units, on = i < 2 * units;
          const int o = (isv ? i - units : i) * 16;
          uint8_t *base = (isv ? vb : kb) + o;
          uint4 v[EV_FLIGHT];
#pragma unroll
          for (int e = 0; e < EV_FLIGHT; ++e) {
            const int64_t xks = __shfl_sync(~0u, ks, x0 + e), xvs = __shfl_sync(~0u, vs, x0 + e);
            if (on && xks >= 0) v[e] = *reinterpret_cast<const uint4 *>(base + (isv ? xvs : xks));
          }
#pragma unroll
          for (int e = 0; e < EV_FLIGHT; ++e) {
            const int64_t xkd = __shfl_sync(~0u, kd, x0 + e), xvd = __shfl_sync(~0u, vd, x0 + e);
            if (on && xkd >= 0) *reinterpret_cast<uint4 *>(base + (isv ? xvd : xkd)) = v[e];
          }
        }
      }
    } else {
      for (int x = 0; x < pairs; ++x) {
        const int64_t xkd = __shfl_sync(~0u, kd, x), xks = __shfl_sync(~0u, ks, x);
        const int64_t xvd = __shfl_sync(~0u, vd, x), xvs = __shfl_sync(~0u, vs, x);
        if (xkd < 0) continue;
        for (int i = lane; i < c.head_dim; i += 32) {
          if (es == 2) {
            reinterpret_cast<uint16_t *>(kb + xkd)[i] = reinterpret_cast<const uint16_t *>(kb + xks)[i];
            reinterpret_cast<uint16_t *>(vb + xvd)[i] = reinterpret_cast<const uint16_t *>(vb + xvs)[i];
          } else {
            reinterpret_cast<uint32_t *>(kb + xkd)[i] = reinterpret_cast<const uint32_t *>(kb + xks)[i];
            reinterpret_cast<uint32_t *>(vb + xvd)[i] = reinterpret_cast<const uint32_t *>(vb + xvs)[i];
          }
        }
      }
    }
  }
  if (S > 1) cluster.sync();  // a CTA's lists are read by the others until here
}

__global__ void evict_lengths_kernel(const __grid_constant__ EvictArgs p) {
  const int b = blockIdx.x * blockDim.x + threadIdx.x;
  if (b >= p.a.cache.batch) return;
  const int len = p.a.lengths[b];
  if (valid_length(len, p.capacity, p.err)) p.a.lengths_out[b] = min(len, p.a.budget);
}

}  // namespace

// A call's kernel arguments but for the error word, and its grid.
static AppendArgs append_plan(const wgx_kv_append_args &a, dim3 &grid) {
  AppendArgs p{};
  const wgx_kv_cache &c = a.cache;
  p.a = a;
  p.capacity = cache_capacity(c);
  const int es = dtype_size(c.dtype);
  p.vec = cache_rows_16b(c);
  const int64_t strides[] = {a.k_batch_stride, a.k_token_stride, a.k_head_stride,
                             a.v_batch_stride, a.v_token_stride, a.v_head_stride};
  for (int64_t s : strides) p.vec = p.vec && (s * es) % 16 == 0;
  p.vec = p.vec && ((reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v)) & 15) == 0;
  // tokens a block takes: AP_UNITS units a thread, and more where that would be
  // over sixteen blocks per SM
  const int all = c.kv_heads * (p.vec ? c.head_dim * es / 16 : c.head_dim);
  const int64_t most = std::max<int64_t>(1, int64_t(device_sm_count()) * 16 / c.batch);
  p.block_tokens = int(std::max<int64_t>(int64_t(std::max(1, AP_THREADS / all)) * AP_UNITS, (int64_t(a.tokens) + most - 1) / most));
  grid = dim3(unsigned((int64_t(a.tokens) + p.block_tokens - 1) / p.block_tokens), unsigned(c.batch));
  p.counters = grid.x == 1 || (a.lengths_out != a.lengths && (!a.seen || a.seen_out != a.seen));
  return p;
}

int kv_append_launches(const wgx_kv_append_args &a) {
  dim3 grid;
  return append_plan(a, grid).counters ? 1 : 2;
}

void launch_kv_append(const wgx_kv_append_args &a, cudaStream_t stream) {
  dim3 grid;
  AppendArgs p = append_plan(a, grid);
  p.err = device_error_word(current_device());
  const int es = dtype_size(a.cache.dtype);
  const int th = timer_begin("append_kernel", stream);
  launch_dependent(p.vec ? (es == 2 ? append_kernel<uint4, 8> : append_kernel<uint4, 4>)
                         : (es == 2 ? append_kernel<uint16_t, 1> : append_kernel<uint32_t, 1>),
                   grid, AP_THREADS, 0, stream, "kv_append launch", p);
  timer_end(th, stream);
  if (!p.counters) {
    advance_kernel<<<unsigned(a.cache.batch + 127) / 128, 128, 0, stream>>>(p);
    check_cuda(cudaGetLastError(), "kv_append counters launch");
  }
}

int cache_evict_launches(const wgx_cache_evict_args &a) { return a.lengths_out != a.lengths ? 1 : 2; }

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
  p.chunk = int(((slots + S - 1) / S + 7) / 8 * 8);
  p.vec = cache_rows_16b(c);
  p.quads = a.slots % 4 == 0 && ((reinterpret_cast<uintptr_t>(a.weights) | reinterpret_cast<uintptr_t>(a.weights_out) |
                                  reinterpret_cast<uintptr_t>(a.positions) |
                                  reinterpret_cast<uintptr_t>(a.positions_out)) & 15) == 0;
  p.counters = cache_evict_launches(a) == 1;
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
  const int th = timer_begin("evict_kernel", stream);
  launch_dependent(evict_kernel, dim3(unsigned(rows * S)), EV_THREADS, size_t(p.chunk) * 6, stream,
                   "cache_evict launch", p, S);
  timer_end(th, stream);
  if (!p.counters) {
    evict_lengths_kernel<<<unsigned(c.batch + 127) / 128, 128, 0, stream>>>(p);
    check_cuda(cudaGetLastError(), "cache_evict counters launch");
  }
}

}  // namespace wgx
