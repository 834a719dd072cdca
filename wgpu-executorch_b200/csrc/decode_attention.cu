// Attention of one new token per sequence over a paged K/V cache:
//   s_j = scale * q . k_j,  p_j = exp(s_j - max s) / sum exp(s - max s),
//   out = sum_j p_j v_j     over the live slots j of the sequence,
// for all query heads that share a K/V head at once.
//
// Every cached byte is read once and used for 2 * group multiply-adds per
// element, so the cache's bytes over the HBM rate are the floor. The work is
// split over the cache's length: a step is TOK slots of one (sequence, K/V
// head), all steps of the batch stand in one line, and every worker (a warp; two
// above 128 channels) of the grid takes an equal, contiguous share of it,
// whatever the lengths are. A worker streams its steps through a ring of its own
// in shared memory, so no block barrier stands between loads and products:
// where a step's rows lie in one page they come by TMA (one copy per operand
// and step, any strides), elsewhere by 16-byte cp.async or element by element.
// The V rows of slots that are not live are cleared in shared memory: stale
// infinities and NaN of a page must not reach a product. The softmax is the
// running one: a reference value and the sum in fp32 per head, the result
// rescaled when a step's scores lie too far from the reference (a few powers of
// two above it, and in fp16 also below it).
//
// The group's heads are the 16 rows of an mma.sync tile (M = heads, N = slots
// for the scores, N = channels for the result). tcgen05 would need 64 or 128
// rows; a decode step has at most a group of them, and its time is the loads'.
// fp16: m16n8k16, exact products of scores, probabilities as a sum of two fp16
// numbers, fp32 sums. fp32: CUDA cores for groups of at
// most 8 heads, above that m16n8k8 tf32 with every operand split in two.
//
// A row of work that lies within one worker's share is finished by it. Rows cut
// by a share's end leave (reference, sum, unnormalised result) in scratch, at
// most two per worker, and join_kernel combines them; it also accumulates the
// probabilities per slot from the scores, kept in scratch for it. Short rows
// are not cut: row mode (below) joins them in shared memory.
//
// Measured (fp16, K and V bytes over the time of the kernel, then the whole
// call): 8 K/V heads x 128 channels, 131071 slots: 84.5 us, 6.35 TB/s, call 97
// us; 64 sequences of 17-8192 slots with weights: 190 us, 5.7 TB/s, call 208;
// 48 sequences of one head of 256 channels x 16, 4096 slots each: steps run at
// 6.4 TB/s, but start, cut rows and join are 20 us of the call's 52:
// neighbouring shares lie in different blocks, and each of some 640 cut rows of
// 16 KB goes through memory. What is left besides is the chain lengths -> page
// table -> rows at the start (about 4 us) and the join (5 us).
#include <cooperative_groups.h>

#include <algorithm>
#include <mutex>

#include "decode.h"
#include "tcgen05.h"
#include "tma.h"

namespace cg = cooperative_groups;

namespace wgx {

namespace {

constexpr int PA_HEADS = 16;        // rows of an mma tile
constexpr int PA_MAX_GROUP = 128;   // query heads per K/V head
// Row mode, a block (or a cluster of 2 or 4) per row instead of equal shares of
// the line and a second kernel: no scratch, no join, but rows must be alike and
// short. Steps a block's part of a row may have: 16; 8 with fp32, 4 above 128
// channels (their steps take longer). Measured, us a call, 8 K/V heads x 4 heads
// of 128, fp16, batch 1 / 8: 128 slots 6.1 / 6.5 in row mode, 11.4 / 11.4
// split; 256: 8.3 / 8.7, 10.8 / 11.6; 512, clusters of 4: 9.6 / 10.6, 10.2 /
// 12.6; 1024: 11.9 / 13.6, 13.2 / 16.3; 2048: 16.5 / 19.5, 12.2 / 24.2. fp32:
// 64 slots 8.1 / 8.2, 9.9 / 10.7; 256, clusters of 4: 11.4 / 12.6, 11.6 / 13.6.
// A lone row is better split from the start of clusters on (one head of 256
// channels x 16, 256 slots: 12.6 in a cluster, 10.2 split).
constexpr int PA_ROW_STEPS = 16;
constexpr int PA_ROW_CLUSTER = 4;
constexpr int PA_ROW_MIN = 8;  // rows from which clusters are used
// fp16 probabilities (see the running softmax), in powers of two: the reference
// value is set PA_ABOVE below a step's maximum, and again when a step's maximum
// is not within PA_FAR of PA_MIDDLE above it; never PA_DEPTH below the highest
// that it has been.
constexpr float PA_ABOVE = 11.f, PA_MIDDLE = 8.f, PA_FAR = 7.f, PA_DEPTH = 60.f;
constexpr int PA_JOIN_THREADS = 256;
constexpr int PA_JOIN_SLOTS = 4096;  // slots per join block of the accumulation

struct AttnArgs {
  CUtensorMap k_map, v_map;  // where tma: [page][head][slot][channel] in boxes of TOK rows
  wgx_paged_attention_args a;
  int64_t capacity;   // slots a table can name
  int group;          // query heads per K/V head
  int chunks;         // ceil(group / PA_HEADS)
  int max_workers;    // warps the scratch has room for
  int min_steps;      // steps a worker takes at least
  int row_blocks;     // row mode: a cluster of so many blocks per row of work; 0: off
  int vec;            // rows move in 16-byte units
  int tma;            // a step's rows lie in one page and move by TMA
  int boxes;          // TMA copies per operand and step
  int q_pairs;        // queries can be read two elements at a time
  float scale2;       // scale * log2(e): the softmax runs in base 2
  float *part_o;      // [worker][2][heads][part_stride]
  int part_stride;    // head_dim rounded up to 4
  float2 *part_ml;    // [worker][2][heads] (max, sum)
  float2 *stats;      // [row][heads]: of rows finished by one warp (accumulation only)
  float *scores;      // [batch][q_heads][score_stride], from a row's first step (accumulation only)
  int64_t score_stride;  // slots of the steps that a row can have
  int weights_quads;  // weights move four slots at a time
  int heads;          // min(group, PA_HEADS): rows a partial result has
  uint32_t *prefix;   // [batch + 1] steps of a row before each sequence (for the join)
  int o_blocks;       // of the join: blocks for the result
  int join_warps;     // of the join: warps per query head
  uint32_t *err;
};

// The line of work: sequence b has steps[b] steps in each of its
// kv_heads * chunks rows. prefix[b] = sum of steps before b (all rows' line
// is prefix[batch] * rows long).
struct Span {
  int first;  // first step (of TOK slots, from slot 0)
  int steps;
  int len;
  int lo;     // first live slot
};
template <int TOK>
__device__ __forceinline__ Span span_of(const AttnArgs &p, int len) {
  Span s;
  s.len = len;
  s.lo = p.a.window > 0 ? max(0, len - p.a.window) : 0;
  s.first = s.lo / TOK;
  s.steps = (len + TOK - 1) / TOK - s.first;
  return s;
}

// prefix[0 .. batch] and lens[0 .. batch - 1] into shared memory.
// Where `leave`, block 0 also leaves the prefix in scratch.
template <int TOK>
__device__ void build_prefix(const AttnArgs &p, uint32_t *prefix, int *lens, bool leave) {
  const int B = p.a.cache.batch, tid = threadIdx.x, nt = blockDim.x;
  __shared__ uint32_t warp_sum[32];
  uint32_t base = 0;
  for (int b0 = 0; b0 < B; b0 += nt) {
    const int b = b0 + tid;
    uint32_t n = 0;
    if (b < B) {
      const int len = slots_in_use(p.a.lengths, b, p.capacity, p.err);
      lens[b] = len;
      n = uint32_t(span_of<TOK>(p, len).steps);
    }
    uint32_t x = n;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const uint32_t y = __shfl_up_sync(~0u, x, d);
      if ((tid & 31) >= d) x += y;
    }
    if ((tid & 31) == 31) warp_sum[tid >> 5] = x;
    __syncthreads();
    uint32_t before = base, all = base;
    for (int w = 0; w < nt / 32; ++w) {
      if (w < (tid >> 5)) before += warp_sum[w];
      all += warp_sum[w];
    }
    if (b < B) {
      prefix[b] = before + x - n;
      if (leave && blockIdx.x == 0) p.prefix[b] = before + x - n;
    }
    base = all;
    __syncthreads();
  }
  if (tid == 0) {
    prefix[B] = base;
    if (leave && blockIdx.x == 0) p.prefix[B] = base;
  }
  __syncthreads();
}

// Whether slot t of sequence b is live. The accumulation of weights asks where a
// head's sum is NaN: its probabilities are NaN then, those of slots that are
// not live (kept as scores of -infinity) zero all the same.
__device__ __forceinline__ bool slot_is_live(const AttnArgs &p, int b, const Span &s, int t) {
  const wgx_kv_cache &c = p.a.cache;
  if (t < s.lo || t >= s.len) return false;
  if (p.a.mask && (t >= p.a.mask_width || !p.a.mask[int64_t(b) * p.a.mask_stride + t])) return false;
  return uint32_t(c.page_table[int64_t(b) * c.table_stride + t / c.page_size]) < uint32_t(c.pages);
}

__device__ __forceinline__ uint32_t worker_count(const AttnArgs &p, uint32_t total) {
  const uint32_t want = (total + uint32_t(p.min_steps) - 1) / uint32_t(p.min_steps);
  return max(1u, min(want, uint32_t(p.max_workers)));
}
// Equal shares of the line: the first `extra` workers take base + 1 steps.
struct Shares {
  uint32_t base, extra;
  __device__ __forceinline__ Shares(uint32_t total, uint32_t workers) {
    base = total / workers;
    extra = total - base * workers;
  }
  __device__ __forceinline__ uint32_t begin(uint32_t worker) const { return base * worker + min(worker, extra); }
  // the worker whose share holds step s (base is at least 1: there are no more
  // workers than steps)
  __device__ __forceinline__ uint32_t of(uint32_t s) const {
    const uint32_t cut = extra * (base + 1);
    return s < cut ? s / (base + 1) : extra + (s - cut) / base;
  }
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(live ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t *r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t *r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void mma16(float *c, const uint32_t *a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma8(float *c, const uint32_t *a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x = head + tail in tf32's 10 mantissa bits each: the head rounded to nearest
// (half of its last place added to the bits), the tail cut by the tensor core,
// which ignores the 13 bits behind it. What is lost is below 2^-21 of x, its sign
// as random as the tail's: errors of 1e-7 in the result, as with rounded tails
// (64 against 67 us at 16 sequences of 3000-5000 slots x 2 x 16 heads x 128).
// A tail must not be rounded by its bits: where x is NaN it is the NaN with all
// mantissa bits set, and half a place more makes that a zero; the head of such
// an x is zero already. Converting (cvt.rna) keeps NaN too, at 112 us.
__device__ __forceinline__ void split_tf32(float x, uint32_t &head, uint32_t &tail) {
  head = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
  tail = __float_as_uint(x - __uint_as_float(head));
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float lds32(uint32_t addr) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

template <typename T, int DP>
struct Tile {
  static constexpr bool kHalf = sizeof(T) == 2;
  static constexpr int TOK = kHalf ? 16 : 8;        // slots per step
  static constexpr uint32_t FULL = (1u << TOK) - 1;
  static constexpr int EPC = 16 / int(sizeof(T));   // elements per 16-byte chunk
  static constexpr int CPR = DP / EPC;              // chunks per staged row
  static constexpr int ROW = DP * int(sizeof(T));   // staged row bytes
  static constexpr int STAGE = 2 * TOK * ROW;       // K and V of one step
  static constexpr int PANEL = 128 / int(sizeof(T));  // channels per 128 bytes
  static constexpr int PANELS = DP / PANEL;
  // Byte of chunk c of row r: panels of 128 bytes x TOK rows, chunks of a row
  // permuted by the row's low bits (the 128-byte swizzle of a TMA copy), so
  // that eight rows' equal chunks lie in different banks.
  __device__ static constexpr uint32_t at(int r, int c) {
    return uint32_t((c >> 3) * (TOK * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4));
  }
};

__device__ __forceinline__ void tma_load_5d(uint32_t dst, const void *map, int x, int y, int z, int w,
                                            int v, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(v), "r"(bar)
      : "memory");
}
// arrives on `bar` when this thread's cp.async copies so far have landed
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

// The steps of a warp's share, from the line's place `begin` on.
template <int TOK>
struct Walk {
  int b, row, step;  // row: kv_head * chunks + chunk
  Span s;

  __device__ __forceinline__ void start(const AttnArgs &p, const uint32_t *prefix, const int *lens,
                                        int rows, uint32_t begin) {
    // the sequence whose rows hold `begin`
    const uint32_t key = begin / uint32_t(rows);
    int lo = 0, hi = p.a.cache.batch - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (prefix[mid] <= key) lo = mid;
      else hi = mid - 1;
    }
    b = lo;
    s = span_of<TOK>(p, lens[lo]);
    const uint32_t rest = begin - prefix[lo] * uint32_t(rows);
    row = int(rest / uint32_t(s.steps));
    step = int(rest) - row * s.steps;
  }
  __device__ __forceinline__ void next_row(const AttnArgs &p, const int *lens, int rows) {
    step = 0;
    if (++row < rows) return;
    row = 0;
    while (++b < p.a.cache.batch) {
      s = span_of<TOK>(p, lens[b]);
      if (s.steps > 0) return;
    }
  }
};

// A worker's loads: its share of the line of work through a ring of STAGES
// steps in shared memory. Every warp of the worker keeps this state; the leader
// issues the copies. What a step needs to know (with scattered rows its page and
// slot per lane, its mask) is fetched one step ahead of its use, page table
// entries 32 pages ahead.
template <typename T, int DP, int STAGES>
struct Loader {
  using L = Tile<T, DP>;
  static constexpr int TOK = L::TOK;
  static_assert(STAGES <= 4, "the live bits of the ring are 4 x 16");
  Walk<TOK> ld;
  uint32_t to_load;
  int head, left;            // K/V head and steps left of the row being loaded
  int t0, slot, page;        // next step: first slot, its place in its page, page
  // the row's page table, 32 entries in a register (one per lane) and the next
  // 32 in another: entry `at` of the first is the next step's
  const int32_t *entries;
  int pages_now, pages_next, at, known;  // known: first entry not yet loaded
  uint32_t mine;             // lane < TOK: its slot `lane` is live
  uint64_t live_ring;        // 16 bits of live slots per step in flight, oldest highest

  __device__ __forceinline__ void fetch_live(const AttnArgs &p, int lane) {
    const int t = t0 + lane;
    mine = lane < TOK && t >= ld.s.lo && t < ld.s.len;
    if (p.a.mask && mine)  // (looked at when the step is issued)
      mine = t < p.a.mask_width ? p.a.mask[int64_t(ld.b) * p.a.mask_stride + t] : 0;
    if (!p.tma) {
      page = -1;
      if (lane < TOK && t >= ld.s.lo && t < ld.s.len) {
        const int pi = int(uint32_t(t) / uint32_t(p.a.cache.page_size));
        slot = t - pi * p.a.cache.page_size;
        page = p.a.cache.page_table[int64_t(ld.b) * p.a.cache.table_stride + pi];
      }
    }
  }
  __device__ __forceinline__ int more_pages(const AttnArgs &p, int lane) {
    const int i = known + lane;
    known += 32;
    return i < p.a.cache.table_width ? entries[i] : -1;
  }
  __device__ __forceinline__ void fetch_row(const AttnArgs &p, int lane) {
    head = ld.row / p.chunks;
    left = ld.s.steps - ld.step;
    t0 = (ld.s.first + ld.step) * TOK;
    if (p.tma) {
      const int pi = int(uint32_t(t0) / uint32_t(p.a.cache.page_size));
      slot = t0 - pi * p.a.cache.page_size;
      entries = p.a.cache.page_table + int64_t(ld.b) * p.a.cache.table_stride;
      known = pi;
      at = 0;
      pages_now = more_pages(p, lane);
      pages_next = more_pages(p, lane);
    }
    fetch_live(p, lane);
  }
  __device__ __forceinline__ void start(const AttnArgs &p, const Walk<TOK> &from, uint32_t steps, int lane) {
    ld = from;
    to_load = steps;
    slot = 0;
    page = -1;
    live_ring = 0;
    fetch_row(p, lane);
  }
  // the live slots of the step that is to be used next
  __device__ __forceinline__ uint32_t oldest() const {
    return uint32_t(live_ring >> (16 * (STAGES - 2))) & 0xffffu;
  }
  __device__ __forceinline__ void issue(const AttnArgs &p, uint8_t *stage_p, uint32_t bar, int lane,
                                        bool leader) {
    const wgx_kv_cache &c = p.a.cache;
    if (p.tma) page = __shfl_sync(~0u, pages_now, at);
    bool on = mine != 0;
    if (on && uint32_t(page) >= uint32_t(c.pages)) {
      atomicOr(p.err, kErrCache);
      on = false;
    }
    const uint32_t bits = __ballot_sync(~0u, on);
    live_ring = (live_ring << 16) | bits;
    if (!bits || !leader) return;  // (no live slot: the step is passed over)
    uint8_t *sk = stage_p, *sv = sk + TOK * L::ROW;
    const T *kbase = static_cast<const T *>(c.k), *vbase = static_cast<const T *>(c.v);
    const int D = c.head_dim;
    if (p.tma) {
      if (lane == 0) {
        const uint32_t ska = smem_u32(sk), sva = smem_u32(sv);
        // (a box counts in full, its part outside the tensor too)
        mbar_expect_tx(bar, uint32_t(2 * TOK * 128) * uint32_t((D + L::PANEL - 1) / L::PANEL));
        for (int j = 0; j < p.boxes; ++j) {
          tma_load_5d(ska + uint32_t(j * TOK * 128), &p.k_map, j * L::PANEL, slot, 0, head, page, bar);
          tma_load_5d(sva + uint32_t(j * TOK * 128), &p.v_map, j * L::PANEL, slot, 0, head, page, bar);
        }
      }
      return;
    }
    const bool live = (bits >> lane) & 1;
    const int64_t ko = live ? int64_t(page) * c.k_page_stride + int64_t(head) * c.k_head_stride +
                                  int64_t(slot) * c.k_slot_stride : 0;
    const int64_t vo = live ? int64_t(page) * c.v_page_stride + int64_t(head) * c.v_head_stride +
                                  int64_t(slot) * c.v_slot_stride : 0;
    if (p.vec) {
      const uint32_t ska = smem_u32(sk), sva = smem_u32(sv);
#pragma unroll 4
      for (int i = 0; i < TOK * L::CPR / 32; ++i) {
        const int idx = i * 32 + lane, r = idx / L::CPR, ch = idx % L::CPR;
        const int64_t kr = __shfl_sync(~0u, ko, r), vr = __shfl_sync(~0u, vo, r);
        const bool ok = (bits >> r) & 1;
        if (ch * L::EPC < D) {
          cp_async16(ska + L::at(r, ch), kbase + kr + ch * L::EPC, ok);
          cp_async16(sva + L::at(r, ch), vbase + vr + ch * L::EPC, ok);
        }
      }
      cp_async_arrive(bar);
    } else {
      for (int r = 0; r < TOK; ++r) {
        const int64_t kr = __shfl_sync(~0u, ko, r), vr = __shfl_sync(~0u, vo, r);
        const bool ok = (bits >> r) & 1;
        for (int e = lane; e < D; e += 32) {
          const uint32_t d = L::at(r, e / L::EPC) + uint32_t(e % L::EPC) * uint32_t(sizeof(T));
          *reinterpret_cast<T *>(sk + d) = ok ? kbase[kr + e] : T(0.f);
          *reinterpret_cast<T *>(sv + d) = ok ? vbase[vr + e] : T(0.f);
        }
      }
      mbar_arrive(bar);
    }
  }
  __device__ __forceinline__ void next(const AttnArgs &p, const int *lens, int rows, uint8_t *ring,
                                       uint64_t *bars, int stage, int lane, bool leader) {
    if (!to_load) {
      live_ring <<= 16;
      return;
    }
    issue(p, ring + stage * L::STAGE, smem_u32(&bars[stage]), lane, leader);
    if (!--to_load) return;
    if (--left == 0) {
      ld.next_row(p, lens, rows);
      fetch_row(p, lane);
    } else {
      t0 += TOK;
      if (p.tma) {
        slot += TOK;
        if (slot == p.a.cache.page_size) {
          slot = 0;
          if (++at == 32) {
            at = 0;
            pages_now = pages_next;
            pages_next = more_pages(p, lane);
          }
        }
      }
      fetch_live(p, lane);
    }
  }
};

// What the pages hold in slots that are not live must not reach 0 * v.
template <typename T, int DP>
__device__ __forceinline__ void clear_dead_rows(uint32_t va, uint32_t live, int lane) {
  using L = Tile<T, DP>;
  for (int r = 0; r < L::TOK; ++r)
    if (!((live >> r) & 1))
      for (int ch = lane; ch < L::CPR; ch += 32)
        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(va + L::at(r, ch)), "r"(0) : "memory");
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncwarp();
}

// A worker after a wait ran out: nothing may be in flight when it leaves, so it
// waits (bounded) for the stages behind the one that did not arrive.
template <int STAGES>
__device__ void drain(uint64_t live_ring, uint64_t *bars, int stage, uint32_t phase) {
  stage = stage + 1 == STAGES ? 0 : stage + 1;
  for (int s = 1; s < STAGES - 1; ++s) {
    const uint32_t live = uint32_t(live_ring >> (16 * (STAGES - 2 - s))) & 0xffffu;
    if (live) mbar_wait(smem_u32(&bars[stage]), (phase >> stage) & 1);
    stage = stage + 1 == STAGES ? 0 : stage + 1;
  }
}

// Shared memory of a block: the workers' rings (1024-byte aligned), what else
// each worker needs, then the sequences' prefix and lengths.
struct BlockSmem {
  uint8_t *ring, *extra;
  uint32_t *prefix;
  int *lens;
};
__device__ __forceinline__ BlockSmem block_smem(uint8_t *raw, int worker, int ring_bytes, int extra_bytes,
                                                int workers, int batch) {
  uint8_t *base = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  BlockSmem m;
  m.ring = base + size_t(worker) * ring_bytes;
  m.extra = base + size_t(workers) * ring_bytes + size_t(worker) * extra_bytes;
  m.prefix = reinterpret_cast<uint32_t *>(base + size_t(workers) * (ring_bytes + extra_bytes));
  m.lens = reinterpret_cast<int *>(m.prefix + batch + 1);
  return m;
}

constexpr int PA_BLOCK_WORKERS = 4;

// Row mode: joins the results of the row's workers, four per block of the
// cluster (o: [head][stride] floats at the front of each worker's ring; ml:
// their maxima and sums), and accumulates the row's probabilities: each block
// takes a share of the output and the slots whose scores it wrote. Every thread
// of the block.
// CLUSTER: more blocks than one.
template <typename T, int TOK, bool CLUSTER>
__device__ void finish_row(const AttnArgs &p, int b, int row, const Span &s, float2 (*ml)[PA_HEADS],
                           uint8_t *rings, int ring_bytes, int stride) {
  constexpr int MOST = PA_BLOCK_WORKERS * PA_ROW_CLUSTER;
  __shared__ float factor[MOST][PA_HEADS], head_m[PA_HEADS], head_inv[PA_HEADS];
  __shared__ bool odd;  // a head without probabilities that are numbers
  cg::cluster_group cluster = cg::this_cluster();
  const int S = CLUSTER ? p.row_blocks : 1, rank = CLUSTER ? int(cluster.block_rank()) : 0;
  auto of = [&](auto *mine, int r) {
    if constexpr (CLUSTER) return cluster.map_shared_rank(mine, r);
    else return mine;
  };
  const int tid = threadIdx.x, D = p.a.cache.head_dim, parts = S * PA_BLOCK_WORKERS;
  const int h = row / p.chunks, chunk = row - h * p.chunks, nh = min(p.heads, p.group - chunk * PA_HEADS);
  if (tid == 0) odd = false;
  if constexpr (CLUSTER) cluster.sync();
  else __syncthreads();
  if (tid < nh) {
    float M = -INFINITY, sum = 0.f;
    for (int w = 0; w < parts; ++w)
      M = fmaxf(M, of(&ml[0][0], w / PA_BLOCK_WORKERS)[w % PA_BLOCK_WORKERS * PA_HEADS + tid].x);
    const float mu = M == -INFINITY ? 0.f : M;
    for (int w = 0; w < parts; ++w) {
      const float2 x = of(&ml[0][0], w / PA_BLOCK_WORKERS)[w % PA_BLOCK_WORKERS * PA_HEADS + tid];
      const float f = exp2_approx(x.x - mu);
      factor[w][tid] = f;
      sum += f * x.y;
    }
    if (sum != sum) odd = true;
    head_m[tid] = mu;
    head_inv[tid] = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
  }
  __syncthreads();
  T *out = static_cast<T *>(p.a.out) + int64_t(b) * p.a.out_batch_stride +
           int64_t(h * p.group + chunk * PA_HEADS) * p.a.out_head_stride;
  for (int i = rank * int(blockDim.x) + tid; i < nh * D; i += S * int(blockDim.x)) {
    const int g = i / D, d = i - g * D;
    float v = 0.f;
#pragma unroll 4
    for (int w = 0; w < parts; ++w) {
      const float f = factor[w][g];  // (zero: the worker may not have written its result)
      const float *o = reinterpret_cast<const float *>(of(rings, w / PA_BLOCK_WORKERS) +
                                                       size_t(w % PA_BLOCK_WORKERS) * ring_bytes);
      if (f != 0.f) v += f * o[g * stride + d];
    }
    out[int64_t(g) * p.a.out_head_stride + d] = T(v * head_inv[g]);
  }
  if (p.scores) {
    const int64_t at = (int64_t(b) * p.a.cache.kv_heads + h) * p.a.slots;
    const float *sc = p.scores + (int64_t(b) * p.a.q_heads + h * p.group) * p.score_stride;
    const bool in_place = p.a.weights == p.a.weights_out;  // (slots in front of the window stay)
    const int t0 = rank || in_place ? (s.first + s.steps * rank / S) * TOK : 0;
    const int t1 = min((s.first + s.steps * (rank + 1) / S) * TOK, int(min(int64_t(s.len), p.a.slots)));
    for (int t = t0 + tid; t < t1; t += int(blockDim.x)) {
      float w = p.a.weights[at + t];
      if (t >= s.first * TOK && (!odd || slot_is_live(p, b, s, t)))
#pragma unroll 4
        for (int g = 0; g < nh; ++g)
          w += exp2_approx(sc[int64_t(g) * p.score_stride + (t - s.first * TOK)] - head_m[g]) * head_inv[g];
      p.a.weights_out[at + t] = w;
    }
  }
  if constexpr (CLUSTER) cluster.sync();  // a block's results are read by the others until here
}

// ROW: row mode, a kernel of its own. In one kernel for both, the registers that
// the end of a row needs were held through the steps: 54.2 against 52 us at 48
// sequences x 4096 slots x 16 heads x 256, 5.14 against 5.02 at one of 77 slots x
// 8 x 64, 63.8 against 60.8 at 16 sequences of 3000-5000 slots x 2 x 16 x 128 in
// fp32; one row of 131072 slots x 8 x 4 x 128 the same within 1 %.
// Tensor-core form: the worker's heads are the 16 rows of an mma tile. A step of
// 16 slots costs a warp about 48 mma of 128 channels and as many other
// instructions; with operand addresses computed in full it was 450 instructions
// and the kernel issue-bound (101 instead of 84.5 us at 131071 slots).
// HALF_ROWS: at most 8 heads (rows 8-15 are padding and their softmax is left
// out). Heads of 256 channels: two warps share a worker, each with half of the
// channels: the halves of the scores are added through shared memory (one
// warp's 128 result registers beside 64 of the query left room for one warp per
// scheduler).
template <typename T, int DP>
struct MmaShape {
  static constexpr int WARPS = DP > 128 ? 2 : 1;  // per worker
  // fp32 rows of 256 channels: the query's registers would not fit beside the
  // result's, so it stays in shared memory
  static constexpr bool kQShared = sizeof(T) == 4 && DP > 128;
  static constexpr int STAGES = kQShared ? 2 : Tile<T, DP>::STAGE > 4096 ? 3 : 4;
  static constexpr int QBYTES = kQShared ? PA_HEADS * Tile<T, DP>::ROW : 0;
  static constexpr int RING = STAGES * Tile<T, DP>::STAGE, EXTRA = QBYTES;
  static constexpr int THREADS = PA_BLOCK_WORKERS * WARPS * 32;
  static_assert(PA_BLOCK_WORKERS * (RING + EXTRA) + 1024 + (2 * 2048 + 1) * 4 + 10 * 1024 <= 227 * 1024, "shared memory of a block");
};

template <typename T, int DP, bool HALF_ROWS, bool ROW>
__global__ void __launch_bounds__(MmaShape<T, DP>::THREADS, DP > 128 ? 1 : 2)
    paged_attention_kernel(const __grid_constant__ AttnArgs p) {
  using L = Tile<T, DP>;
  using M = MmaShape<T, DP>;
  constexpr int TOK = L::TOK, STAGES = M::STAGES, PANEL = L::PANEL;
  constexpr int WP = L::PANELS / M::WARPS, NT = DP / 8 / M::WARPS;  // this warp's panels and tiles of the result
  constexpr int HALVES = HALF_ROWS ? 1 : 2, ST = TOK / 8;
  extern __shared__ uint8_t pa_smem_raw[];
  __shared__ __align__(8) uint64_t all_bars[PA_BLOCK_WORKERS][STAGES];
  __shared__ float2 row_ml[PA_BLOCK_WORKERS][PA_HEADS];
  __shared__ __align__(16) float4 halves[M::WARPS == 2 ? PA_BLOCK_WORKERS : 1][2][M::WARPS == 2 ? ST : 1][32];
  const wgx_kv_cache &c = p.a.cache;
  const int lane = threadIdx.x % 32, worker = threadIdx.x / (32 * M::WARPS);
  const int part = threadIdx.x / 32 % M::WARPS;  // of the worker
  const BlockSmem sm = block_smem(pa_smem_raw, worker, M::RING, M::EXTRA, PA_BLOCK_WORKERS, c.batch);
  uint64_t *bars = all_bars[worker];
  const int D = c.head_dim;
  // barrier among the worker's warps; true when all of their threads say so
  auto worker_all = [&](bool mine) -> bool {
    if constexpr (M::WARPS == 1) {
      return __all_sync(~0u, mine);
    } else {
      uint32_t all;
      asm volatile(
          "{\n\t.reg .pred a, b;\n\t"
          "setp.ne.u32 a, %1, 0;\n\t"
          "barrier.cta.red.and.pred b, %2, %3, a;\n\t"
          "selp.u32 %0, 1, 0, b;\n\t}"
          : "=r"(all)
          : "r"(uint32_t(mine)), "r"(worker + 1), "n"(M::WARPS * 32)
          : "memory");
      return all != 0;
    }
  };
  if (part == 0 && lane == 0) {
    for (int s = 0; s < STAGES; ++s) mbar_init(smem_u32(&bars[s]), p.tma ? 1 : 32);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (D < DP && !p.tma && part == 0) {
    // chunks behind the rows' ends: read by the products (with zero queries),
    // never loaded
    for (int i = lane * 16; i < M::RING; i += 512)
      *reinterpret_cast<uint4 *>(sm.ring + i) = make_uint4(0u, 0u, 0u, 0u);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (p.tma && threadIdx.x == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&p.k_map) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&p.v_map) : "memory");
  }
  wait_for_prior_kernel();
  let_dependents_launch();
  const int rows = c.kv_heads * p.chunks;
  Walk<TOK> cur;
  uint32_t to_do, me = 0;
  if constexpr (ROW) {
    // this cluster's row, this block's part of it, a quarter of that per worker
    const int unit = int(blockIdx.x) / p.row_blocks, rank = int(blockIdx.x) - unit * p.row_blocks;
    cur.b = unit / rows;
    cur.row = unit - cur.b * rows;
    cur.s = span_of<TOK>(p, slots_in_use(p.a.lengths, cur.b, p.capacity, p.err));
    // (steps * blocks * workers is small: row mode is for short tables)
    const int lo = cur.s.steps * rank / p.row_blocks, hi = cur.s.steps * (rank + 1) / p.row_blocks;
    cur.step = lo + (hi - lo) * worker / PA_BLOCK_WORKERS;
    to_do = uint32_t(lo + (hi - lo) * (worker + 1) / PA_BLOCK_WORKERS - cur.step);
    if (part == 0 && lane < PA_HEADS) row_ml[worker][lane] = make_float2(-INFINITY, 0.f);
    __syncthreads();
  } else {
    build_prefix<TOK>(p, sm.prefix, sm.lens, p.scores != nullptr);  // (ends with a block barrier)
    const uint32_t total = sm.prefix[c.batch] * uint32_t(rows);
    const uint32_t workers = worker_count(p, total);
    me = uint32_t(worker) * gridDim.x + blockIdx.x;
    if (total == 0 || me >= workers) return;
    const Shares shares(total, workers);
    const uint32_t begin = shares.begin(me);
    cur.start(p, sm.prefix, sm.lens, rows, begin);
    to_do = shares.begin(me + 1) - begin;
  }
  Loader<T, DP, STAGES> loader;
  loader.to_load = 0;
  // the queries of the row at hand
  constexpr int QK = DP / M::WARPS / (L::kHalf ? 16 : 8);  // this warp's operand columns
  const int d0 = part * WP * PANEL;                        // and first channel
  uint32_t qf[M::kQShared ? 1 : QK][4];
  auto load_q = [&]() {
    const int h = cur.row / p.chunks, chunk = cur.row - h * p.chunks;
    const int nh = min(p.heads, p.group - chunk * PA_HEADS);
    const T *q = static_cast<const T *>(p.a.q) + int64_t(cur.b) * p.a.q_batch_stride +
                 int64_t(h * p.group + chunk * PA_HEADS) * p.a.q_head_stride;
    auto qv = [&](int g, int d) -> T {
      return (g < nh && d < D) ? q[int64_t(g) * p.a.q_head_stride + d] : T(0.f);
    };
    const int r0 = lane >> 2, kq = lane & 3;
    if constexpr (L::kHalf) {
#pragma unroll
      for (int kk = 0; kk < QK; ++kk)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int g = r0 + (j & 1) * 8, d = d0 + kk * 16 + 2 * kq + (j >> 1) * 8;
          if ((j & 1) && HALF_ROWS) {
            qf[kk][j] = 0u;
          } else if (p.q_pairs) {
            qf[kk][j] = g < nh && d < D ? *reinterpret_cast<const uint32_t *>(
                                              q + int64_t(g) * p.a.q_head_stride + d)
                                        : 0u;
          } else {
            const __half2 v = __half2(qv(g, d), qv(g, d + 1));
            qf[kk][j] = *reinterpret_cast<const uint32_t *>(&v);
          }
        }
    } else if constexpr (!M::kQShared) {
#pragma unroll
      for (int kk = 0; kk < QK; ++kk)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          qf[kk][j] = __float_as_uint(qv(r0 + (j & 1) * 8, d0 + kk * 8 + kq + (j >> 1) * 4));
    } else {
      // (this warp's channels; it alone reads them)
      __syncwarp();
      const uint32_t q_a = smem_u32(sm.extra);
      for (int g = 0; g < PA_HEADS; ++g)
        for (int d = d0 + lane; d < d0 + WP * PANEL; d += 32) {
          const bool in = g < nh && d < D;
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(
                           q_a + uint32_t(g * L::ROW + (((d / 4) ^ (g & 7)) << 4) + (d % 4) * 4)),
                       "l"(in ? q + int64_t(g) * p.a.q_head_stride + d : q), "r"(in ? 4 : 0)
                       : "memory");
        }
    }
  };
  if (to_do) {
    load_q();  // (in flight beside the first steps' page table entries)
    loader.start(p, cur, to_do, lane);
  }
#pragma unroll 1
  for (int s = 0; s < STAGES - 1; ++s) loader.next(p, sm.lens, rows, sm.ring, bars, s, lane, part == 0);

  float o[NT][4];
  const uint32_t ring_a = smem_u32(sm.ring);
  // Bytes of this lane's chunks within a panel of K and of V (L::at): the
  // permutation is an exclusive or, so a panel's four operand columns cost four
  // numbers, and panels are constant offsets.
  uint32_t kx[4], vx[L::kHalf ? 4 : 8];
  {
    uint32_t k0, v0, v1 = 0;
    if constexpr (L::kHalf) {
      const int kt = ((lane >> 4) << 3) + (lane & 7), vt = (((lane >> 3) & 1) << 3) + (lane & 7);
      k0 = uint32_t(kt * 128 + ((((lane >> 3) & 1) ^ (kt & 7)) << 4));
      v0 = uint32_t(vt * 128 + (((lane >> 4) ^ (vt & 7)) << 4));
    } else {
      const int kt = lane >> 2, vt = 2 * (lane & 3), in = ((lane >> 2) & 3) * 4;
      k0 = uint32_t(kt * 128 + (kt << 4) + (lane & 3) * 4);
      v0 = uint32_t(vt * 128 + (((lane >> 4) ^ vt) << 4) + in);
      v1 = uint32_t((vt + 1) * 128 + (((lane >> 4) ^ (vt + 1)) << 4) + in);
    }
    const uint32_t mine = uint32_t(part * WP * TOK * 128);  // this warp's panels
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      kx[i] = (k0 ^ uint32_t(32 * i)) + mine;
      vx[i] = (v0 ^ uint32_t(32 * i)) + mine;
      if constexpr (!L::kHalf) vx[4 + i] = (v1 ^ uint32_t(32 * i)) + mine;
    }
  }
  int stage = 0;
  uint32_t phase = 0;  // bit s: parity of stage s's next wait
  bool ok = true;

  while (to_do && ok) {
    const int h = cur.row / p.chunks, chunk = cur.row - h * p.chunks;
    const bool from_begin = cur.step == 0;  // this share holds the row's first step
    const int nh = min(p.heads, p.group - chunk * PA_HEADS);
    float m[HALVES], l[HALVES], high[L::kHalf ? HALVES : 1];
#pragma unroll
    for (int n = 0; n < NT; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
#pragma unroll
    for (int x = 0; x < HALVES; ++x) {
      m[x] = -INFINITY, l[x] = 0.f;
      if constexpr (L::kHalf) high[x] = -INFINITY;
    }
    if constexpr (M::kQShared) {
      asm volatile("cp.async.wait_all;" ::: "memory");
      __syncwarp();
    }
    const uint32_t here = min(uint32_t(cur.s.steps - cur.step), to_do);
    const bool whole = from_begin && cur.step + int(here) == cur.s.steps;
#pragma unroll 1
    for (uint32_t i = 0; i < here; ++i) {
      const uint32_t live = loader.oldest();
      if (live) {
        ok = mbar_wait(smem_u32(&bars[stage]), (phase >> stage) & 1);
        phase ^= 1u << stage;
      }
      // (also: the stage before this one is free)
      if (!worker_all(ok)) {
        if (lane == 0) atomicOr(p.err, kErrLoadTimeout);
        ok = false;
        break;
      }
      loader.next(p, sm.lens, rows, sm.ring, bars, stage == 0 ? STAGES - 1 : stage - 1, lane, part == 0);
      const uint32_t ka = ring_a + uint32_t(stage * L::STAGE), va = ka + uint32_t(TOK * L::ROW);
      stage = stage + 1 == STAGES ? 0 : stage + 1;
      if (!live && !p.scores) continue;
      if (live != L::FULL) clear_dead_rows<T, DP>(va, live, lane);
      // ---- scores: s[t][.] are slots t * 8 + 2 * (lane % 4) + {0, 1} of head
      // lane / 4 ([0], [1]) and lane / 4 + 8 ([2], [3])
      float s[ST][4];
#pragma unroll
      for (int t = 0; t < ST; ++t) s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.f;
      if constexpr (L::kHalf) {
        float s2[2][4] = {};  // odd columns: sums of their own, for the pipeline
#pragma unroll
        for (int pn = 0; pn < WP; ++pn) {
          if (d0 + pn * PANEL < D) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t b[4];
              ldsm4(ka + kx[i] + uint32_t(pn * TOK * 128), b);
              mma16(i & 1 ? s2[0] : s[0], qf[pn * 4 + i], b[0], b[1]);
              mma16(i & 1 ? s2[1] : s[ST - 1], qf[pn * 4 + i], b[2], b[3]);
            }
          }
        }
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 2 * HALVES; ++e) s[t % ST][e] += s2[t][e];
      } else {
        const int r = lane >> 2;
        // the tensor core cuts its running sums instead of rounding them: the
        // small products have sums of their own, and the large ones two
        float lo[4] = {}, lo2[4] = {}, odd[4] = {};
#pragma unroll
        for (int pn = 0; pn < WP; ++pn) {
          if (d0 + pn * PANEL < D) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int kk = pn * 4 + i;
              uint32_t ah[4], al[4], bh[2], bl[2];
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                if constexpr (M::kQShared) {
                  const int g = r + (j & 1) * 8;
                  const uint32_t qa = smem_u32(sm.extra) + uint32_t(g * L::ROW + ((g & 7) << 4) + (lane & 3) * 4);
                  split_tf32(lds32(qa ^ uint32_t((d0 / 4 + 2 * kk + (j >> 1)) << 4)), ah[j], al[j]);
                } else {
                  split_tf32(__uint_as_float(qf[kk][j]), ah[j], al[j]);
                }
              }
#pragma unroll
              for (int j = 0; j < 2; ++j)
                split_tf32(lds32((ka + kx[i] + uint32_t(pn * TOK * 128)) ^ uint32_t(16 * j)), bh[j], bl[j]);
              mma8(lo, al, bh[0], bh[1]);
              mma8(lo2, ah, bl[0], bl[1]);
              mma8(i & 1 ? odd : s[0], ah, bh[0], bh[1]);
            }
          }
        }
#pragma unroll
        for (int j = 0; j < 2 * HALVES; ++j) s[0][j] += odd[j] + (lo[j] + lo2[j]);
      }
      if constexpr (M::WARPS == 2) {
        // the other warp's half of the channels
#pragma unroll
        for (int t = 0; t < ST; ++t)
          halves[worker][part][t][lane] = make_float4(s[t][0], s[t][1], s[t][2], s[t][3]);
        worker_all(true);
#pragma unroll
        for (int t = 0; t < ST; ++t) {
          const float4 y = halves[worker][part ^ 1][t][lane];
          s[t][0] += y.x;
          s[t][1] += y.y;
          s[t][2] += y.z;
          s[t][3] += y.w;
        }
      }
      // ---- running softmax, base 2. The reference value m follows the
      // maximum only when that has grown by a few powers of two, so that the
      // result is rescaled a few times per row instead of at every new maximum
      // of any head. fp32: by more than 2^8.
      // fp16: the probabilities 2^(s - m) enter the product as fp16 numbers, with
      // 22 bits down to 2^-14 and none below 2^-25, so a step's largest has to
      // lie well inside fp16's range, also where it is far below the row's
      // maximum: a row of one dominant slot, whose value is near zero, has the
      // sum of all the small probabilities for a result. m is set 2^11 below a
      // step's maximum, up again when a later one is over 2^15 above it, down
      // when one is less than 2 above it: a step's probabilities are below 2^15
      // and keep 22 bits, or 2^-26 of its largest. Sums and results grow by
      // as much in fp32; 2^60 is the limit, beyond which a step no longer
      // counts. (Probabilities held relative to the row's maximum alone, below
      // 2^8, were off by 6 % at 2^-23 of it, and zero from 2^-26 on.)
#pragma unroll
      for (int t = 0; t < ST; ++t)
#pragma unroll
        for (int e = 0; e < 2 * HALVES; ++e) s[t][e] *= p.scale2;
      if (live != L::FULL) {
#pragma unroll
        for (int t = 0; t < ST; ++t)
#pragma unroll
          for (int e = 0; e < 2 * HALVES; ++e)
            if (!((live >> (t * 8 + 2 * (lane & 3) + (e & 1))) & 1)) s[t][e] = -INFINITY;
      }
      if (p.scores) {
        const int t0 = (cur.step + int(i)) * TOK + 2 * (lane & 3);
        if (part == 0) {
#pragma unroll
          for (int x = 0; x < HALVES; ++x) {
            const int g = (lane >> 2) + 8 * x;
            if (g < nh) {
              float *w = p.scores + (int64_t(cur.b) * p.a.q_heads + h * p.group + chunk * PA_HEADS + g) *
                                        p.score_stride + t0;
#pragma unroll
              for (int t = 0; t < ST; ++t)
                *reinterpret_cast<float2 *>(w + t * 8) = make_float2(s[t][2 * x], s[t][2 * x + 1]);
            }
          }
        }
        if (!live) continue;
      }
      // (false where neither has a score yet: the difference is NaN)
      auto out_of_range = [](float most, float ref) { return fabsf(most - ref - PA_MIDDLE) > PA_FAR; };
      bool far = false;
      float mx[HALVES];
#pragma unroll
      for (int x = 0; x < HALVES; ++x) {
        mx[x] = fmaxf(s[0][2 * x], s[0][2 * x + 1]);
        if constexpr (ST > 1) mx[x] = fmaxf(mx[x], fmaxf(s[1][2 * x], s[1][2 * x + 1]));
        mx[x] = fmaxf(mx[x], __shfl_xor_sync(~0u, mx[x], 1));
        mx[x] = fmaxf(mx[x], __shfl_xor_sync(~0u, mx[x], 2));
        if constexpr (L::kHalf) far |= out_of_range(mx[x], m[x]);
        else far |= mx[x] > m[x] + 8.f;
      }
      if (__any_sync(~0u, far)) {
#pragma unroll
        for (int x = 0; x < HALVES; ++x) {
          float mn = fmaxf(m[x], mx[x]);
          if constexpr (L::kHalf) {
            mn = out_of_range(mx[x], m[x]) ? fmaxf(mx[x] - PA_ABOVE, high[x] - PA_DEPTH) : m[x];
            high[x] = fmaxf(high[x], mn);
          }
          const float f = mn != m[x] ? exp2_approx(m[x] - mn) : 1.f;
          l[x] *= f;
          m[x] = mn;
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            o[n][2 * x] *= f;
            o[n][2 * x + 1] *= f;
          }
        }
      }
#pragma unroll
      for (int x = 0; x < HALVES; ++x) {
        const float mu = m[x] == -INFINITY ? 0.f : m[x];
#pragma unroll
        for (int t = 0; t < ST; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float &v = s[t][2 * x + e];
            v = exp2_approx(v - mu);
            l[x] += v;
          }
      }
      if (HALF_ROWS) {
#pragma unroll
        for (int t = 0; t < ST; ++t) s[t][2] = s[t][3] = 0.f;
      }
      // ---- result += p v
      if constexpr (L::kHalf) {
        // the probabilities go in as a sum of two fp16 numbers: one alone would
        // add an error as large as the output's own rounding
        uint32_t ph[4], pl[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int t = (j >> 1) * (ST - 1), x = j & 1;
          if (x && HALF_ROWS) {
            ph[j] = pl[j] = 0u;
            continue;
          }
          ph[j] = pack2(s[t][2 * x], s[t][2 * x + 1]);
          const float2 hf = __half22float2(*reinterpret_cast<const __half2 *>(&ph[j]));
          pl[j] = pack2(s[t][2 * x] - hf.x, s[t][2 * x + 1] - hf.y);
        }
#pragma unroll
        for (int pn = 0; pn < WP; ++pn) {
          if (d0 + pn * PANEL < D) {
            uint32_t b[4][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) ldsm4_t(va + vx[i] + uint32_t(pn * TOK * 128), b[i]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              mma16(o[pn * 8 + 2 * i], ph, b[i][0], b[i][1]);
              mma16(o[pn * 8 + 2 * i + 1], ph, b[i][2], b[i][3]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              mma16(o[pn * 8 + 2 * i], pl, b[i][0], b[i][1]);
              mma16(o[pn * 8 + 2 * i + 1], pl, b[i][2], b[i][3]);
            }
          }
        }
      } else {
        // the k index of the product runs over the slots in the order 0, 2, 4,
        // 6, 1, 3, 5, 7, which is how the scores' accumulator holds them
        uint32_t ah[4], al[4];
        split_tf32(s[0][0], ah[0], al[0]);
        split_tf32(s[0][2], ah[1], al[1]);
        split_tf32(s[0][1], ah[2], al[2]);
        split_tf32(s[0][3], ah[3], al[3]);
#pragma unroll
        for (int pn = 0; pn < WP; ++pn) {
          if (d0 + pn * PANEL < D) {
            uint32_t bh[4][2], bl[4][2];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int j = 0; j < 2; ++j)
                split_tf32(lds32(va + vx[4 * j + i] + uint32_t(pn * TOK * 128)), bh[i][j], bl[i][j]);
            // a sum of its own per step, added in fp32 with rounding: cut sums
            // drift over thousands of slots
            float acc[4][4] = {};
#pragma unroll
            for (int i = 0; i < 4; ++i) mma8(acc[i], al, bh[i][0], bh[i][1]);
#pragma unroll
            for (int i = 0; i < 4; ++i) mma8(acc[i], ah, bl[i][0], bl[i][1]);
#pragma unroll
            for (int i = 0; i < 4; ++i) mma8(acc[i], ah, bh[i][0], bh[i][1]);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int j = 0; j < 2 * HALVES; ++j) o[pn * 4 + i][j] += acc[i][j];
          }
        }
      }
    }
    to_do -= here;
    if (ROW) worker_all(true);  // (the ring becomes the result's place)
#pragma unroll
    for (int x = 0; x < HALVES; ++x) {
      float sum = l[x];
      sum += __shfl_xor_sync(~0u, sum, 1);
      sum += __shfl_xor_sync(~0u, sum, 2);
      const int g = (lane >> 2) + 8 * x;
      if (g >= nh || !ok) continue;
      if (ROW) {
        float *ro = reinterpret_cast<float *>(sm.ring) + g * DP;
#pragma unroll
        for (int n = 0; n < NT; ++n)
          *reinterpret_cast<float2 *>(ro + d0 + n * 8 + 2 * (lane & 3)) = make_float2(o[n][2 * x], o[n][2 * x + 1]);
        if (part == 0 && (lane & 3) == 0) row_ml[worker][g] = make_float2(m[x], sum);
      } else if (whole) {
        const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
        T *out = static_cast<T *>(p.a.out) + int64_t(cur.b) * p.a.out_batch_stride +
                 int64_t(h * p.group + chunk * PA_HEADS + g) * p.a.out_head_stride;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int d = d0 + n * 8 + 2 * (lane & 3) + e;
            if (d < D) out[d] = T(o[n][2 * x + e] * inv);
          }
        if (p.stats && part == 0 && (lane & 3) == 0)
          p.stats[(int64_t(cur.b) * rows + cur.row) * PA_HEADS + g] = make_float2(m[x], sum);
      } else {
        const int64_t at = (int64_t(me) * 2 + (from_begin ? 1 : 0)) * p.heads + g;
        float *po = p.part_o + at * p.part_stride;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int d = d0 + n * 8 + 2 * (lane & 3) + e;
            if (d < D) po[d] = o[n][2 * x + e];
          }
        if (part == 0 && (lane & 3) == 0) p.part_ml[at] = make_float2(m[x], sum);
      }
    }
    if (ROW || !to_do) break;
    cur.next_row(p, sm.lens, rows);
    load_q();
  }
  if (!ok) drain<STAGES>(loader.live_ring, bars, stage, phase);
  if constexpr (ROW) {
    uint8_t *rings = sm.ring - size_t(worker) * M::RING;
    if (p.row_blocks == 1) finish_row<T, TOK, false>(p, cur.b, cur.row, cur.s, row_ml, rings, M::RING, DP);
    else finish_row<T, TOK, true>(p, cur.b, cur.row, cur.s, row_ml, rings, M::RING, DP);
  }
}

// CUDA-core form for fp32 caches and groups of at most 8 heads (G: the group
// rounded up to 1, 2, 4, 8): 2 * G multiply-adds per cached element, exact
// products. On the tensor cores a step of 8 slots costs the same whatever the
// group (about 450 instructions, most of them the operands' splitting); here
// about 100 and 64 * G more at 128 channels. 12 sequences of 129-2001 slots x 5
// heads x 80 channels, 2 query heads each: a call takes 32.4 us on the tensor
// cores, 22.4 here (34 MB; the rest is latency: six or seven steps per worker,
// whose masks are fetched one step ahead). 116 sequences x 2 heads x
// 128 channels, 762-1525 slots: 52 us a call, 5.2 TB/s.
template <int DP, int G>
struct SimtShape {
  static constexpr int STAGES = DP > 128 && G > 2 ? 2 : Tile<float, DP>::STAGE > 4096 ? 3 : 4;
  static constexpr int QBYTES = G * DP * 4;
  static constexpr int PBYTES = 8 * G * 4;
  static constexpr int RING = STAGES * Tile<float, DP>::STAGE, EXTRA = QBYTES + PBYTES;
  static constexpr int THREADS = PA_BLOCK_WORKERS * 32;
  static_assert(PA_BLOCK_WORKERS * (RING + EXTRA) + 1024 + (2 * 2048 + 1) * 4 + 2 * 1024 <= 227 * 1024, "shared memory of a block");
};

__device__ __forceinline__ float4 lds128(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

template <int DP, int G, bool ROW>
__global__ void __launch_bounds__(SimtShape<DP, G>::THREADS)
    paged_attention_simt_kernel(const __grid_constant__ AttnArgs p) {
  using L = Tile<float, DP>;
  using M = SimtShape<DP, G>;
  constexpr int TOK = 8, STAGES = M::STAGES, CHUNKS = DP / 4;
  constexpr int LANES = CHUNKS < 32 ? CHUNKS : 32;  // lanes over a row of V
  constexpr int SPLIT = 32 / LANES;                 // slots at a time
  constexpr int OV = CHUNKS / LANES;                // chunks of the result per lane
  extern __shared__ uint8_t pa_smem_raw[];
  __shared__ __align__(8) uint64_t all_bars[PA_BLOCK_WORKERS][STAGES];
  __shared__ float2 row_ml[PA_BLOCK_WORKERS][PA_HEADS];
  const wgx_kv_cache &c = p.a.cache;
  const int lane = threadIdx.x % 32, worker = threadIdx.x / 32;
  const BlockSmem sm = block_smem(pa_smem_raw, worker, M::RING, M::EXTRA, PA_BLOCK_WORKERS, c.batch);
  uint64_t *bars = all_bars[worker];
  const int D = c.head_dim;
  if (lane == 0) {
    for (int s = 0; s < STAGES; ++s) mbar_init(smem_u32(&bars[s]), p.tma ? 1 : 32);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (D < DP && !p.tma) {
    // chunks behind the rows' ends are read but never loaded
    for (int i = lane * 16; i < M::RING; i += 512)
      *reinterpret_cast<uint4 *>(sm.ring + i) = make_uint4(0u, 0u, 0u, 0u);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (p.tma && threadIdx.x == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&p.k_map) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&p.v_map) : "memory");
  }
  wait_for_prior_kernel();
  let_dependents_launch();
  const int rows = c.kv_heads;  // (p.chunks is 1)
  Walk<TOK> cur;
  uint32_t to_do, me = 0;
  if constexpr (ROW) {
    // this cluster's row, this block's part of it, a quarter of that per worker
    const int unit = int(blockIdx.x) / p.row_blocks, rank = int(blockIdx.x) - unit * p.row_blocks;
    cur.b = unit / rows;
    cur.row = unit - cur.b * rows;
    cur.s = span_of<TOK>(p, slots_in_use(p.a.lengths, cur.b, p.capacity, p.err));
    // (steps * blocks * workers is small: row mode is for short tables)
    const int lo = cur.s.steps * rank / p.row_blocks, hi = cur.s.steps * (rank + 1) / p.row_blocks;
    cur.step = lo + (hi - lo) * worker / PA_BLOCK_WORKERS;
    to_do = uint32_t(lo + (hi - lo) * (worker + 1) / PA_BLOCK_WORKERS - cur.step);
    if (lane < PA_HEADS) row_ml[worker][lane] = make_float2(-INFINITY, 0.f);
    __syncthreads();
  } else {
    build_prefix<TOK>(p, sm.prefix, sm.lens, p.scores != nullptr);  // (ends with a block barrier)
    const uint32_t total = sm.prefix[c.batch] * uint32_t(rows);
    const uint32_t workers = worker_count(p, total);
    me = uint32_t(worker) * gridDim.x + blockIdx.x;
    if (total == 0 || me >= workers) return;
    const Shares shares(total, workers);
    const uint32_t begin = shares.begin(me);
    cur.start(p, sm.prefix, sm.lens, rows, begin);
    to_do = shares.begin(me + 1) - begin;
  }
  Loader<float, DP, STAGES> loader;
  loader.to_load = 0;
  const uint32_t ring_a = smem_u32(sm.ring);
  const uint32_t q_a = smem_u32(sm.extra);              // [head][channel]
  const uint32_t p_a = q_a + uint32_t(M::QBYTES);             // [slot][head]
  float *p_s = reinterpret_cast<float *>(sm.extra + M::QBYTES);
  // the queries of the row at hand, zeros behind the group and the channels
  auto load_q = [&]() {
    const float *q = static_cast<const float *>(p.a.q) + int64_t(cur.b) * p.a.q_batch_stride +
                     int64_t(cur.row) * p.group * p.a.q_head_stride;
    __syncwarp();
#pragma unroll
    for (int g = 0; g < G; ++g)
      for (int d = lane; d < DP; d += 32) {
        const bool in = g < p.group && d < D;
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(q_a + uint32_t((g * DP + d) * 4)),
                     "l"(in ? q + int64_t(g) * p.a.q_head_stride + d : q), "r"(in ? 4 : 0)
                     : "memory");
      }
  };
  if (to_do) {
    load_q();  // (in flight beside the first steps' page table entries)
    loader.start(p, cur, to_do, lane);
  }
#pragma unroll 1
  for (int s = 0; s < STAGES - 1; ++s) loader.next(p, sm.lens, rows, sm.ring, bars, s, lane, true);

  // scores: lane = quarter * 8 + slot, chunks 4 * i + quarter of the slot's row
  const int ks = lane & 7, quarter = lane >> 3;
  const uint32_t k0 = uint32_t(ks * 128 + ((quarter ^ ks) << 4));
  // result: lane = half * LANES + chunk, slots SPLIT * j + half
  const int vc = lane % LANES, half = lane / LANES;
  int stage = 0;
  uint32_t phase = 0;
  bool ok = true;

  while (to_do && ok) {
    const int h = cur.row;
    const bool from_begin = cur.step == 0;
    const int nh = p.group;
    float m[G], l[G];
    float4 o[OV][G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      m[g] = -INFINITY;
      l[g] = 0.f;
#pragma unroll
      for (int k = 0; k < OV; ++k) o[k][g] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();
    const uint32_t here = min(uint32_t(cur.s.steps - cur.step), to_do);
#pragma unroll 1
    for (uint32_t i = 0; i < here; ++i) {
      const uint32_t live = loader.oldest();
      if (live) {
        ok = mbar_wait(smem_u32(&bars[stage]), (phase >> stage) & 1);
        phase ^= 1u << stage;
      }
      // (also: the stage before this one is free)
      if (!__all_sync(~0u, ok)) {
        if (lane == 0) atomicOr(p.err, kErrLoadTimeout);
        ok = false;
        break;
      }
      loader.next(p, sm.lens, rows, sm.ring, bars, stage == 0 ? STAGES - 1 : stage - 1, lane, true);
      const uint32_t ka = ring_a + uint32_t(stage * L::STAGE), va = ka + uint32_t(TOK * L::ROW);
      stage = stage + 1 == STAGES ? 0 : stage + 1;
      if (!live && !p.scores) continue;
      if (live != L::FULL) clear_dead_rows<float, DP>(va, live, lane);
      // ---- scores of this lane's slot, a quarter of the channels each
      float s[G];
#pragma unroll
      for (int g = 0; g < G; ++g) s[g] = 0.f;
#pragma unroll
      for (int pn = 0; pn < L::PANELS; ++pn) {
        if (pn * L::PANEL < D) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float4 k = lds128(ka + uint32_t(pn * TOK * 128) + (k0 ^ uint32_t(64 * e)));
            const uint32_t qc = q_a + uint32_t((pn * 8 + e * 4 + quarter) * 16);
#pragma unroll
            for (int g = 0; g < G; ++g) {
              const float4 q = lds128(qc + uint32_t(g * DP * 4));
              s[g] = fmaf(k.x, q.x, s[g]);
              s[g] = fmaf(k.y, q.y, s[g]);
              s[g] = fmaf(k.z, q.z, s[g]);
              s[g] = fmaf(k.w, q.w, s[g]);
            }
          }
        }
      }
      const bool on = (live >> ks) & 1;
      bool grew = false;
      float mx[G];
#pragma unroll
      for (int g = 0; g < G; ++g) {
        s[g] += __shfl_xor_sync(~0u, s[g], 8);
        s[g] += __shfl_xor_sync(~0u, s[g], 16);
        s[g] = on ? s[g] * p.scale2 : -INFINITY;
        mx[g] = fmaxf(s[g], __shfl_xor_sync(~0u, s[g], 1));
        mx[g] = fmaxf(mx[g], __shfl_xor_sync(~0u, mx[g], 2));
        mx[g] = fmaxf(mx[g], __shfl_xor_sync(~0u, mx[g], 4));
        grew |= mx[g] > m[g] + 8.f;
      }
      if (p.scores) {
        if (quarter == 0) {
          float *w = p.scores + (int64_t(cur.b) * p.a.q_heads + h * nh) * p.score_stride +
                     (cur.step + int(i)) * TOK + ks;
          for (int g = 0; g < G; ++g)
            if (g < nh) w[int64_t(g) * p.score_stride] = s[g];
        }
        if (!live) continue;
      }
      // ---- running softmax (see paged_attention_kernel)
      if (grew) {  // (the same in every lane)
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const float mn = fmaxf(m[g], mx[g]);
          const float f = mn > m[g] ? exp2_approx(m[g] - mn) : 1.f;
          l[g] *= f;
          m[g] = mn;
#pragma unroll
          for (int k = 0; k < OV; ++k) {
            o[k][g].x *= f;
            o[k][g].y *= f;
            o[k][g].z *= f;
            o[k][g].w *= f;
          }
        }
      }
#pragma unroll
      for (int g = 0; g < G; ++g) {
        s[g] = exp2_approx(s[g] - (m[g] == -INFINITY ? 0.f : m[g]));
        l[g] += s[g];
        if (quarter == 0) p_s[ks * G + g] = s[g];
      }
      __syncwarp();
      // ---- result += p v
#pragma unroll
      for (int j = 0; j < TOK / SPLIT; ++j) {
        const int t = j * SPLIT + half;
        float pg[G];
        if constexpr (G >= 4) {
#pragma unroll
          for (int g = 0; g < G; g += 4) {
            const float4 y = lds128(p_a + uint32_t((t * G + g) * 4));
            pg[g] = y.x;
            pg[g + 1] = y.y;
            pg[g + 2] = y.z;
            pg[g + 3] = y.w;
          }
        } else {
#pragma unroll
          for (int g = 0; g < G; ++g) pg[g] = lds32(p_a + uint32_t((t * G + g) * 4));
        }
#pragma unroll
        for (int k = 0; k < OV; ++k) {
          if ((vc + 32 * k) * 4 < D) {
            const float4 v = lds128(va + L::at(t, vc + 32 * k));
#pragma unroll
            for (int g = 0; g < G; ++g) {
              o[k][g].x = fmaf(pg[g], v.x, o[k][g].x);
              o[k][g].y = fmaf(pg[g], v.y, o[k][g].y);
              o[k][g].z = fmaf(pg[g], v.z, o[k][g].z);
              o[k][g].w = fmaf(pg[g], v.w, o[k][g].w);
            }
          }
        }
      }
    }
    to_do -= here;
    const bool whole = from_begin && cur.step + int(here) == cur.s.steps;
    if (ROW) __syncwarp();  // (the ring becomes the result's place)
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float sum = l[g];
      sum += __shfl_xor_sync(~0u, sum, 1);
      sum += __shfl_xor_sync(~0u, sum, 2);
      sum += __shfl_xor_sync(~0u, sum, 4);
      if constexpr (SPLIT == 2) {
        o[0][g].x += __shfl_xor_sync(~0u, o[0][g].x, 16);
        o[0][g].y += __shfl_xor_sync(~0u, o[0][g].y, 16);
        o[0][g].z += __shfl_xor_sync(~0u, o[0][g].z, 16);
        o[0][g].w += __shfl_xor_sync(~0u, o[0][g].w, 16);
      }
      if (g >= nh || !ok) continue;
      const int64_t at = (int64_t(me) * 2 + (from_begin ? 1 : 0)) * p.heads + g;
      const float inv = ROW || !whole ? 1.f : sum > 0.f || sum != sum ? 1.f / sum : 0.f;
      float *to = ROW ? reinterpret_cast<float *>(sm.ring) + g * DP
                  : whole ? static_cast<float *>(p.a.out) + int64_t(cur.b) * p.a.out_batch_stride +
                              int64_t(h * nh + g) * p.a.out_head_stride
                        : p.part_o + at * p.part_stride;
      if (half == 0) {
#pragma unroll
        for (int k = 0; k < OV; ++k) {
          const int d = (vc + 32 * k) * 4;
          if (d < D) to[d] = o[k][g].x * inv;
          if (d + 1 < D) to[d + 1] = o[k][g].y * inv;
          if (d + 2 < D) to[d + 2] = o[k][g].z * inv;
          if (d + 3 < D) to[d + 3] = o[k][g].w * inv;
        }
      }
      if (lane == 0) {
        if (ROW) row_ml[worker][g] = make_float2(m[g], sum);
        else if (!whole) p.part_ml[at] = make_float2(m[g], sum);
        else if (p.stats) p.stats[(int64_t(cur.b) * rows + cur.row) * PA_HEADS + g] = make_float2(m[g], sum);
      }
    }
    if (ROW || !to_do) break;
    cur.next_row(p, sm.lens, rows);
    load_q();
  }
  if (!ok) drain<STAGES>(loader.live_ring, bars, stage, phase);
  if constexpr (ROW) {
    uint8_t *rings = sm.ring - size_t(worker) * M::RING;
    if (p.row_blocks == 1) finish_row<float, TOK, false>(p, cur.b, cur.row, cur.s, row_ml, rings, M::RING, DP);
    else finish_row<float, TOK, true>(p, cur.b, cur.row, cur.s, row_ml, rings, M::RING, DP);
  }
}

// Rows cut between workers: out = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i.
// Blocks below o_blocks join query heads, join_warps warps each (one where a
// row has few partial results, the whole block for a lone long row that most
// of the grid worked on); the others add the probabilities of PA_JOIN_SLOTS
// slots of a K/V head to its weights. Where the rows lie in the line of work
// was left in scratch by the attention.
// KQ: groups of 128 channels.
template <typename T, int TOK, int KQ>
__global__ void __launch_bounds__(PA_JOIN_THREADS) join_kernel(const __grid_constant__ AttnArgs p) {
  constexpr int WARPS = PA_JOIN_THREADS / 32, FLIGHT = 8;
  extern __shared__ __align__(16) uint8_t jn_smem[];
  __shared__ float head_m[PA_MAX_GROUP], head_inv[PA_MAX_GROUP];
  __shared__ __align__(16) float sums[WARPS][128 * KQ];
  const wgx_kv_cache &c = p.a.cache;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int rows = c.kv_heads * p.chunks, D = c.head_dim;

  // the workers that worked on row (h, chunk) of b
  auto locate = [&](const uint32_t *prefix, int b, int h, int chunk, const Span &s, int &w0, int &w1) {
    const uint32_t total = prefix[c.batch] * uint32_t(rows);
    const Shares shares(total, worker_count(p, total));
    const uint32_t r0 = prefix[b] * uint32_t(rows) + uint32_t(h * p.chunks + chunk) * uint32_t(s.steps);
    w0 = int(shares.of(r0));
    w1 = int(shares.of(r0 + uint32_t(s.steps) - 1));
  };
  // row `g` of worker w0 + i's partial result of a row: the first worker began
  // the row, the others were in it when their shares began
  auto part_of = [&](int w0, int i, int g) { return (int64_t(w0 + i) * 2 + (i == 0 ? 1 : 0)) * p.heads + g; };
  // (maximum, sum) of head g's n partial results; all lanes get them
  auto stats_of = [&](int w0, int n, int g) {
    float M = -INFINITY, sum = 0.f;
    for (int i = lane; i < n; i += 32) M = fmaxf(M, p.part_ml[part_of(w0, i, g)].x);
    M = warp_max(M);
    const float mu = M == -INFINITY ? 0.f : M;
    for (int i = lane; i < n; i += 32) {
      const float2 ml = p.part_ml[part_of(w0, i, g)];
      sum += ml.y * exp2_approx(ml.x - mu);
    }
    return make_float2(mu, warp_sum(sum));
  };

  if (int(blockIdx.x) < p.o_blocks) {
    // (all of this from the call's inputs, while the attention ends)
    uint32_t *prefix = reinterpret_cast<uint32_t *>(jn_smem);
    int *lens = reinterpret_cast<int *>(prefix + c.batch + 1);
    build_prefix<TOK>(p, prefix, lens, false);
    const int per = p.join_warps, sub = warp % per;
    const int unit = blockIdx.x * (WARPS / per) + warp / per;
    const bool real = unit < c.batch * p.a.q_heads;
    const int b = real ? unit / p.a.q_heads : 0, i = unit - b * p.a.q_heads;
    const int h = i / p.group, gi = i - h * p.group, chunk = gi / PA_HEADS, g = gi % PA_HEADS;
    const Span s = span_of<TOK>(p, lens[b]);
    T *out = static_cast<T *>(p.a.out) + int64_t(b) * p.a.out_batch_stride + int64_t(i) * p.a.out_head_stride;
    int w0 = 0, w1 = 0;
    if (real && s.steps > 0) locate(prefix, b, h, chunk, s, w0, w1);
    const bool split = w0 != w1;
    float4 acc[KQ] = {};
    float inv = 0.f;
    const int quads = (D + 3) / 4;
    int at_quad[KQ];  // (lanes behind the row's end repeat its last four channels)
#pragma unroll
    for (int k = 0; k < KQ; ++k) at_quad[k] = min(lane + 32 * k, quads - 1);
    wait_for_prior_kernel();
    let_dependents_launch();
    if (split) {
      const int n = w1 - w0 + 1;
      const float2 st = stats_of(w0, n, g);
      inv = st.y > 0.f || st.y != st.y ? 1.f / st.y : 0.f;
      for (int base = sub; base < n; base += 32 * per) {
        const int mine = base + lane * per;
        const float f = mine < n ? exp2_approx(p.part_ml[part_of(w0, mine, g)].x - st.x) : 0.f;
        const int cnt = min(32, (n - base + per - 1) / per);
        for (int j0 = 0; j0 < cnt; j0 += FLIGHT) {
          float4 v[FLIGHT][KQ];
#pragma unroll
          for (int j = 0; j < FLIGHT; ++j) {
            const float4 *po = reinterpret_cast<const float4 *>(
                p.part_o + part_of(w0, base + min(j0 + j, cnt - 1) * per, g) * p.part_stride);
#pragma unroll
            for (int k = 0; k < KQ; ++k) v[j][k] = po[at_quad[k]];
          }
#pragma unroll
          for (int j = 0; j < FLIGHT; ++j) {
            const float fj = __shfl_sync(~0u, f, j0 + j);  // (zero behind the last)
            if (j0 + j < cnt) {
#pragma unroll
              for (int k = 0; k < KQ; ++k) {
                acc[k].x += fj * v[j][k].x;
                acc[k].y += fj * v[j][k].y;
                acc[k].z += fj * v[j][k].z;
                acc[k].w += fj * v[j][k].w;
              }
            }
          }
        }
      }
    }
    if (per > 1) {
#pragma unroll
      for (int k = 0; k < KQ; ++k)
        if (lane + 32 * k < quads) *reinterpret_cast<float4 *>(&sums[warp][4 * (lane + 32 * k)]) = acc[k];
      __syncthreads();
      if (sub) return;
      for (int w = 1; w < per; ++w)
#pragma unroll
        for (int k = 0; k < KQ; ++k)
          if (lane + 32 * k < quads) {
            const float4 v = *reinterpret_cast<const float4 *>(&sums[warp + w][4 * (lane + 32 * k)]);
            acc[k].x += v.x;
            acc[k].y += v.y;
            acc[k].z += v.z;
            acc[k].w += v.w;
          }
    }
    if (!real || (s.steps > 0 && !split)) return;
#pragma unroll
    for (int k = 0; k < KQ; ++k) {
      const int d = 4 * (lane + 32 * k);
      if (d < D) out[d] = T(acc[k].x * inv);
      if (d + 1 < D) out[d + 1] = T(acc[k].y * inv);
      if (d + 2 < D) out[d + 2] = T(acc[k].z * inv);
      if (d + 3 < D) out[d + 3] = T(acc[k].w * inv);
    }
    return;
  }

  const int at_row = (int(blockIdx.x) - p.o_blocks) % (c.batch * c.kv_heads);
  const int slice = (int(blockIdx.x) - p.o_blocks) / (c.batch * c.kv_heads) * PA_JOIN_SLOTS;
  const int b = at_row / c.kv_heads, h = at_row % c.kv_heads;
  const Span s = span_of<TOK>(p, slots_in_use(p.a.lengths, b, p.capacity, p.err));
  // (in place, slots in front of the window stay; first * TOK keeps quads aligned)
  const int t0 = p.a.weights == p.a.weights_out ? max(slice, s.first * TOK) : slice;
  const int t1 = min(slice + PA_JOIN_SLOTS, int(min(int64_t(s.len), p.a.slots)));
  if (t0 >= t1) return;
  wait_for_prior_kernel();
  let_dependents_launch();
  bool odd = false;  // a head without probabilities that are numbers
  for (int g = warp; g < p.group; g += WARPS) {
    const int chunk = g / PA_HEADS, gr = g % PA_HEADS;
    int w0, w1;
    locate(p.prefix, b, h, chunk, s, w0, w1);
    float2 st;
    if (w0 == w1) {
      st = p.stats[(int64_t(b) * rows + h * p.chunks + chunk) * PA_HEADS + gr];
      if (st.x == -INFINITY) st.x = 0.f;
    } else {
      st = stats_of(w0, w1 - w0 + 1, gr);
    }
    odd |= st.y != st.y;
    if (lane == 0) {
      head_m[g] = st.x;
      head_inv[g] = st.y > 0.f || st.y != st.y ? 1.f / st.y : 0.f;
    }
  }
  odd = __syncthreads_or(odd);
  const int64_t at = int64_t(at_row) * p.a.slots;
  const float *sc = p.scores + (int64_t(b) * p.a.q_heads + h * p.group) * p.score_stride;
  auto one = [&](int t) {
    float w = p.a.weights[at + t];
    // (slots in front of the window have scores of -infinity)
    if (t >= s.first * TOK && (!odd || slot_is_live(p, b, s, t)))
      for (int g = 0; g < p.group; ++g)
        w += exp2_approx(sc[int64_t(g) * p.score_stride + (t - s.first * TOK)] - head_m[g]) * head_inv[g];
    p.a.weights_out[at + t] = w;
  };
  int t = t0 + 4 * tid;
  if (p.weights_quads && !odd) {
    // four slots of four heads at a time (2^(-infinity) times a number is zero)
    for (; t + 4 <= t1; t += 4 * PA_JOIN_THREADS) {
      float4 w = *reinterpret_cast<const float4 *>(p.a.weights + at + t);
      if (t >= s.first * TOK) {
#pragma unroll 4
        for (int g = 0; g < p.group; ++g) {
          const float4 x = __ldcs(reinterpret_cast<const float4 *>(sc + int64_t(g) * p.score_stride + (t - s.first * TOK)));
          const float m = head_m[g], inv = head_inv[g];
          w.x += exp2_approx(x.x - m) * inv;
          w.y += exp2_approx(x.y - m) * inv;
          w.z += exp2_approx(x.z - m) * inv;
          w.w += exp2_approx(x.w - m) * inv;
        }
      }
      *reinterpret_cast<float4 *>(p.a.weights_out + at + t) = w;
    }
    // (the row's last one to three slots: t is theirs in one thread)
    for (; t < t1; ++t) one(t);
  } else {
    for (t = t0 + tid; t < t1; t += PA_JOIN_THREADS) one(t);
  }
}

struct Config {
  void (*kernel)(AttnArgs), (*row_kernel)(AttnArgs);  // shares of the line; row mode
  int ring, tok, threads, ctas_per_sm;
};

template <typename T, int DP, bool HALF_ROWS>
Config mma_config() {
  Config c{};
  c.kernel = paged_attention_kernel<T, DP, HALF_ROWS, false>;
  c.row_kernel = paged_attention_kernel<T, DP, HALF_ROWS, true>;
  c.ring = PA_BLOCK_WORKERS * (MmaShape<T, DP>::RING + MmaShape<T, DP>::EXTRA) + 1024;  // + alignment
  c.tok = Tile<T, DP>::TOK;
  c.threads = MmaShape<T, DP>::THREADS;
  return c;
}
template <int DP, int G>
Config simt_config() {
  Config c{};
  c.kernel = paged_attention_simt_kernel<DP, G, false>;
  c.row_kernel = paged_attention_simt_kernel<DP, G, true>;
  c.ring = PA_BLOCK_WORKERS * (SimtShape<DP, G>::RING + SimtShape<DP, G>::EXTRA) + 1024;
  c.tok = 8;
  c.threads = SimtShape<DP, G>::THREADS;
  return c;
}
template <int DP>
Config config_of(int dtype, int heads) {
  if (dtype == WGX_FLOAT16) return heads <= 8 ? mma_config<__half, DP, true>() : mma_config<__half, DP, false>();
  if (heads <= 1) return simt_config<DP, 1>();
  if (heads <= 2) return simt_config<DP, 2>();
  if (heads <= 4) return simt_config<DP, 4>();
  if (heads <= 8) return simt_config<DP, 8>();
  return mma_config<float, DP, false>();
}

constexpr int kPaMaxBatch = 2048;
inline int prefix_bytes(int batch) { return (2 * batch + 1) * 4; }

// The kernel for a call's type, head size and group; its attributes are set
// and its occupancy read once per device.
const Config &config_for(int dtype, int head_dim, int heads) {
  static std::mutex mu;
  static Config table[64][2][3][5];
  static bool ready[64][2][3][5] = {};
  const int dev = current_device();
  if (dev >= 64) fail("paged_attention: device ordinal out of range");
  const int dt = dtype == WGX_FLOAT16, dp = head_dim <= 64 ? 0 : head_dim <= 128 ? 1 : 2;
  const int hk = heads <= 1 ? 0 : heads <= 2 ? 1 : heads <= 4 ? 2 : heads <= 8 ? 3 : 4;
  std::lock_guard<std::mutex> lock(mu);
  if (!ready[dev][dt][dp][hk]) {
    Config c = dp == 0 ? config_of<64>(dtype, heads)
                       : dp == 1 ? config_of<128>(dtype, heads) : config_of<256>(dtype, heads);
    for (auto *kernel : {c.kernel, c.row_kernel})
      check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      c.ring + prefix_bytes(kPaMaxBatch)),
                 "paged_attention smem attr");
    check_cuda(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&c.ctas_per_sm, c.kernel, c.threads,
                                                             c.ring + prefix_bytes(256)),
               "paged_attention occupancy");
    if (c.ctas_per_sm < 1) c.ctas_per_sm = 1;
    table[dev][dt][dp][hk] = c;
    ready[dev][dt][dp][hk] = true;
  }
  return table[dev][dt][dp][hk];
}

struct Layout {
  AttnArgs p;
  int grid;
  const Config *cfg;
  uint64_t bytes;
};

Layout layout_of(const wgx_paged_attention_args &a, bool for_launch) {
  Layout l{};
  AttnArgs &p = l.p;
  const wgx_kv_cache &c = a.cache;
  p.a = a;
  p.capacity = cache_capacity(c);
  p.group = a.q_heads / c.kv_heads;
  p.chunks = (p.group + PA_HEADS - 1) / PA_HEADS;
  p.heads = std::min(p.group, PA_HEADS);
  p.vec = cache_rows_16b(c);
  const int es = dtype_size(c.dtype);
  p.q_pairs = c.dtype == WGX_FLOAT16 && c.head_dim % 2 == 0 && a.q_batch_stride % 2 == 0 &&
              a.q_head_stride % 2 == 0 && (reinterpret_cast<uintptr_t>(a.q) & 3) == 0;
  p.scale2 = a.scale * 1.4426950408889634f;
  l.cfg = &config_for(c.dtype, c.head_dim, p.heads);
  // TMA: a step's rows must lie in one page. Rows of whole 128-byte panels move
  // as one box per operand, others panel by panel with zeros behind the row.
  if (for_launch && p.vec && c.page_size % l.cfg->tok == 0) {
    const int panel = 128 / es, panels = c.head_dim % panel == 0 ? c.head_dim / panel : 1;
    p.boxes = panels * panel == c.head_dim ? 1 : (c.head_dim + panel - 1) / panel;
    p.tma = encode_rows_tmap(&p.k_map, c.k, c, c.k_page_stride, c.k_head_stride, c.k_slot_stride, panels, l.cfg->tok) &&
            encode_rows_tmap(&p.v_map, c.v, c, c.v_page_stride, c.v_head_stride, c.v_slot_stride, panels, l.cfg->tok);
  }
  const int64_t rows = int64_t(c.batch) * c.kv_heads * p.chunks;
  // steps a row can have: of the table's slots, or of the window (which may
  // begin inside a step)
  int64_t row_steps = (p.capacity + l.cfg->tok - 1) / l.cfg->tok;
  if (a.window > 0) row_steps = std::min<int64_t>(row_steps, (int64_t(a.window) + l.cfg->tok - 1) / l.cfg->tok + 1);
  // Row mode where a row's table is short (see the constants). Blocks that share
  // a K/V head's weights cannot accumulate them (chunks > 1), and one block would
  // be long copying the weights in front of a window.
  const int per = c.head_dim > 128 ? PA_ROW_STEPS / 4 : l.cfg->tok == 16 ? PA_ROW_STEPS : PA_ROW_STEPS / 2;
  if (!a.weights_out || (p.chunks == 1 && (a.weights == a.weights_out || p.capacity <= 4 * per * l.cfg->tok))) {
    const int64_t room = int64_t(device_sm_count()) * l.cfg->ctas_per_sm;
    if (row_steps <= per) p.row_blocks = 1;
    else if (rows >= PA_ROW_MIN && rows * 4 <= room && row_steps <= 4 * per) p.row_blocks = 4;
    else if (rows >= PA_ROW_MIN && rows * 2 <= room && row_steps <= 2 * per) p.row_blocks = 2;
  }
  p.min_steps = 1;
  const uint64_t steps = uint64_t(row_steps) * uint64_t(rows);
  if (steps >= uint64_t(1) << 31) fail("paged_attention: too many slots");
  const int resident = device_sm_count() * l.cfg->ctas_per_sm;
  p.max_workers = int(std::min<uint64_t>(std::max<uint64_t>(steps, 1), uint64_t(resident) * PA_BLOCK_WORKERS));
  l.grid = p.row_blocks ? int(rows) * p.row_blocks : std::min(resident, p.max_workers);
  uint64_t off = 0;
  const uint64_t parts = p.row_blocks ? 0 : uint64_t(p.max_workers) * 2 * p.heads;
  auto take = [&](uint64_t bytes) {
    const uint64_t at = off;
    off += align256(bytes);
    return static_cast<uint8_t *>(a.scratch) + at;
  };
  p.part_stride = (c.head_dim + 3) / 4 * 4;
  p.part_o = reinterpret_cast<float *>(take(parts * p.part_stride * 4));
  p.part_ml = reinterpret_cast<float2 *>(take(parts * 8));
  p.prefix = reinterpret_cast<uint32_t *>(take((uint64_t(c.batch) + 1) * 4));
  // warps per head of the join, by the partial results a row can have when the
  // rows are alike
  const int64_t expect = p.max_workers / (int64_t(c.batch) * c.kv_heads * p.chunks);
  p.join_warps = expect > 64 ? 8 : expect > 32 ? 4 : expect > 16 ? 2 : 1;
  const int per_block = PA_JOIN_THREADS / 32 / p.join_warps;
  p.o_blocks = int((int64_t(c.batch) * a.q_heads + per_block - 1) / per_block);
  if (a.weights_out) {
    p.stats = reinterpret_cast<float2 *>(take(uint64_t(c.batch) * c.kv_heads * p.chunks * PA_HEADS * 8));
    p.score_stride = (row_steps * l.cfg->tok + 15) / 16 * 16;
    p.weights_quads = a.slots % 4 == 0 && ((reinterpret_cast<uintptr_t>(a.weights) |
                                            reinterpret_cast<uintptr_t>(a.weights_out)) & 15) == 0;
    p.scores = reinterpret_cast<float *>(take(uint64_t(c.batch) * a.q_heads * p.score_stride * 4));
  }
  l.bytes = off;
  return l;
}

}  // namespace

uint64_t paged_attention_scratch_bytes(const wgx_paged_attention_args &a) { return layout_of(a, false).bytes; }
int paged_attention_launches(const wgx_paged_attention_args &a) { return layout_of(a, false).p.row_blocks ? 1 : 2; }

void launch_paged_attention(const wgx_paged_attention_args &a, cudaStream_t stream) {
  Layout l = layout_of(a, true);
  if (a.scratch_bytes < l.bytes || (reinterpret_cast<uintptr_t>(a.scratch) & 255))
    fail("paged_attention: scratch of " + std::to_string(l.bytes) + " bytes, 256-byte aligned, needed");
  l.p.err = device_error_word(current_device());
  const wgx_kv_cache &c = a.cache;
  const int pre = prefix_bytes(c.batch);
  const int th = timer_begin("paged_attention_kernel", stream);
  launch_dependent(l.p.row_blocks ? l.cfg->row_kernel : l.cfg->kernel, dim3(unsigned(l.grid)), l.cfg->threads,
                   size_t(l.cfg->ring + pre), stream, "paged_attention launch", l.p, l.p.row_blocks);
  timer_end(th, stream);
  if (l.p.row_blocks) return;
  int64_t blocks = l.p.o_blocks;
  if (a.weights_out)
    blocks += int64_t(c.batch) * c.kv_heads * ((l.p.capacity + PA_JOIN_SLOTS - 1) / PA_JOIN_SLOTS);
  const bool wide = c.head_dim > 128, half = c.dtype == WGX_FLOAT16;
  launch_dependent(half ? (wide ? join_kernel<__half, 16, 2> : join_kernel<__half, 16, 1>)
                        : (wide ? join_kernel<float, 8, 2> : join_kernel<float, 8, 1>),
                   dim3(unsigned(blocks)), PA_JOIN_THREADS, size_t(pre), stream, "paged_attention join launch", l.p);
}

}  // namespace wgx
