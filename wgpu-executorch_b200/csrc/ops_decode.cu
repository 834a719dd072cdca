// Front end of the text-decoding operators: argument checks, the C entry
// points and the recorders (wgx.kv_append / paged_attention / cache_evict /
// beam_search_step). Checks look at the host's arguments only; lengths, page
// ids and masks are device data and are checked where they are used.
#include <algorithm>
#include <atomic>
#include <initializer_list>

#include "decode.h"

namespace wgx {

int device_sm_count() {
  static std::atomic<int> counts[64];
  const int dev = current_device();
  if (dev < 64 && counts[dev].load(std::memory_order_relaxed)) return counts[dev].load(std::memory_order_relaxed);
  int n = 0;
  check_cuda(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev), "SM count");
  if (dev < 64) counts[dev].store(n, std::memory_order_relaxed);
  return n;
}

namespace {

constexpr int64_t kMaxSlots = int64_t(1) << 30;  // slots a table names: indices are 32-bit

void need(bool ok, const char *op, const char *what) {
  if (!ok) fail(std::string(op) + ": " + what);
}
bool aligned(const void *p, int bytes) { return reinterpret_cast<uintptr_t>(p) % uintptr_t(bytes) == 0; }

void check_cache(const wgx_kv_cache &c, const char *op) {
  need(c.dtype == WGX_FLOAT32 || c.dtype == WGX_FLOAT16, op,
       "Tensors must have matching float32 or float16 dtype");
  need(c.k && c.v && c.page_table, op, "null cache or page table");
  const int es = c.dtype == WGX_FLOAT16 ? 2 : 4;
  need(aligned(c.k, es) && aligned(c.v, es) && aligned(c.page_table, 4), op, "misaligned pointer");
  need(c.batch >= 1 && c.batch <= 65535, op, "batch must be in [1, 65535]");
  need(c.kv_heads >= 1 && c.pages >= 1 && c.page_size >= 1 && c.table_width >= 1 && c.layers >= 1, op,
       "cache dimensions must be positive");
  need(c.kv_heads <= 65535, op, "at most 65535 K/V heads");
  need(c.head_dim >= 1 && c.head_dim <= 256, op, "head size must be in [1, 256]");
  need(cache_capacity(c) <= kMaxSlots, op, "page table names more than 2^30 slots");
  // kernels count rows, and elements of a page's row of heads, in 32 bits
  need(int64_t(c.batch) * c.kv_heads <= int64_t(1) << 27, op, "more than 2^27 sequences x K/V heads");
  need(int64_t(c.page_size) * c.head_dim <= int64_t(1) << 30 &&
           int64_t(c.layers) * c.kv_heads <= int64_t(1) << 30,
       op, "cache extents too large");
}

void check_append(const wgx_kv_append_args *a) {
  const char *op = "kv_append";
  need(a, op, "null arguments");
  check_cache(a->cache, op);
  const int es = a->cache.dtype == WGX_FLOAT16 ? 2 : 4;
  need(a->tokens >= 1, op, "at least one token");
  need(a->k && a->v && a->lengths && a->lengths_out, op, "null pointer");
  need(aligned(a->k, es) && aligned(a->v, es), op, "misaligned pointer");
  need(!a->seen == !a->seen_out, op, "seen and seen_out come together");
  need(!a->positions || a->seen, op, "positions need seen");
  need(!(a->weights || a->positions) || a->slots >= cache_capacity(a->cache), op,
       "weights and positions must cover every slot of the page table");
}

void check_attention(const wgx_paged_attention_args *a) {
  const char *op = "paged_attention";
  need(a, op, "null arguments");
  const wgx_kv_cache &c = a->cache;
  check_cache(c, op);
  const int es = c.dtype == WGX_FLOAT16 ? 2 : 4;
  need(a->q && a->out && a->lengths, op, "null pointer");
  need(aligned(a->q, es) && aligned(a->out, es), op, "misaligned pointer");
  need(c.batch <= 2048, op, "batch must be in [1, 2048]");
  need(a->q_heads >= 1 && a->q_heads % c.kv_heads == 0, op,
       "query heads must be a multiple of the K/V heads");
  need(a->q_heads / c.kv_heads <= 128, op, "at most 128 query heads per K/V head");
  need(cache_capacity(c) * c.batch <= int64_t(1) << 33, op, "page tables name more than 2^33 slots");
  need(int64_t(c.batch) * a->q_heads <= int64_t(1) << 30, op, "more than 2^30 sequences x query heads");
  need(a->window >= 0, op, "window must not be negative");
  need(a->scale == a->scale, op, "scale is NaN");
  need(!a->mask || a->mask_width >= 0, op, "mask width must not be negative");
  need(!a->weights == !a->weights_out, op, "weights and weights_out come together");
  need(!a->weights_out || a->slots >= cache_capacity(c), op,
       "weights must cover every slot of the page table");
  need(!a->weights_out || cache_capacity(c) <= int64_t(1) << 25, op,
       "weights are accumulated over at most 2^25 slots");
}

void check_evict(const wgx_cache_evict_args *a) {
  const char *op = "cache_evict";
  need(a, op, "null arguments");
  check_cache(a->cache, op);
  need(a->lengths && a->lengths_out && a->seen && a->weights && a->weights_out && a->positions &&
           a->positions_out,
       op, "null pointer");
  need(a->budget >= 1, op, "budget must be positive");
  need(a->recent >= 0 && a->sinks >= 0 && int64_t(a->recent) + a->sinks <= a->budget, op,
       "recent + sinks must be in [0, budget]");
  need(a->slots >= cache_capacity(a->cache), op,
       "weights and positions must cover every slot of the page table");
  need(cache_capacity(a->cache) <= kEvictMaxSlots, op, "more than 262144 slots per sequence are not supported");
}

void check_beam(const wgx_beam_search_args *a) {
  const char *op = "beam_search_step";
  need(a, op, "null arguments");
  need(a->dtype == WGX_FLOAT32 || a->dtype == WGX_FLOAT16, op, "logits must be float32 or float16");
  need(a->logits && a->scores && a->finished && a->scores_out && a->parents && a->tokens &&
           a->finished_out,
       op, "null pointer");
  need(aligned(a->logits, a->dtype == WGX_FLOAT16 ? 2 : 4), op, "misaligned pointer");
  need(a->beams >= 1 && a->beams <= WGX_MAX_BEAMS, op, "beams must be in [1, 32]");
  need(a->batch >= 1 && int64_t(a->batch) * a->beams <= 65535, op,
       "batch * beams must be in [1, 65535]");
  need(a->vocab >= 1 && a->vocab <= 1 << 24, op, "vocabulary must be in [1, 2^24]");
  need(a->scores_out != a->scores && a->finished_out != a->finished, op,
       "outputs must not overlap inputs");
  if (!a->cache.k) return;
  check_cache(a->cache, op);
  need(a->cache.batch == a->batch * a->beams, op, "the cache must hold batch * beams sequences");
  need(a->lengths && a->spare && a->page_table_out && a->lengths_out, op, "null pointer");
  need(a->page_table_out != a->cache.page_table && a->lengths_out != a->lengths, op,
       "outputs must not overlap inputs");
}

}  // namespace

}  // namespace wgx

using namespace wgx;

extern "C" {

int wgx_kv_append(const wgx_kv_append_args *a, void *stream) {
  return guarded([&] {
    check_append(a);
    launch_kv_append(*a, static_cast<cudaStream_t>(stream));
  });
}

int wgx_paged_attention_scratch_bytes(const wgx_paged_attention_args *a, uint64_t *bytes) {
  return guarded([&] {
    check_attention(a);
    if (!bytes) fail("paged_attention: null pointer");
    *bytes = paged_attention_scratch_bytes(*a);
  });
}

int wgx_paged_attention(const wgx_paged_attention_args *a, void *stream) {
  return guarded([&] {
    check_attention(a);
    launch_paged_attention(*a, static_cast<cudaStream_t>(stream));
  });
}

int wgx_cache_evict(const wgx_cache_evict_args *a, void *stream) {
  return guarded([&] {
    check_evict(a);
    launch_cache_evict(*a, static_cast<cudaStream_t>(stream));
  });
}

int wgx_beam_search_scratch_bytes(const wgx_beam_search_args *a, uint64_t *bytes) {
  return guarded([&] {
    check_beam(a);
    if (!bytes) fail("beam_search_step: null pointer");
    *bytes = beam_search_scratch_bytes(*a);
  });
}

int wgx_beam_search_step(const wgx_beam_search_args *a, void *stream) {
  return guarded([&] {
    check_beam(a);
    launch_beam_search_step(*a, static_cast<cudaStream_t>(stream));
  });
}

}  // extern "C"

namespace wgx {

namespace {

// ---------------------------------------------------------------- recorders
// Recorded tensors are dense. A cache is [pages, kv_heads, page_size,
// head_dim] (beam_search_step also takes [layers, pages, ...]), a page table
// [batch, pages per sequence] int32, lengths [batch] int32, weights and
// positions [batch, kv_heads, slots] float32 / int32.
struct Reader {
  const std::vector<wgx_arg> &args;
  const char *op;

  const wgx_arg &at(size_t i) const {
    if (i >= args.size()) fail(std::string(op) + ": missing argument " + std::to_string(i));
    return args[i];
  }
  wgx_tensor *opt(size_t i, const char *what, std::initializer_list<int> dtypes,
                  std::initializer_list<int64_t> shape) const {
    const wgx_arg &x = at(i);
    if (x.kind == WGX_ARG_NULL) return nullptr;
    if (x.kind != WGX_ARG_TENSOR || !x.v.tensor) fail(std::string(op) + ": " + what + " must be a Tensor");
    wgx_tensor *t = x.v.tensor;
    bool ok = false;
    for (int d : dtypes) ok = ok || t->dtype == d;
    if (!ok) fail(std::string(op) + ": " + what + " has dtype " + dtype_name(t->dtype));
    bool same = size_t(t->ndim) == shape.size();
    size_t k = 0;
    for (int64_t n : shape) {
      same = same && (n < 0 || t->shape[k] == n);  // -1: any extent
      ++k;
    }
    if (!same) {
      std::string got, want;
      for (int d = 0; d < t->ndim; ++d) got += (d ? ", " : "") + std::to_string(t->shape[d]);
      for (int64_t n : shape) want += (want.empty() ? "" : ", ") + (n < 0 ? std::string("*") : std::to_string(n));
      fail(std::string(op) + ": " + what + " shape [" + got + "] !== expected [" + want + "]");
    }
    return t;
  }
  wgx_tensor *tensor(size_t i, const char *what, std::initializer_list<int> dtypes,
                     std::initializer_list<int64_t> shape) const {
    wgx_tensor *t = opt(i, what, dtypes, shape);
    if (!t) fail(std::string(op) + ": " + what + " must be a Tensor");
    return t;
  }
  double number(size_t i, double otherwise) const {
    const wgx_arg &x = at(i);
    if (x.kind == WGX_ARG_NULL) return otherwise;
    if (x.kind == WGX_ARG_NUMBER) return x.v.number;
    fail(std::string(op) + ": argument " + std::to_string(i) + " must be a number");
  }
  int integer(size_t i, int otherwise) const {
    const double v = number(i, otherwise);
    if (!(v >= -2147483648.0 && v <= 2147483647.0) || v != std::floor(v))
      fail(std::string(op) + ": argument " + std::to_string(i) + " must be an integer");
    return int(v);
  }
  void count(size_t n) const {
    if (args.size() != n)
      fail(std::string(op) + ": expected " + std::to_string(n) + " args, got " + std::to_string(args.size()));
  }
};

template <typename T>
T *ptr(wgx_tensor *t) { return t ? static_cast<T *>(t->data()) : nullptr; }

// k and v: [pages, kv_heads, page_size, head_dim], or with a leading extent
// of layers where `layered`.
wgx_kv_cache dense_cache(const Reader &r, size_t k_at, size_t v_at, size_t table_at, bool layered) {
  wgx_kv_cache c{};
  const std::initializer_list<int> fl = {WGX_FLOAT32, WGX_FLOAT16};
  const wgx_arg &x = r.at(k_at);
  const bool five = layered && x.kind == WGX_ARG_TENSOR && x.v.tensor && x.v.tensor->ndim == 5;
  wgx_tensor *k = five ? r.tensor(k_at, "k_cache", fl, {-1, -1, -1, -1, -1})
                       : r.tensor(k_at, "k_cache", fl, {-1, -1, -1, -1});
  const int64_t *s = k->shape + (five ? 1 : 0);
  const int64_t layers = five ? k->shape[0] : 1;
  wgx_tensor *v = five ? r.tensor(v_at, "v_cache", {k->dtype}, {layers, s[0], s[1], s[2], s[3]})
                       : r.tensor(v_at, "v_cache", {k->dtype}, {s[0], s[1], s[2], s[3]});
  wgx_tensor *table = r.tensor(table_at, "page_table", {WGX_INT32}, {-1, -1});
  for (int d = 0; d < k->ndim; ++d)
    if (k->shape[d] > 0x7fffffff) fail(std::string(r.op) + ": cache extent too large");
  if (table->shape[0] > 0x7fffffff || table->shape[1] > 0x7fffffff)
    fail(std::string(r.op) + ": page table extent too large");
  c.k = k->data();
  c.v = v->data();
  c.page_table = ptr<const int32_t>(table);
  c.k_slot_stride = c.v_slot_stride = s[3];
  c.k_head_stride = c.v_head_stride = s[2] * s[3];
  c.k_page_stride = c.v_page_stride = s[1] * s[2] * s[3];
  c.k_layer_stride = c.v_layer_stride = s[0] * s[1] * s[2] * s[3];
  c.table_stride = table->shape[1];
  c.batch = int32_t(table->shape[0]);
  c.kv_heads = int32_t(s[1]);
  c.head_dim = int32_t(s[3]);
  c.dtype = k->dtype;
  c.pages = int32_t(s[0]);
  c.page_size = int32_t(s[2]);
  c.table_width = int32_t(table->shape[1]);
  c.layers = int32_t(layers);
  return c;
}

void push(wgx_context *ctx, const char *name, int launches, uint64_t workspace,
          std::function<void(const ExecEnv &)> run) {
  Command c;
  c.name = name;
  c.kernel_launches = launches;
  c.workspace_bytes = workspace;
  c.run = std::move(run);
  ctx->commands.push_back(std::move(c));
}

// [k, v, page_table, lengths, positions?, seen?, weights?, k_cache, v_cache,
//  seen_out?, lengths_out]
void record_kv_append(wgx_context *ctx, const std::vector<wgx_arg> &args) {
  const char *name = "wgx.kv_append.default";
  const Reader r{args, name};
  r.count(11);
  wgx_kv_append_args a{};
  a.cache = dense_cache(r, 7, 8, 2, false);
  const wgx_kv_cache &c = a.cache;
  wgx_tensor *k = r.tensor(0, "k", {c.dtype}, {c.batch, -1, c.kv_heads, c.head_dim});
  if (k->shape[1] > 0x7fffffff) fail(std::string(name) + ": too many tokens");
  wgx_tensor *v = r.tensor(1, "v", {c.dtype}, {c.batch, k->shape[1], c.kv_heads, c.head_dim});
  a.k = k->data();
  a.v = v->data();
  a.tokens = int32_t(k->shape[1]);
  a.k_head_stride = a.v_head_stride = c.head_dim;
  a.k_token_stride = a.v_token_stride = int64_t(c.kv_heads) * c.head_dim;
  a.k_batch_stride = a.v_batch_stride = a.k_token_stride * a.tokens;
  a.lengths = ptr<const int32_t>(r.tensor(3, "lengths", {WGX_INT32}, {c.batch}));
  wgx_tensor *pos = r.opt(4, "positions", {WGX_INT32}, {c.batch, c.kv_heads, -1});
  a.seen = ptr<const int32_t>(r.opt(5, "seen", {WGX_INT32}, {c.batch}));
  wgx_tensor *w = r.opt(6, "weights", {WGX_FLOAT32}, {c.batch, c.kv_heads, pos ? pos->shape[2] : -1});
  a.positions = ptr<int32_t>(pos);
  a.weights = ptr<float>(w);
  a.slots = pos ? pos->shape[2] : w ? w->shape[2] : 0;
  a.seen_out = ptr<int32_t>(r.opt(9, "seen_out", {WGX_INT32}, {c.batch}));
  a.lengths_out = ptr<int32_t>(r.tensor(10, "lengths_out", {WGX_INT32}, {c.batch}));
  check_append(&a);
  push(ctx, name, kv_append_launches(a), 0, [a](const ExecEnv &env) { launch_kv_append(a, env.stream); });
}

// [q, k_cache, v_cache, page_table, lengths, mask?, scale?, window?, weights?,
//  weights_out?, out]
void record_paged_attention(wgx_context *ctx, const std::vector<wgx_arg> &args) {
  const char *name = "wgx.paged_attention.default";
  const Reader r{args, name};
  r.count(11);
  wgx_paged_attention_args a{};
  a.cache = dense_cache(r, 1, 2, 3, false);
  const wgx_kv_cache &c = a.cache;
  wgx_tensor *q = r.tensor(0, "q", {c.dtype}, {c.batch, -1, c.head_dim});
  if (q->shape[1] > 65535) fail(std::string(name) + ": too many query heads");
  a.q = q->data();
  a.q_heads = int32_t(q->shape[1]);
  a.lengths = ptr<const int32_t>(r.tensor(4, "lengths", {WGX_INT32}, {c.batch}));
  wgx_tensor *mask = r.opt(5, "mask", {WGX_BOOL, WGX_UINT8}, {c.batch, -1});
  if (mask) {
    a.mask = ptr<const uint8_t>(mask);
    a.mask_stride = mask->shape[1];
    a.mask_width = int32_t(std::min<int64_t>(mask->shape[1], 0x7fffffff));
  }
  a.scale = float(r.number(6, 1.0 / std::sqrt(double(c.head_dim))));
  a.window = r.integer(7, 0);
  wgx_tensor *w = r.opt(8, "weights", {WGX_FLOAT32}, {c.batch, c.kv_heads, -1});
  wgx_tensor *wo = r.opt(9, "weights_out", {WGX_FLOAT32}, {c.batch, c.kv_heads, w ? w->shape[2] : -1});
  a.weights = ptr<const float>(w);
  a.weights_out = ptr<float>(wo);
  a.slots = w ? w->shape[2] : 0;
  a.out = r.tensor(10, "out", {c.dtype}, {c.batch, a.q_heads, c.head_dim})->data();
  a.q_head_stride = a.out_head_stride = c.head_dim;
  a.q_batch_stride = a.out_batch_stride = int64_t(a.q_heads) * c.head_dim;
  check_attention(&a);
  push(ctx, name, paged_attention_launches(a), paged_attention_scratch_bytes(a), [a](const ExecEnv &env) {
    wgx_paged_attention_args x = a;
    x.scratch = env.workspace;
    x.scratch_bytes = env.workspace_bytes;
    launch_paged_attention(x, env.stream);
  });
}

// [page_table, lengths, seen, weights, positions, budget, recent?, sinks?,
//  k_cache, v_cache, weights_out, positions_out, lengths_out]
void record_cache_evict(wgx_context *ctx, const std::vector<wgx_arg> &args) {
  const char *name = "wgx.cache_evict.default";
  const Reader r{args, name};
  r.count(13);
  wgx_cache_evict_args a{};
  a.cache = dense_cache(r, 8, 9, 0, false);
  const wgx_kv_cache &c = a.cache;
  a.lengths = ptr<const int32_t>(r.tensor(1, "lengths", {WGX_INT32}, {c.batch}));
  a.seen = ptr<const int32_t>(r.tensor(2, "seen", {WGX_INT32}, {c.batch}));
  wgx_tensor *w = r.tensor(3, "weights", {WGX_FLOAT32}, {c.batch, c.kv_heads, -1});
  a.slots = w->shape[2];
  a.weights = ptr<const float>(w);
  a.positions = ptr<const int32_t>(r.tensor(4, "positions", {WGX_INT32}, {c.batch, c.kv_heads, a.slots}));
  a.budget = r.integer(5, 0);
  a.recent = r.integer(6, 0);
  a.sinks = r.integer(7, 0);
  a.weights_out = ptr<float>(r.tensor(10, "weights_out", {WGX_FLOAT32}, {c.batch, c.kv_heads, a.slots}));
  a.positions_out =
      ptr<int32_t>(r.tensor(11, "positions_out", {WGX_INT32}, {c.batch, c.kv_heads, a.slots}));
  a.lengths_out = ptr<int32_t>(r.tensor(12, "lengths_out", {WGX_INT32}, {c.batch}));
  check_evict(&a);
  push(ctx, name, cache_evict_launches(a), 0, [a](const ExecEnv &env) { launch_cache_evict(a, env.stream); });
}

// [logits, scores, finished, eos, lengths?, page_table?, spare?, k_cache?,
//  v_cache?, scores_out, parents, tokens, finished_out, page_table_out?,
//  lengths_out?]: all of the state's or none
void record_beam_search_step(wgx_context *ctx, const std::vector<wgx_arg> &args) {
  const char *name = "wgx.beam_search_step.default";
  const Reader r{args, name};
  r.count(15);
  wgx_beam_search_args a{};
  wgx_tensor *x = r.tensor(0, "logits", {WGX_FLOAT32, WGX_FLOAT16}, {-1, -1, -1});
  for (int d = 0; d < 3; ++d)
    if (x->shape[d] > 0x7fffffff) fail(std::string(name) + ": logits extent too large");
  a.logits = x->data();
  a.dtype = x->dtype;
  a.batch = int32_t(x->shape[0]);
  a.beams = int32_t(x->shape[1]);
  a.vocab = int32_t(x->shape[2]);
  a.logits_beam_stride = a.vocab;
  a.logits_batch_stride = int64_t(a.beams) * a.vocab;
  const int64_t B = a.batch, W = a.beams;
  const std::initializer_list<int> flag = {WGX_BOOL, WGX_UINT8};
  a.scores = ptr<const float>(r.tensor(1, "scores", {WGX_FLOAT32}, {B, W}));
  a.finished = ptr<const uint8_t>(r.tensor(2, "finished", flag, {B, W}));
  a.eos = r.integer(3, -1);
  a.scores_out = ptr<float>(r.tensor(9, "scores_out", {WGX_FLOAT32}, {B, W}));
  a.parents = ptr<int32_t>(r.tensor(10, "parents", {WGX_INT32}, {B, W}));
  a.tokens = ptr<int32_t>(r.tensor(11, "tokens", {WGX_INT32}, {B, W}));
  a.finished_out = ptr<uint8_t>(r.tensor(12, "finished_out", flag, {B, W}));
  const bool state = r.at(7).kind != WGX_ARG_NULL;
  if (state) {
    a.cache = dense_cache(r, 7, 8, 5, true);
    a.lengths = ptr<const int32_t>(r.tensor(4, "lengths", {WGX_INT32}, {B * W}));
    a.spare = ptr<const int32_t>(r.tensor(6, "spare", {WGX_INT32}, {B * W}));
    a.page_table_out =
        ptr<int32_t>(r.tensor(13, "page_table_out", {WGX_INT32}, {B * W, a.cache.table_width}));
    a.lengths_out = ptr<int32_t>(r.tensor(14, "lengths_out", {WGX_INT32}, {B * W}));
  } else {
    for (size_t i : {4, 5, 6, 8, 13, 14})
      if (r.at(i).kind != WGX_ARG_NULL)
        fail(std::string(name) + ": the cache's arguments come together");
  }
  check_beam(&a);
  push(ctx, name, state ? 3 : 2, beam_search_scratch_bytes(a), [a](const ExecEnv &env) {
    wgx_beam_search_args y = a;
    y.scratch = env.workspace;
    y.scratch_bytes = env.workspace_bytes;
    launch_beam_search_step(y, env.stream);
  });
}

}  // namespace

// The arguments that an operator writes, by position in the lists above: more
// than the last one, and most of them are read too (caches, and what an
// operator may update in place).
const std::vector<size_t> &decode_written_args(const std::string &op) {
  static const std::unordered_map<std::string, std::vector<size_t>> table = {
      {"wgx.kv_append.default", {4, 6, 7, 8, 9, 10}},
      {"wgx.paged_attention.default", {9, 10}},
      {"wgx.cache_evict.default", {8, 9, 10, 11, 12}},
      {"wgx.beam_search_step.default", {7, 8, 9, 10, 11, 12, 13, 14}},
  };
  static const std::vector<size_t> none;
  const auto it = table.find(op);
  return it == table.end() ? none : it->second;
}

void register_decode_ops(std::unordered_map<std::string, OpRecorder> &r) {
  r["wgx.kv_append.default"] = record_kv_append;
  r["wgx.paged_attention.default"] = record_paged_attention;
  r["wgx.cache_evict.default"] = record_cache_evict;
  r["wgx.beam_search_step.default"] = record_beam_search_step;
}

}  // namespace wgx
