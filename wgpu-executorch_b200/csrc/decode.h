// Text decoding over a paged key/value cache: declarations shared by the
// kernels (decode_attention.cu, decode_cache.cu, decode_beam.cu) and their
// front end (ops_decode.cu: checks, C entry points, recorders).
#pragma once
#include <cuda.h>

#include "internal.h"

namespace wgx {

// 5-D map over the rows of a cache's K or V: dimension 0 the channels (all of
// them, or with panels > 1 one 128-byte panel), 1 a page's slots, 2 the panels,
// 3 the heads, 4 the pages; box = one panel's width x `rows` slots x panels,
// 128-byte swizzle, zeros behind a row's end. False when the driver does not
// take the strides.
bool encode_rows_tmap(CUtensorMap *map, const void *base, const wgx_kv_cache &c, int64_t page_stride,
                      int64_t head_stride, int64_t slot_stride, int panels, int rows);

// All enqueue on `stream`, expect checked arguments and throw Error when a
// launch fails.
uint64_t paged_attention_scratch_bytes(const wgx_paged_attention_args &a);
void launch_paged_attention(const wgx_paged_attention_args &a, cudaStream_t stream);
void launch_kv_append(const wgx_kv_append_args &a, cudaStream_t stream);
void launch_cache_evict(const wgx_cache_evict_args &a, cudaStream_t stream);
// Kernels that a call launches.
int paged_attention_launches(const wgx_paged_attention_args &a);
int kv_append_launches(const wgx_kv_append_args &a);
int cache_evict_launches(const wgx_cache_evict_args &a);
uint64_t beam_search_scratch_bytes(const wgx_beam_search_args &a);
void launch_beam_search_step(const wgx_beam_search_args &a, cudaStream_t stream);

constexpr int64_t kEvictMaxSlots = 262144;  // of a sequence that cache_evict can order

// Slots one sequence's table can name.
inline int64_t cache_capacity(const wgx_kv_cache &c) { return int64_t(c.table_width) * c.page_size; }

// K and V rows can be moved in 16-byte units.
inline bool cache_rows_16b(const wgx_kv_cache &c) {
  const int e = c.dtype == WGX_FLOAT16 ? 2 : 4;
  const int64_t strides[] = {c.k_layer_stride, c.k_page_stride, c.k_head_stride, c.k_slot_stride,
                             c.v_layer_stride, c.v_page_stride, c.v_head_stride, c.v_slot_stride};
  int64_t bits = int64_t(c.head_dim) * e;
  for (int64_t s : strides) bits |= s * e;
  return ((bits | int64_t(reinterpret_cast<uintptr_t>(c.k)) |
           int64_t(reinterpret_cast<uintptr_t>(c.v))) & 15) == 0;
}

int device_sm_count();  // of the current device
inline int current_device() {
  int dev = 0;
  check_cuda(cudaGetDevice(&dev), "cudaGetDevice");
  return dev;
}

inline uint64_t align256(uint64_t x) { return (x + 255) / 256 * 256; }  // parts of a scratch buffer

#ifdef __CUDACC__
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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

// Programmatic dependent launch: the next kernel's blocks may be set up while
// this one's work ends (every block of this kernel has started); wait returns
// when all of the prior kernel's work is done and visible. Every kernel here
// lets its dependents launch after its own wait: what a kernel reads before its
// wait may then come from anything but its direct predecessor, which is what
// the join and reorder_kernel rely on for the call's inputs.
__device__ __forceinline__ void let_dependents_launch() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void wait_for_prior_kernel() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// Launches a kernel that may be set up while the stream's previous kernel ends
// (it calls griddepcontrol.wait before it touches what that one writes).
// cluster > 1: in clusters of so many blocks.
template <typename P>
void launch_dependent(void (*kernel)(P), dim3 grid, int threads, size_t smem, cudaStream_t stream,
                      const char *what, const P &arg, int cluster = 0) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(unsigned(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = unsigned(cluster);
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  check_cuda(cudaLaunchKernelEx(&cfg, kernel, arg), what);
}

// Whether n is a length that a table of so many slots can have; noted where not.
// The operators that write leave a sequence of another length as it is: what
// its table names may be other sequences' rows.
__device__ __forceinline__ bool valid_length(int n, int64_t capacity, uint32_t *err) {
  if (n >= 0 && n <= capacity) return true;
  atomicOr(err, kErrCache);
  return false;
}
// Slots in use of sequence b, held within [0, capacity] (for reading).
__device__ __forceinline__ int slots_in_use(const int32_t *lengths, int b, int64_t capacity,
                                            uint32_t *err) {
  const int n = lengths[b];
  if (valid_length(n, capacity, err)) return n;
  return n < 0 ? 0 : int(capacity);
}
#endif

}  // namespace wgx
