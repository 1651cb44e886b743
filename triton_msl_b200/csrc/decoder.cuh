// Host-side calls between the C entry points of the decoder-serving operators
// (capi_decoder.cu) and their kernels.
#pragma once
#include <cuda_runtime.h>
#include <atomic>
#include <cstddef>
#include <cstdint>

namespace b2 {

// Runs `set` (a cudaError_t call on the current device) once per device, for
// settings such as a kernel's shared-memory limit that a launch needs every time
// and that cost a microsecond; a failure is returned and tried again next time.
class OncePerDevice {
 public:
  template <typename F>
  cudaError_t operator()(F&& set) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = 1ull << (dev & 63);
    if (dev < 64 && (done_.load(std::memory_order_acquire) & bit)) return cudaSuccess;
    e = set();
    if (e == cudaSuccess && dev < 64) done_.fetch_or(bit, std::memory_order_release);
    return e;
  }

 private:
  std::atomic<uint64_t> done_{0};
};

// From capi.cu: the name behind b2_last_kernel(), and whether the current
// device runs the tcgen05 kernels.
void set_last_kernel(const char* name);
bool device_is_sm100();

// Division by a number known at launch, n < 2^31: a multiply and a shift in place of
// the twenty instructions of a 32-bit division (Granlund and Montgomery 1994).
struct FastDiv {
  uint32_t d = 1, mul = 1, shift = 0;
  FastDiv() = default;
  explicit FastDiv(uint32_t by) : d(by) {
    while ((1ull << shift) < by) ++shift;
    mul = (uint32_t)(((1ull << 32) * ((1ull << shift) - by)) / by + 1);
  }
#ifdef __CUDACC__
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(n, mul) + n) >> shift; }
#endif
};

struct RopeCall {
  const void *q, *k;
  void *qo, *ko;
  const void *qw, *kw;
  const float* table;
  const void* positions;
  int pos64;
  int64_t T, Hq, Hk, D, R, P;
  const int64_t* strides;  // q.t q.h k.t k.h qo.t qo.h ko.t ko.h
  float eps;
  int interleaved, dtype;
};
int rope_launch(const RopeCall& c, cudaStream_t st);
uint32_t rope_read_status(bool clear);

// The 4-bit paged cache: codes [pages, H, page, D/2] uint8 and scales
// [pages, H, page, D/group, 2] bf16 for keys and for values, contiguous.
struct CacheShape {
  int64_t pages, page_size, H, D, group;
};
struct CacheRowsCall {  // write: k, v -> cache; read: cache -> k, v
  void *k_codes, *k_scales, *v_codes, *v_scales;
  void *k, *v;
  const void* slots;
  int slots64;
  int64_t T;
  CacheShape shape;
  const int64_t* strides;  // k.t k.h v.t v.h
  int dtype;
};
int kv_cache_write_launch(const CacheRowsCall& c, cudaStream_t st);
int kv_cache_read_launch(const CacheRowsCall& c, cudaStream_t st);
uint32_t kv_cache_read_status(bool clear);

struct CacheAttnCall {
  const void* q;
  void* o;
  const void *k_codes, *k_scales, *v_codes, *v_scales;
  const int32_t *page_table, *lengths;
  int64_t B, N, Hq, max_pages, table_stride;
  CacheShape shape;
  const int64_t* strides;  // q.b q.n q.h o.b o.n o.h
  float sm_scale;
  int dtype;
  void* workspace;
  size_t ws_bytes;
};
size_t kv_cache_attn_workspace(int64_t B, int64_t rows, int64_t kv_heads, int64_t D);
int kv_cache_attn_launch(const CacheAttnCall& c, cudaStream_t st, const char** kernel);
uint32_t kv_cache_attn_read_status(bool clear);

struct PackedCall {
  const void *q, *k, *v;
  void* o;
  const int32_t *cu_q, *cu_k;
  int64_t B, Tq, Tk, Hq, Hk, D;
  const int64_t* strides;  // t, h, d of q, k, v, o
  float sm_scale;
  int causal, dtype;
  void* workspace;
  size_t ws_bytes;
};
size_t fa_packed_workspace(int64_t B, int64_t Tq, int64_t share);
bool fa_packed_sm100_eligible(const PackedCall& c);
int fa_packed_sm100_launch(const PackedCall& c, cudaStream_t st);
uint32_t fa_packed_read_status(bool clear);
int fa_packed_simt_launch(const PackedCall& c, cudaStream_t st);
uint32_t fa_packed_simt_read_status(bool clear);

// OR of the status words of all kernels above (capi_decoder.cu).
uint32_t decoder_read_status(bool clear);

}  // namespace b2
