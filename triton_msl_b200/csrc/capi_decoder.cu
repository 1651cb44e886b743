// C ABI entry points of the decoder-serving operators (include/b2msl.h): q/k norm
// with rotary positions, the 4-bit paged cache, attention over it, and attention
// over packed sequences. Validation is complete before any launch.
#include <climits>
#include <cmath>

#include "b2_common.cuh"
#include "decoder.cuh"

namespace b2 {
namespace {

bool float_dtype(int dt) { return dt == B2_F32 || dt == B2_F16 || dt == B2_BF16; }
bool index_dtype(int dt) { return dt == B2_I32 || dt == B2_I64; }
bool misaligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) != 0; }

// Shape of the paged cache, {pages, H, page_size, D, group}; `fn` names the caller.
int cache_shape(const char* fn, const int64_t c[5], const void* kc, const void* ks, const void* vc,
                const void* vs, CacheShape* out) {
  if (!c) {
    set_error("%s: null cache shape", fn);
    return B2_EINVAL;
  }
  *out = {c[0], c[2], c[1], c[3], c[4]};
  if (out->pages < 0 || out->H <= 0 || out->page_size <= 0 || out->D <= 0) {
    set_error("%s: invalid cache shape pages=%lld H=%lld page=%lld D=%lld", fn, (long long)out->pages,
              (long long)out->H, (long long)out->page_size, (long long)out->D);
    return B2_EINVAL;
  }
  if (out->D != 64 && out->D != 128) {
    set_error("%s: the 4-bit cache holds head_dim 64 or 128, got %lld", fn, (long long)out->D);
    return B2_EUNSUPPORTED;
  }
  if (out->group != 64 && out->group != out->D) {
    set_error("%s: groups of 64 channels or of the whole head (%lld), got %lld", fn, (long long)out->D,
              (long long)out->group);
    return B2_EUNSUPPORTED;
  }
  if (out->H > INT_MAX || out->pages > INT_MAX || out->page_size > INT_MAX ||
      out->pages * out->page_size > INT_MAX) {
    set_error("%s: pages * page_size must be < 2^31", fn);
    return B2_EINVAL;
  }
  if (out->pages > 0 && (!kc || !ks || !vc || !vs)) {
    set_error("%s: null cache pointer", fn);
    return B2_EINVAL;
  }
  if (misaligned(kc, 16) || misaligned(ks, 16) || misaligned(vc, 16) || misaligned(vs, 16)) {
    set_error("%s: the cache's arrays must start on 16-byte boundaries", fn);
    return B2_EINVAL;
  }
  return B2_OK;
}

bool finite_scale(const char* fn, float s) {
  if (std::isfinite(s)) return true;
  set_error("%s: sm_scale must be finite", fn);
  return false;
}

int cache_rows(const char* fn, bool write, CacheRowsCall& c, const int64_t cache[5], int slots_dtype,
               cudaStream_t st) {
  clear_error();
  const int rc = cache_shape(fn, cache, c.k_codes, c.k_scales, c.v_codes, c.v_scales, &c.shape);
  if (rc != B2_OK) return rc;
  if (!float_dtype(c.dtype)) {
    set_error("%s: unsupported dtype %d", fn, c.dtype);
    return B2_EINVAL;
  }
  if (!index_dtype(slots_dtype)) {
    set_error("%s: slots must be int32 or int64", fn);
    return B2_EINVAL;
  }
  if (c.T < 0) {
    set_error("%s: invalid token count %lld", fn, (long long)c.T);
    return B2_EINVAL;
  }
  if (c.T == 0) return B2_OK;
  if (!c.k || !c.v || !c.slots || !c.strides) {
    set_error("%s: null pointer argument", fn);
    return B2_EINVAL;
  }
  if (c.T > INT_MAX || c.T * c.shape.H * (c.shape.D / 8) > INT_MAX - 1024) {
    set_error("%s: tokens * heads * head_dim / 8 must be < 2^31", fn);
    return B2_EINVAL;
  }
  c.slots64 = slots_dtype == B2_I64;
  const int r = write ? kv_cache_write_launch(c, st) : kv_cache_read_launch(c, st);
  if (r == B2_OK) set_last_kernel(write ? "kv_cache_write" : "kv_cache_read");
  return r;
}

}  // namespace

uint32_t decoder_read_status(bool clear) {
  return rope_read_status(clear) | kv_cache_read_status(clear) | kv_cache_attn_read_status(clear) |
         fa_packed_read_status(clear) | fa_packed_simt_read_status(clear);
}

}  // namespace b2

using namespace b2;

extern "C" {

int b2_qk_norm_rope(const void* q, const void* k, void* q_out, void* k_out, const void* q_weight,
                    const void* k_weight, const float* table, const void* positions, int pos_dtype,
                    int64_t T, int64_t Hq, int64_t Hk, int64_t D, int64_t R, int64_t P,
                    const int64_t strides[8], float eps, int interleaved, int dtype, void* stream) {
  clear_error();
  if (T < 0 || Hq < 0 || Hk < 0 || P < 0 || D <= 0 || R < 0 || R > D || (R & 1) || (D & 1)) {
    set_error("b2_qk_norm_rope: invalid shape T=%lld Hq=%lld Hk=%lld D=%lld R=%lld P=%lld (D and R even, R <= D)",
              (long long)T, (long long)Hq, (long long)Hk, (long long)D, (long long)R, (long long)P);
    return B2_EINVAL;
  }
  if (!float_dtype(dtype) || !index_dtype(pos_dtype)) {
    set_error("b2_qk_norm_rope: unsupported dtype %d or position dtype %d", dtype, pos_dtype);
    return B2_EINVAL;
  }
  if (D > 512) {
    set_error("b2_qk_norm_rope: head_dim %lld > 512 is not supported", (long long)D);
    return B2_EUNSUPPORTED;
  }
  if (T > INT_MAX || Hq > INT_MAX || Hk > INT_MAX) {
    set_error("b2_qk_norm_rope: tokens and heads must be < 2^31");
    return B2_EINVAL;
  }
  if (T == 0 || Hq + Hk == 0) return B2_OK;
  if ((Hq && (!q || !q_out)) || (Hk && (!k || !k_out)) || !positions || !strides ||
      (R > 0 && P > 0 && !table)) {
    set_error("b2_qk_norm_rope: null pointer argument");
    return B2_EINVAL;
  }
  const RopeCall c = {q, k, q_out, k_out, q_weight, k_weight, table, positions, pos_dtype == B2_I64,
                      T, Hq, Hk, D, R, P, strides, eps, interleaved ? 1 : 0, dtype};
  const int rc = rope_launch(c, reinterpret_cast<cudaStream_t>(stream));
  if (rc == B2_OK) set_last_kernel("qk_norm_rope");
  return rc;
}

int b2_kv_cache_write(const void* k, const void* v, void* k_codes, void* k_scales, void* v_codes,
                      void* v_scales, const void* slots, int slots_dtype, int64_t T,
                      const int64_t cache[5], const int64_t strides[4], int dtype, void* stream) {
  CacheRowsCall c = {k_codes, k_scales, v_codes, v_scales, const_cast<void*>(k), const_cast<void*>(v),
                     slots, 0, T, {}, strides, dtype};
  return cache_rows("b2_kv_cache_write", true, c, cache, slots_dtype,
                    reinterpret_cast<cudaStream_t>(stream));
}

int b2_kv_cache_read(void* k, void* v, const void* k_codes, const void* k_scales, const void* v_codes,
                     const void* v_scales, const void* slots, int slots_dtype, int64_t T,
                     const int64_t cache[5], const int64_t strides[4], int dtype, void* stream) {
  CacheRowsCall c = {const_cast<void*>(k_codes), const_cast<void*>(k_scales), const_cast<void*>(v_codes),
                     const_cast<void*>(v_scales), k, v, slots, 0, T, {}, strides, dtype};
  return cache_rows("b2_kv_cache_read", false, c, cache, slots_dtype,
                    reinterpret_cast<cudaStream_t>(stream));
}

int b2_kv_cache_attn(const void* q, void* o, const void* k_codes, const void* k_scales,
                     const void* v_codes, const void* v_scales, const int32_t* page_table,
                     const int32_t* lengths, int64_t B, int64_t N, int64_t Hq, int64_t max_pages,
                     int64_t table_stride, const int64_t cache[5], const int64_t strides[6],
                     float sm_scale, int dtype, void* workspace, size_t ws_bytes, void* stream) {
  clear_error();
  const char* fn = "b2_kv_cache_attn";
  CacheAttnCall c = {q, o, k_codes, k_scales, v_codes, v_scales, page_table, lengths, B, N, Hq,
                     max_pages, table_stride, {}, strides, sm_scale, dtype, workspace, ws_bytes};
  const int rc = cache_shape(fn, cache, k_codes, k_scales, v_codes, v_scales, &c.shape);
  if (rc != B2_OK) return rc;
  if (B < 0 || N < 0 || Hq < 0 || max_pages < 0 || Hq % c.shape.H) {
    set_error("%s: invalid shape B=%lld N=%lld Hq=%lld H=%lld max_pages=%lld (Hq a multiple of H)", fn,
              (long long)B, (long long)N, (long long)Hq, (long long)c.shape.H, (long long)max_pages);
    return B2_EINVAL;
  }
  if (!float_dtype(dtype)) {
    set_error("%s: unsupported dtype %d", fn, dtype);
    return B2_EINVAL;
  }
  if (c.shape.page_size % 16) {
    set_error("%s: page_size %lld is not a multiple of 16", fn, (long long)c.shape.page_size);
    return B2_EUNSUPPORTED;
  }
  if (!finite_scale(fn, sm_scale)) return B2_EINVAL;
  if (B == 0 || N == 0 || Hq == 0) return B2_OK;
  if (!q || !o || !lengths || !strides || (max_pages > 0 && !page_table)) {
    set_error("%s: null pointer argument", fn);
    return B2_EINVAL;
  }
  if (B > INT_MAX || N > INT_MAX || Hq > INT_MAX || max_pages > INT_MAX || B * N > INT_MAX ||
      B * N * Hq > INT_MAX) {
    set_error("%s: B * N * Hq must be < 2^31", fn);
    return B2_EINVAL;
  }
  if (max_pages * c.shape.page_size > INT_MAX - 4096) {
    set_error("%s: max_pages * page_size must be below 2^31 - 4096", fn);
    return B2_EINVAL;
  }
  if (c.shape.pages * c.shape.page_size * c.shape.H > UINT_MAX || c.shape.page_size * c.shape.H > UINT_MAX) {
    set_error("%s: pages * H * page_size must be < 2^32", fn);
    return B2_EINVAL;
  }
  const char* kernel = "";
  const int r = kv_cache_attn_launch(c, reinterpret_cast<cudaStream_t>(stream), &kernel);
  if (r == B2_OK) set_last_kernel(kernel);
  return r;
}

int b2_fa_packed(const void* q, const void* k, const void* v, void* o, const int32_t* cu_q,
                 const int32_t* cu_k, int64_t B, int64_t Tq, int64_t Tk, int64_t Hq, int64_t Hk,
                 int64_t D, const int64_t strides[12], float sm_scale, int causal, int dtype,
                 void* workspace, size_t ws_bytes, void* stream) {
  clear_error();
  if (B < 0 || Tq < 0 || Tk < 0 || Hq < 0 || Hk <= 0 || D <= 0 || Hq % Hk) {
    set_error("b2_fa_packed: invalid shape B=%lld Tq=%lld Tk=%lld Hq=%lld Hk=%lld D=%lld (Hq a multiple of Hk)",
              (long long)B, (long long)Tq, (long long)Tk, (long long)Hq, (long long)Hk, (long long)D);
    return B2_EINVAL;
  }
  if (!float_dtype(dtype)) {
    set_error("b2_fa_packed: unsupported dtype %d", dtype);
    return B2_EINVAL;
  }
  if (D > 128) {
    set_error("b2_fa_packed: head_dim %lld > 128 is not supported", (long long)D);
    return B2_EUNSUPPORTED;
  }
  if (!finite_scale("b2_fa_packed", sm_scale)) return B2_EINVAL;
  if (Tq >= (1LL << 30) || Tk >= (1LL << 30) || B >= (1LL << 30) || Hq > 65535) {
    set_error("b2_fa_packed: Tq, Tk and B must be < 2^30 and Hq < 65536");
    return B2_EINVAL;
  }
  if (Tq == 0 || Hq == 0) return B2_OK;
  if (!q || !o || !cu_q || !cu_k || !strides || (Tk > 0 && (!k || !v))) {
    set_error("b2_fa_packed: null pointer argument");
    return B2_EINVAL;
  }
  const PackedCall c = {q, k, v, o, cu_q, cu_k, B, Tq, Tk, Hq, Hk, D, strides, sm_scale,
                        causal ? 1 : 0, dtype, workspace, ws_bytes};
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool tensor = device_is_sm100() && fa_packed_sm100_eligible(c);
  const int rc = tensor ? fa_packed_sm100_launch(c, st) : fa_packed_simt_launch(c, st);
  if (rc == B2_OK) set_last_kernel(tensor ? "fa_packed_sm100" : "fa_packed_simt");
  return rc;
}

}  // extern "C"
