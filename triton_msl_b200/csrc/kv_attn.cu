// Attention of the newest N tokens of each sequence over the 4-bit paged cache.
//
//   o_r = sum_j softmax_j(scale * q_r . k_j) v_j,  j < L - N + 1 + n(r),
//   k_j = ck_j * sk_j + lok_j, v_j = cv_j * sv_j + lov_j (kv_cache.cu)
// for the rows r = (n, head); L counts the new tokens, which are in the cache
// already. A row without a key gives zeros.
//
// fp16 and bf16 queries run kv_attn_mma.cu. The kernel here serves fp32 queries:
// one CTA per row, one warp per key in turn, each lane D/32 channels, the running
// maximum and sum of the softmax per warp and one merge at the end. It reads a key
// head once per query head.
#include "b2_common.cuh"
#include "decoder.cuh"
#include "kv_attn.cuh"

namespace b2 {
namespace {

__device__ uint32_t g_kv_attn_status;

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kRowWarps = 4;

template <typename T, int D, int GROUP>
__global__ void __launch_bounds__(kRowWarps * 32) kv_attn_row_kernel(const __grid_constant__ AttnArgs a) {
  constexpr int CH = D / 32;  // channels per lane: 2 or 4, inside one code word
  __shared__ float sm[kRowWarps], sl[kRowWarps], so[kRowWarps][D];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int head = blockIdx.x % a.Hq;
  const int n = (blockIdx.x / a.Hq) % a.N;
  const int b = blockIdx.x / (a.Hq * a.N);
  const int kvh = head / (a.Hq / a.H);
  const int c0 = lane * CH;
  const int word = (c0 % 64 / 8) * (D / 64) + c0 / 64, shift = (c0 & 7) * 4, grp = c0 / GROUP;

  const int held = a.lengths[b];
  const long long room = (long long)a.max_pages * a.page_size;
  bool bad = held < 0 || held > room;
  const int len = bad ? 0 : held;
  const int keys = max(0, len - a.N + 1 + n);

  const T* q = static_cast<const T*>(a.q) + b * a.qb + n * a.qn + head * a.qh;
  float qv[CH];
#pragma unroll
  for (int i = 0; i < CH; ++i) qv[i] = to_f32<T>(q[c0 + i]) * a.scale_log2;

  float m = -INFINITY, l = 0.f, acc[CH] = {};
  for (int j = warp; j < keys; j += kRowWarps) {
    const int page = a.page_table[b * a.table_stride + j / a.page_size];
    if (page < 0 || page >= a.num_pages) {
      bad = true;
      break;
    }
    const size_t at = ((size_t)page * a.H + kvh) * a.page_size + j % a.page_size;
    const uint32_t wk = reinterpret_cast<const uint32_t*>(a.k_codes)[at * (D / 8) + word] >> shift;
    const uint32_t wv = reinterpret_cast<const uint32_t*>(a.v_codes)[at * (D / 8) + word] >> shift;
    const uint32_t mk = a.k_scales[at * (D / GROUP) + grp], mv = a.v_scales[at * (D / GROUP) + grp];
    const float ks = __uint_as_float(mk << 16), kl = __uint_as_float(mk & 0xffff0000u);
    const float vs = __uint_as_float(mv << 16), vl = __uint_as_float(mv & 0xffff0000u);
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < CH; ++i) s = fmaf(qv[i], fmaf((float)((wk >> (4 * i)) & 15u), ks, kl), s);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const float mn = fmaxf(m, s);
    const float base = mn == -INFINITY ? 0.f : mn;
    const float al = exp2f(m - base), p = exp2f(s - base);
    m = mn;
    l = l * al + p;
#pragma unroll
    for (int i = 0; i < CH; ++i) acc[i] = acc[i] * al + p * fmaf((float)((wv >> (4 * i)) & 15u), vs, vl);
  }
  if (bad && lane == 0) atomicOr(&g_kv_attn_status, DEV_BAD_INDEX);
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = bad ? __int_as_float(0x7fffffff) : l;
  }
#pragma unroll
  for (int i = 0; i < CH; ++i) so[warp][c0 + i] = acc[i];
  __syncthreads();
  float top = sm[0];
  for (int w = 1; w < kRowWarps; ++w) top = fmaxf(top, sm[w]);
  if (top == -INFINITY) top = 0.f;
  T* o = static_cast<T*>(a.o) + b * a.ob + n * a.on + head * a.oh;
  for (int d = threadIdx.x; d < D; d += kRowWarps * 32) {
    float sum = 0.f, val = 0.f;
    for (int w = 0; w < kRowWarps; ++w) {
      const float f = exp2f(sm[w] - top);
      sum += f * sl[w];
      val += f * so[w][d];
    }
    // keys whose scores are all -inf leave no weight either: 0/0
    o[d] = from_f32<T>(keys > 0 || sum != sum ? val / sum : 0.f);
  }
}

template <typename T, int D, int GROUP>
int launch_row(const AttnArgs& a, long long rows, cudaStream_t st) {
  kv_attn_row_kernel<T, D, GROUP><<<(unsigned)rows, kRowWarps * 32, 0, st>>>(a);
  B2_CHECK_LAUNCH();
  return B2_OK;
}

template <typename T>
int launch_row_typed(const AttnArgs& a, const CacheShape& s, long long rows, cudaStream_t st) {
  if (s.D == 64) return launch_row<T, 64, 64>(a, rows, st);
  if (s.group == 64) return launch_row<T, 128, 64>(a, rows, st);
  return launch_row<T, 128, 128>(a, rows, st);
}

}  // namespace

size_t kv_cache_attn_workspace(int64_t B, int64_t rows, int64_t kv_heads, int64_t D) {
  if (B <= 0 || rows <= 0 || kv_heads <= 0 || (D != 64 && D != 128)) return 0;
  return kv_attn_mma_workspace(rows, D);
}

int kv_cache_attn_launch(const CacheAttnCall& c, cudaStream_t st, const char** kernel) {
  const CacheShape& s = c.shape;
  AttnArgs a = {};
  a.q = c.q;
  a.o = c.o;
  a.k_codes = static_cast<const uint8_t*>(c.k_codes);
  a.v_codes = static_cast<const uint8_t*>(c.v_codes);
  a.k_scales = static_cast<const uint32_t*>(c.k_scales);
  a.v_scales = static_cast<const uint32_t*>(c.v_scales);
  a.page_table = c.page_table;
  a.lengths = c.lengths;
  a.qb = c.strides[0];
  a.qn = c.strides[1];
  a.qh = c.strides[2];
  a.ob = c.strides[3];
  a.on = c.strides[4];
  a.oh = c.strides[5];
  a.table_stride = c.table_stride;
  a.B = (int)c.B;
  a.N = (int)c.N;
  a.Hq = (int)c.Hq;
  a.H = (int)s.H;
  a.G = (int)(c.Hq / s.H);
  a.rows = (int)(c.N * a.G);
  a.page_size = (int)s.page_size;
  a.num_pages = (int)s.pages;
  a.max_pages = (int)c.max_pages;
  a.scale_log2 = c.sm_scale * kLog2e;
  B2_CUDA_TRY(cudaGetSymbolAddress(reinterpret_cast<void**>(&a.status), g_kv_attn_status));
  // fp32 queries would lose bits as fp16 operands; a cache without pages has
  // nothing that the other kernel could load in place of a page that is not there
  if (c.dtype != B2_F32 && s.pages > 0) {
    const size_t need = kv_attn_mma_workspace(a.rows, s.D);
    if (!c.workspace || c.ws_bytes < need || (reinterpret_cast<uintptr_t>(c.workspace) & 15)) {
      set_error("b2_kv_cache_attn: needs a 16-byte aligned workspace of %zu bytes", need);
      return B2_EINVAL;
    }
    a.partials = static_cast<float*>(c.workspace);
    a.q_vec = (reinterpret_cast<uintptr_t>(c.q) & 15) == 0 && a.qb % 8 == 0 && a.qn % 8 == 0 && a.qh % 8 == 0;
    a.page_div = FastDiv((uint32_t)a.page_size);
    *kernel = "kv_attn_mma";
    return kv_attn_mma_launch(a, (int)s.D, (int)s.group, c.dtype, st);
  }
  const long long rows = c.B * c.N * c.Hq;
  *kernel = "kv_attn_row";
  switch (c.dtype) {
    case B2_F32: return launch_row_typed<float>(a, s, rows, st);
    case B2_F16: return launch_row_typed<__half>(a, s, rows, st);
    default: return launch_row_typed<__nv_bfloat16>(a, s, rows, st);
  }
}

uint32_t kv_cache_attn_read_status(bool clear) {
  uint32_t v = 0;
  cudaMemcpyFromSymbol(&v, g_kv_attn_status, sizeof(v));
  if (clear) {
    const uint32_t z = 0;
    cudaMemcpyToSymbol(g_kv_attn_status, &z, sizeof(z));
  }
  return v;
}

}  // namespace b2
