// The paged key/value cache in 4 bits: quantising rows as they are written, and
// reading rows back.
//
// A row is one token's D channels of one head. Each group of 64 or 128 channels
// is held as codes c in 0..15 with a scale s and a lowest value lo in bf16:
//   lo = min rounded down to bf16, s = (max - lo) * (1/15) rounded up to bf16,
//   c = clamp(rint((x - lo) * (1/s)), 0, 15) in fp32, read back as c*s + lo.
// Rounding lo down and s up keeps the whole range inside codes 0..15, so no
// value is clipped by more than half a step; bf16 because it has fp32's range
// (an outlier cannot overflow it) at 4 bytes a group, and its 8 bits widen the
// step by at most 1/64. A group with a NaN or an infinity, or whose range max - min
// passes fp32's, reads back as NaN.
//
// Layout: codes [pages, H, page, D/2]; the row's 32-bit words hold 8 channels,
// the first in the lowest bits; the word with channels 64g+8i.. is stored at
// word i*(D/64)+g, so that the 16 bytes which an attention lane loads hold words
// of every 64-channel group and each tensor-core step stays inside one group
// (kv_attn.cu). Scales [pages, H, page, D/group, 2].
//
// Bound: HBM and, for 16-bit rows, instructions. One thread owns two words of keys and
// the same two of values: a group's extremes, scale and reciprocal are then found by 4
// or 8 lanes (8 or 16 with one word a thread: a write of 32768 tokens of 8 heads of 128 took
// 42 us where it takes 28, 6.2 TB/s). The read back takes 33, 5.3 TB/s.
#include <type_traits>

#include "b2_common.cuh"
#include "decoder.cuh"
#include "fa_math.cuh"
#include "vec16.cuh"

namespace b2 {
namespace {

using namespace fa;

__device__ uint32_t g_kv_cache_status;

constexpr int kCacheThreads = 256;

// max that keeps NaN (a group with a NaN has to be seen)
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// x rounded toward -inf to a bf16 value (finite x)
__device__ __forceinline__ float bf16_down(float x) {
  const int bits = __float_as_int(x), cut = bits & 0xffff0000;
  return __int_as_float(bits < 0 && cut != bits ? cut + 0x10000 : cut);
}
// x >= 0 rounded up to a bf16 value
__device__ __forceinline__ float bf16_up(float x) {
  return __int_as_float((__float_as_int(x) + 0xffff) & 0xffff0000);
}

struct RowsArgs {
  uint32_t *k_codes, *k_scales, *v_codes, *v_scales;  // words of 8 codes; (scale, lo) pairs
  void *k, *v;
  const void* slots;
  long long kt, kh, vt, vh;
  unsigned rows, H, page_size, capacity;
  FastDiv by_heads, by_page;
  int slots64;
};

// A lane's channels of one row: two words of 8.
constexpr int kPer = 16;
template <typename T, bool VEC>
__device__ __forceinline__ void load_row(const T* p, T (&x)[kPer]) {
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T); ++i) reinterpret_cast<uint4*>(x)[i] = reinterpret_cast<const uint4*>(p)[i];
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i) x[i] = p[i];
  }
}
__device__ __forceinline__ __nv_bfloat162 max2(__nv_bfloat162 a, __nv_bfloat162 b) { return __hmax2_nan(a, b); }
__device__ __forceinline__ __half2 max2(__half2 a, __half2 b) { return __hmax2_nan(a, b); }
__device__ __forceinline__ __nv_bfloat162 min2(__nv_bfloat162 a, __nv_bfloat162 b) { return __hmin2_nan(a, b); }
__device__ __forceinline__ __half2 min2(__half2 a, __half2 b) { return __hmin2_nan(a, b); }

__device__ __forceinline__ __nv_bfloat162 low_pair(__nv_bfloat162 a, __nv_bfloat162 b) { return __lows2bfloat162(a, b); }
__device__ __forceinline__ __half2 low_pair(__half2 a, __half2 b) { return __lows2half2(a, b); }
__device__ __forceinline__ __nv_bfloat162 high_pair(__nv_bfloat162 a, __nv_bfloat162 b) { return __highs2bfloat162(a, b); }
__device__ __forceinline__ __half2 high_pair(__half2 a, __half2 b) { return __highs2half2(a, b); }

// Largest and lowest value of a group of LANES * 16 values; NaN when it holds one.
// 16-bit types: compared two at a time in their own type, (max, -min) in one word, so
// that one shuffle and one packed maximum serve both (every step is exact).
template <int LANES, typename T>
__device__ __forceinline__ void extremes(const T (&x)[kPer], float& hi, float& lo) {
  if constexpr (sizeof(T) == 2) {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    const T2* p = reinterpret_cast<const T2*>(x);
    T2 up = p[0], dn = p[0];
#pragma unroll
    for (int i = 1; i < kPer / 2; ++i) {
      up = max2(up, p[i]);
      dn = min2(dn, p[i]);
    }
    dn = __hneg2(dn);
    T2 m = max2(low_pair(up, dn), high_pair(up, dn));
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) {
      const uint32_t y = __shfl_xor_sync(0xffffffffu, *reinterpret_cast<uint32_t*>(&m), o);
      m = max2(m, *reinterpret_cast<const T2*>(&y));
    }
    hi = to_f32<T>(m.x);
    lo = -to_f32<T>(m.y);
  } else {
    hi = lo = x[0];
#pragma unroll
    for (int i = 1; i < kPer; ++i) {
      hi = max_nan(hi, x[i]);
      lo = fminf(lo, x[i]);
    }
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) {
      hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
      lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    }
  }
}

// The code words of 16 values and the group's (scale, lo) as two packed bf16.
template <int LANES, typename T>
__device__ __forceinline__ void quantise(const T (&x)[kPer], uint32_t (&word)[2], uint32_t& meta) {
  float hi, lo;
  extremes<LANES>(x, hi, lo);
  const float low = bf16_down(lo);
  const float step = (hi - low) * (1.0f / 15.0f);
  const float scale = bf16_up(step);
  if (!(step < INFINITY) || !(scale < INFINITY)) {  // a NaN or an infinity in the group
    meta = 0x7fff7fffu;
    word[0] = word[1] = 0u;
    return;
  }
  meta = (__float_as_uint(scale) >> 16) | (__float_as_uint(low) & 0xffff0000u);
  // below 2^-126 the reciprocal may overflow; the group reads back as lo then
  const float inv = scale >= 1.17549435e-38f ? __frcp_rn(scale) : 0.0f;
  // (x - low) * inv is at most 15 (1 + 2^-21), scale being rounded up. Adding
  // 1.5 * 2^23 rounds it to the nearest integer (ties to even) and leaves that in
  // the low bits; what the constant's own bits add to the word is subtracted.
  constexpr uint32_t kMagic = 0x4b400000u;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    uint32_t sum = 0, bias = 0;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      float y0, y1;
      if constexpr (sizeof(T) == 2) {
        widen2<T>(reinterpret_cast<const uint32_t*>(x)[4 * w + i / 2], y0, y1);
      } else {
        y0 = x[8 * w + i];
        y1 = x[8 * w + i + 1];
      }
      f2_t y = f2_add(f2_pack(y0, y1), f2_pack(-low, -low));
      f2_unpack(y, y0, y1);
      // the product is rounded by itself: a packed product and sum come out fused,
      // which decides values half way between two codes differently
      y = f2_add(f2_pack(__fmul_rn(y0, inv), __fmul_rn(y1, inv)), f2_pack(12582912.0f, 12582912.0f));
      f2_unpack(y, y0, y1);
      sum += (__float_as_uint(y0) << (4 * i)) + (__float_as_uint(y1) << (4 * i + 4));
      bias += (kMagic << (4 * i)) + (kMagic << (4 * i + 4));
    }
    word[w] = sum - bias;
  }
}

// Where the lane's first word lies in the row; its second is D/64 further.
template <int D>
__device__ __forceinline__ int stored_word(int lane) {
  return (lane & 3) * 2 * (D / 64) + (lane >> 2);
}

template <typename T, int D, int GROUP, bool VEC>
__global__ void __launch_bounds__(kCacheThreads) kv_write_kernel(const __grid_constant__ RowsArgs a) {
  constexpr int LPR = D / kPer, LPG = GROUP / kPer;  // lanes of a row, of a group
  const unsigned tid = blockIdx.x * kCacheThreads + threadIdx.x;
  const unsigned row = tid / LPR;
  const int lane = tid % LPR;
  // threads past the last row repeat it without storing: the shuffles need them
  const unsigned r = row < a.rows ? row : a.rows - 1;
  const unsigned token = a.by_heads.div(r), head = r - token * a.H;
  __align__(16) T k[kPer], v[kPer];
  load_row<T, VEC>(static_cast<const T*>(a.k) + (long long)token * a.kt + (long long)head * a.kh + lane * kPer, k);
  load_row<T, VEC>(static_cast<const T*>(a.v) + (long long)token * a.vt + (long long)head * a.vh + lane * kPer, v);
  const long long slot = a.slots64 ? static_cast<const long long*>(a.slots)[token]
                                   : static_cast<const int*>(a.slots)[token];
  uint32_t mk, mv, wk[2], wv[2];
  quantise<LPG>(k, wk, mk);
  quantise<LPG>(v, wv, mv);
  if (row >= a.rows || slot < 0) return;
  if (slot >= (long long)a.capacity) {
    if (lane == 0) atomicOr(&g_kv_cache_status, DEV_BAD_INDEX);
    return;
  }
  const unsigned page = a.by_page.div((unsigned)slot), place = (unsigned)slot - page * a.page_size;
  const size_t at = ((size_t)page * a.H + head) * a.page_size + place;
  uint32_t* kc = a.k_codes + at * (D / 8) + stored_word<D>(lane);
  uint32_t* vc = a.v_codes + at * (D / 8) + stored_word<D>(lane);
  kc[0] = wk[0];
  kc[D / 64] = wk[1];
  vc[0] = wv[0];
  vc[D / 64] = wv[1];
  if (lane % LPG == 0) {
    a.k_scales[at * (D / GROUP) + lane / LPG] = mk;
    a.v_scales[at * (D / GROUP) + lane / LPG] = mv;
  }
}

// The 8 values of one word.
template <typename T, bool VEC>
__device__ __forceinline__ void put_values(T* p, uint32_t word, uint32_t meta) {
  const float s = __uint_as_float(meta << 16), lo = __uint_as_float(meta & 0xffff0000u);
  __align__(16) T x[8];
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    // 2^23 + c minus 2^23 is the code as a float
    f2_t y = f2_pack(__uint_as_float(0x4b000000u | ((word >> (4 * i)) & 15u)),
                     __uint_as_float(0x4b000000u | ((word >> (4 * i + 4)) & 15u)));
    y = f2_fma(f2_add(y, f2_pack(-8388608.0f, -8388608.0f)), f2_pack(s, s), f2_pack(lo, lo));
    float y0, y1;
    f2_unpack(y, y0, y1);
    if constexpr (sizeof(T) == 2) {
      reinterpret_cast<uint32_t*>(x)[i / 2] = narrow2<T>(y0, y1);
    } else {
      x[i] = y0;
      x[i + 1] = y1;
    }
  }
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(x)[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = x[i];
  }
}

// A lane takes two words that are stored side by side, of one group (D = 64) or of two.
template <typename T, int D, int GROUP, bool VEC>
__global__ void __launch_bounds__(kCacheThreads) kv_read_kernel(const __grid_constant__ RowsArgs a) {
  constexpr int LPR = D / kPer, NG = D / GROUP;
  const unsigned tid = blockIdx.x * kCacheThreads + threadIdx.x;
  const unsigned row = tid / LPR;
  const int lane = tid % LPR;
  if (row >= a.rows) return;
  const unsigned token = a.by_heads.div(row), head = row - token * a.H;
  const long long slot = a.slots64 ? static_cast<const long long*>(a.slots)[token]
                                   : static_cast<const int*>(a.slots)[token];
  T* k = static_cast<T*>(a.k) + (long long)token * a.kt + (long long)head * a.kh;
  T* v = static_cast<T*>(a.v) + (long long)token * a.vt + (long long)head * a.vh;
  const int c0 = D == 128 ? 8 * lane : 16 * lane, c1 = D == 128 ? 64 + 8 * lane : 16 * lane + 8;
  if (slot >= 0 && slot < (long long)a.capacity) {
    const unsigned page = a.by_page.div((unsigned)slot), place = (unsigned)slot - page * a.page_size;
    const size_t at = ((size_t)page * a.H + head) * a.page_size + place;
    const uint2 wk = reinterpret_cast<const uint2*>(a.k_codes)[at * LPR + lane];
    const uint2 wv = reinterpret_cast<const uint2*>(a.v_codes)[at * LPR + lane];
    uint2 mk, mv;
    if constexpr (NG == 2) {
      mk = reinterpret_cast<const uint2*>(a.k_scales)[at];
      mv = reinterpret_cast<const uint2*>(a.v_scales)[at];
    } else {
      mk.x = mk.y = a.k_scales[at];
      mv.x = mv.y = a.v_scales[at];
    }
    put_values<T, VEC>(k + c0, wk.x, mk.x);
    put_values<T, VEC>(k + c1, wk.y, mk.y);
    put_values<T, VEC>(v + c0, wv.x, mv.x);
    put_values<T, VEC>(v + c1, wv.y, mv.y);
  } else {
    // a negative slot is padding and reads as zero; one past the cache as NaN: scale 0,
    // lowest value 0 or NaN
    const uint32_t fill = slot < 0 ? 0u : 0x7fff0000u;
    if (slot >= 0 && lane == 0) atomicOr(&g_kv_cache_status, DEV_BAD_INDEX);
    put_values<T, VEC>(k + c0, 0u, fill);
    put_values<T, VEC>(k + c1, 0u, fill);
    put_values<T, VEC>(v + c0, 0u, fill);
    put_values<T, VEC>(v + c1, 0u, fill);
  }
}

template <bool WRITE, typename T, int D, int GROUP>
int launch(const RowsArgs& a, bool vec, cudaStream_t st) {
  const unsigned long long threads = (unsigned long long)a.rows * (D / kPer);
  const unsigned grid = (unsigned)((threads + kCacheThreads - 1) / kCacheThreads);
  if constexpr (WRITE) {
    if (vec) kv_write_kernel<T, D, GROUP, true><<<grid, kCacheThreads, 0, st>>>(a);
    else kv_write_kernel<T, D, GROUP, false><<<grid, kCacheThreads, 0, st>>>(a);
  } else {
    if (vec) kv_read_kernel<T, D, GROUP, true><<<grid, kCacheThreads, 0, st>>>(a);
    else kv_read_kernel<T, D, GROUP, false><<<grid, kCacheThreads, 0, st>>>(a);
  }
  B2_CHECK_LAUNCH();
  return B2_OK;
}

template <bool WRITE, typename T>
int launch_typed(const RowsArgs& a, const CacheShape& s, bool vec, cudaStream_t st) {
  if (s.D == 64) return launch<WRITE, T, 64, 64>(a, vec, st);
  if (s.group == 64) return launch<WRITE, T, 128, 64>(a, vec, st);
  return launch<WRITE, T, 128, 128>(a, vec, st);
}

template <bool WRITE>
int rows_launch(const CacheRowsCall& c, cudaStream_t st) {
  const CacheShape& s = c.shape;
  RowsArgs a = {};
  a.k_codes = static_cast<uint32_t*>(c.k_codes);
  a.k_scales = static_cast<uint32_t*>(c.k_scales);
  a.v_codes = static_cast<uint32_t*>(c.v_codes);
  a.v_scales = static_cast<uint32_t*>(c.v_scales);
  a.k = c.k;
  a.v = c.v;
  a.slots = c.slots;
  a.slots64 = c.slots64;
  a.kt = c.strides[0];
  a.kh = c.strides[1];
  a.vt = c.strides[2];
  a.vh = c.strides[3];
  a.rows = (unsigned)(c.T * s.H);
  a.H = (unsigned)s.H;
  a.page_size = (unsigned)s.page_size;
  a.capacity = (unsigned)(s.pages * s.page_size);
  a.by_heads = FastDiv(a.H);
  a.by_page = FastDiv(a.page_size);
  const long long per = 16 / dtype_size(c.dtype);
  const bool vec = ((reinterpret_cast<uintptr_t>(c.k) | reinterpret_cast<uintptr_t>(c.v)) & 15) == 0 &&
                   a.kt % per == 0 && a.kh % per == 0 && a.vt % per == 0 && a.vh % per == 0;
  switch (c.dtype) {
    case B2_F32: return launch_typed<WRITE, float>(a, s, vec, st);
    case B2_F16: return launch_typed<WRITE, __half>(a, s, vec, st);
    default: return launch_typed<WRITE, __nv_bfloat16>(a, s, vec, st);
  }
}

}  // namespace

int kv_cache_write_launch(const CacheRowsCall& c, cudaStream_t st) { return rows_launch<true>(c, st); }
int kv_cache_read_launch(const CacheRowsCall& c, cudaStream_t st) { return rows_launch<false>(c, st); }

uint32_t kv_cache_read_status(bool clear) {
  uint32_t v = 0;
  cudaMemcpyFromSymbol(&v, g_kv_cache_status, sizeof(v));
  if (clear) {
    const uint32_t z = 0;
    cudaMemcpyToSymbol(g_kv_cache_status, &z, sizeof(z));
  }
  return v;
}

}  // namespace b2
