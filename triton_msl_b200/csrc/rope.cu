// Per-head RMSNorm of queries and keys and their rotary positions, in one pass.
//
//   y = x * rsqrt(mean_d(x^2) + eps) * w          (only where a weight is given)
//   for each of R/2 pairs (a, b) of y: a' = a*c - b*s, b' = b*c + a*s, with
//   (c, s) = table[position]; channels R..D-1 keep y.
//   Pairs: (i, i + R/2) in the half layout, (2i, 2i+1) in the interleaved one.
//
// Bound: HBM. Each value is read once and written once; the table row of a
// token (4R bytes) is shared by its heads and mostly served by the L1 cache.
// A lane group owns HPT heads of one token: each lane holds the two vectors
// whose channels rotate into one another, so the rotation needs no exchange,
// and the norm one shuffle tree; the lane's table values are loaded once for
// all HPT heads, whose loads are issued together before any arithmetic.
// The arithmetic is fp32 throughout; only the result is rounded to x's type.
#include "b2_common.cuh"
#include "decoder.cuh"

namespace b2 {
namespace {

__device__ uint32_t g_rope_status;

constexpr int kRopeThreads = 256;
constexpr int kRopeMaxDim = 512;

template <int BYTES> struct RawVec;
template <> struct RawVec<16> { using type = uint4; };
template <> struct RawVec<8> { using type = uint2; };
template <> struct RawVec<4> { using type = uint32_t; };
template <> struct RawVec<2> { using type = uint16_t; };

struct RopeTensor {
  const void* x;
  void* y;
  const void* w;  // null: no norm
  long long xt, xh, yt, yh;  // token and head strides, elements
  int heads;
};

struct RopeArgs {
  RopeTensor in[2];      // queries, keys
  const float* table;    // [P, R]: cos | sin
  const void* positions;
  long long P;
  unsigned items;        // lane groups per token (both tensors)
  unsigned items_q;      // of these, the queries'
  unsigned total;        // items * tokens
  int pos64, D, R, log_tpr, heads_per_group;
  float eps;
};

// One lane holds NP units of 2*VE values of each head. Unit u < R/(2 VE) is
// rotated: channels [u VE, u VE + VE) with those R/2 above (half layout), or the
// 2 VE neighbours from 2 u VE (interleaved). The other units are copied.
template <typename T, int VE, int NP, int HPT, bool INTER>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const __grid_constant__ RopeArgs a) {
  using Raw = typename RawVec<VE * (int)sizeof(T)>::type;
  const int tpr = 1 << a.log_tpr;
  const unsigned gid = (blockIdx.x * kRopeThreads + threadIdx.x) >> a.log_tpr;
  const int lane = threadIdx.x & (tpr - 1);
  // Lanes past the last group stay for the shuffles and load nothing.
  const bool live = gid < a.total;
  const unsigned token = live ? gid / a.items : 0;
  const unsigned item = live ? gid - token * a.items : 0;
  const bool is_k = item >= a.items_q;
  const RopeTensor& in = a.in[is_k ? 1 : 0];
  const int h0 = (int)(is_k ? item - a.items_q : item) * a.heads_per_group;
  const int nh = live ? min(a.heads_per_group, in.heads - h0) : 0;
  const T* x = static_cast<const T*>(in.x) + (long long)token * in.xt + (long long)h0 * in.xh;
  T* y = static_cast<T*>(in.y) + (long long)token * in.yt + (long long)h0 * in.yh;
  const T* w = static_cast<const T*>(in.w);
  const int units = a.D / (2 * VE), turned = a.R / (2 * VE);

  auto first = [&](int u) { return INTER || u >= turned ? 2 * u * VE : u * VE; };
  auto second = [&](int u) { return INTER || u >= turned ? 2 * u * VE + VE : u * VE + a.R / 2; };

  Raw raw[HPT][NP][2];
#pragma unroll
  for (int i = 0; i < HPT; ++i)
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const int u = lane + p * tpr;
      raw[i][p][0] = raw[i][p][1] = Raw{};
      if (i < nh && u < units) {
        raw[i][p][0] = *reinterpret_cast<const Raw*>(x + i * in.xh + first(u));
        raw[i][p][1] = *reinterpret_cast<const Raw*>(x + i * in.xh + second(u));
      }
    }

  long long pos = 0;
  if (live) pos = a.pos64 ? static_cast<const long long*>(a.positions)[token]
                          : static_cast<const int*>(a.positions)[token];
  // A position outside the table has no angle: the rotated channels become NaN
  // and the status word records it; nothing is read out of range.
  const bool in_table = pos >= 0 && pos < a.P;
  if (live && !in_table && lane == 0) atomicOr(&g_rope_status, DEV_BAD_INDEX);
  const float* row = a.table + (in_table ? pos : 0) * a.R;
  float cs[NP][VE], sn[NP][VE];
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    const int u = lane + p * tpr;
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      cs[p][e] = 1.f;
      sn[p][e] = 0.f;
    }
    if (live && u < turned) {
      if (in_table) {
        if constexpr (VE >= 4) {
#pragma unroll
          for (int e = 0; e < VE; e += 4) {
            *reinterpret_cast<float4*>(&cs[p][e]) = __ldg(reinterpret_cast<const float4*>(row + u * VE + e));
            *reinterpret_cast<float4*>(&sn[p][e]) = __ldg(reinterpret_cast<const float4*>(row + a.R / 2 + u * VE + e));
          }
        } else {
#pragma unroll
          for (int e = 0; e < VE; ++e) {
            cs[p][e] = __ldg(row + u * VE + e);
            sn[p][e] = __ldg(row + a.R / 2 + u * VE + e);
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < VE; ++e) cs[p][e] = sn[p][e] = __int_as_float(0x7fffffff);
      }
    }
  }

#pragma unroll
  for (int i = 0; i < HPT; ++i) {
    float v[NP][2 * VE];
    float ss = 0.f;
#pragma unroll
    for (int p = 0; p < NP; ++p)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const T* e = reinterpret_cast<const T*>(&raw[i][p][c]);
#pragma unroll
        for (int j = 0; j < VE; ++j) {
          v[p][c * VE + j] = to_f32<T>(e[j]);
          ss = fmaf(v[p][c * VE + j], v[p][c * VE + j], ss);
        }
      }
    if (w) {  // uniform in the lane group
      // lanes of other groups may take the other branch: a group's shuffles
      // name its own lanes only
      const unsigned mask = tpr == 32 ? 0xffffffffu : ((1u << tpr) - 1u) << (threadIdx.x & 31 & ~(tpr - 1));
      for (int o = tpr >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
      const float r = rsqrtf(ss / (float)a.D + a.eps);
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        const int u = lane + p * tpr;
        if (u < units) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const Raw wr = __ldg(reinterpret_cast<const Raw*>(w + (c ? second(u) : first(u))));
            const T* e = reinterpret_cast<const T*>(&wr);
#pragma unroll
            for (int j = 0; j < VE; ++j) v[p][c * VE + j] *= r * to_f32<T>(e[j]);
          }
        }
      }
    }
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const int u = lane + p * tpr;
      // units that are not rotated have c = 1, s = 0 but are left alone: 0 * inf
      if (u < turned) {
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          float& lo = v[p][INTER ? 2 * e : e];
          float& hi = v[p][INTER ? 2 * e + 1 : VE + e];
          const float t = lo * cs[p][e] - hi * sn[p][e];
          hi = hi * cs[p][e] + lo * sn[p][e];
          lo = t;
        }
      }
      if (i < nh && u < units) {
        Raw out[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          T* e = reinterpret_cast<T*>(&out[c]);
#pragma unroll
          for (int j = 0; j < VE; ++j) e[j] = from_f32<T>(v[p][c * VE + j]);
        }
        *reinterpret_cast<Raw*>(y + i * in.yh + first(u)) = out[0];
        *reinterpret_cast<Raw*>(y + i * in.yh + second(u)) = out[1];
      }
    }
  }
}

template <typename T, int VE, int HPT>
int launch(RopeArgs& a, long long tokens, bool inter, cudaStream_t st) {
  constexpr int NP = kRopeMaxDim / (2 * VE * 32) > 0 ? kRopeMaxDim / (2 * VE * 32) : 1;
  const int units = a.D / (2 * VE);
  a.log_tpr = 0;
  while ((1 << a.log_tpr) < units && a.log_tpr < 5) ++a.log_tpr;
  a.heads_per_group = HPT;
  a.items_q = (unsigned)((a.in[0].heads + HPT - 1) / HPT);
  a.items = a.items_q + (unsigned)((a.in[1].heads + HPT - 1) / HPT);
  const long long total = tokens * a.items;
  const long long threads = total << a.log_tpr;
  if (threads + kRopeThreads >= (1LL << 31)) {
    set_error("b2_qk_norm_rope: %lld tokens x %u lane groups are too many for one launch", tokens, a.items);
    return B2_EINVAL;
  }
  a.total = (unsigned)total;
  const unsigned grid = (unsigned)((threads + kRopeThreads - 1) / kRopeThreads);
  if (inter) rope_kernel<T, VE, NP, HPT, true><<<grid, kRopeThreads, 0, st>>>(a);
  else rope_kernel<T, VE, NP, HPT, false><<<grid, kRopeThreads, 0, st>>>(a);
  B2_CHECK_LAUNCH();
  return B2_OK;
}

template <typename T>
int launch_typed(RopeArgs& a, long long tokens, bool inter, int ve, cudaStream_t st) {
  constexpr int HPT = sizeof(T) == 2 ? 4 : 2;
  if constexpr (sizeof(T) == 2) {
    if (ve >= 8) return launch<T, 8, HPT>(a, tokens, inter, st);
  }
  if (ve >= 4) return launch<T, 4, HPT>(a, tokens, inter, st);
  if (ve >= 2) return launch<T, 2, HPT>(a, tokens, inter, st);
  return launch<T, 1, HPT>(a, tokens, inter, st);
}

}  // namespace

int rope_launch(const RopeCall& c, cudaStream_t st) {
  RopeArgs a = {};
  const int64_t* s = c.strides;
  a.in[0] = {c.q, c.qo, c.qw, s[0], s[1], s[4], s[5], (int)c.Hq};
  a.in[1] = {c.k, c.ko, c.kw, s[2], s[3], s[6], s[7], (int)c.Hk};
  a.table = c.table;
  a.positions = c.positions;
  a.P = c.P;
  a.pos64 = c.pos64;
  a.D = (int)c.D;
  a.R = (int)c.R;
  a.eps = c.eps;
  // Widest vector that divides the rotated half, the row and every stride and
  // pointer (16 bytes at most).
  const int es = dtype_size(c.dtype);
  int ve = 16 / es;
  auto fits = [&](int v) {
    if ((c.R / 2) % v || c.D % (2 * v)) return false;
    if (v >= 4 && (reinterpret_cast<uintptr_t>(c.table) & 15)) return false;
    for (int i = 0; i < 2; ++i) {
      if (a.in[i].heads == 0) continue;
      const uintptr_t bytes = (uintptr_t)v * es;
      if ((reinterpret_cast<uintptr_t>(a.in[i].x) | reinterpret_cast<uintptr_t>(a.in[i].y) |
           reinterpret_cast<uintptr_t>(a.in[i].w)) % bytes)
        return false;
      if (a.in[i].xt % v || a.in[i].xh % v || a.in[i].yt % v || a.in[i].yh % v) return false;
    }
    return true;
  };
  while (ve > 1 && !fits(ve)) ve >>= 1;
  switch (c.dtype) {
    case B2_F32: return launch_typed<float>(a, c.T, c.interleaved, ve, st);
    case B2_F16: return launch_typed<__half>(a, c.T, c.interleaved, ve, st);
    default: return launch_typed<__nv_bfloat16>(a, c.T, c.interleaved, ve, st);
  }
}

uint32_t rope_read_status(bool clear) {
  uint32_t v = 0;
  cudaMemcpyFromSymbol(&v, g_rope_status, sizeof(v));
  if (clear) {
    const uint32_t z = 0;
    cudaMemcpyToSymbol(g_rope_status, &z, sizeof(z));
  }
  return v;
}

}  // namespace b2
