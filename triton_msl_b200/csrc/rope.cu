// Per-head RMSNorm of queries and keys and their rotary positions, in one pass.
//
//   y = x * rsqrt(mean_d(x^2) + eps) * w          (only where a weight is given)
//   for each of R/2 pairs (a, b) of y: a' = a*c - b*s, b' = b*c + a*s, with
//   (c, s) = table[position]; channels R..D-1 keep y.
//   Pairs: (i, i + R/2) in the half layout, (2i, 2i+1) in the interleaved one.
//
// Bound: HBM. Each value is read once and written once; the table row of a
// token (4R bytes) is shared by its heads and mostly served by the L1 cache.
// A lane group owns heads of one token, four at a time: each lane holds the two
// vectors whose channels rotate into one another, so the rotation needs no
// exchange, and the norm one shuffle tree; the lane's table values are loaded once
// for all heads, and four heads' loads are issued together before any arithmetic.
// 16-bit inputs are bound by instructions as much as by HBM (converting, norm and
// rotation, 14 a value): vectors of 4 channels, 16 lanes a head of 128, leave
// registers for 24 warps per SM. Measured on 16384 tokens, 32 + 8 heads of 128, norm,
// half layout: bf16 56 us, 6.1 TB/s (4 heads a group 74; vectors of 8, 16 warps, and a
// division per head in the norm 92); fp32 102 to 111 us, 6.7 to 6.1 TB/s.
#include <algorithm>
#include <type_traits>

#include "b2_common.cuh"
#include "decoder.cuh"
#include "fa_math.cuh"
#include "vec16.cuh"

namespace b2 {
namespace {

using namespace fa;

__device__ uint32_t g_rope_status;

template <int BYTES> struct RawVec;
template <> struct RawVec<16> { using type = uint4; };
template <> struct RawVec<8> { using type = uint2; };
template <> struct RawVec<4> { using type = uint32_t; };
template <> struct RawVec<2> { using type = uint16_t; };

// Heads of a lane group at once, and CTAs per SM below. When they were chosen (the same
// case, groups of 4 heads), 4 heads and 3 CTAs (80 registers) took 81 us; 2 heads and 4
// CTAs 91; 2 and 5 83; 4 and 4 (64 registers, spills) 110.
constexpr int kHeads = 4;
// A LOOP kernel's groups take several times 4 heads of a token, the next ones' loads in
// flight while these are worked on: the angles and addresses, a third of the
// instructions of 4 heads, are made once for all, and no warp waits for a load it has
// just asked for. Smaller CTAs end the grid more evenly there (56.1 us; 3 of 256 threads
// 56.9). With 4 heads a group it is 3 to 8 % slower than a kernel without the loop.
template <bool LOOP>
constexpr int kThreadsOf = LOOP ? 128 : 256;
template <bool LOOP>
constexpr int kCtasOf = LOOP ? 6 : 3;

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
  unsigned blocks_q;     // CTAs of the queries; the keys' follow
  unsigned groups[2];    // lane groups of each tensor
  unsigned items[2];     // of a token
  FastDiv by_items[2];
  int pos64, D, R, log_tpr;
  int heads_per_group[2];  // of each tensor's lane groups; at most kHeads without LOOP
  float eps, inv_dim;
};

// VE values, two to a packed fp32 pair where VE is even.
template <int VE>
struct Vals {
  static constexpr bool kPacked = VE % 2 == 0;
  static constexpr int N = kPacked ? VE / 2 : VE;
  using E = typename std::conditional<kPacked, f2_t, float>::type;
  E v[N];
  __device__ __forceinline__ Vals() {}
  __device__ __forceinline__ explicit Vals(const float (&x)[VE]) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if constexpr (kPacked) v[i] = f2_pack(x[2 * i], x[2 * i + 1]);
      else v[i] = x[i];
  }
  __device__ __forceinline__ void fill(float x) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if constexpr (kPacked) v[i] = f2_pack(x, x);
      else v[i] = x;
  }
  __device__ __forceinline__ void get(float (&x)[VE]) const {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if constexpr (kPacked) f2_unpack(v[i], x[2 * i], x[2 * i + 1]);
      else x[i] = v[i];
  }
};
template <int VE>
__device__ __forceinline__ Vals<VE> mul(const Vals<VE>& a, const Vals<VE>& b) {
  Vals<VE> r;
#pragma unroll
  for (int i = 0; i < Vals<VE>::N; ++i)
    if constexpr (Vals<VE>::kPacked) r.v[i] = f2_mul(a.v[i], b.v[i]);
    else r.v[i] = a.v[i] * b.v[i];
  return r;
}
template <int VE>
__device__ __forceinline__ Vals<VE> fma(const Vals<VE>& a, const Vals<VE>& b, const Vals<VE>& c) {
  Vals<VE> r;
#pragma unroll
  for (int i = 0; i < Vals<VE>::N; ++i)
    if constexpr (Vals<VE>::kPacked) r.v[i] = f2_fma(a.v[i], b.v[i], c.v[i]);
    else r.v[i] = fmaf(a.v[i], b.v[i], c.v[i]);
  return r;
}

// The first and second values of a unit's pairs from its two vectors, and back.
template <typename T, int VE, bool INTER, typename Raw>
__device__ __forceinline__ void widen(const Raw (&x)[2], float (&a)[VE], float (&b)[VE]) {
  if constexpr (sizeof(T) == 2 && VE % 2 == 0) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(x);
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      if constexpr (INTER) widen2<T>(w[e], a[e], b[e]);
      else if (e % 2 == 0) {
        widen2<T>(w[e / 2], a[e], a[e + 1]);
        widen2<T>(w[(VE + e) / 2], b[e], b[e + 1]);
      }
    }
  } else {
    const T* v = reinterpret_cast<const T*>(x);
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      a[e] = to_f32<T>(v[INTER ? 2 * e : e]);
      b[e] = to_f32<T>(v[INTER ? 2 * e + 1 : VE + e]);
    }
  }
}
template <typename T, int VE, bool INTER, typename Raw>
__device__ __forceinline__ void narrow(const float (&a)[VE], const float (&b)[VE], Raw (&x)[2]) {
  if constexpr (sizeof(T) == 2 && VE % 2 == 0) {
    uint32_t* w = reinterpret_cast<uint32_t*>(x);
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      if constexpr (INTER) w[e] = narrow2<T>(a[e], b[e]);
      else if (e % 2 == 0) {
        w[e / 2] = narrow2<T>(a[e], a[e + 1]);
        w[(VE + e) / 2] = narrow2<T>(b[e], b[e + 1]);
      }
    }
  } else {
    T* v = reinterpret_cast<T*>(x);
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      v[INTER ? 2 * e : e] = from_f32<T>(a[e]);
      v[INTER ? 2 * e + 1 : VE + e] = from_f32<T>(b[e]);
    }
  }
}

// One lane holds NP units of 2*VE values of each head. Unit u < R/(2 VE) is
// rotated: channels [u VE, u VE + VE) with those R/2 above (half layout), or the
// 2 VE neighbours from 2 u VE (interleaved). The other units are copied.
// TPR lanes share a head (0: 1 << log_tpr).
template <typename T, int VE, int NP, int TPR, bool INTER, bool LOOP>
__global__ void __launch_bounds__(kThreadsOf<LOOP>, NP == 1 ? kCtasOf<LOOP> : 1) rope_kernel(const __grid_constant__ RopeArgs a) {
  using Raw = typename RawVec<VE * (int)sizeof(T)>::type;
  const int tpr = TPR ? TPR : 1 << a.log_tpr;
  // A CTA has heads of one tensor, so what belongs to the tensor is uniform in it.
  const int which = blockIdx.x >= a.blocks_q ? 1 : 0;
  const RopeTensor& in = a.in[which];
  const unsigned tid = (blockIdx.x - (which ? a.blocks_q : 0)) * kThreadsOf<LOOP> + threadIdx.x;
  const unsigned gid = TPR ? tid / TPR : tid >> a.log_tpr;
  const int lane = threadIdx.x & (tpr - 1);
  // Lanes past the last group stay for the shuffles and load nothing.
  const bool live = gid < a.groups[which];
  const unsigned token = live ? a.by_items[which].div(gid) : 0;
  const int per = a.heads_per_group[which];
  const int h0 = live ? (int)(gid - token * a.items[which]) * per : 0;
  const int nh = live ? min(per, in.heads - h0) : 0;
  const T* x = static_cast<const T*>(in.x) + (long long)token * in.xt + (long long)h0 * in.xh;
  T* y = static_cast<T*>(in.y) + (long long)token * in.yt + (long long)h0 * in.yh;
  // between a group's heads; the host keeps this within 32 bits
  const int xh = (int)in.xh, yh = (int)in.yh;
  const T* w = static_cast<const T*>(in.w);
  const int units = a.D / (2 * VE), turned = a.R / (2 * VE);

  auto first = [&](int u) { return INTER || u >= turned ? 2 * u * VE : u * VE; };
  auto second = [&](int u) { return INTER || u >= turned ? 2 * u * VE + VE : u * VE + a.R / 2; };

  Raw raw[kHeads][NP][2];
  auto load = [&](int h) {
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const int u = lane + p * tpr;
      const T* const x0 = x + first(u);
      const int gap = second(u) - first(u);
#pragma unroll
      for (int i = 0; i < kHeads; ++i) {
        raw[i][p][0] = raw[i][p][1] = Raw{};
        if (h + i < nh && u < units) {
          raw[i][p][0] = *reinterpret_cast<const Raw*>(x0 + i * xh);
          raw[i][p][1] = *reinterpret_cast<const Raw*>(x0 + i * xh + gap);
        }
      }
    }
  };
  load(0);

  long long pos = 0;
  if (live) pos = a.pos64 ? static_cast<const long long*>(a.positions)[token]
                          : static_cast<const int*>(a.positions)[token];
  // A position outside the table has no angle: the rotated channels become NaN
  // and the status word records it; nothing is read out of range.
  const bool in_table = pos >= 0 && pos < a.P;
  if (live && !in_table && lane == 0) atomicOr(&g_rope_status, DEV_BAD_INDEX);
  const float* row = a.table + (in_table ? pos : 0) * a.R;
  // Per lane and token, for all of its heads: with the weight w folded into the
  // angles, a' = r (a c w_a - b s w_b) and b' = r (b c w_b + a s w_a), r the head's
  // 1/rms: six operations a pair in place of eight, and four heads share these.
  float ca[NP][VE], sb[NP][VE], cb[NP][VE], sa[NP][VE];
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    const int u = lane + p * tpr;
    float wa[VE], wb[VE];
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      ca[p][e] = cb[p][e] = wa[e] = wb[e] = 1.f;
      sa[p][e] = sb[p][e] = 0.f;
    }
    if (live && u < turned) {
      float cs[VE], sn[VE];
      if (in_table) {
        if constexpr (VE >= 4) {
#pragma unroll
          for (int e = 0; e < VE; e += 4) {
            *reinterpret_cast<float4*>(&cs[e]) = __ldg(reinterpret_cast<const float4*>(row + u * VE + e));
            *reinterpret_cast<float4*>(&sn[e]) = __ldg(reinterpret_cast<const float4*>(row + a.R / 2 + u * VE + e));
          }
        } else {
#pragma unroll
          for (int e = 0; e < VE; ++e) {
            cs[e] = __ldg(row + u * VE + e);
            sn[e] = __ldg(row + a.R / 2 + u * VE + e);
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < VE; ++e) cs[e] = sn[e] = __int_as_float(0x7fffffff);
      }
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        ca[p][e] = cb[p][e] = cs[e];
        sa[p][e] = sn[e];
        sb[p][e] = -sn[e];
      }
    }
    if (w && live && u < units) {
      const Raw wr[2] = {__ldg(reinterpret_cast<const Raw*>(w + first(u))), __ldg(reinterpret_cast<const Raw*>(w + second(u)))};
      const T* e0 = reinterpret_cast<const T*>(wr);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        wa[e] = to_f32<T>(e0[INTER ? 2 * e : e]);
        wb[e] = to_f32<T>(e0[INTER ? 2 * e + 1 : VE + e]);
        ca[p][e] *= wa[e];
        sa[p][e] *= wa[e];
        cb[p][e] *= wb[e];
        sb[p][e] *= wb[e];
      }
    }
  }

  for (int h = 0; h < (LOOP ? per : 1); h += kHeads) {
    // the pairs' first and second values, each head's
    float va[kHeads][NP][VE], vb[kHeads][NP][VE];
#pragma unroll
    for (int i = 0; i < kHeads; ++i)
#pragma unroll
      for (int p = 0; p < NP; ++p) widen<T, VE, INTER>(raw[i][p], va[i][p], vb[i][p]);
    if (LOOP && h + kHeads < per) {
      x += (long long)kHeads * xh;
      load(h + kHeads);
    }
    // 1/rms of each head; the heads' shuffle trees run beside one another
    float r[kHeads];
#pragma unroll
    for (int i = 0; i < kHeads; ++i) r[i] = 1.f;
    if (w) {  // the whole CTA alike, so every lane takes part
#pragma unroll
      for (int i = 0; i < kHeads; ++i) {
        Vals<VE> s2;
        s2.fill(0.f);
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          const Vals<VE> ya(va[i][p]), yb(vb[i][p]);
          s2 = fma(ya, ya, s2);
          s2 = fma(yb, yb, s2);
        }
        float t[VE];
        s2.get(t);
        r[i] = t[0];
#pragma unroll
        for (int e = 1; e < VE; ++e) r[i] += t[e];
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
        if (o < tpr)
#pragma unroll
          for (int i = 0; i < kHeads; ++i) r[i] += __shfl_xor_sync(0xffffffffu, r[i], o);
#pragma unroll
      for (int i = 0; i < kHeads; ++i) r[i] = rsqrtf(fmaf(r[i], a.inv_dim, a.eps));
    }
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const int u = lane + p * tpr;
      const Vals<VE> kca(ca[p]), ksb(sb[p]), kcb(cb[p]), ksa(sa[p]);
      T* const y0 = y + first(u);
      const int gap = second(u) - first(u);
#pragma unroll
      for (int i = 0; i < kHeads; ++i) {
        if (!(h + i < nh && u < units)) continue;
        const Vals<VE> xa(va[i][p]), xb(vb[i][p]);
        Vals<VE> scale;
        scale.fill(r[i]);
        Vals<VE> ya = mul(xa, kca), yb = mul(xb, kcb);
        if (u < turned) {  // the others only take the norm: 0 * inf is not 0
          ya = fma(xb, ksb, ya);
          yb = fma(xa, ksa, yb);
        }
        float oa[VE], ob[VE];
        mul(ya, scale).get(oa);
        mul(yb, scale).get(ob);
        Raw out[2];
        narrow<T, VE, INTER>(oa, ob, out);
        *reinterpret_cast<Raw*>(y0 + i * yh) = out[0];
        *reinterpret_cast<Raw*>(y0 + i * yh + gap) = out[1];
      }
    }
    if (LOOP) y += (long long)kHeads * yh;
  }
}

template <typename T, int VE, int NP>
int launch(RopeArgs& a, long long tokens, bool inter, cudaStream_t st) {
  // Heads further apart than 32 bits allow go to a group each.
  const long long far = 1LL << 28;
  const bool near = a.in[0].xh < far && a.in[0].yh < far && a.in[1].xh < far && a.in[1].yh < far &&
                    a.in[0].xh > -far && a.in[0].yh > -far && a.in[1].xh > -far && a.in[1].yh > -far;
  const int units = a.D / (2 * VE);
  a.log_tpr = 0;
  while ((1 << a.log_tpr) < units && a.log_tpr < 5) ++a.log_tpr;
  auto items_of = [&](int i, int per) { return ((long long)a.in[i].heads + per - 1) / per; };
  int per = near ? kHeads : 1;
  bool loop = false;
  if constexpr (sizeof(T) == 2 && VE == 4 && NP == 1) {
    // As many heads a group, up to 8 times 4, as leave 5/4 of the warps that the GPU
    // holds at once. With 32 + 8 heads of 128 and 4 / 8 / 16 / 32 heads a group, in us:
    // 700 tokens 4.1 / 4.4 / 5.6 / 7.9, 2048 8.6 / 7.9 / 8.5 / 10.4, 4096 16.8 / 14.6 /
    // 13.4 / 15.1, 16384 76 / 61 / 59 / 56. fp32 is at HBM's rate without (102 us; 105).
    const long long full = (long long)device_sm_count() * kCtasOf<true> * kThreadsOf<true> * 5 / 4;
    for (int p = kHeads * 8; near && p > kHeads; p /= 2) {
      if (((tokens * (items_of(0, p) + items_of(1, p))) << a.log_tpr) < full) continue;
      per = p;
      loop = true;
      break;
    }
  }
  const int cta = loop ? kThreadsOf<true> : kThreadsOf<false>;
  unsigned blocks[2];
  for (int i = 0; i < 2; ++i) {
    a.heads_per_group[i] = std::max(1, std::min(per, a.in[i].heads));
    a.items[i] = (unsigned)items_of(i, per);
    const long long groups = tokens * a.items[i], threads = groups << a.log_tpr;
    if (groups >= (1LL << 31) || threads + cta >= (1LL << 32)) {
      set_error("b2_qk_norm_rope: %lld tokens x %u lane groups are too many for one launch", tokens, a.items[i]);
      return B2_EINVAL;
    }
    a.groups[i] = (unsigned)groups;
    a.by_items[i] = FastDiv(a.items[i] ? a.items[i] : 1);
    blocks[i] = (unsigned)((threads + cta - 1) / cta);
  }
  a.blocks_q = blocks[0];
  const unsigned grid = blocks[0] + blocks[1];
  auto run = [&](auto kernel) { kernel<<<grid, cta, 0, st>>>(a); };
  // The widths of a head of 64 and of 128 in vectors of four are known to the compiler.
  if constexpr (VE == 4 && NP == 1) {
    auto wide = [&](auto LOOP) {
      constexpr bool L = decltype(LOOP)::value;
      if (a.log_tpr == 4) run(inter ? rope_kernel<T, 4, 1, 16, true, L> : rope_kernel<T, 4, 1, 16, false, L>);
      else if (a.log_tpr == 3) run(inter ? rope_kernel<T, 4, 1, 8, true, L> : rope_kernel<T, 4, 1, 8, false, L>);
      else run(inter ? rope_kernel<T, 4, 1, 0, true, L> : rope_kernel<T, 4, 1, 0, false, L>);
    };
    if constexpr (sizeof(T) == 2) {
      if (loop) wide(std::true_type{});
      else wide(std::false_type{});
    } else {
      wide(std::false_type{});
    }
  } else {
    run(inter ? rope_kernel<T, VE, NP, 0, true, false> : rope_kernel<T, VE, NP, 0, false, false>);
  }
  B2_CHECK_LAUNCH();
  return B2_OK;
}

// A head of up to 64 VE channels is one unit a lane; the longest take several.
template <typename T>
int launch_typed(RopeArgs& a, long long tokens, bool inter, int ve, cudaStream_t st) {
  if (ve == 4) return a.D <= 256 ? launch<T, 4, 1>(a, tokens, inter, st) : launch<T, 4, 2>(a, tokens, inter, st);
  if (ve == 2) return a.D <= 128 ? launch<T, 2, 1>(a, tokens, inter, st) : launch<T, 2, 4>(a, tokens, inter, st);
  return a.D <= 128 ? launch<T, 1, 2>(a, tokens, inter, st) : launch<T, 1, 8>(a, tokens, inter, st);
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
  a.inv_dim = 1.0f / (float)c.D;
  // Widest vector, up to four values, that divides the rotated half, the row and
  // every stride and pointer.
  const int es = dtype_size(c.dtype);
  int ve = 4;
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
