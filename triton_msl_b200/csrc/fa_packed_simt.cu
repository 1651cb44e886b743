// Attention over packed sequences on the CUDA cores: fp32 inputs, strides and
// head dims that the tensor-core kernel (fa_packed_sm100.cu) does not take.
//
//   o_i = sum_j softmax_j(scale * q_i . k_j) v_j over the keys j of i's own
//   sequence, with j <= i + (Lk - Lq) when causal; no key: zeros.
//
// One CTA owns 16 queries of one head and walks the keys 32 at a time, staged in
// shared memory as fp32. A warp owns 4 queries; lane = key for the scores (one
// key row read serves 4 queries) and lane = channel for the values. Masked keys
// are skipped in the value sum, so what they hold cannot reach a result. Bound by
// shared-memory reads and FFMA; it is the general path, not the fast one.
#include "b2_common.cuh"
#include "decoder.cuh"
#include "packed.cuh"

namespace b2 {
namespace {

__device__ uint32_t g_packed_simt_status;

constexpr int kRows = 16, kKeys = 32, kThreads = 128, kMaxD = 128;
constexpr float kLog2e = 1.4426950408889634f;

struct SimtArgs {
  const void *q, *k, *v;
  void* o;
  const int32_t *cu_q, *cu_k;
  long long s[12];  // t, h, d strides of q, k, v, o
  int B, Tq, Tk, Hq, Hk, D, causal;
  float scale_log2;
};

template <typename T>
__global__ void __launch_bounds__(kThreads) fa_packed_simt_kernel(const __grid_constant__ SimtArgs a) {
  __shared__ float Qs[kRows][kMaxD], Ks[kKeys][kMaxD + 1], Vs[kKeys][kMaxD];
  __shared__ int s_seq, s_blk;
  __shared__ packed::Span s_span;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // The CTA's sequence and block: 32 sequences at a time, where the ones before them
  // end, prefix sums of their block counts. The grid has a CTA for every block that can
  // exist, so the last ones find none.
  if (warp == 0) {
    int left = (int)blockIdx.x, seq = -2, blk = 0, before = 0;
    packed::Span own = {0, 0};
    for (int b0 = -1; b0 <= a.B && seq == -2; b0 += 32) {
      const int b = b0 + lane;
      packed::Span q = b <= a.B ? packed::span_of(a.cu_q, b, a.B, a.Tq) : packed::Span{0, 0};
      int end = q.start + q.len;
      for (int o = 1; o < 32; o <<= 1) end = max(end, __shfl_up_sync(0xffffffffu, end, o));
      end = max(end, before);
      const int up = __shfl_up_sync(0xffffffffu, end, 1);
      q = q.after(lane ? up : before);
      before = __shfl_sync(0xffffffffu, end, 31);
      const int cnt = (q.len + kRows - 1) / kRows;
      int inc = cnt;
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += up;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, left < inc);
      if (hit) {
        const int w = __ffs(hit) - 1;
        seq = b0 + w;
        own = {__shfl_sync(0xffffffffu, q.start, w), __shfl_sync(0xffffffffu, q.len, w)};
        blk = left - (__shfl_sync(0xffffffffu, inc, w) - __shfl_sync(0xffffffffu, cnt, w));
      } else {
        left -= __shfl_sync(0xffffffffu, inc, 31);
      }
    }
    if (lane == 0) {
      s_seq = seq;
      s_blk = blk;
      s_span = own;
    }
    if (blockIdx.x == 0 && blockIdx.y == 0)
      for (int b = lane; b < a.B; b += 32)
        if (packed::span_bad(a.cu_q, b, a.Tq) || packed::span_bad(a.cu_k, b, a.Tk))
          atomicOr(&g_packed_simt_status, DEV_BAD_INDEX);
  }
  __syncthreads();
  const int seq = s_seq;
  if (seq == -2) return;
  const packed::Span sq = s_span;
  const packed::Span sk = seq < 0 || seq >= a.B ? packed::Span{0, 0} : packed::span_of(a.cu_k, seq, a.B, a.Tk);
  const int head = blockIdx.y, kvh = head / (a.Hq / a.Hk);
  const int i0 = s_blk * kRows, off = sk.len - sq.len;
  const T* q = static_cast<const T*>(a.q) + sq.start * a.s[0] + head * a.s[1];
  const T* k = static_cast<const T*>(a.k) + sk.start * a.s[3] + kvh * a.s[4];
  const T* v = static_cast<const T*>(a.v) + sk.start * a.s[6] + kvh * a.s[7];
  T* o = static_cast<T*>(a.o) + sq.start * a.s[9] + head * a.s[10];

  for (int e = threadIdx.x; e < kRows * kMaxD; e += kThreads) {
    const int r = e / kMaxD, d = e % kMaxD;
    Qs[r][d] = i0 + r < sq.len && d < a.D ? to_f32<T>(q[(i0 + r) * a.s[0] + d * a.s[2]]) * a.scale_log2 : 0.f;
  }
  // keys [0, lim) for query i; a block needs those of its last query
  auto limit = [&](int i) { return a.causal ? min(sk.len, max(0, i + off + 1)) : sk.len; };
  const int last = min(i0 + kRows, sq.len) - 1;
  const int n = limit(last);
  int lim[4];
  float m[4], l[4], acc[4][kMaxD / 32];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    lim[r] = limit(i0 + warp * 4 + r);
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int c = 0; c < kMaxD / 32; ++c) acc[r][c] = 0.f;
  }
  for (int j0 = 0; j0 < n; j0 += kKeys) {
    __syncthreads();
    for (int e = threadIdx.x; e < kKeys * kMaxD; e += kThreads) {
      const int r = e / kMaxD, d = e % kMaxD;
      const bool in = j0 + r < sk.len && d < a.D;
      Ks[r][d] = in ? to_f32<T>(k[(j0 + r) * a.s[3] + d * a.s[5]]) : 0.f;
      Vs[r][d] = in ? to_f32<T>(v[(j0 + r) * a.s[6] + d * a.s[8]]) : 0.f;
    }
    __syncthreads();
    float s[4] = {};
    for (int d = 0; d < a.D; ++d) {
      const float kd = Ks[lane][d];
#pragma unroll
      for (int r = 0; r < 4; ++r) s[r] = fmaf(Qs[warp * 4 + r][d], kd, s[r]);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int kept = min(kKeys, lim[r] - j0);  // uniform in the warp
      if (kept <= 0) continue;
      if (lane >= kept) s[r] = -INFINITY;
      float mx = s[r];
      for (int x = 16; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
      const float mn = fmaxf(m[r], mx), base = mn == -INFINITY ? 0.f : mn;
      const float al = exp2f(m[r] - base), p = exp2f(s[r] - base);
      m[r] = mn;
      float sum = p;
      for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
      l[r] = l[r] * al + sum;
#pragma unroll
      for (int c = 0; c < kMaxD / 32; ++c) acc[r][c] *= al;
      for (int x = 0; x < kept; ++x) {
        const float px = __shfl_sync(0xffffffffu, p, x);
#pragma unroll
        for (int c = 0; c < kMaxD / 32; ++c) acc[r][c] = fmaf(px, Vs[x][lane + 32 * c], acc[r][c]);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int i = i0 + warp * 4 + r;
    if (i >= sq.len) continue;
#pragma unroll
    for (int c = 0; c < kMaxD / 32; ++c) {
      const int d = lane + 32 * c;
      if (d < a.D) o[i * a.s[9] + d * a.s[11]] = from_f32<T>(lim[r] > 0 ? acc[r][c] / l[r] : 0.f);
    }
  }
}

template <typename T>
int launch(const SimtArgs& a, cudaStream_t st) {
  const long long blocks = (long long)a.Tq / kRows + a.B + 2;  // at most: one partial block a sequence
  fa_packed_simt_kernel<T><<<dim3((unsigned)blocks, (unsigned)a.Hq), kThreads, 0, st>>>(a);
  B2_CHECK_LAUNCH();
  return B2_OK;
}

}  // namespace

int fa_packed_simt_launch(const PackedCall& c, cudaStream_t st) {
  SimtArgs a = {};
  a.q = c.q;
  a.k = c.k;
  a.v = c.v;
  a.o = c.o;
  a.cu_q = c.cu_q;
  a.cu_k = c.cu_k;
  for (int i = 0; i < 12; ++i) a.s[i] = c.strides[i];
  a.B = (int)c.B;
  a.Tq = (int)c.Tq;
  a.Tk = (int)c.Tk;
  a.Hq = (int)c.Hq;
  a.Hk = (int)c.Hk;
  a.D = (int)c.D;
  a.causal = c.causal;
  a.scale_log2 = c.sm_scale * kLog2e;
  switch (c.dtype) {
    case B2_F32: return launch<float>(a, st);
    case B2_F16: return launch<__half>(a, st);
    default: return launch<__nv_bfloat16>(a, st);
  }
}

uint32_t fa_packed_simt_read_status(bool clear) {
  uint32_t v = 0;
  cudaMemcpyFromSymbol(&v, g_packed_simt_status, sizeof(v));
  if (clear) {
    const uint32_t z = 0;
    cudaMemcpyToSymbol(g_packed_simt_status, &z, sizeof(z));
  }
  return v;
}

}  // namespace b2
