// Attention of the newest N tokens of each sequence over the 4-bit paged cache, fp16
// and bf16 queries (the row kernel of kv_attn.cu serves fp32).
//
// With k_j = ck_j s_j + lo_j per group g of channels (kv_cache.cu), and likewise v:
//   score_rj = sum_g sk_jg (q_r . ck_j)_g + lok_jg (sum of q_r)_g
//   o_rd     = sum_j (p_rj sv_jg) cv_jd + sum_j p_rj lov_jg
// so the codes themselves are what is multiplied, and scales and lowest values
// touch one number per key and group, not one per channel. A 4-bit code in the low
// mantissa bits of an fp16 is the subnormal c * 2^-24 (or c * 2^-20 four bits up),
// exactly, so two codes become a tensor-core operand by one AND; the powers of two
// go into q (a sixteenth for the odd codes) and into the last multiplication.
//
// Tensor work is mma.sync m16n8k16 with the codes as the A operand, straight from
// registers: S^T = K.Q^T (16 keys x 8 rows) and O^T = V^T.P^T (16 channels x 8
// rows). tcgen05 would need the widened codes written to shared or tensor memory
// first, four times the bytes that came in, and M = 128 rows where 1 to 16 exist.
// P^T comes from S^T's registers by one 8x8 transpose (movmatrix). The rows are the
// (token, head) pairs that share a key head: a key is read once for all of them.
//
// Work is split along the keys: all sequences' tiles of 128 keys form one line that
// is cut evenly among the CTAs (two per SM), whatever the lengths. Inside a tile
// each of 8 warps takes 16 keys. A warp's codes and scales come by cp.async into its
// own ring of shared memory, kStages deep, so no barrier is needed in the loop. At a
// sequence's end, or the CTA's, the warps' partial results are merged; a sequence
// cut between CTAs is joined by kv_attn_join_kernel from partials in the workspace,
// in the order of the keys.
//
// Softmax: the running maximum of a row is only raised when a score passes it by 2^8
// (one vote a step), P = 2^(s - m) then stays below 2^8. P * sv is rounded to fp16
// (the one rounding of weights, 2^-11); F, a power of two per warp, keeps sv * F
// within [.., 64] so that the product stays in fp16's range. Scores, sums, the lowest
// values' part and the accumulators are fp32.
#include "b2_common.cuh"
#include "decoder.cuh"
#include "kv_attn.cuh"

namespace b2 {
namespace {

constexpr int kWarps = 8, kThreads = 32 * kWarps, kStages = 4;
constexpr int kTile = 16 * kWarps;  // keys

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 8x8 transpose of 16-bit values across the warp
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float scale_of(uint32_t meta) { return __uint_as_float(meta << 16); }
__device__ __forceinline__ float low_of(uint32_t meta) { return __uint_as_float(meta & 0xffff0000u); }

template <int D, int GROUP>
struct Ring {
  static constexpr int NG = D / GROUP;
  static constexpr int kCodes = 16 * D / 2;        // bytes of 16 keys
  static constexpr int kScales = 16 * NG * 4;
  static constexpr int kStage = 2 * kCodes + 2 * kScales;
  static constexpr int kVCodes = kCodes, kKScales = 2 * kCodes, kVScales = 2 * kCodes + kScales;
};
// Where the V codes of key `row` (0..15), 16-byte piece `seg`, lie in their stage:
// the four keys 2t that the lanes t read together fall into different banks.
template <int D>
__device__ __forceinline__ int v_place(int row, int seg) {
  const int r = ((row >> 1) & 3) | ((row & 1) << 2) | (row & 8);
  if (D == 128) seg ^= ((r >> 1) & 1) << 1;
  return r * (D / 2) + seg * 16;
}

// Sum over the CTA of two numbers per thread.
struct Pair {
  long long a, b;
};
template <int WARPS>
__device__ __forceinline__ Pair block_sum(long long a, long long b, Pair* scratch) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = {a, b};
  __syncthreads();
  Pair s = {0, 0};
  for (int w = 0; w < WARPS; ++w) {
    s.a += scratch[w].a;
    s.b += scratch[w].b;
  }
  return s;
}

// A sequence's keys: 0 when the length is not one the page table can hold.
__device__ __forceinline__ int keys_of(const AttnArgs& a, int b) {
  const int n = a.lengths[b];
  return n < 0 || n > (long long)a.max_pages * a.page_size ? 0 : n;
}
__device__ __forceinline__ int tiles_of(const AttnArgs& a, int b) { return (keys_of(a, b) + kTile - 1) / kTile; }

// One row of the group: its token among the new ones and its query head.
__device__ __forceinline__ int row_token(const AttnArgs& a, int row) { return row / a.G; }

template <typename T, int D, int GROUP, int NT>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 2 : 1) kv_attn_kernel(const __grid_constant__ AttnArgs a) {
  using R = Ring<D, GROUP>;
  constexpr int NG = R::NG, N64 = D / 64, WPT = D / 32, ROWS = 8 * NT;
  extern __shared__ __align__(16) uint8_t smem[];
  float* s_o = reinterpret_cast<float*>(smem + kWarps * kStages * R::kStage);  // [warp][row][D + 4]
  float* s_m = s_o + kWarps * ROWS * (D + 4);                                  // [warp][row]
  float* s_l = s_m + kWarps * ROWS;
  __shared__ Pair s_sum[kWarps];
  __shared__ int s_seq;
  __shared__ long long s_first;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int segs = a.H * a.row_blocks;  // lines of tiles per sequence

  // ---- this CTA's part of the line of all tiles
  asm volatile("griddepcontrol.launch_dependents;");
  long long total = 0;
  {
    long long mine = 0;
    for (int b = threadIdx.x; b < a.B; b += kThreads) mine += tiles_of(a, b);
    total = block_sum<kWarps>(mine, 0, s_sum).a * segs;
  }
  const long long ctas = total < gridDim.x ? total : gridDim.x;
  if (blockIdx.x >= ctas) return;
  const long long begin = blockIdx.x * total / ctas, end = (blockIdx.x + 1) * total / ctas;
  {
    // the sequence that holds tile `begin`: prefix sums, kThreads sequences at a time
    long long before = 0;
    for (int b0 = 0; b0 < a.B; b0 += kThreads) {
      const int b = b0 + threadIdx.x;
      const long long n = b < a.B ? (long long)tiles_of(a, b) * segs : 0;
      long long inc = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += up;
      }
      __syncthreads();
      if (lane == 31) s_sum[warp] = {inc, 0};
      __syncthreads();
      long long base = before;
      for (int w = 0; w < warp; ++w) base += s_sum[w].a;
      if (n > 0 && begin >= base + inc - n && begin < base + inc) {
        s_seq = b;
        s_first = base + inc - n;
      }
      for (int w = 0; w < kWarps; ++w) before += s_sum[w].a;
      if (before > begin) break;
    }
    __syncthreads();
  }

  // A place on the line: sequence, segment (key head and row block), tile.
  struct Cursor {
    int b, seg, tile, tiles, keys;
  };
  auto settle = [&](Cursor& c) {  // at the end of a segment: to the next one that has tiles
    if (c.tile < c.tiles) return;
    c.tile = 0;
    if (++c.seg < segs) return;
    c.seg = 0;
    do {
      if (++c.b >= a.B) {
        c.tiles = 0;
        return;
      }
      c.keys = keys_of(a, c.b);
      c.tiles = (c.keys + kTile - 1) / kTile;
    } while (c.tiles == 0);
  };
  Cursor at;
  at.b = s_seq;
  at.keys = keys_of(a, at.b);
  at.tiles = (at.keys + kTile - 1) / kTile;
  at.seg = (int)((begin - s_first) / at.tiles);
  at.tile = (int)((begin - s_first) - (long long)at.seg * at.tiles);

  // ---- loads, kStages - 1 tiles ahead
  uint8_t* ring = smem + warp * (kStages * R::kStage);
  const uint32_t ring_addr = (uint32_t)__cvta_generic_to_shared(ring);
  const int cpp = a.page_size / 16;  // chunks per page
  Cursor ld = at;
  long long ld_pos = begin;
  int ld_page = 0, ld_off = 0;
  bool ld_has = false;
  unsigned bad_stages = 0;  // a stage whose page lies outside the cache
  auto ld_lookup = [&] {    // the page of this warp's 16 keys of the tile; used one step later
    const int chunk = ld.tile * kWarps + warp;
    ld_has = ld_pos < end && chunk * 16 < ld.keys;
    if (ld_has) {
      const int idx = chunk / cpp;
      ld_off = chunk - idx * cpp;
      ld_page = a.page_table[ld.b * a.table_stride + idx];
    }
  };
  auto ld_issue = [&](int stage) {
    if (ld_has) {
      const bool bad = ld_page < 0 || ld_page >= a.num_pages;
      bad_stages = (bad_stages & ~(1u << stage)) | ((bad ? 1u : 0u) << stage);
      const int kvh = ld.seg / a.row_blocks;
      const size_t row = ((size_t)(bad ? 0 : ld_page) * a.H + kvh) * a.page_size + ld_off * 16;
      const uint8_t* kc = a.k_codes + row * (D / 2);
      const uint8_t* vc = a.v_codes + row * (D / 2);
      const uint32_t dst = ring_addr + stage * R::kStage;
#pragma unroll
      for (int i = 0; i < R::kCodes / 512; ++i) {
        const int piece = i * 32 + lane;
        cp_async16(dst + piece * 16, kc + piece * 16);
        constexpr int kSegs = D / 32;  // 16-byte pieces of a row
        cp_async16(dst + R::kVCodes + v_place<D>(piece / kSegs, piece % kSegs), vc + piece * 16);
      }
      constexpr int kPieces = R::kScales / 16;
      if (lane < 2 * kPieces) {
        const int p = lane % kPieces;
        const uint8_t* src = reinterpret_cast<const uint8_t*>(lane < kPieces ? a.k_scales : a.v_scales) + row * (NG * 4);
        cp_async16(dst + (lane < kPieces ? R::kKScales : R::kVScales) + p * 16, src + p * 16);
      }
    }
    cp_async_commit();
    if (ld_pos < end) {
      ++ld_pos;
      ++ld.tile;
      settle(ld);
      ld_lookup();
    }
  };
  ld_lookup();
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) ld_issue(s);

  // ---- a segment's state
  uint32_t qf[NT][WPT][2][2];          // B operands: code word, low or high byte pair, register
  float f[NT][2], qs[NT][NG][2];       // per column: factor of the code part, scaled sums of q
  int lim[NT][2];                      // keys each column's row keeps
  float m[NT][2], mu[NT][2], l[NT][2], lo[NT][NG][2];
  float o[N64 * 4][NT][4];
  float F = 0.f;
  int keys_all = 0;                    // keys that every row keeps

  auto begin_segment = [&](const Cursor& c) {
    const int kvh = c.seg / a.row_blocks, rb = c.seg - kvh * a.row_blocks;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = rb * ROWS + nt * 8 + g;
      float x[N64][16];
      if (row < a.rows) {
        const int n = row_token(a, row);
        const T* q = static_cast<const T*>(a.q) + (long long)c.b * a.qb + n * a.qn +
                     (long long)(kvh * a.G + row - n * a.G) * a.qh + 16 * t;
#pragma unroll
        for (int w = 0; w < N64; ++w) {
          if (a.q_vec) {
            uint4 r[2];
            r[0] = *reinterpret_cast<const uint4*>(q + 64 * w);
            r[1] = *reinterpret_cast<const uint4*>(q + 64 * w + 8);
            const T* e = reinterpret_cast<const T*>(r);
#pragma unroll
            for (int i = 0; i < 16; ++i) x[w][i] = to_f32<T>(e[i]);
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) x[w][i] = to_f32<T>(q[64 * w + i]);
          }
        }
      } else {
#pragma unroll
        for (int w = 0; w < N64; ++w)
#pragma unroll
          for (int i = 0; i < 16; ++i) x[w][i] = 0.f;
      }
      // A power of two per row brings its largest value to 2^14 .. 2^15 in fp16: no
      // value down to 2^-28 of it becomes subnormal, and a sixteenth of it fits too.
      float top = 0.f;
#pragma unroll
      for (int w = 0; w < N64; ++w)
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(x[w][i]));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int e = min(max(268 - (int)(__float_as_uint(top) >> 23), 1), 254);
      const float up = __int_as_float(e << 23), down = __int_as_float((254 - e) << 23);
      float sum[NG] = {};
#pragma unroll
      for (int w = 0; w < N64; ++w)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          sum[NG == 2 ? w : 0] += x[w][i];
          x[w][i] *= up;
        }
#pragma unroll
      for (int k = 0; k < NG; ++k) {
        sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], 1);
        sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], 2);
      }
      // word ii*N64 + w of the lane holds channels 64w + 16t + 8ii ..; its codes pair
      // up as (0,4) (1,5) | (2,6) (3,7)
#pragma unroll
      for (int w = 0; w < N64; ++w)
#pragma unroll
        for (int ii = 0; ii < 2; ++ii)
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            const int c0 = 8 * ii + 2 * s;
            qf[nt][ii * N64 + w][s][0] = half2_bits(x[w][c0], x[w][c0 + 4]);
            qf[nt][ii * N64 + w][s][1] = half2_bits(x[w][c0 + 1] * 0.0625f, x[w][c0 + 5] * 0.0625f);
          }
      // to the lanes that hold the row's scores: columns 2t, 2t + 1
#pragma unroll
      for (int c2 = 0; c2 < 2; ++c2) {
        const int src = (2 * t + c2) * 4;
        f[nt][c2] = __shfl_sync(0xffffffffu, down, src) * (16777216.f * a.scale_log2);
#pragma unroll
        for (int k = 0; k < NG; ++k) qs[nt][k][c2] = __shfl_sync(0xffffffffu, sum[k], src) * a.scale_log2;
        const int r = rb * ROWS + nt * 8 + 2 * t + c2;
        // rows that do not exist keep what the last token keeps
        lim[nt][c2] = r < a.rows ? max(0, c.keys - a.N + 1 + row_token(a, r)) : c.keys;
        m[nt][c2] = -INFINITY;
        mu[nt][c2] = 0.f;
        l[nt][c2] = 0.f;
#pragma unroll
        for (int k = 0; k < NG; ++k) lo[nt][k][c2] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < N64 * 4; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) o[i][nt][k] = 0.f;
    }
    F = __int_as_float(254 << 23);
    keys_all = max(0, c.keys - a.N + 1);
  };

  // ---- 16 keys
  auto step = [&](const uint8_t* st, int key0, int keys, bool bad) {
    // scores
    uint32_t k0[WPT], k1[WPT];
    if constexpr (D == 128) {
      *reinterpret_cast<uint4*>(k0) = *reinterpret_cast<const uint4*>(st + g * 64 + t * 16);
      *reinterpret_cast<uint4*>(k1) = *reinterpret_cast<const uint4*>(st + (g + 8) * 64 + t * 16);
    } else {
      *reinterpret_cast<uint2*>(k0) = *reinterpret_cast<const uint2*>(st + g * 32 + t * 8);
      *reinterpret_cast<uint2*>(k1) = *reinterpret_cast<const uint2*>(st + (g + 8) * 32 + t * 8);
    }
    uint32_t km[2][NG], vm[2][NG];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int k = 0; k < NG; ++k) {
        km[h][k] = *reinterpret_cast<const uint32_t*>(st + R::kKScales + ((g + 8 * h) * NG + k) * 4);
        vm[h][k] = *reinterpret_cast<const uint32_t*>(st + R::kVScales + ((g + 8 * h) * NG + k) * 4);
      }
    float acc[NG][NT][4] = {};
#pragma unroll
    for (int w = 0; w < WPT; ++w)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const uint32_t x0 = s ? k0[w] >> 8 : k0[w], x1 = s ? k1[w] >> 8 : k1[w];
        const uint32_t a0 = x0 & 0x000f000fu, a1 = x1 & 0x000f000fu;
        const uint32_t a2 = x0 & 0x00f000f0u, a3 = x1 & 0x00f000f0u;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          mma16816(acc[NG == 2 ? w % N64 : 0][nt], a0, a1, a2, a3, qf[nt][w][s][0], qf[nt][w][s][1]);
      }
    float sc[NT][4], sv[2][NG], lv[2][NG];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int k = 0; k < NG; ++k) {
        sv[h][k] = scale_of(vm[h][k]);
        lv[h][k] = low_of(vm[h][k]);
      }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int h = i >> 1, c2 = i & 1;
        float x = scale_of(km[h][0]) * acc[0][nt][i], y = low_of(km[h][0]) * qs[nt][0][c2];
        if constexpr (NG == 2) {
          x = fmaf(scale_of(km[h][1]), acc[1][nt][i], x);
          y = fmaf(low_of(km[h][1]), qs[nt][1][c2], y);
        }
        sc[nt][i] = fmaf(x, f[nt][c2], y);
      }
    const bool edge = key0 + 16 > keys_all;  // some row keeps only a part
    if (edge) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int key = key0 + g + 8 * h;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c2 = 0; c2 < 2; ++c2)
            if (key >= lim[nt][c2]) sc[nt][2 * h + c2] = -INFINITY;
        // past the sequence the page holds anything
        if (key >= keys)
#pragma unroll
          for (int k = 0; k < NG; ++k) sv[h][k] = lv[h][k] = 0.f;
      }
    }
    // raise the maxima, or lower F, where needed
    bool raise = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c2 = 0; c2 < 2; ++c2) raise = raise || fmaxf(sc[nt][c2], sc[nt][2 + c2]) > m[nt][c2] + 8.f;
#pragma unroll
    for (int k = 0; k < NG; ++k) raise = raise || fmaxf(sv[0][k], sv[1][k]) * F > 64.f;
    if (__any_sync(0xffffffffu, raise)) {
      float top = 0.f;
#pragma unroll
      for (int k = 0; k < NG; ++k) top = fmaxf(top, fmaxf(sv[0][k], sv[1][k]));  // NaN is left aside
      const uint32_t top_bits = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
      float ratio = 1.f;
      if (__uint_as_float(top_bits) * F > 64.f) {
        const float to = __int_as_float(min(max(259 - (int)(top_bits >> 23), 1), 254) << 23);
        ratio = to / F;
        F = to;
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c2 = 0; c2 < 2; ++c2) {
          float x = fmaxf(sc[nt][c2], sc[nt][2 + c2]);
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
          const float to = fmaxf(m[nt][c2], x);
          const float base = to == -INFINITY ? 0.f : to;
          const float al = ex2(m[nt][c2] - base);
          m[nt][c2] = to;
          mu[nt][c2] = base;
          l[nt][c2] *= al;
#pragma unroll
          for (int k = 0; k < NG; ++k) lo[nt][k][c2] *= al;
#pragma unroll
          for (int i = 0; i < N64 * 4; ++i) {
            o[i][nt][c2] *= al * ratio;
            o[i][nt][2 + c2] *= al * ratio;
          }
        }
    }
    // weights, and their products with the values' scales as the B operand
    uint32_t pf[NT][NG][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float p[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[i] = ex2(sc[nt][i] - mu[nt][i & 1]);
        l[nt][i & 1] += p[i];
      }
#pragma unroll
      for (int k = 0; k < NG; ++k) {
        float w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = p[i] * (sv[i >> 1][k] * F);
        float y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = p[i] * lv[i >> 1][k];
        if (edge) {
          // a row's own masked keys count for nothing, NaN or not
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (key0 + g + 8 * (i >> 1) >= lim[nt][i & 1]) w[i] = y[i] = 0.f;
        }
        lo[nt][k][0] += y[0] + y[2];
        lo[nt][k][1] += y[1] + y[3];
        pf[nt][k][0] = transpose8(half2_bits(w[0], w[1]));
        pf[nt][k][1] = transpose8(half2_bits(w[2], w[3]));
      }
    }
    if (bad) {  // no such page: every row that reaches it is undefined
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c2 = 0; c2 < 2; ++c2)
          if (key0 < lim[nt][c2]) l[nt][c2] = __int_as_float(0x7fffffff);
    }
    // values
#pragma unroll
    for (int w = 0; w < N64; ++w) {
      uint32_t x[4];  // keys 2t, 2t+1, 2t+8, 2t+9: channels 64w + 8g ..
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 2 * t + (i & 1) + 8 * (i >> 1);
        if constexpr (D == 128) {
          const uint2 y = *reinterpret_cast<const uint2*>(st + R::kVCodes + v_place<D>(row, g >> 1) + (g & 1) * 8);
          x[i] = w ? y.y : y.x;
        } else {
          x[i] = *reinterpret_cast<const uint32_t*>(st + R::kVCodes + v_place<D>(row, g >> 2) + (g & 3) * 4);
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {  // codes 4h .. 4h+3 of each word
        uint32_t p0 = __byte_perm(x[0], x[1], h ? 0x7632 : 0x5410);
        uint32_t p1 = __byte_perm(x[2], x[3], h ? 0x7632 : 0x5410);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const uint32_t a0 = p0 & 0x000f000fu, a1 = p0 & 0x00f000f0u;
          const uint32_t a2 = p1 & 0x000f000fu, a3 = p1 & 0x00f000f0u;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            mma16816(o[w * 4 + 2 * h + s][nt], a0, a1, a2, a3, pf[nt][NG == 2 ? w : 0][0], pf[nt][NG == 2 ? w : 0][1]);
          p0 >>= 8;
          p1 >>= 8;
        }
      }
    }
  };

  // ---- merge the warps' results of a segment
  auto end_segment = [&](const Cursor& c, long long seg_begin) {
    const int kvh = c.seg / a.row_blocks, rb = c.seg - kvh * a.row_blocks;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c2 = 0; c2 < 2; ++c2) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
          l[nt][c2] += __shfl_xor_sync(0xffffffffu, l[nt][c2], d);
#pragma unroll
          for (int k = 0; k < NG; ++k) lo[nt][k][c2] += __shfl_xor_sync(0xffffffffu, lo[nt][k][c2], d);
        }
        const int r = nt * 8 + 2 * t + c2;
        if (g == 0) {
          s_m[warp * ROWS + r] = m[nt][c2];
          s_l[warp * ROWS + r] = l[nt][c2];
        }
        const float down = 1.f / F;  // a power of two, in range; 2^24 / F need not be
#pragma unroll
        for (int i = 0; i < N64 * 4; ++i) {
          const int d = 64 * (i / 4) + 8 * g + 2 * (i % 4);
          const float y = lo[nt][NG == 2 ? i / 4 : 0][c2];
          const float2 v = {fmaf(o[i][nt][c2] * 16777216.f, down, y), fmaf(o[i][nt][2 + c2] * 1048576.f, down, y)};
          *reinterpret_cast<float2*>(s_o + (warp * ROWS + r) * (D + 4) + d) = v;
        }
      }
    __syncthreads();
    const bool whole = seg_begin >= begin && seg_begin + c.tiles <= end;
    // the CTA's first cut segment goes to its slot 0 when it began before the CTA
    const int slot = seg_begin < begin ? 0 : 1;
    float* part = a.partials + (size_t)(2 * blockIdx.x + slot) * ROWS * (D + 2);
    for (int e = threadIdx.x; e < ROWS * (D / 4); e += kThreads) {
      const int r = e / (D / 4), d = (e % (D / 4)) * 4;
      const int row = rb * ROWS + r;
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_m[w * ROWS + r]);
      const float base = top == -INFINITY ? 0.f : top;
      float sum = 0.f;
      float4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float x = ex2(s_m[w * ROWS + r] - base);
        const float4 y = *reinterpret_cast<const float4*>(s_o + (w * ROWS + r) * (D + 4) + d);
        sum = fmaf(x, s_l[w * ROWS + r], sum);
        v.x = fmaf(x, y.x, v.x);
        v.y = fmaf(x, y.y, v.y);
        v.z = fmaf(x, y.z, v.z);
        v.w = fmaf(x, y.w, v.w);
      }
      if (whole) {
        if (row < a.rows) {
          const int n = row_token(a, row);
          const bool any = c.keys - a.N + 1 + n > 0;
          T* out = static_cast<T*>(a.o) + (long long)c.b * a.ob + n * a.on + (long long)(kvh * a.G + row - n * a.G) * a.oh + d;
          const float inv = any ? 1.f / sum : 0.f;
          out[0] = from_f32<T>(any ? v.x * inv : 0.f);
          out[1] = from_f32<T>(any ? v.y * inv : 0.f);
          out[2] = from_f32<T>(any ? v.z * inv : 0.f);
          out[3] = from_f32<T>(any ? v.w * inv : 0.f);
        }
      } else {
        *reinterpret_cast<float4*>(part + r * D + d) = v;
        if (d == 0) {
          part[ROWS * D + r] = top;
          part[ROWS * D + ROWS + r] = sum;
        }
      }
    }
    __syncthreads();
  };

  // ---- the line
  long long seg_begin = begin - at.tile;  // of the segment at hand
  begin_segment(at);
  int stage = 0;
  for (long long pos = begin; pos < end; ++pos) {
    cp_async_wait<kStages - 2>();
    __syncwarp();  // the other lanes' pieces have landed, and all are done with the oldest stage
    const bool bad = (bad_stages >> stage) & 1;  // before the next issue reuses the bit
    ld_issue((stage + kStages - 1) % kStages);
    const int key0 = (at.tile * kWarps + warp) * 16;
    if (key0 < at.keys) {
      if (bad && lane == 0) atomicOr(a.status, DEV_BAD_INDEX);
      step(ring + stage * R::kStage, key0, at.keys, bad);
    }
    stage = (stage + 1) % kStages;
    const bool last = at.tile + 1 == at.tiles;
    if (last || pos + 1 == end) {
      end_segment(at, seg_begin);
      if (pos + 1 < end) {
        seg_begin = pos + 1;
        ++at.tile;
        settle(at);
        begin_segment(at);
      }
    } else {
      ++at.tile;
    }
  }
  cp_async_wait<0>();
}

// Joins the parts of the segments that were cut between CTAs; writes the rows of
// sequences without tiles (no key, or a length that cannot be).
template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(kThreads) kv_attn_join_kernel(const __grid_constant__ AttnArgs a, long long grid) {
  __shared__ Pair s_sum[kWarps];
  const int segs = a.H * a.row_blocks;
  const int b = blockIdx.x / segs, seg = blockIdx.x - b * segs;
  const int kvh = seg / a.row_blocks, rb = seg - kvh * a.row_blocks;
  const int tiles = tiles_of(a, b);
  long long before = 0, total = 0;
  if (tiles > 0) {
    long long mine_before = 0, mine = 0;
    for (int i = threadIdx.x; i < a.B; i += kThreads) {
      const int n = tiles_of(a, i);
      mine += n;
      if (i < b) mine_before += n;
    }
    const Pair s = block_sum<kWarps>(mine, mine_before, s_sum);
    total = s.a * segs;
    before = s.b * segs + (long long)seg * tiles;
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int held = a.lengths[b];
  const bool wrong = tiles == 0 && held != 0;
  long long c0 = 0, c1 = 0;
  if (tiles > 0) {
    const long long ctas = total < grid ? total : grid;
    // CTA c holds tiles [c * total / ctas, (c + 1) * total / ctas)
    c0 = ((before + 1) * ctas - 1) / total;
    c1 = ((before + tiles) * ctas - 1) / total;
    if (c0 == c1) return;  // whole in one CTA, which wrote it
  } else if (wrong && threadIdx.x == 0) {
    atomicOr(a.status, DEV_BAD_INDEX);
  }
  const size_t stride = (size_t)ROWS * (D + 2);
  for (int e = threadIdx.x; e < ROWS * (D / 4); e += kThreads) {
    const int r = e / (D / 4), d = (e % (D / 4)) * 4;
    const int row = rb * ROWS + r;
    if (row >= a.rows) continue;
    const int n = row_token(a, row);
    float4 v = {0.f, 0.f, 0.f, 0.f};
    if (tiles > 0 && held - a.N + 1 + n > 0) {
      // the first CTA's part began in it (slot 1), the others' began before them
      auto part = [&](long long c) { return a.partials + (size_t)(2 * c + (c == c0 ? 1 : 0)) * stride; };
      float top = -INFINITY;
      for (long long c = c0; c <= c1; ++c) top = fmaxf(top, part(c)[ROWS * D + r]);
      const float base = top == -INFINITY ? 0.f : top;
      float sum = 0.f;
#pragma unroll 4
      for (long long c = c0; c <= c1; ++c) {
        const float* p = part(c);
        const float x = ex2(p[ROWS * D + r] - base);
        const float4 y = *reinterpret_cast<const float4*>(p + r * D + d);
        sum = fmaf(x, p[ROWS * D + ROWS + r], sum);
        v.x = fmaf(x, y.x, v.x);
        v.y = fmaf(x, y.y, v.y);
        v.z = fmaf(x, y.z, v.z);
        v.w = fmaf(x, y.w, v.w);
      }
      v.x /= sum;
      v.y /= sum;
      v.z /= sum;
      v.w /= sum;
    } else if (wrong) {
      v.x = v.y = v.z = v.w = __int_as_float(0x7fffffff);
    }
    T* out = static_cast<T*>(a.o) + (long long)b * a.ob + n * a.on + (long long)(kvh * a.G + row - n * a.G) * a.oh + d;
    out[0] = from_f32<T>(v.x);
    out[1] = from_f32<T>(v.y);
    out[2] = from_f32<T>(v.z);
    out[3] = from_f32<T>(v.w);
  }
}

constexpr int kMaxGrid = 2 * 160;  // CTAs that the workspace has room for

template <typename T, int D, int GROUP, int NT>
int launch(AttnArgs& a, cudaStream_t st) {
  using R = Ring<D, GROUP>;
  constexpr int ROWS = 8 * NT;
  constexpr size_t smem = (size_t)kWarps * kStages * R::kStage + (size_t)kWarps * ROWS * (D + 6) * sizeof(float);
  a.row_blocks = (a.rows + ROWS - 1) / ROWS;
  const long long segs = (long long)a.B * a.H * a.row_blocks;
  if (segs >= (1LL << 31)) {
    set_error("b2_kv_cache_attn: B * H * row blocks must be < 2^31");
    return B2_EINVAL;
  }
  auto kern = kv_attn_kernel<T, D, GROUP, NT>;
  B2_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  int grid = device_sm_count() * (NT == 1 ? 2 : 1);
  if (grid > kMaxGrid) grid = kMaxGrid;
  kern<<<grid, kThreads, smem, st>>>(a);
  B2_CHECK_LAUNCH();
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)segs);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  B2_CUDA_TRY(cudaLaunchKernelEx(&cfg, kv_attn_join_kernel<T, D, ROWS>, a, (long long)grid));
  return B2_OK;
}

template <typename T>
int launch_typed(AttnArgs& a, int D, int group, cudaStream_t st) {
  const bool one = a.rows <= 8;
  if (D == 64) return one ? launch<T, 64, 64, 1>(a, st) : launch<T, 64, 64, 2>(a, st);
  if (group == 64) return one ? launch<T, 128, 64, 1>(a, st) : launch<T, 128, 64, 2>(a, st);
  return one ? launch<T, 128, 128, 1>(a, st) : launch<T, 128, 128, 2>(a, st);
}

}  // namespace

size_t kv_attn_mma_workspace(int64_t rows, int64_t D) {
  return sizeof(float) * 2 * kMaxGrid * (size_t)(rows <= 8 ? 8 : 16) * (size_t)(D + 2);
}

int kv_attn_mma_launch(AttnArgs& a, int D, int group, int dtype, cudaStream_t st) {
  return dtype == B2_F16 ? launch_typed<__half>(a, D, group, st) : launch_typed<__nv_bfloat16>(a, D, group, st);
}

}  // namespace b2
