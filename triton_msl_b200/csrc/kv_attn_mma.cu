// Attention of the newest N tokens of each sequence over the 4-bit paged cache, fp16
// and bf16 queries (the row kernel of kv_attn.cu serves fp32).
//
// With k_j = ck_j s_j + lo_j per group g of channels (kv_cache.cu), and likewise v:
//   score_rj = sum_g sk_jg (q_r . ck_j)_g + lok_jg (sum of q_r)_g
//   o_rd     = sum_j (p_rj sv_jg) cv_jd + sum_j p_rj lov_jg
// so the codes themselves are what is multiplied, and scales and lowest values
// touch one number per key and group, not one per channel. A 4-bit code c0 in the low
// mantissa bits of an fp16 is the subnormal c0 * 2^-24, exactly, 16 c1 beside it is
// 16 c1 * 2^-24, and a byte of two codes is (c0 + 16 c1) * 2^-24. So a word of 8 codes
// becomes tensor-core operands by 5 instructions for keys, q0 c0 + q1/16 (16 c1), and by 4
// for values, whose bytes give sums from which the c0's are taken at the end. q0 and
// q1/16 are exact in fp16. (Bytes for the keys too want q0 - q1/16, which has to be
// rounded: 1 to 1.5 % faster, 36.5 us where this takes 37.0, 116.4 where 118.2, but scores
// of bf16 queries of 30 were off by up to 0.1.) For fp16 the values take more as well
// (kBytes below). The powers of two go into the last multiplication.
//
// Tensor work is mma.sync m16n8k16 with the codes as the A operand, straight from
// registers: S^T = K.Q^T (16 keys x 8 rows) and O^T = V^T.P^T (16 channels x 8
// rows). tcgen05 would need the widened codes written to shared or tensor memory
// first, four times the bytes that came in, and M = 128 rows where 1 to 16 exist.
// P^T comes from S^T's registers by one 8x8 transpose (movmatrix). The rows are the
// (token, head) pairs that share a key head: a key is read once for all of them.
//
// Work is split along the keys: all sequences' tiles of 128 keys form one line that
// is cut evenly among the CTAs (two to four per SM), whatever the lengths. Inside a tile
// each of 4 warps takes 32 keys. A warp's codes and scales come by cp.async into its
// own two buffers of shared memory, so no barrier is needed in the loop. At a
// sequence's end, or the CTA's, the warps' partial results are merged; a sequence cut
// between CTAs is joined by kv_attn_join_kernel from partials in the workspace, in the
// order of the keys.
//
// Bound: instructions, a third of which widen codes, and the waits between dependent ones
// at 16 warps an SM (ALU pipe 56 %, issue slots 58 %), and, on long sequences, HBM.
// Measured, 32 query heads on 8, D = 128, groups of 64, bf16: 32 sequences of up to 8192
// tokens 37.2 us, 4.2 TB/s; of up to 32768 118.8 us, 5.3.
//
// Softmax: P = 2^(s - m), and P * sv is rounded to fp16 (the one rounding of weights,
// 2^-11). So m follows the largest product P * sv of a row and not its largest score: the
// first keys' lies at 2^7 to 2^8, and m is raised when one passes 2^15.5 (one vote a step).
// A product of 2^-21 of the largest so far is not yet subnormal, and large values of small
// weight leave the others their bits. Scores, sums, the lowest values' part and the
// accumulators are fp32; P itself, at most 2^85.5, only meets those.
#include <type_traits>

#include "b2_common.cuh"
#include "decoder.cuh"
#include "fa_math.cuh"
#include "kv_attn.cuh"

namespace b2 {
namespace {

using namespace fa;

constexpr int kWarps = 4, kThreads = 32 * kWarps, kStages = 2;
constexpr int kSteps = 2;                    // of 16 keys a warp and tile
constexpr int kTile = 16 * kSteps * kWarps;  // keys
// Maximum of no scores.
constexpr float kNoMax = -3e38f;
// Bounds of log2(P * sv): where a row's m puts the largest, and where m is raised.
constexpr float kPut = 8.f, kRaise = 15.5f;

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

// A sequence's keys: 0 when the length is not one the page table can hold.
__device__ __forceinline__ int keys_of(const AttnArgs& a, int b) {
  const int n = a.lengths[b];
  return n < 0 || n > (long long)a.max_pages * a.page_size ? 0 : n;
}
__device__ __forceinline__ int tiles_of(const AttnArgs& a, int b) { return (keys_of(a, b) + kTile - 1) / kTile; }

// The line of all work: sequence after sequence, in each segment after segment (key
// head, block of rows), a segment kSetup units for its start and end, then its tiles.
// CTA c of n holds units [share * c + min(c, more), ...). Measured on 32 sequences of
// up to 2048 / 8192 keys: kSetup 1: 15.7 / 37.7 us, 2: 15.6 / 36.7, 3: 16.6 / 37.7.
constexpr int kSetup = 2;
struct Line {
  unsigned share, more, ctas;
  __device__ Line(unsigned total, unsigned grid) {
    ctas = min(total, grid);
    share = ctas ? total / ctas : 0;
    more = total - share * ctas;
  }
  __device__ unsigned begin(unsigned c) const { return share * c + min(c, more); }
  __device__ unsigned owner(unsigned unit) const {
    const unsigned big = more * (share + 1);
    return unit < big ? unit / (share + 1) : more + (unit - big) / share;
  }
};
__device__ __forceinline__ unsigned units_of(int tiles) { return tiles ? tiles + kSetup : 0; }
// Units per segment of all sequences, and of those before b; the whole warp.
__device__ __forceinline__ unsigned count_units(const AttnArgs& a, int b, unsigned* before) {
  unsigned all = 0, some = 0;
#pragma unroll 4
  for (int i = threadIdx.x & 31; i < a.B; i += 32) {
    const unsigned n = units_of(tiles_of(a, i));
    all += n;
    if (i < b) some += n;
  }
  if (before) *before = __reduce_add_sync(0xffffffffu, some);
  return __reduce_add_sync(0xffffffffu, all);
}
// Bytes 0 and 2, or 1 and 3, of a word as the low bytes of two halves
__device__ __forceinline__ uint32_t byte_pair(uint32_t x, int odd) {
  return odd ? __byte_perm(x, 0, 0x4341) : x & 0x00ff00ffu;
}

// One row of the group: its token among the new ones and its query head.
__device__ __forceinline__ int row_token(const AttnArgs& a, int row) { return row / a.G; }

// CTAs per SM that the registers allow.
template <int D, int NT>
constexpr int kCtasPerSm = NT == 1 ? 4 : D == 64 ? 3 : 2;

// NT tiles of 8 columns (query rows). COLS = 2: every column is a row, a lane has two of
// each tile. COLS = 1, for at most 4 rows: rows are the even columns, so that a lane has
// one live column and the scores, exponentials and weights of the dead one are not
// computed (half of that work for the common 4 heads on a key head).
template <typename T, int D, int GROUP, int NT, int COLS>
__global__ void __launch_bounds__(kThreads, kCtasPerSm<D, NT>) kv_attn_kernel(const __grid_constant__ AttnArgs a) {
  using R = Ring<D, GROUP>;
  constexpr int NG = R::NG, N64 = D / 64, WPT = D / 32, ROWS = COLS * 4 * NT;
  // What bf16 results do not resolve and fp16 ones do (relative error of their output's
  // rounding 2.1e-4):
  // - Values' bytes as subnormals: their products' sums come out low by 2^-18 of their
  //   size. For fp16 the bytes lie 3 bits higher, where the largest are normal numbers
  //   (4 sequences of up to 42677 tokens: 3.9e-4 -> 2.4e-4).
  // - The accumulators are cut, not rounded, at every step: low by 2^-25 of a sum of codes
  //   for each 16 keys a warp takes. For fp16 the codes' middle is taken from the sums
  //   after each tile, by the weights' own sum (64 key heads of 30000 tokens: 3.4e-4 ->
  //   2.9e-4, shift 7e-6 -> 5e-7 of values of 1).
  // The two cost 32 sequences of up to 8192 tokens 40.2 us for bf16's 37.2, of up to
  // 32768 130 for 119.
  constexpr bool kBytes = std::is_same<T, __nv_bfloat16>::value;
  constexpr float kUnit = kBytes ? 16777216.f : 2097152.f;  // of the sums of codes
  // With a column to spare per row, the weights of a row's second group take it: one
  // operand then serves both groups, whose sums are in columns of their own (118 ->
  // 117 us for 32 sequences of up to 32768 tokens).
  constexpr bool kBoth = COLS == 1 && NG == 2;
  auto column = [](int i, int c2) { return kBoth ? i / 4 : c2; };  // of o[i] and a row
  extern __shared__ __align__(16) uint8_t smem[];
  float* s_o = reinterpret_cast<float*>(smem + kWarps * kStages * kSteps * R::kStage);  // [warp][row][D + 4]
  float* s_m = s_o + kWarps * ROWS * (D + 4);                                  // [warp][row]
  float* s_l = s_m + kWarps * ROWS;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int segs = a.H * a.row_blocks;  // lines of tiles per sequence

  // ---- this CTA's part of the line of all tiles; every warp finds it by itself
  asm volatile("griddepcontrol.launch_dependents;");
  const Line line(count_units(a, 0, nullptr) * segs, gridDim.x);
  if (blockIdx.x >= line.ctas) return;
  const unsigned begin = line.begin(blockIdx.x), end = line.begin(blockIdx.x + 1);
  // The segment at hand: sequence, key head and block of rows.
  struct Segment {
    int b, kvh, rb, keys, tiles;
  } sg = {};
  int at = 0;  // the unit of it at which this CTA begins
  {
    unsigned base = 0;
    for (int b0 = 0; b0 < a.B; b0 += 32) {
      const int keys = b0 + lane < a.B ? keys_of(a, b0 + lane) : 0;
      const unsigned n = units_of((keys + kTile - 1) / kTile) * segs;
      unsigned inc = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned up = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += up;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, begin < base + inc);
      if (hit) {
        const int w = __ffs(hit) - 1;
        sg.b = b0 + w;
        sg.keys = __shfl_sync(0xffffffffu, keys, w);
        const unsigned first = base + __shfl_sync(0xffffffffu, inc - n, w);
        sg.tiles = (sg.keys + kTile - 1) / kTile;
        const int seg = (int)((begin - first) / units_of(sg.tiles));
        sg.kvh = a.row_blocks == 1 ? seg : seg / a.row_blocks;
        sg.rb = seg - sg.kvh * a.row_blocks;
        at = (int)(begin - first) - seg * (int)units_of(sg.tiles);
        break;
      }
      base += __shfl_sync(0xffffffffu, inc, 31);
    }
  }
  int left = (int)(end - begin);  // units of this CTA

  // ---- loads, one tile ahead
  uint8_t* ring = smem + warp * (kStages * kSteps * R::kStage);
  const uint32_t ring_addr = (uint32_t)__cvta_generic_to_shared(ring);
  const uint32_t page_rows = (uint32_t)a.H * a.page_size;
  constexpr int kSegs = D / 32;  // 16-byte pieces of a row of codes
  constexpr int kPieces = R::kScales / 16;
  const uint32_t v_dst = R::kVCodes + v_place<D>(lane / kSegs, lane % kSegs);
  const bool s_lane = lane < 2 * kPieces;  // lanes that load scales: first the keys', then the values'
  const uint32_t s_dst = (lane < kPieces ? R::kKScales : R::kVScales) + (lane % kPieces) * 16;
  const uint8_t *k_src, *v_src, *s_src;  // the segment's head in page 0, and this lane's piece
  const int32_t* pages;                  // the sequence's row of the page table
  int page[kSteps];                      // of the tile to be loaded next
  bool wrong = false;                    // a page of the segment lies outside the cache
  auto lookup = [&](int tl) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int key = tl * kTile + (warp * kSteps + s) * 16;
      if (key < sg.keys) page[s] = pages[a.page_div.div(key)];
    }
  };
  auto load = [&](int tl, int stage) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int key = tl * kTile + (warp * kSteps + s) * 16;
      if (key < sg.keys) {
        const bool bad = (unsigned)page[s] >= (unsigned)a.num_pages;
        wrong |= bad;
        const uint32_t in_page = key - a.page_div.div(key) * a.page_size;
        const uint32_t row = (bad ? 0u : (unsigned)page[s]) * page_rows + in_page;  // the cache has < 2^32
        const uint8_t* kc = k_src + (uint64_t)row * (D / 2);
        const uint8_t* vc = v_src + (uint64_t)row * (D / 2);
        const uint32_t dst = ring_addr + (stage * kSteps + s) * R::kStage;
#pragma unroll
        for (int i = 0; i < R::kCodes / 512; ++i) {
          cp_async16(dst + lane * 16 + i * 512, kc + i * 512);
          cp_async16(dst + v_dst + i * 512, vc + i * 512);  // 8 rows further: the same place, 512 bytes on
        }
        if (s_lane) cp_async16(dst + s_dst, s_src + (uint64_t)row * (NG * 4));
      }
    }
    cp_async_commit();
  };

  // ---- a segment's state
  uint32_t qf[NT][WPT][2][2];          // B operands: code word, low or high byte pair, register
  float f[NT][COLS], qs[NT][NG][COLS]; // per column: factor of the code part, scaled sums of q
  int lim[NT][COLS];                   // keys each column's row keeps
  float m[NT][COLS], l[NT][COLS], lo[NT][NG][COLS];  // the scores' reference, sums
  float o[N64 * 4][NT][4];
  int keys_all = 0;                    // keys that every row keeps
  bool fresh = true;                   // no key yet

  uint4 raw[NT][N64][sizeof(T)];       // the lane's 16 channels of each 64, as they come
  auto load_rows = [&](const Segment& c) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = COLS == 2 ? c.rb * ROWS + nt * 8 + g : g >> 1;
      const bool live = row < a.rows && (COLS == 2 || g % 2 == 0);
      const int n = live ? row_token(a, row) : 0;
      const T* q = static_cast<const T*>(a.q) + (long long)c.b * a.qb + n * a.qn +
                   (long long)(c.kvh * a.G + (live ? row : 0) - n * a.G) * a.qh + 16 * t;
#pragma unroll
      for (int w = 0; w < N64; ++w) {
        raw[nt][w][0] = raw[nt][w][1] = make_uint4(0, 0, 0, 0);
        if (live) {
          if (a.q_vec) {
            raw[nt][w][0] = *reinterpret_cast<const uint4*>(q + 64 * w);
            raw[nt][w][1] = *reinterpret_cast<const uint4*>(q + 64 * w + 8);
          } else {
            T* e = reinterpret_cast<T*>(raw[nt][w]);
#pragma unroll
            for (int i = 0; i < 16; ++i) e[i] = q[64 * w + i];
          }
        }
      }
    }
  };
  auto begin_segment = [&](const Segment& c) {
    const int rb = c.rb;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float x[N64][16];
#pragma unroll
      for (int w = 0; w < N64; ++w)
#pragma unroll
        for (int i = 0; i < 16; ++i) x[w][i] = to_f32<T>(reinterpret_cast<const T*>(raw[nt][w])[i]);
      // A power of two per row brings its largest value to 2^14 .. 2^15 in fp16: no
      // value down to 2^-28 of it becomes subnormal, and a sixteenth of it fits too.
      float top = 0.f;
#pragma unroll
      for (int w = 0; w < N64; ++w)
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(x[w][i]));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // (both powers, up and down, are normal numbers)
      const int e = min(max(268 - (int)(__float_as_uint(top) >> 23), 1), 253);
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
      for (int c2 = 0; c2 < COLS; ++c2) {
        const int src = (2 * t + c2) * 4;
        f[nt][c2] = __shfl_sync(0xffffffffu, down, src) * (16777216.f * a.scale_log2);
#pragma unroll
        for (int k = 0; k < NG; ++k) qs[nt][k][c2] = __shfl_sync(0xffffffffu, sum[k], src) * a.scale_log2;
        const int r = COLS == 2 ? rb * ROWS + nt * 8 + 2 * t + c2 : t;
        // rows that do not exist keep what the last token keeps
        lim[nt][c2] = r < a.rows ? max(0, c.keys - a.N + 1 + row_token(a, r)) : c.keys;
        m[nt][c2] = 0.f;
        l[nt][c2] = 0.f;
#pragma unroll
        for (int k = 0; k < NG; ++k) lo[nt][k][c2] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < N64 * 4; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) o[i][nt][k] = 0.f;
    }
    fresh = true;
    keys_all = max(0, c.keys - a.N + 1);
  };

  const int k_off = g * (D / 2) + t * (D / 8), m_off = R::kKScales + g * NG * 4;
  const int v_off = R::kVCodes + v_place<D>(2 * t, D == 128 ? g >> 1 : g >> 2) + (D == 128 ? (g & 1) * 8 : (g & 3) * 4);

  // ---- 32 keys: two times 16, whose instructions fill one another's waits
  auto step = [&](const uint8_t* st, int key0, int keys) {
    float x[kSteps][NT][4], sv[kSteps][2][NG], lv[kSteps][2][NG];  // x: scores less the running maximum
#pragma unroll
    for (int u = 0; u < kSteps; ++u) {
      const uint8_t* p0 = st + u * R::kStage;
      uint32_t k0[WPT], k1[WPT], km[2][NG], vm[2][NG];
      if constexpr (D == 128) {
        *reinterpret_cast<uint4*>(k0) = *reinterpret_cast<const uint4*>(p0 + k_off);
        *reinterpret_cast<uint4*>(k1) = *reinterpret_cast<const uint4*>(p0 + k_off + 8 * (D / 2));
      } else {
        *reinterpret_cast<uint2*>(k0) = *reinterpret_cast<const uint2*>(p0 + k_off);
        *reinterpret_cast<uint2*>(k1) = *reinterpret_cast<const uint2*>(p0 + k_off + 8 * (D / 2));
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint8_t* p = p0 + m_off + 8 * h * NG * 4;
        if constexpr (NG == 2) {
          *reinterpret_cast<uint2*>(km[h]) = *reinterpret_cast<const uint2*>(p);
          *reinterpret_cast<uint2*>(vm[h]) = *reinterpret_cast<const uint2*>(p + R::kScales);
        } else {
          km[h][0] = *reinterpret_cast<const uint32_t*>(p);
          vm[h][0] = *reinterpret_cast<const uint32_t*>(p + R::kScales);
        }
      }
      float acc[NG][NT][4] = {};
#pragma unroll
      for (int w = 0; w < WPT; ++w)
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const uint32_t x0 = s ? byte_pair(k0[w], 1) : k0[w], x1 = s ? byte_pair(k1[w], 1) : k1[w];
          const uint32_t a0 = x0 & 0x000f000fu, a1 = x1 & 0x000f000fu;
          const uint32_t a2 = x0 & 0x00f000f0u, a3 = x1 & 0x00f000f0u;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            mma16816(acc[NG == 2 ? w % N64 : 0][nt], a0, a1, a2, a3, qf[nt][w][s][0], qf[nt][w][s][1]);
        }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int k = 0; k < NG; ++k) {
          sv[u][h][k] = scale_of(vm[h][k]);
          lv[u][h][k] = low_of(vm[h][k]);
        }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; i += 3 - COLS) {
          const int h = i >> 1, c2 = i & 1;
          float w = scale_of(km[h][0]) * acc[0][nt][i], y = fmaf(low_of(km[h][0]), qs[nt][0][c2], -m[nt][c2]);
          if constexpr (NG == 2) {
            w = fmaf(scale_of(km[h][1]), acc[1][nt][i], w);
            y = fmaf(low_of(km[h][1]), qs[nt][1][c2], y);
          }
          x[u][nt][i] = fmaf(w, f[nt][c2], y);
        }
    }
    const bool edge = key0 + 16 * kSteps > keys_all;  // some row keeps only a part
    if (edge) {
#pragma unroll
      for (int u = 0; u < kSteps; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int key = key0 + 16 * u + g + 8 * h;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c2 = 0; c2 < COLS; ++c2)
              if (key >= lim[nt][c2]) x[u][nt][2 * h + c2] = -INFINITY;
          // past the sequence the page, or a buffer that nothing was loaded into,
          // holds anything
          if (key >= keys)
#pragma unroll
            for (int k = 0; k < NG; ++k) sv[u][h][k] = lv[u][h][k] = 0.f;
        }
    }
    // raise the references where needed
    float log_sv[kSteps][2];  // of the larger scale, at least -70: 0.1 too low at most
#pragma unroll
    for (int u = 0; u < kSteps; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float y = fmax3(sv[u][h][0], sv[u][h][NG - 1], 8.5e-22f);  // NaN is left aside, here and below
        // exponent and first bits of the mantissa, as they lie in the word, behind 2^23
        log_sv[u][h] = fmaf(__uint_as_float(__byte_perm(__float_as_uint(y), 0x4b000000u, 0x7632)), 0.0078125f, -65663.f);
      }
    float over = -INFINITY;
#pragma unroll
    for (int u = 0; u < kSteps; ++u)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c2 = 0; c2 < COLS; ++c2)
          over = fmax3(over, x[u][nt][c2] + log_sv[u][0], x[u][nt][2 + c2] + log_sv[u][1]);
    if (__any_sync(0xffffffffu, over > kRaise) || fresh) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c2 = 0; c2 < COLS; ++c2) {
          float y = -INFINITY, top = -INFINITY;  // of the products, of the scores
#pragma unroll
          for (int u = 0; u < kSteps; ++u) {
            y = fmax3(y, x[u][nt][c2] + log_sv[u][0], x[u][nt][2 + c2] + log_sv[u][1]);
            top = fmax3(top, x[u][nt][c2], x[u][nt][2 + c2]);
          }
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) {
            y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, d));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
          }
          // The step leaves a new largest score a whole number above m, and otherwise is
          // one: the largest weight is then a power of two and its product exact (fp16, 2
          // to 3000 keys: 2.1e-4 from the exact result; with m a whole number 2.9e-4).
          // The first keys may set m below its start of 0.
          const float by = y - kPut, step = fresh || top > 12.f ? top + ceilf(by - top) : ceilf(by);
          const float up = (fresh ? y > -INFINITY : by > 0.f) ? step : 0.f;
          // what is summed so far shrinks by the step; before the first keys that is
          // nothing, and a step far down would make it 0 * inf
          const float al = fresh ? 1.f : ex2(-up);
          m[nt][c2] += up;
#pragma unroll
          for (int u = 0; u < kSteps; ++u) {
            x[u][nt][c2] -= up;
            x[u][nt][2 + c2] -= up;
          }
          l[nt][c2] *= al;
#pragma unroll
          for (int k = 0; k < NG; ++k) lo[nt][k][c2] *= al;
#pragma unroll
          for (int i = 0; i < N64 * 4; ++i) {
            o[i][nt][column(i, c2)] *= al;
            o[i][nt][2 + column(i, c2)] *= al;
          }
        }
      fresh = false;
    }
    float sums[NT][kBoth ? 1 : NG][4] = {};  // of the weights of these keys
#pragma unroll
    for (int u = 0; u < kSteps; ++u) {
      // weights, and their products with the values' scales as the B operand
      uint32_t pf[NT][kBoth ? 1 : NG][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float p[4], both[NG][2];
#pragma unroll
        for (int i = 0; i < 4; i += 3 - COLS) {
          p[i] = ex2(x[u][nt][i]);
          l[nt][i & 1] += p[i];
        }
#pragma unroll
        for (int k = 0; k < NG; ++k) {
          float w[4] = {};
#pragma unroll
          for (int i = 0; i < 4; i += 3 - COLS) w[i] = p[i] * sv[u][i >> 1][k];
          if (edge) {
            // a row's own masked keys count for nothing, NaN or not
#pragma unroll
            for (int i = 0; i < 4; i += 3 - COLS) {
              const bool out = key0 + 16 * u + g + 8 * (i >> 1) >= lim[nt][i & 1];
              if (out) w[i] = 0.f;
              lo[nt][k][i & 1] += out ? 0.f : p[i] * lv[u][i >> 1][k];
            }
          } else {
#pragma unroll
            for (int i = 0; i < 4; i += 3 - COLS) lo[nt][k][i & 1] = fmaf(p[i], lv[u][i >> 1][k], lo[nt][k][i & 1]);
          }
          if constexpr (kBoth) {
            both[k][0] = w[0];
            both[k][1] = w[2];
            if (k == 0) continue;
            w[1] = w[0], w[3] = w[2];
            w[0] = both[0][0], w[2] = both[0][1];
          }
          uint32_t packed[2] = {half2_bits(w[0], w[1]), half2_bits(w[2], w[3])};
          if constexpr (std::is_same<T, __half>::value) {
            // What the rounding took from a weight, times the middle of the codes, goes
            // to the lowest values' sum: the rounding then counts for the code's distance
            // from 7.5 and not for the whole code. fp16 results resolve that (16 sequences
            // of up to 4095 keys: relative error 4.5e-4 without, 2.6e-4 with, 2.1e-4 of it
            // the output's rounding); bf16 ones do not.
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float2 r = __half22float2(*reinterpret_cast<const __half2*>(&packed[h]));
              lo[nt][kBoth ? 0 : k][0] = fmaf(w[2 * h] - r.x, 7.5f, lo[nt][kBoth ? 0 : k][0]);
              if constexpr (kBoth) lo[nt][1][0] = fmaf(w[2 * h + 1] - r.y, 7.5f, lo[nt][1][0]);
              if constexpr (COLS == 2) lo[nt][k][1] = fmaf(w[2 * h + 1] - r.y, 7.5f, lo[nt][k][1]);
            }
          }
          pf[nt][kBoth ? 0 : k][0] = transpose8(packed[0]);
          pf[nt][kBoth ? 0 : k][1] = transpose8(packed[1]);
          if constexpr (!kBytes) {
            constexpr uint32_t kOnes = 0x3c003c00u;
            mma16816(sums[nt][kBoth ? 0 : k], kOnes, kOnes, kOnes, kOnes, pf[nt][kBoth ? 0 : k][0], pf[nt][kBoth ? 0 : k][1]);
          }
        }
      }
      // values
      uint32_t vw[4][N64];
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // keys 2t + (i & 1) + 8 (i >> 1): v_place keeps their distances
        const uint8_t* p = st + u * R::kStage + v_off + ((i & 1) * 4 + (i >> 1) * 8) * (D / 2);
        if constexpr (D == 128) *reinterpret_cast<uint2*>(vw[i]) = *reinterpret_cast<const uint2*>(p);
        else vw[i][0] = *reinterpret_cast<const uint32_t*>(p);
      }
#pragma unroll
      for (int w = 0; w < N64; ++w) {  // channels 64w + 8g ..
#pragma unroll
        for (int h = 0; h < 2; ++h) {  // codes 4h .. 4h+3 of each word
          const uint32_t p0 = __byte_perm(vw[0][w], vw[1][w], h ? 0x7632 : 0x5410);
          const uint32_t p1 = __byte_perm(vw[2][w], vw[3][w], h ? 0x7632 : 0x5410);
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            uint32_t a0, a1, a2, a3;
            if constexpr (kBytes) {
              a1 = byte_pair(p0, s), a3 = byte_pair(p1, s);
              a0 = (s ? a1 : p0) & 0x000f000fu, a2 = (s ? a3 : p1) & 0x000f000fu;
            } else {
              const uint32_t y0 = s ? p0 >> 5 : p0 << 3, y1 = s ? p1 >> 5 : p1 << 3;
              a0 = y0 & 0x00780078u, a1 = y0 & 0x07f807f8u;
              a2 = y1 & 0x00780078u, a3 = y1 & 0x07f807f8u;
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mma16816(o[w * 4 + 2 * h + s][nt], a0, a1, a2, a3, pf[nt][kBoth || NG == 1 ? 0 : w][0], pf[nt][kBoth || NG == 1 ? 0 : w][1]);
          }
        }
      }
    }
    if constexpr (!kBytes) {  // 7.5, and 127.5 of a byte, from the sums to the lowest values'
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c2 = 0; c2 < COLS; ++c2) {
#pragma unroll
          for (int i = 0; i < N64 * 4; ++i) {
            const int c = column(i, c2);
            const float w = sums[nt][kBoth || NG == 1 ? 0 : i / 4][c];
            o[i][nt][c] = fmaf(w, -7.5f / kUnit, o[i][nt][c]);
            o[i][nt][2 + c] = fmaf(w, -127.5f / kUnit, o[i][nt][2 + c]);
          }
          // all eight lanes of a column have its sum
#pragma unroll
          for (int k = 0; k < NG; ++k)
            lo[nt][k][c2] = fmaf(sums[nt][kBoth ? 0 : k][kBoth ? k : c2], 0.125f * 7.5f, lo[nt][k][c2]);
        }
    }
  };

  // ---- merge the warps' results of a segment
  auto end_segment = [&](const Segment& c, bool cut_front, bool cut_back) {
    const int kvh = c.kvh, rb = c.rb;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c2 = 0; c2 < COLS; ++c2) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
          l[nt][c2] += __shfl_xor_sync(0xffffffffu, l[nt][c2], d);
#pragma unroll
          for (int k = 0; k < NG; ++k) lo[nt][k][c2] += __shfl_xor_sync(0xffffffffu, lo[nt][k][c2], d);
        }
        if (wrong) l[nt][c2] = __int_as_float(0x7fffffff);  // no such page: the rows are undefined
        const int r = COLS == 2 ? nt * 8 + 2 * t + c2 : t;
        // l is brought to 1 .. 2, by a power of two, and m to the logarithm of the whole
        // sum: the warps' references follow their own products and may lie far apart
        const int e = (int)(__float_as_uint(l[nt][c2]) >> 23);
        const float down = __int_as_float((254 - e) << 23);
        if (g == 0) {
          s_m[warp * ROWS + r] = l[nt][c2] == 0.f ? kNoMax : m[nt][c2] + (float)(e - 127);
          s_l[warp * ROWS + r] = l[nt][c2] * down;
        }
#pragma unroll
        for (int i = 0; i < N64 * 4; ++i) {
          const int d = 64 * (i / 4) + 8 * g + 2 * (i % 4);
          const float y = lo[nt][NG == 2 ? i / 4 : 0][c2];
          const int c = column(i, c2);
          const float2 v = {fmaf(o[i][nt][c], kUnit, y) * down, fmaf(o[i][nt][2 + c] - o[i][nt][c], kUnit / 16.f, y) * down};
          *reinterpret_cast<float2*>(s_o + (warp * ROWS + r) * (D + 4) + d) = v;
        }
      }
    __syncthreads();
    const bool whole = !cut_front && !cut_back;
    // a CTA has at most two cut segments: one that began before it, one that goes on
    float* part = a.partials + (size_t)(2 * blockIdx.x + (cut_front ? 0 : 1)) * ROWS * (D + 2);
    for (int e = threadIdx.x; e < ROWS * (D / 4); e += kThreads) {
      const int r = e / (D / 4), d = (e % (D / 4)) * 4;
      const int row = rb * ROWS + r;
      float top = kNoMax;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_m[w * ROWS + r]);
      float sum = 0.f;
      float4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float x = ex2(s_m[w * ROWS + r] - top);
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

  // ---- the segments of this CTA's part of the line
  while (true) {
    const int until = min((int)units_of(sg.tiles), at + left);
    left -= until - at;
    const int start = max(0, at - kSetup), stop = max(0, until - kSetup);  // tiles
    if (start < stop) {
      {
        const size_t head = (size_t)sg.kvh * a.page_size;
        k_src = a.k_codes + head * (D / 2) + lane * 16;
        v_src = a.v_codes + head * (D / 2) + lane * 16;
        s_src = reinterpret_cast<const uint8_t*>(lane < kPieces ? a.k_scales : a.v_scales) + head * (NG * 4) + (lane % kPieces) * 16;
        pages = a.page_table + sg.b * a.table_stride;
      }
      wrong = false;
      lookup(start);
      load_rows(sg);
      load(start, 0);
      if (start + 1 < stop) lookup(start + 1);
      begin_segment(sg);
      int stage = 0;
      for (int tile = start; tile < stop; ++tile) {
        cp_async_wait<0>();
        __syncwarp();  // the other lanes' pieces have landed, and all are done with the other buffer
        if (tile + 1 < stop) {
          load(tile + 1, stage ^ 1);
          if (tile + 2 < stop) lookup(tile + 2);
        }
        const int key0 = tile * kTile + warp * kSteps * 16;
        if (key0 < sg.keys) step(ring + stage * kSteps * R::kStage, key0, sg.keys);
        stage ^= 1;
      }
      if (wrong && lane == 0) atomicOr(a.status, DEV_BAD_INDEX);
      end_segment(sg, start > 0, stop < sg.tiles);
    }
    if (left == 0) break;
    // the next segment that has tiles
    at = 0;
    if (++sg.rb == a.row_blocks) {
      sg.rb = 0;
      if (++sg.kvh == a.H) {
        sg.kvh = 0;
        do {
          if (++sg.b >= a.B) return;
          sg.keys = keys_of(a, sg.b);
          sg.tiles = (sg.keys + kTile - 1) / kTile;
        } while (sg.tiles == 0);
      }
    }
  }
}

// Joins the parts of the segments that were cut between CTAs; writes the rows of
// sequences without tiles (no key, or a length that cannot be). One CTA per row: its
// threads take the row's channels four at a time and the parts kJoin / (D/4) at once.
constexpr int kJoin = 128;
constexpr int kJoinMax = 1024;  // parts whose weights are kept; a segment has at most the grid's CTAs
template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(kJoin) kv_attn_join_kernel(const __grid_constant__ AttnArgs a, int grid) {
  constexpr int LANES = D / 4, LINES = kJoin / LANES;
  __shared__ float s_w[kJoinMax], s_l[kJoinMax], s_top[kJoin / 32], s_total[kJoin / 32];
  __shared__ float4 s_v[LINES][LANES];
  const int per_seq = a.H * a.rows;
  const int b = blockIdx.x / per_seq, rest = blockIdx.x - b * per_seq;
  const int kvh = rest / a.rows, row = rest - kvh * a.rows;
  const int rb = row / ROWS, r = row - rb * ROWS;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int segs = a.H * a.row_blocks, seg = kvh * a.row_blocks + rb;
  const int held = a.lengths[b], tiles = tiles_of(a, b);
  const int n = row_token(a, row);
  T* out = static_cast<T*>(a.o) + (long long)b * a.ob + n * a.on + (long long)(kvh * a.G + row - n * a.G) * a.oh;
  // every CTA waits for the attention kernel, so that this one's end is the call's
  if (tiles == 0) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const bool wrong = held != 0;
    if (wrong && threadIdx.x == 0) atomicOr(a.status, DEV_BAD_INDEX);
    for (int d = threadIdx.x; d < D; d += kJoin) out[d] = from_f32<T>(wrong ? __int_as_float(0x7fffffff) : 0.f);
    return;
  }
  unsigned before;
  const Line line(count_units(a, b, &before) * segs, grid);
  before = before * segs + (unsigned)seg * units_of(tiles) + kSetup;  // the first tile
  const int c0 = (int)line.owner(before), c1 = (int)line.owner(before + tiles - 1);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (c0 == c1) return;  // whole in one CTA, which wrote it
  const int parts = c1 - c0 + 1;
  // the first CTA's part began in it (slot 1), the others' began before them (slot 0)
  const size_t stride = (size_t)ROWS * (D + 2);
  auto part = [&](int i) { return a.partials + (size_t)(2 * (c0 + i) + (i == 0 ? 1 : 0)) * stride; };
  const int col = threadIdx.x % LANES, first = threadIdx.x / LANES;
  // Everything a thread can ask for without the weights is asked for first.
  constexpr int kAhead = 4;
  float4 ahead[kAhead];
#pragma unroll
  for (int j = 0; j < kAhead; ++j)
    if (first + j * LINES < parts) ahead[j] = *reinterpret_cast<const float4*>(part(first + j * LINES) + r * D + 4 * col);
  float top = kNoMax, sum = 0.f;
  for (int i = threadIdx.x; i < parts; i += kJoin) {
    const float* p = part(i) + ROWS * D + r;
    s_w[i] = p[0];
    s_l[i] = p[ROWS];
    top = fmaxf(top, s_w[i]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) s_top[warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kJoin / 32; ++w) top = fmaxf(top, s_top[w]);
  for (int i = threadIdx.x; i < parts; i += kJoin) {
    s_w[i] = ex2(s_w[i] - top);
    sum = fmaf(s_w[i], s_l[i], sum);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) s_total[warp] = sum;
  __syncthreads();
  float4 v = {0.f, 0.f, 0.f, 0.f};
  auto add = [&](const float4& y, float w) {
    v.x = fmaf(w, y.x, v.x);
    v.y = fmaf(w, y.y, v.y);
    v.z = fmaf(w, y.z, v.z);
    v.w = fmaf(w, y.w, v.w);
  };
#pragma unroll
  for (int j = 0; j < kAhead; ++j)
    if (first + j * LINES < parts) add(ahead[j], s_w[first + j * LINES]);
#pragma unroll 8
  for (int i = first + kAhead * LINES; i < parts; i += LINES)
    add(*reinterpret_cast<const float4*>(part(i) + r * D + 4 * col), s_w[i]);
  s_v[first][col] = v;
  __syncthreads();
  if (first == 0) {
    float all = 0.f;
#pragma unroll
    for (int w = 0; w < kJoin / 32; ++w) all += s_total[w];
#pragma unroll
    for (int i = 1; i < LINES; ++i) {
      const float4 y = s_v[i][col];
      v.x += y.x;
      v.y += y.y;
      v.z += y.z;
      v.w += y.w;
    }
    const bool any = held - a.N + 1 + n > 0;
    out[4 * col] = from_f32<T>(any ? v.x / all : 0.f);
    out[4 * col + 1] = from_f32<T>(any ? v.y / all : 0.f);
    out[4 * col + 2] = from_f32<T>(any ? v.z / all : 0.f);
    out[4 * col + 3] = from_f32<T>(any ? v.w / all : 0.f);
  }
}

constexpr int kMaxGrid = 4 * 160;  // CTAs that the workspace has room for
static_assert(kMaxGrid <= kJoinMax, "a segment's parts");

template <typename T, int D, int GROUP, int NT, int COLS>
int launch(AttnArgs& a, cudaStream_t st) {
  using R = Ring<D, GROUP>;
  constexpr int ROWS = COLS * 4 * NT;
  constexpr size_t smem = (size_t)kWarps * kStages * kSteps * R::kStage + (size_t)kWarps * ROWS * (D + 6) * sizeof(float);
  a.row_blocks = (a.rows + ROWS - 1) / ROWS;
  const double tiles = (double)a.B * a.H * a.row_blocks * (((double)a.max_pages * a.page_size + kTile) / kTile + kSetup);
  if (tiles >= 2147483648.0) {
    set_error("b2_kv_cache_attn: B * H * row blocks * (max_pages * page_size / %d) must be < 2^31", kTile);
    return B2_EINVAL;
  }
  auto kern = kv_attn_kernel<T, D, GROUP, NT, COLS>;
  static OncePerDevice ready;
  B2_CUDA_TRY(ready([&] { return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem); }));
  int grid = device_sm_count() * kCtasPerSm<D, NT>;
  if (grid > kMaxGrid) grid = kMaxGrid;
  kern<<<grid, kThreads, smem, st>>>(a);
  B2_CHECK_LAUNCH();
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((long long)a.B * a.H * a.rows));
  cfg.blockDim = dim3(kJoin);
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  B2_CUDA_TRY(cudaLaunchKernelEx(&cfg, kv_attn_join_kernel<T, D, ROWS>, a, grid));
  return B2_OK;
}

template <typename T, int D, int GROUP>
int launch_rows(AttnArgs& a, cudaStream_t st) {
  if (a.rows <= 4) return launch<T, D, GROUP, 1, 1>(a, st);
  if (a.rows <= 8) return launch<T, D, GROUP, 1, 2>(a, st);
  // More rows: blocks of 16, each reading the keys again (from L2). Blocks of 32 with
  // D = 64 (255 registers) measured 62 us against 67 for 16 sequences of up to 32768
  // keys and 32 rows, but 19.3 against 18.5 up to 4095 and 10.2 against 7.8 up to 64.
  return launch<T, D, GROUP, 2, 2>(a, st);
}

template <typename T>
int launch_typed(AttnArgs& a, int D, int group, cudaStream_t st) {
  if (D == 64) return launch_rows<T, 64, 64>(a, st);
  return group == 64 ? launch_rows<T, 128, 64>(a, st) : launch_rows<T, 128, 128>(a, st);
}

}  // namespace

size_t kv_attn_mma_workspace(int64_t rows, int64_t D) {
  const size_t block = rows <= 8 ? 8 : 16;
  return sizeof(float) * 2 * kMaxGrid * block * (size_t)(D + 2);
}

int kv_attn_mma_launch(AttnArgs& a, int D, int group, int dtype, cudaStream_t st) {
  return dtype == B2_F16 ? launch_typed<__half>(a, D, group, st) : launch_typed<__nv_bfloat16>(a, D, group, st);
}

}  // namespace b2
