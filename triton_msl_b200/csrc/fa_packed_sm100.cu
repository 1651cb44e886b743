// Attention over packed sequences on 5th-generation tensor cores (fp16 / bf16 in,
// fp32 accumulate), grouped heads, causal or not, head_dim up to 128.
//
//   o_i = sum_j softmax_j(scale * q_i . k_j) v_j over the keys j of i's own
//   sequence, with j <= i + (Lk - Lq) when causal; no key: zeros.
//
// The pipeline is that of fa_sm100.cu: a persistent CTA per SM, two 128-row
// query tiles ping-ponged, TMA loads (warp 0), one issuing warp for tcgen05.mma
// (warp 1), S and P in TMEM (P aliases S), eight softmax warps, O in TMEM. What
// differs is what a tile holds:
//  * Rows of a tile are (token, query head of the group) pairs: with G query
//    heads on a key head, a tile is floor(128/G) tokens x G heads, one TMA box of
//    {channels, G heads, tokens}. K and V are then loaded once for the whole
//    group, short sequences fill their tiles, and the causal diagonal wastes
//    floor(128/G) + 128 keys a tile instead of 256.
//  * The work list (fa_packed_plan_kernel): one entry per 2*floor(128/G) tokens
//    of a sequence, most key blocks first, made on the device from the offsets,
//    so the host needs no lengths. Heads vary fastest, CTAs take the entries in
//    serpentine order.
//  * Keys past a sequence's end belong to the next one. Their scores are
//    replaced by -inf; their V rows, whose weights are zero but which may hold
//    NaN or infinities, are zeroed in shared memory by warp 2 before the MMA.
//  * V rows of later tokens of the same sequence (causal) cannot be zeroed, as
//    later queries of the tile use them. A result row that is not finite is
//    looked at again: if a masked key of its last blocks is not finite, the row
//    is computed anew over its own keys, at the end.
//  * NaN scores make the row NaN: the running maximum propagates NaN, since the
//    polynomial exponential would not.
// D <= 64 runs on 64-channel tiles, D <= 128 on 128; TMA fills the channels
// past D with zeros.
#include <climits>

#include "decoder.cuh"
#include "fa_math.cuh"
#include "packed.cuh"
#include "sm100.cuh"

namespace b2 {
namespace {

using namespace sm100;
using namespace fa;

__device__ uint32_t g_packed_status;

constexpr int kBM = 128, kBN = 128, kThreads = 384;
// Registers per thread: 128 * (56 + 2 * 224) = 384 * 168, the launch allocation.
constexpr int kRegsProducer = 56, kRegsSoftmax = 224, kLaunchRegs = 168;
static_assert(128 * (kRegsProducer + 2 * kRegsSoftmax) <= kThreads * kLaunchRegs,
              "register split exceeds the launch allocation");
constexpr uint32_t kTmemCols = 512;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRescaleThreshold = 8.0f;  // log2 units

// ------------------------------------------------------------- the work list
// One entry: 2*R consecutive queries of one sequence (R tokens a tile).
struct __align__(16) Entry {
  int q0, nq;      // first token of q and tokens, 1 .. 2R
  int k0, Lk;      // the sequence's keys
  int lim0;        // keys of the entry's first query (may be <= 0); query i has lim0 + i
  int n0, n1;      // key blocks of the two tiles
  int pad;
};
static_assert(sizeof(Entry) == 32, "two 16-byte loads");
constexpr int kPlanHeader = 64;      // bytes before the entries: the number of them
constexpr int kPlanClasses = 256;    // key-block counts told apart by the sort

struct PlanArgs {
  const int32_t *cu_q, *cu_k;
  int B, Tq, Tk, R, causal;
  int* ws;
};

__device__ __forceinline__ Entry make_entry(const PlanArgs& a, const packed::Span& q, const packed::Span& k, int blk) {
  Entry e;
  const int i0 = blk * 2 * a.R;
  e.q0 = q.start + i0;
  e.nq = min(2 * a.R, q.len - i0);
  e.k0 = k.start;
  e.Lk = k.len;
  e.lim0 = a.causal ? i0 + k.len - q.len + 1 : k.len;
  auto blocks = [&](int tile) {
    const int last = min((tile + 1) * a.R, e.nq) - 1;  // the tile's last query
    if (last < tile * a.R) return 0;
    const int lim = a.causal ? min(k.len, e.lim0 + last) : k.len;
    return lim > 0 ? (lim + kBN - 1) / kBN : 0;
  };
  e.n0 = blocks(0);
  e.n1 = blocks(1);
  e.pad = 0;
  return e;
}

// Counts up to 127 have a class each, above that 32 share one.
__device__ __forceinline__ int plan_class(int blocks) {
  return kPlanClasses - 1 - (blocks < 128 ? blocks : min(128 + ((blocks - 128) >> 5), kPlanClasses - 1));
}

// One CTA: a counting sort of the entries by key blocks, most first. The order
// within a class is the atomics' and changes nothing but the schedule.
__global__ void __launch_bounds__(1024) fa_packed_plan_kernel(const PlanArgs a) {
  __shared__ int hist[kPlanClasses];
  __shared__ int part[kPlanClasses / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  asm volatile("griddepcontrol.launch_dependents;");
  if (threadIdx.x < kPlanClasses) hist[threadIdx.x] = 0;
  bool bad = false, bad_q = false;
  for (int b = threadIdx.x; b < a.B; b += blockDim.x) {
    bad_q |= packed::span_bad(a.cu_q, b, a.Tq);
    bad |= packed::span_bad(a.cu_k, b, a.Tk);
  }
  if (bad || bad_q) atomicOr(&g_packed_status, DEV_BAD_INDEX);
  // Also the barrier behind hist. With query offsets that descend one warp walks the
  // sequences in order, since where one begins depends on all before it.
  const bool in_order = __syncthreads_or(bad_q);
  auto for_entries = [&](auto&& f) {
    int end = 0;
    for (int b = in_order ? (warp == 0 ? -1 : a.B + 1) : warp - 1; b <= a.B; b += in_order ? 1 : warps) {
      packed::Span q = packed::span_of(a.cu_q, b, a.B, a.Tq);
      if (in_order) {
        q = q.after(end);
        end = q.start + q.len;
      }
      const packed::Span k = b < 0 || b >= a.B ? packed::Span{0, 0} : packed::span_of(a.cu_k, b, a.B, a.Tk);
      for (int blk = lane; blk * 2 * a.R < q.len; blk += 32) {
        const Entry e = make_entry(a, q, k, blk);
        f(e, plan_class(max(e.n0, e.n1)));
      }
    }
  };
  for_entries([&](const Entry&, int cls) { atomicAdd(&hist[cls], 1); });
  __syncthreads();
  // prefix sums of the classes, one per thread of the first eight warps
  int own = 0, inc = 0;
  if (threadIdx.x < kPlanClasses) {
    own = inc = hist[threadIdx.x];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += up;
    }
    if (lane == 31) part[warp] = inc;
  }
  __syncthreads();
  if (threadIdx.x < kPlanClasses) {
    for (int w = 0; w < warp; ++w) inc += part[w];
    hist[threadIdx.x] = inc - own;
  }
  __syncthreads();
  Entry* list = reinterpret_cast<Entry*>(reinterpret_cast<char*>(a.ws) + kPlanHeader);
  // The spans cover every token once: at most as many entries as the list has room for,
  // unless something writes the offsets meanwhile.
  const int room = a.Tq / (2 * a.R) + a.B + 2;
  for_entries([&](const Entry& e, int cls) {
    const int at = atomicAdd(&hist[cls], 1);
    if (at < room) list[at] = e;
  });
  if (threadIdx.x == kPlanClasses - 1) a.ws[0] = min(inc, room);
}

// ------------------------------------------------------------- the attention
struct __align__(8) Barriers {
  uint64_t q_full, q_empty;
  uint64_t k_full[2], k_empty[2];
  uint64_t v_full[2], v_empty[2];
  // a sequence's last V block lands on vt_full; warp 2 zeroes the rows past the
  // sequence's end and then arrives on v_full in the copy's place
  uint64_t vt_full[2];
  uint64_t s_full[2], p_full[2];
  uint64_t o_full[2], o_empty[2];
  uint64_t done;
  uint32_t tmem_base;
  int abort_flag;
  uint32_t blocks;  // that warp 0 has asked for
};

template <int D>
struct Cfg {
  static constexpr int kAtoms = D / 64;                     // 64 channels: 128-byte swizzle rows
  static constexpr uint32_t kTileBytes = 128 * D * 2;
  static constexpr uint32_t kAtomTileBytes = 128 * 128;
  static constexpr uint32_t kSBO = 8 * 128;
  static constexpr uint32_t kOutStageBytes = 32 * 128;      // per softmax warp
  static constexpr bool kSumMma = D <= 64;                  // row sums on the tensor core
  static constexpr uint32_t kOnesBytes = kSumMma ? 1024 : 0;
  static constexpr size_t kSmem = 1024 + 6 * kTileBytes + 8 * kOutStageBytes + kOnesBytes + sizeof(Barriers);
  static_assert(2 * (kBN + D + (kSumMma ? 16 : 0)) <= (int)kTmemCols, "TMEM columns exceeded");
  static_assert(kSmem <= 227 * 1024, "shared memory per CTA exceeded");
};

struct KernelArgs {
  const int* ws;
  const void *q, *k, *v;
  void* o;
  long long qt, qh, kt, kh, vt, vh, ot, oh;
  int G, R, Hk, D, causal;
  unsigned most;  // units that the work list has room for
  float scale_log2;
};

// Three-input maximum that propagates NaN.
__device__ __forceinline__ float fmax3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

template <int D, bool BF16>
__global__ void __launch_bounds__(kThreads, 1)
fa_packed_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                 const __grid_constant__ CUtensorMap tmV, const __grid_constant__ KernelArgs a) {
  using C = Cfg<D>;
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;                         // 2 tiles
  uint8_t* sK = smem + 2 * C::kTileBytes;     // 2 stages
  uint8_t* sV = smem + 4 * C::kTileBytes;     // 2 stages
  uint8_t* sO = smem + 6 * C::kTileBytes;     // output staging, 8 warps
  uint8_t* sOnes = sO + 8 * C::kOutStageBytes;
  Barriers* bars = reinterpret_cast<Barriers*>(sOnes + C::kOnesBytes);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort_flag = &bars->abort_flag;
  volatile uint32_t* blocks = &bars->blocks;

  if (threadIdx.x == 0) {
    mbar_init(&bars->q_full, 1);
    mbar_init(&bars->q_empty, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars->k_full[i], 1);
      mbar_init(&bars->k_empty[i], 1);
      mbar_init(&bars->v_full[i], 1);
      mbar_init(&bars->v_empty[i], 1);
      mbar_init(&bars->vt_full[i], 1);
      mbar_init(&bars->s_full[i], 1);
      mbar_init(&bars->p_full[i], 4);
      mbar_init(&bars->o_full[i], 1);
      mbar_init(&bars->o_empty[i], 4);
    }
    mbar_init(&bars->done, 1);
    bars->abort_flag = 0;
    bars->blocks = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (warp == 1) {
    tmem_alloc(&bars->tmem_base, kTmemCols);
    tmem_relinquish();
  }
  if (a.G * a.R < kBM) {
    // a box of G*R rows leaves the tile's last rows: zeros, never written again
    for (int i = threadIdx.x; i < (int)(2 * C::kTileBytes / 16); i += kThreads)
      reinterpret_cast<uint4*>(sQ)[i] = make_uint4(0, 0, 0, 0);
    fence_proxy_async_smem();
  }
  if constexpr (C::kSumMma) {
    if (threadIdx.x < C::kOnesBytes / 16) {
      const uint32_t w = BF16 ? 0x3F803F80u : 0x3C003C00u;
      reinterpret_cast<uint4*>(sOnes)[threadIdx.x] = make_uint4(w, w, w, w);
      fence_proxy_async_smem();
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;
  // columns of tile t: S_t (and P_t), O_t, and the row sums L_t (D <= 64 only)
  auto tS = [&](int t) { return tmem + t * 128; };
  auto tO = [&](int t) { return tmem + 256 + t * D; };
  auto tL = [&](int t) { return tmem + 256 + 2 * D + t * 16; };

  // the work list is the plan kernel's
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const unsigned num_units = (unsigned)a.ws[0] * (unsigned)a.Hk;  // < 2^31: the host checks
  const Entry* list = reinterpret_cast<const Entry*>(reinterpret_cast<const char*>(a.ws) + kPlanHeader);
  // CTA c takes, in round r, unit r*grid + c (even r) or r*grid + grid-1-c (odd
  // r): with the heaviest units first this pairs heavy and light ones.
  struct Unit {
    Entry e;
    int kvh;
    bool valid;
  };
  auto fetch = [&](uint32_t r) -> Unit {
    Unit u;
    const unsigned at = r * gridDim.x + ((r & 1) ? (gridDim.x - 1 - blockIdx.x) : blockIdx.x);
    u.valid = at < num_units;
    // loaded without waiting for the number of units: the list has room for a.most
    if (at < a.most) {
      const unsigned row = at / (unsigned)a.Hk;
      u.kvh = (int)(at - row * a.Hk);
      const int4* p = reinterpret_cast<const int4*>(list + row);
      // plain loads: they must not move above the wait, as invariant ones may
      *reinterpret_cast<int4*>(&u.e.q0) = p[0];
      *reinterpret_cast<int4*>(&u.e.lim0) = p[1];
    }
    return u;
  };
  // the unit's last key block reaches past the sequence
  auto has_tail = [&](const Entry& e, int n) { return n * kBN > e.Lk; };

  if (warp == 0) {
    // ---------------------------------------------------------------- TMA
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsProducer));
    if (lane == 0) {
      bool ok = true;
      uint32_t g = 0, uq = 0;       // K/V blocks issued, query loads
      uint32_t tails = 0, tailed = 0;  // bit s: phase of V buffer s's vt_full; used at all
      const uint32_t q_bytes = 2 * C::kAtoms * (uint32_t)(a.G * a.R) * 128;
      Unit next = fetch(0);
      for (uint32_t ui = 0; next.valid && ok; ++ui) {
        const Unit u = next;
        next = fetch(ui + 1);
        const int n = max(u.e.n0, u.e.n1);
        if (n == 0) continue;
        if (!mbar_wait(&bars->q_empty, (uq & 1) ^ 1u, abort_flag, &g_packed_status, DEV_TIMEOUT_SLOT)) break;
        mbar_arrive_expect_tx(&bars->q_full, q_bytes);
        ++uq;
        for (int t = 0; t < 2; ++t)
          for (int at = 0; at < C::kAtoms; ++at)
            tma_load_3d(sQ + t * C::kTileBytes + at * C::kAtomTileBytes, &tmQ, &bars->q_full, at * 64,
                        u.kvh * a.G, u.e.q0 + t * a.R);
        for (int j = 0; j < n; ++j, ++g) {
          const int s = g & 1;
          const uint32_t par = ((g >> 1) & 1) ^ 1u;
          if (!mbar_wait(&bars->k_empty[s], par, abort_flag, &g_packed_status, DEV_TIMEOUT_SLOT)) { ok = false; break; }
          mbar_arrive_expect_tx(&bars->k_full[s], C::kTileBytes);
          for (int at = 0; at < C::kAtoms; ++at)
            tma_load_3d(sK + s * C::kTileBytes + at * C::kAtomTileBytes, &tmK, &bars->k_full[s], at * 64,
                        u.kvh, u.e.k0 + j * kBN);
          if (!mbar_wait(&bars->v_empty[s], par, abort_flag, &g_packed_status, DEV_TIMEOUT_SLOT)) {
            // aborted: K of this position is in flight, and only it
            const unsigned long long t0 = globaltimer();
            while (!mbar_test(smem_addr(&bars->k_full[s]), (g >> 1) & 1) && globaltimer() - t0 < kWaitLimitNs) {}
            ok = false;
            break;
          }
          const bool tail = j == n - 1 && has_tail(u.e, n);
          uint64_t* vbar = tail ? &bars->vt_full[s] : &bars->v_full[s];
          if (tail) {
            tails ^= 1u << s;
            tailed |= 1u << s;
          }
          mbar_arrive_expect_tx(vbar, C::kTileBytes);
          for (int at = 0; at < C::kAtoms; ++at)
            tma_load_3d(sV + s * C::kTileBytes + at * C::kAtomTileBytes, &tmV, vbar, at * 64, u.kvh,
                        u.e.k0 + j * kBN);
          *blocks = g + 1;
        }
      }
      // Bounded drain of copies still in flight into this CTA's shared memory.
      const unsigned long long t0 = globaltimer();
      auto drain = [&](uint64_t* bar, uint32_t par) {
        while (!mbar_test(smem_addr(bar), par)) {
          if (globaltimer() - t0 > kWaitLimitNs) { atomicOr(&g_packed_status, DEV_TIMEOUT_TMA); return; }
        }
      };
      if (uq > 0) drain(&bars->q_full, (uq - 1) & 1);
      for (uint32_t j = (g > 2 ? g - 2 : 0); j < g; ++j) {
        drain(&bars->k_full[j & 1], (j >> 1) & 1);
        drain(&bars->v_full[j & 1], (j >> 1) & 1);
      }
      for (int i = 0; i < 2; ++i)
        if ((tailed >> i) & 1u) drain(&bars->vt_full[i], ((tails >> i) & 1u) ^ 1u);
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsProducer));
    // The whole warp runs the loop and one elected lane issues.
    const bool leader = elect_one();
    constexpr uint32_t idS = idesc_f16(kBM, kBN, BF16, false, false);
    constexpr uint32_t idO = idesc_f16(kBM, D, BF16, false, true);
    constexpr uint32_t idL = idesc_f16(kBM, 16, BF16, false, false);
    const uint64_t dq0 = sdesc(smem_addr(sQ), 16, C::kSBO, kSwizzle128);
    const uint64_t dq1 = sdesc(smem_addr(sQ) + C::kTileBytes, 16, C::kSBO, kSwizzle128);
    const uint64_t dk0 = sdesc(smem_addr(sK), 16, C::kSBO, kSwizzle128);
    const uint64_t dk1 = sdesc(smem_addr(sK) + C::kTileBytes, 16, C::kSBO, kSwizzle128);
    const uint64_t dv0 = sdesc(smem_addr(sV), C::kAtomTileBytes, C::kSBO, kSwizzle128);
    const uint64_t dv1 = sdesc(smem_addr(sV) + C::kTileBytes, C::kAtomTileBytes, C::kSBO, kSwizzle128);
    const uint64_t dones = sdesc(smem_addr(sOnes), 128, 256, 0);
    (void)dones;
    auto qk = [&](int t, int ks) {
      const uint64_t da = t ? dq1 : dq0, db = ks ? dk1 : dk0;
      const uint32_t d = tS(t);
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        const uint32_t off16 = ((k / 4) * C::kAtomTileBytes + (k % 4) * 32) >> 4;
        if (leader) mma_f16_ss(d, da + off16, db + off16, idS, k > 0 ? 1u : 0u);
      }
      if (leader) mma_commit(&bars->s_full[t]);
    };
    auto pv = [&](int t, int vs, bool accumulate) {
      const uint64_t db = vs ? dv1 : dv0;
      const uint32_t d = tO(t), pa = tS(t);
#pragma unroll
      for (int k = 0; k < kBN / 16; ++k)
        if (leader) mma_f16_ts(d, pa + k * 8, db + ((k * 16 * 128) >> 4), idO, (k > 0 || accumulate) ? 1u : 0u);
      if constexpr (C::kSumMma) {
#pragma unroll
        for (int k = 0; k < kBN / 16; ++k)
          if (leader) mma_f16_ts(tL(t), pa + k * 8, dones, idL, (k > 0 || accumulate) ? 1u : 0u);
      }
    };
    bool ok = true, issued = false;
    uint32_t g = 0, uq = 0;
    uint32_t p_phase = 0, o_phase = 0;  // bit t: phase of tile t's p_full, of its o_empty
    Unit next = fetch(0);
    for (uint32_t ui = 0; next.valid && ok; ++ui) {
      const int n0 = next.e.n0, n1 = next.e.n1, n = max(n0, n1);
      if (n == 0) {
        next = fetch(ui + 1);
        continue;
      }
      if (!mbar_wait(&bars->q_full, uq & 1, abort_flag, &g_packed_status, DEV_TIMEOUT_TMA)) break;
      ++uq;
      if (!mbar_wait(&bars->k_full[g & 1], (g >> 1) & 1, abort_flag, &g_packed_status, DEV_TIMEOUT_TMA)) break;
      tc_fence_after();
      // S_t's TMEM held the previous unit's last P_t, whose P.V was issued earlier
      // (tcgen05.mma executes in order).
      if (n0 > 0) qk(0, g & 1);
      if (n1 > 0) qk(1, g & 1);
      if (leader) mma_commit(&bars->k_empty[g & 1]);
      if (n == 1 && leader) mma_commit(&bars->q_empty);
      next = fetch(ui + 1);  // while the tensor core works
      issued = true;
      for (int j = 0; j < n; ++j) {
        const uint32_t gj = g + j, gk = gj + 1;
        const int vs = gj & 1, ks = gk & 1;
        if (!mbar_wait(&bars->v_full[vs], (gj >> 1) & 1, abort_flag, &g_packed_status, DEV_TIMEOUT_TMA)) { ok = false; break; }
        // Both tiles' steps as straight code: a loop over them left their phases in
        // local memory, read before every P.V.
        if (j < n0) {
          // O_t holds the previous output until its softmax warps have read it
          if (j == 0) {
            if (!mbar_wait(&bars->o_empty[0], (o_phase & 1u) ^ 1u, abort_flag, &g_packed_status, DEV_TIMEOUT_EPI)) { ok = false; break; }
            o_phase ^= 1u;
          }
          if (!mbar_wait(&bars->p_full[0], p_phase & 1u, abort_flag, &g_packed_status, DEV_TIMEOUT_EPI)) { ok = false; break; }
          p_phase ^= 1u;
          tc_fence_after();
          pv(0, vs, j > 0);
          if (j == n0 - 1 && leader) mma_commit(&bars->o_full[0]);
        }
        if (j + 1 < n) {
          if (!mbar_wait(&bars->k_full[ks], (gk >> 1) & 1, abort_flag, &g_packed_status, DEV_TIMEOUT_TMA)) { ok = false; break; }
          tc_fence_after();
          if (j + 1 < n0) qk(0, ks);
        }
        if (j < n1) {
          if (j == 0) {
            if (!mbar_wait(&bars->o_empty[1], (o_phase >> 1) ^ 1u, abort_flag, &g_packed_status, DEV_TIMEOUT_EPI)) { ok = false; break; }
            o_phase ^= 2u;
          }
          if (!mbar_wait(&bars->p_full[1], p_phase >> 1, abort_flag, &g_packed_status, DEV_TIMEOUT_EPI)) { ok = false; break; }
          p_phase ^= 2u;
          tc_fence_after();
          pv(1, vs, j > 0);
          if (j == n1 - 1 && leader) mma_commit(&bars->o_full[1]);
        }
        if (leader) mma_commit(&bars->v_empty[vs]);
        if (j + 1 < n) {
          if (j + 1 < n1) qk(1, ks);
          if (leader) mma_commit(&bars->k_empty[ks]);
          if (j + 2 == n && leader) mma_commit(&bars->q_empty);  // last Q.K^T of the unit
        }
      }
      g += n;
    }
    if (issued) {
      if (leader) mma_commit(&bars->done);
      const unsigned long long t0 = globaltimer();
      while (!mbar_test(smem_addr(&bars->done), 0)) {
        if (globaltimer() - t0 > kWaitLimitNs) { atomicOr(&g_packed_status, DEV_TIMEOUT_MMA); break; }
      }
    }
  } else if (warp == 2) {
    // ------------------------------------------- V rows past the sequence's end
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsProducer));
    uint32_t g = 0;
    uint32_t tails = 0;  // bit s: phase of vt_full[s]
    // Units without such rows are passed over, so a wait can span many of them: seconds
    // in a batch of prompts of a million tokens. It ends when no block is asked for any more.
    auto wait_tail = [&](uint64_t* bar, uint32_t parity) {
      const uint32_t at = smem_addr(bar);
      uint32_t seen = *blocks;
      unsigned long long t0 = globaltimer();
      for (uint32_t it = 1; !mbar_test(at, parity); ++it) {
        if ((it & 63u) != 0) continue;
        if (*abort_flag) return false;
        const uint32_t now = *blocks;
        if (now != seen) {
          seen = now;
          t0 = globaltimer();
        } else if (globaltimer() - t0 > kWaitLimitNs) {
          *abort_flag = 1;
          atomicOr(&g_packed_status, DEV_TIMEOUT_TMA);
          return false;
        }
      }
      return true;
    };
    Unit next = fetch(0);
    for (uint32_t ui = 0; next.valid; ++ui) {
      const Unit u = next;
      next = fetch(ui + 1);
      const int n = max(u.e.n0, u.e.n1);
      g += n;
      if (n == 0 || !has_tail(u.e, n)) continue;
      const int s = (g - 1) & 1;
      if (!__all_sync(0xffffffffu, wait_tail(&bars->vt_full[s], (tails >> s) & 1u))) break;
      tails ^= 1u << s;
      const int first = u.e.Lk - (n - 1) * kBN;  // 1 .. 127: rows from here on are not the sequence's
      uint8_t* v = sV + s * C::kTileBytes;
      for (int i = lane; i < (kBN - first) * 8 * C::kAtoms; i += 32) {
        const int at = i / ((kBN - first) * 8), r = i % ((kBN - first) * 8);
        *reinterpret_cast<uint4*>(v + at * C::kAtomTileBytes + first * 128 + r * 16) = make_uint4(0, 0, 0, 0);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->v_full[s]);
    }
  } else if (warp >= 4) {
    // ------------------------------------------------- softmax / correction
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    const int t = (warp >= 8) ? 1 : 0;
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const int tok = row / a.G;  // of the tile
    const int gh = row - tok * a.G;
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const float scale_log2 = a.scale_log2;
    uint8_t* stg = sO + (warp - 4) * C::kOutStageBytes;
    bool ok = true;
    uint32_t gs = 0, co = 0;  // S blocks of this tile seen, outputs read
    bool odd = false;         // a row's result may hold what its masked keys hold
    Unit next = fetch(0);
    for (uint32_t ui = 0; next.valid && ok; ++ui) {
      const Unit u = next;
      next = fetch(ui + 1);
      const int i = t * a.R + tok;  // query of the entry
      const bool live = tok < a.R && i < u.e.nq;
      const int n_t = t == 0 ? u.e.n0 : u.e.n1;
      // keys [0, lim) are the row's; rows that hold no query keep none
      const int lim = !live ? 0 : a.causal ? min(u.e.Lk, u.e.lim0 + i) : u.e.Lk;
      // the first block that a row of the tile does not keep whole
      const int whole = a.causal ? min(u.e.Lk, u.e.lim0 + t * a.R) : u.e.Lk;
      float m_run = -INFINITY;  // running max in log2 units (possibly stale)
      float l_run = 0.f;
      for (int j = 0; j < n_t; ++j) {
        if (!mbar_wait(&bars->s_full[t], gs & 1, abort_flag, &g_packed_status, DEV_TIMEOUT_MMA)) { ok = false; break; }
        ++gs;
        tc_fence_after();
        uint32_t sr[kBN];
#pragma unroll
        for (int c = 0; c < kBN / 32; ++c)
          tmem_ld32(tS(t) + lane_off + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&sr[c * 32]));
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < kBN; ++e) asm volatile("" : "+r"(sr[e]));
        float s[kBN];
#pragma unroll
        for (int e = 0; e < kBN; ++e) s[e] = __uint_as_float(sr[e]);
        const int kbase = j * kBN;
        if (kbase + kBN > whole) {
          const int keep = lim - kbase;  // keys [0, keep) of the block
#pragma unroll
          for (int e = 0; e < kBN; ++e)
            if (e >= keep) s[e] = -INFINITY;
        }
        // Row max: four independent 3-input max chains.
        float mq[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int e = 4; e < kBN; e += 8) {
          mq[0] = fmax3_nan(mq[0], s[e], s[e + 1]);
          mq[1] = fmax3_nan(mq[1], s[e + 2], s[e + 3]);
          mq[2] = fmax3_nan(mq[2], e + 4 < kBN ? s[e + 4] : -INFINITY, e + 5 < kBN ? s[e + 5] : -INFINITY);
          mq[3] = fmax3_nan(mq[3], e + 6 < kBN ? s[e + 6] : -INFINITY, e + 7 < kBN ? s[e + 7] : -INFINITY);
        }
        const float mx = fmax3_nan(fmax3_nan(mq[0], mq[1], mq[2]), mq[3], -INFINITY) * scale_log2;
        // Rescale only when some row of this warp grew its max by > 2^8 (or is NaN).
        const bool grow = !(mx <= m_run + kRescaleThreshold);
        const bool warp_rescale = __any_sync(0xffffffffu, grow);
        float alpha = 1.f;
        if (warp_rescale) {
          float m_new = fmax3_nan(m_run, mx, -INFINITY);
          // an infinite score has no softmax (inf - inf)
          if (m_new == INFINITY) m_new = __int_as_float(0x7fffffff);
          alpha = (m_run == -INFINITY) ? 0.f : ex2(m_run - m_new);
          m_run = m_new;
        }
        const float m_use = m_run == -INFINITY ? 0.f : m_run;
        const f2_t sc2 = f2_pack(scale_log2, scale_log2), nm2 = f2_pack(-m_use, -m_use);
        f2_t acc2[4] = {0ull, 0ull, 0ull, 0ull};
        uint32_t p[kBN / 2];
        // 5/8 (D = 128) or 1/2 of the exponentials on the MUFU, the rest on the FMA
        // pipe: the split measured best for this loop in fa_sm100.cu.
#pragma unroll
        for (int e = 0; e < kBN / 2; ++e) {
          const f2_t x2 = f2_fma(f2_pack(s[2 * e], s[2 * e + 1]), sc2, nm2);
          float x0, x1, p0, p1;
          f2_unpack(x2, x0, x1);
          if (D == 128 ? (e & 7) < 5 : (e & 1) == 0) {
            p0 = ex2(x0);
            p1 = ex2(x1);
          } else {
            exp2_poly2(x0, x1, p0, p1);
          }
          if constexpr (!C::kSumMma) acc2[e & 3] = f2_add(acc2[e & 3], f2_pack(p0, p1));
          p[e] = BF16 ? pack_bf162(p0, p1) : pack_half2(p0, p1);
        }
        if constexpr (!C::kSumMma) {
          const f2_t a01 = f2_add(acc2[0], acc2[1]), a23 = f2_add(acc2[2], acc2[3]);
          float u0, u1;
          f2_unpack(f2_add(a01, a23), u0, u1);
          l_run = l_run * alpha + (u0 + u1);
        }
#pragma unroll
        for (int c = 0; c < kBN / 2 / 32; ++c) {
          uint32_t r[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) r[e] = p[c * 32 + e];
          tmem_st32(tS(t) + lane_off + c * 32, r);
        }
        if (warp_rescale && j > 0) {
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            uint32_t r[32];
            tmem_ld32(tO(t) + lane_off + c * 32, r);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) * alpha);
            tmem_st32(tO(t) + lane_off + c * 32, r);
          }
          if constexpr (C::kSumMma) {
            const uint32_t lc = tmem_ld1(tL(t) + lane_off);
            tmem_ld_wait();
            tmem_st1(tL(t) + lane_off, __float_as_uint(__uint_as_float(lc) * alpha));
          }
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->p_full[t]);
      }
      if (!ok) break;
      // the row's place in the output, elements; -1: no query
      T* const obase = static_cast<T*>(a.o) + (long long)u.e.q0 * a.ot + (long long)u.kvh * a.G * a.oh;
      const long long ooff = live ? (long long)i * a.ot + (long long)gh * a.oh : -1;
      if (n_t > 0) {
        if (!mbar_wait(&bars->o_full[t], co & 1, abort_flag, &g_packed_status, DEV_TIMEOUT_MMA)) { ok = false; break; }
        ++co;
        tc_fence_after();
        if constexpr (C::kSumMma) {
          l_run = __uint_as_float(tmem_ld1(tL(t) + lane_off));
          tmem_ld_wait();
        }
      }
      // no key: zeros; keys whose scores are all -inf, or NaN: NaN
      const float inv = lim <= 0 ? 0.f : l_run > 0.f ? 1.f / l_run : __int_as_float(0x7fffffff);
      // All of the row first, so that the next unit's P.V may overwrite O early.
      uint32_t r[D];
      if (n_t > 0) {
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
          tmem_ld32(tO(t) + lane_off + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&r[c * 32]));
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < D; ++e) asm volatile("" : "+r"(r[e]));
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->o_empty[t]);
        // a row without a key in a tile with keys: its weights are 0, which a value that
        // is not finite turns into NaN
        if (lim <= 0) {
#pragma unroll
          for (int e = 0; e < D; ++e) r[e] = 0u;
        }
      } else {
#pragma unroll
        for (int e = 0; e < D; ++e) r[e] = 0u;
      }
      float probe = 0.f;  // NaN once a value of the row is not finite
#pragma unroll
      for (int at = 0; at < C::kAtoms; ++at) {
        __syncwarp();
#pragma unroll
        for (int v = 0; v < 8; ++v) {
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float f0 = __uint_as_float(r[at * 64 + v * 8 + 2 * e]) * inv;
            const float f1 = __uint_as_float(r[at * 64 + v * 8 + 2 * e + 1]) * inv;
            probe = fmaf(f0, 0.f, probe);
            probe = fmaf(f1, 0.f, probe);
            w[e] = BF16 ? pack_bf162(f0, f1) : pack_half2(f0, f1);
          }
          *reinterpret_cast<uint4*>(stg + lane * 128 + ((v ^ (lane & 7)) * 16)) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        __syncwarp();
        // 8 lanes write a row's 128 bytes, four rows at a time
#pragma unroll
        for (int it = 0; it < 8; ++it) {
          const int line = it * 4 + (lane >> 3), ch = lane & 7;
          const long long off = __shfl_sync(0xffffffffu, ooff, line);
          const uint4 val = *reinterpret_cast<const uint4*>(stg + line * 128 + ((ch ^ (line & 7)) * 16));
          if (off >= 0 && at * 64 + ch * 8 < a.D)
            *reinterpret_cast<uint4*>(obase + off + at * 64 + ch * 8) = val;
        }
      }
      odd = odd || (lim > 0 && lim < min(n_t * kBN, u.e.Lk) && probe != probe);
    }
    if (__any_sync(0xffffffffu, odd)) {
      // A result of this warp was not finite, in a row with masked keys in its blocks.
      // Walk its units again: where a row is not finite and a masked value is not
      // either, the row is computed anew in fp32. Out of the loop above, where even a
      // call cost its registers (causal [4, 16, 2048, 128] 78 -> 85 us).
      __syncwarp();
      const int c = lane * 4;
      const bool on = c < a.D;
      auto load4 = [&](const void* base, long long at, float (&x)[4]) {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = on ? to_f32<T>(static_cast<const T*>(base)[at + c + e]) : 0.f;
      };
      auto unfinished = [&](const float (&x)[4]) {
        return __any_sync(0xffffffffu, !(isfinite(x[0]) && isfinite(x[1]) && isfinite(x[2]) && isfinite(x[3])));
      };
      for (uint32_t ui = 0;; ++ui) {
        const Unit u = fetch(ui);
        if (!u.valid) break;
        const int hi = min((t == 0 ? u.e.n0 : u.e.n1) * kBN, u.e.Lk);
        for (int x = 0; x < 32; ++x) {
          const int w = (quarter * 32 + x) / a.G, i = t * a.R + w;
          const int n = a.causal ? min(u.e.Lk, u.e.lim0 + i) : u.e.Lk;
          if (w >= a.R || i >= u.e.nq || n <= 0 || n >= hi) continue;
          const long long token = u.e.q0 + i, head = u.kvh * a.G + (quarter * 32 + x) - w * a.G;
          const long long k0 = u.e.k0 * a.kt + u.kvh * a.kh, v0 = u.e.k0 * a.vt + u.kvh * a.vh;
          float f[4];
          load4(a.o, token * a.ot + head * a.oh, f);
          if (!unfinished(f)) continue;
          bool found = false;
          for (int j = n; j < hi && !found; ++j) {
            load4(a.v, v0 + j * a.vt, f);
            found = unfinished(f);
          }
          if (!found) continue;
          float q[4], acc[4] = {}, m = -INFINITY, l = 0.f;
          load4(a.q, token * a.qt + head * a.qh, q);
          for (int j = 0; j < n; ++j) {
            load4(a.k, k0 + j * a.kt, f);
            float s = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) s = fmaf(q[e], f[e], s);
#pragma unroll
            for (int y = 16; y > 0; y >>= 1) s += __shfl_xor_sync(0xffffffffu, s, y);
            s *= scale_log2;
            const float mn = fmaxf(m, s), base = mn == -INFINITY ? 0.f : mn;
            const float al = exp2f(m - base), p = exp2f(s - base);
            m = mn;
            l = l * al + p;
            load4(a.v, v0 + j * a.vt, f);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] = acc[e] * al + p * f[e];
          }
          if (on)
#pragma unroll
            for (int e = 0; e < 4; ++e) static_cast<T*>(a.o)[token * a.ot + head * a.oh + c + e] = from_f32<T>(acc[e] / l);
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsProducer));
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

template <int D, bool BF16>
int launch(const PackedCall& c, cudaStream_t st) {
  const int G = (int)(c.Hq / c.Hk), R = kBM / G;
  const long long most = (c.Tq / (2 * R) + c.B + 2) * c.Hk;
  if (most >= (1LL << 31)) {
    set_error("b2_fa_packed: %lld units of work are too many for one launch", most);
    return B2_EINVAL;
  }
  const CUtensorMapDataType tdt = BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const void* ptrs[3] = {c.q, c.k, c.v};
  const int64_t heads[3] = {c.Hq, c.Hk, c.Hk}, tokens[3] = {c.Tq, c.Tk, c.Tk};
  CUtensorMap tm[3];
  for (int i = 0; i < 3; ++i) {
    const int64_t* s = c.strides + 3 * i;  // t, h, d
    const uint64_t dims[3] = {(uint64_t)c.D, (uint64_t)heads[i], (uint64_t)tokens[i]};
    const uint64_t strides[2] = {(uint64_t)s[1] * 2, (uint64_t)s[0] * 2};
    const uint32_t box[3] = {64, i == 0 ? (uint32_t)G : 1u, i == 0 ? (uint32_t)R : (uint32_t)kBN};
    if (!encode_tmap(&tm[i], tdt, 3, ptrs[i], dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)) return B2_ELAUNCH;
  }
  auto kern = fa_packed_kernel<D, BF16>;
  static OncePerDevice ready;
  B2_CUDA_TRY(ready([&] {
    // setmaxnreg.inc waits until the block's register pool can serve it: only
    // launch when the compiled allocation covers the split.
    cudaFuncAttributes fa;
    cudaError_t e = cudaFuncGetAttributes(&fa, kern);
    if (e != cudaSuccess) return e;
    if (fa.numRegs < kLaunchRegs) return cudaErrorInvalidKernelImage;
    return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Cfg<D>::kSmem);
  }));
  int* ws = static_cast<int*>(c.workspace);
  const PlanArgs pa = {c.cu_q, c.cu_k, (int)c.B, (int)c.Tq, (int)c.Tk, R, c.causal, ws};
  const int64_t planners = 32 * (c.B + 2);  // a warp per sequence, and for what lies before and after them
  // 12 prompts: 12.7 us a call, 12.8 with 1024 threads
  fa_packed_plan_kernel<<<1, (int)(planners < kPlanClasses ? kPlanClasses : planners > 1024 ? 1024 : planners), 0, st>>>(pa);
  B2_CHECK_LAUNCH();
  KernelArgs a = {ws, c.q, c.k, c.v, c.o};
  a.qt = c.strides[0];
  a.qh = c.strides[1];
  a.kt = c.strides[3];
  a.kh = c.strides[4];
  a.vt = c.strides[6];
  a.vh = c.strides[7];
  a.ot = c.strides[9];
  a.oh = c.strides[10];
  a.G = G;
  a.R = R;
  a.Hk = (int)c.Hk;
  a.D = (int)c.D;
  a.causal = c.causal;
  a.scale_log2 = c.sm_scale * kLog2e;
  a.most = (unsigned)most;
  const int sms = device_sm_count();
  // The kernel's prologue (barriers, TMEM, descriptors) runs beside the plan kernel.
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(most < sms ? most : sms));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Cfg<D>::kSmem;
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  B2_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, tm[0], tm[1], tm[2], a));
  return B2_OK;
}

}  // namespace

size_t fa_packed_workspace(int64_t B, int64_t Tq, int64_t share) {
  if (B < 0 || Tq <= 0 || share < 1 || share > kBM) return 0;
  return kPlanHeader + sizeof(Entry) * (size_t)(Tq / (2 * (kBM / share)) + B + 2);
}

bool fa_packed_sm100_eligible(const PackedCall& c) {
  if (c.dtype != B2_F16 && c.dtype != B2_BF16) return false;
  if (c.D % 8 || c.D > 128 || !(c.sm_scale > 0.f) || c.Tk == 0 || c.Hq / c.Hk > kBM) return false;
  const void* p[4] = {c.q, c.k, c.v, c.o};
  for (int i = 0; i < 4; ++i) {
    if ((reinterpret_cast<uintptr_t>(p[i]) & 15) != 0) return false;
    const int64_t *s = c.strides + 3 * i;
    if (s[2] != 1 || s[0] % 8 || s[1] % 8) return false;
    // a tensor map wants positive strides below 2^40 bytes
    if (i < 3 && (s[0] <= 0 || s[0] >= (1LL << 38) || s[1] <= 0 || s[1] >= (1LL << 38))) return false;
  }
  const size_t need = fa_packed_workspace(c.B, c.Tq, c.Hq / c.Hk);
  return c.workspace && c.ws_bytes >= need && (reinterpret_cast<uintptr_t>(c.workspace) & 15) == 0;
}

int fa_packed_sm100_launch(const PackedCall& c, cudaStream_t st) {
  const bool bf = c.dtype == B2_BF16;
  if (c.D <= 64) return bf ? launch<64, true>(c, st) : launch<64, false>(c, st);
  return bf ? launch<128, true>(c, st) : launch<128, false>(c, st);
}

uint32_t fa_packed_read_status(bool clear) {
  uint32_t v = 0;
  cudaMemcpyFromSymbol(&v, g_packed_status, sizeof(v));
  if (clear) {
    const uint32_t z = 0;
    cudaMemcpyToSymbol(g_packed_status, &z, sizeof(z));
  }
  return v;
}

}  // namespace b2
