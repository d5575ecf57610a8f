// Cross-attention gradient on the tensor cores.
//
//   S = Q K^T, dP = dO V^T                         (tensor memory, 32 bits)
//   P = 2^(c S + bias - lse), dS = P (dP - delta)  (registers; delta = sum_k P dP)
//   dV += P^T dO, dK += dS^T Q, dQ = dS K
//
// A block of 256 threads owns one head's tile of up to 128 keys (kKeys, kBoth) and
// walks over 128-query tiles with dK and dV in tensor memory, or owns a query tile
// and walks over the keys with dQ there (kQueries).  A tensor-memory lane is a
// query; two threads share it, half of the keys each.  Where all keys fit one tile
// one walk does everything (kBoth): delta is summed from P and dP themselves and O
// is not read.  More keys take a row-sum pass (delta = dO . O), then kKeys and
// kQueries, which both form S and dP: seven products instead of five, and no sum
// whose order could change.
//
// P and dS go through shared memory as [query][key] tiles in the swizzle that the
// products read, with the queries as the contraction (dV, dK: the contiguous index
// is the operand's M) or the keys (dQ).  S and dP of the next tile are started
// behind the products of this one, where tensor memory has room for dQ beside them.
//
// Rounding.  P and dS are rounded to the element type once, for the products.
// FP16's range is short for that: P is held 2^kLift times larger, and dS is scaled
// by a power of two that follows the largest |dP| and |delta| of the block's walk.
//
// What bounds it.  8 x 1024 queries x 8 heads x 80, 77 keys, FP16, forward and gradient:
// 41.5 us.  One block to an SM, and a tile's steps follow one another; before arithmetic
// was paired a 128-query tile took about 9,000 cycles: scores and dP waited for 1,700 to
// 2,400, P 2,100, exchange 490, dS 860, products 1,600, dQ 1,800.  Pairing, with row sums by
// groups of lanes, took 3 x 1021 queries to 333 keys from 89 us to 76; their additive
// biases' largest, and what it is taken off, cost 3 again (80).  The products are too small
// to keep the tensor cores busy (9 % of their cycles).
#include <cuda_runtime.h>

#include "nova_attention.cuh"

namespace nova {
namespace xattn {

using namespace tc;

namespace {

constexpr int kRows = 128;
constexpr int kThreads = 256;
constexpr float kLift = 10.f;
constexpr int kMaxExp = 60;

enum Mode : int { kBoth = 0, kKeys = 1, kQueries = 2 };

struct BwdParams {
  Args a;
  Pick qp, kp, vp, gp;
  int KT, nkt;        // keys per tile, tiles
  int DB, DP;         // 64-element blocks and padded width of a head
  int qtiles;         // query tiles of a head
  int chunk, splits;  // query tiles per block, blocks per head and key tile
  int stages;         // of the walked pair
  int early;          // S and dP of the next tile before dQ of this one is read
  uint32_t c_dv, c_dk, c_dq;  // tensor-memory columns (S at 0, dP at KT)
  uint32_t q_bytes, k_bytes;  // one tile of Q or dO, of K or V
  float *part_dk, *part_dv;   // [splits][B][Nk][H][D]
};

__device__ int g_status;

template <typename T, bool MASK, int MODE>
__global__ void __launch_bounds__(kThreads, 1)
    backward_tc(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                const __grid_constant__ CUtensorMap mv, const __grid_constant__ CUtensorMap mg,
                const __grid_constant__ CUtensorMap mdq, const __grid_constant__ BwdParams p) {
  constexpr bool kBf16 = !std::is_same<T, __half>::value;
  constexpr bool kWalkQ = MODE != kQueries;
  extern __shared__ unsigned char raw[];
  __shared__ uint64_t bars[5];  // fixed pair, walked pair [2], S and dP, the other products
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  __shared__ alignas(8) float bias[2][kRows];
  __shared__ float red[2][kRows];
  __shared__ uint32_t peak[kThreads / 32];
  __shared__ float refs[kThreads / 32];  // largest biases of the sample, a part for each warp
  const int tid = threadIdx.x, half = tid >> 7, r = tid & (kRows - 1);
  const int warp = __shfl_sync(~0u, tid >> 5, 0);
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
  // Fixed pair, walked pairs, P, dS.
  const uint32_t fixed_bytes = kWalkQ ? p.k_bytes : p.q_bytes;
  const uint32_t walk_bytes = kWalkQ ? p.q_bytes : p.k_bytes;
  const uint32_t s_fix = base, s_walk = base + 2 * fixed_bytes;
  const uint32_t s_p = s_walk + 2 * p.stages * walk_bytes;
  const uint32_t s_ds = MODE == kQueries ? s_p : s_p + 2 * kRows * 128;
  const uint32_t bf = smem_u32(&bars[0]), bx = smem_u32(&bars[1]), bs = smem_u32(&bars[3]),
                 bd = smem_u32(&bars[4]);
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&tmem_slot)),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (tid == 32) {
    for (int i = 0; i < 5; ++i) mbar_init(smem_u32(&bars[i]), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    abort_flag = 0;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(~0u, tmem_slot, 0);
  // Warp 0 starts copies and products; one lane of it, always the same, does.
  bool one = false;
  if (warp == 0) one = elect_one();
  const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
  pdl_trigger();
  pdl_wait();

  unsigned id = blockIdx.x;
  int split = 0, kt_fix = 0, t_first, steps;
  if (kWalkQ) {
    split = id % p.splits;
    id /= p.splits;
    kt_fix = id % p.nkt;
    id /= p.nkt;
    t_first = split * p.chunk;
    steps = min(p.qtiles, t_first + p.chunk) - t_first;
  } else {
    t_first = id % p.qtiles;
    id /= p.qtiles;
    steps = p.nkt;
  }
  const int h = id % p.a.H, b = id / p.a.H;
  const long long row0 = ((long long)b * p.a.H + h) * p.a.Nq;

  // A pair of tiles: (Q, dO) of query tile t, or (K, V) of key tile t.
  auto load_q = [&](int t, uint32_t at, uint32_t bar) {
    mbar_expect_tx(bar, 2 * p.q_bytes);
    for (int d = 0; d < p.DB; ++d)
      tma_load_4d(at + d * (kRows * 128), &mq, d * 64, t * kRows, h * p.qp.h, b * p.qp.b, bar);
    for (int d = 0; d < p.DB; ++d)
      tma_load_4d(at + p.q_bytes + d * (kRows * 128), &mg, d * 64, t * kRows, h * p.gp.h,
                  b * p.gp.b, bar);
  };
  auto load_k = [&](int t, uint32_t at, uint32_t bar) {
    mbar_expect_tx(bar, 2 * p.k_bytes);
    for (int d = 0; d < p.DB; ++d)
      tma_load_4d(at + d * (p.KT * 128), &mk, d * 64, t * p.KT, h * p.kp.h, b * p.kp.b, bar);
    for (int d = 0; d < p.DB; ++d)
      tma_load_4d(at + p.k_bytes + d * (p.KT * 128), &mv, d * 64, t * p.KT, h * p.vp.h, b * p.vp.b,
                  bar);
  };
  auto load_step = [&](int i) {
    const int st = i % p.stages;
    const uint32_t at = s_walk + 2 * st * walk_bytes;
    if (kWalkQ) load_q(t_first + i, at, bx + 8u * st);
    else load_k(i, at, bx + 8u * st);
  };
  const uint32_t idesc_s = instr_desc(kBf16, kRows, p.KT, false, false);
  const uint32_t idesc_d = instr_desc(kBf16, kRows, p.DP, true, true);
  const uint32_t idesc_q = instr_desc(kBf16, kRows, p.DP, false, true);
  const int chunks = p.KT / 16;
  // S and dP of step i, by warp 0; its tiles have landed when this returns true.
  auto start_scores = [&](int i) {
    const int st = i % p.stages;
    if (!wait_phase(bx + 8u * st, (i / p.stages) & 1, &abort_flag, &g_status, kDevTimeoutProducer))
      return false;
    tc_fence_after();
    const uint32_t x = s_walk + 2 * st * walk_bytes;
    const uint32_t q_at = kWalkQ ? x : s_fix, k_at = kWalkQ ? s_fix : x;
    if (one) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint64_t ad = smem_desc_sw128(q_at + u * p.q_bytes);
        const uint64_t kd = smem_desc_sw128(k_at + u * p.k_bytes);
#pragma unroll
        for (int s = 0; s < kMaxD / 16; ++s)
          if (s < p.DP / 16)
            umma_f16(tmem + u * p.KT, ad + (uint32_t)((s >> 2) * (kRows * 8) + (s & 3) * 2),
                     kd + (uint32_t)((s >> 2) * (p.KT * 8) + (s & 3) * 2), idesc_s, s != 0);
      }
      umma_commit(bs);
    }
    return true;
  };

  int loaded = 0;  // started walked pairs
  bool ok = true;
  if (one) {
    if (kWalkQ) load_k(kt_fix, s_fix, bf);
    else load_q(t_first, s_fix, bf);
    for (int u = 0; u < p.stages && u < steps; ++u) load_step(u);
  }
  loaded = min(p.stages, steps);
  // Bias of key tile `t` into bias[slot], minus infinity for a key that is out.
  auto set_bias = [&](int t, int slot) {
    const int keys = min(p.KT, p.a.Nk - t * p.KT);
    if (tid < p.KT) {
      float x = -INFINITY;
      const bool in = tid < keys && key_bias(p.a, b, t * p.KT + tid, &x);
      bias[slot][tid] = in ? x : -INFINITY;
    }
  };
  // Clears the rows of K (and of V behind it) of keys that are out: P and dS are zero
  // there, and zero times infinity is not.
  auto clear_masked = [&](uint32_t k_at, int slot, bool both) {
    if (tid < p.KT && bias[slot][tid] == -INFINITY) {
      for (int u = 0; u < (both ? 2 : 1); ++u)
        for (int d = 0; d < p.DB; ++d)
          for (int i = 0; i < 8; ++i)
            st_shared_v4(k_at + u * p.k_bytes + d * (p.KT * 128) + sw128(tid, i), 0, 0, 0, 0);
      fence_async_smem();
    }
  };
  // lse is relative to the sample's largest bias.
  if (MASK && kWalkQ) set_bias(kt_fix, 0);
  if (MASK && is_additive(p.a)) {
    const float part = warp_most(largest_bias(p.a, b, tid, kThreads));
    if ((tid & 31) == 0) refs[warp] = part;
  }
  ok = wait_phase(bf, 0, &abort_flag, &g_status, kDevTimeoutProducer);
  if (MASK && kWalkQ && ok) clear_masked(s_fix, 0, true);
  if (!__syncthreads_and(ok)) ok = false;
  if (warp == 0 && ok) ok = start_scores(0);
  float ref = 0.f;
  if (MASK && is_additive(p.a)) {
    ref = refs[0];
#pragma unroll
    for (int w = 1; w < kThreads / 32; ++w) ref = fmaxf(ref, refs[w]);
    if (ref == -INFINITY) ref = 0.f;  // no key takes part
  }

  const float c = p.a.scale * kLog2e;
  const int n0 = (chunks + 1) / 2;
  const int first = half ? n0 : 0, count = half ? chunks - n0 : n0;  // this thread's 16-key chunks
  int exp_now = 0;
  bool exp_set = false;

  // The row's lse (no contribution from rows past the end or without keys) and delta.
  auto row_lse = [&](int t) {
    const int row = t * kRows + r;
    if (row >= p.a.Nq) return INFINITY;
    const float v = p.a.lse_in[row0 + row];
    return v == -INFINITY ? INFINITY : v;
  };
  auto row_delta = [&](int t) {
    const int row = t * kRows + r;
    return row < p.a.Nq ? p.a.delta[row0 + row] : 0.f;
  };
  // A sample without keys (all its rows are) passes nothing on, whatever its q and do hold.
  const uint32_t keep = MASK && p.a.lse_in[row0] == -INFINITY ? 0u : ~0u;
  float lse = row_lse(t_first);
  float delta = MODE == kBoth ? 0.f : row_delta(t_first);

  int i = 0;
  for (; i < steps; ++i) {  // leaves early only where all threads do
    const int st = i % p.stages, slot = kWalkQ ? 0 : (i & 1);
    const uint32_t x = s_walk + 2 * st * walk_bytes;
    const uint32_t q_at = kWalkQ ? x : s_fix, k_at = kWalkQ ? s_fix : x;
    const int kt = kWalkQ ? kt_fix : i;
    const int keys = min(p.KT, p.a.Nk - kt * p.KT);
    if (MASK && !kWalkQ) {
      set_bias(i, slot);
      __syncthreads();
    }
    float lse_next = 0.f, delta_next = 0.f;
    if (kWalkQ && i + 1 < steps) {
      lse_next = row_lse(t_first + i + 1);
      if (MODE == kKeys) delta_next = row_delta(t_first + i + 1);
    }
    ok = wait_phase(bs, i & 1, &abort_flag, &g_status, kDevTimeoutMma);
    __syncwarp();
    tc_fence_after();

    // P (times 2^kLift) and dP of this thread's keys.
    uint32_t s[4][16], g[4][16];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (u < count) {
        tmem_ld16_issue(lanes + 16u * (first + u), s[u]);
        tmem_ld16_issue(lanes + p.KT + 16u * (first + u), g[u]);
      }
    tmem_wait_ld();
    tc_fence_before();
    float2 sums = make_float2(0.f, 0.f);
    float top = 0.f;
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (u < count) {
        const int col = 16 * (first + u);
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          float2 dp = make_float2(__uint_as_float(g[u][e]), __uint_as_float(g[u][e + 1]));
          float2 x = make_float2(__uint_as_float(s[u][e]), __uint_as_float(s[u][e + 1]));
          // The product is rounded before lse is taken off, as it was when lse was
          // formed: a single key's probability is then exactly one.
          if (MASK) {
            const float2 add = *reinterpret_cast<const float2*>(&bias[slot][col + e]);
            x = __ffma2_rn(x, make_float2(c, c), add);
            x = __fadd2_rn(x, make_float2(-ref, -ref));
            if (MODE == kQueries) {  // K and V of a key that is out hold anything here
              if (add.x == -INFINITY) x.x = -INFINITY, dp.x = 0.f;
              if (add.y == -INFINITY) x.y = -INFINITY, dp.y = 0.f;
            }
          } else {
            x = __fmul2_rn(x, make_float2(c, c));
          }
          x = __fadd2_rn(x, make_float2(-lse, -lse));
          x = __fadd2_rn(x, make_float2(kLift, kLift));
          s[u][e] = __float_as_uint(ex2(x.x));
          s[u][e + 1] = __float_as_uint(ex2(x.y));
          g[u][e] = __float_as_uint(dp.x);
          g[u][e + 1] = __float_as_uint(dp.y);
        }
        if (!MASK && col + 16 > keys) {
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (col + e >= keys) s[u][e] = 0u;
        }
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          const float2 dp = make_float2(__uint_as_float(g[u][e]), __uint_as_float(g[u][e + 1]));
          if (MODE == kBoth)
            sums = __ffma2_rn(make_float2(__uint_as_float(s[u][e]), __uint_as_float(s[u][e + 1])), dp,
                              sums);
          if (!kBf16) top = fmaxf(top, fmaxf(fabsf(dp.x), fabsf(dp.y)));
        }
      }
    const float sum = sums.x + sums.y;
    if (MODE == kBoth) red[half][r] = sum;
    if (!kBf16) {
      // delta comes from all tiles, and may be far above this one's dP.
      if (MODE != kBoth) top = fmaxf(top, fabsf(delta));
      // A row that is not finite has no say in the scale of the others.
      const uint32_t bits = isfinite(top) && isfinite(sum) ? __float_as_uint(top) : 0u;
      const uint32_t most = __reduce_max_sync(~0u, bits);
      if ((tid & 31) == 0) peak[warp] = most;
    }
    // The rows of dQ staged over P and dS have left before these are written.
    if (MODE == kBoth && one) bulk_wait_read_all();
    if (!__syncthreads_and(ok)) {
      ok = false;
      break;
    }
    if (MODE == kBoth) delta = (red[0][r] + red[1][r]) * (1.f / 1024.f);
    float lift = 1.f / 1024.f;  // 2^-kLift, times 2^exp_now
    if (!kBf16) {
      uint32_t most = 0;
#pragma unroll
      for (int w = 0; w < kThreads / 32; ++w) most = max(most, peak[w]);
      const int ex = (int)(most >> 23) - 127;  // |dP|, |delta| < 2^(ex + 1), |dS| < 2^(ex + 2)
      if (!exp_set || exp_now > 13 - ex) {
        int to = 9 - ex;
        to = to > kMaxExp ? kMaxExp : to < -kMaxExp ? -kMaxExp : to;
        if (exp_set && i > 0 && to != exp_now) {
          const float f = exp2f((float)(to - exp_now));
          const uint32_t acc = MODE == kQueries ? p.c_dq : p.c_dk;
          for (int u = half; u < p.DP / 16; u += 2) {
            uint32_t o[16];
            tmem_ld16_issue(lanes + acc + 16u * u, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            tmem_st16(lanes + acc + 16u * u, o);
          }
          tmem_wait_st();
        }
        exp_now = to;
        exp_set = true;
      }
      lift *= exp2f((float)exp_now);
    }
    if (MASK && MODE == kQueries) clear_masked(k_at, slot, false);
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (u < count) {
        const int ck = first + u;
        const uint32_t at = (uint32_t)(ck >> 2) * (kRows * 128);
        uint32_t w[8];
        if (MODE != kQueries) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            w[e] = pack2<T>(__uint_as_float(s[u][2 * e]), __uint_as_float(s[u][2 * e + 1]));
          st_shared_v4(s_p + at + sw128(r, (ck & 3) * 2), w[0], w[1], w[2], w[3]);
          st_shared_v4(s_p + at + sw128(r, (ck & 3) * 2 + 1), w[4], w[5], w[6], w[7]);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float2 d = make_float2(__uint_as_float(g[u][2 * e]), __uint_as_float(g[u][2 * e + 1]));
          d = __fmul2_rn(__fadd2_rn(d, make_float2(-delta, -delta)), make_float2(lift, lift));
          d = __fmul2_rn(d, make_float2(__uint_as_float(s[u][2 * e]), __uint_as_float(s[u][2 * e + 1])));
          w[e] = pack2<T>(d.x, d.y);
        }
        st_shared_v4(s_ds + at + sw128(r, (ck & 3) * 2), w[0], w[1], w[2], w[3]);
        st_shared_v4(s_ds + at + sw128(r, (ck & 3) * 2 + 1), w[4], w[5], w[6], w[7]);
      }
    fence_async_smem();
    tc_fence_before();
    __syncthreads();

    if (warp == 0) {
      tc_fence_after();
      if (one) {
        if (MODE != kQueries) {
          // dV += P^T dO, dK += dS^T Q: the queries are the contraction.
          const uint64_t pd = smem_desc_mn(s_p, kRows * 128), sd = smem_desc_mn(s_ds, kRows * 128);
          const uint64_t gd = smem_desc_mn(q_at + p.q_bytes, kRows * 128),
                         qd = smem_desc_mn(q_at, kRows * 128);
#pragma unroll
          for (int u = 0; u < kRows / 16; ++u)
            umma_f16(tmem + p.c_dv, pd + 128ull * u, gd + 128ull * u, idesc_d, u != 0 || i != 0);
#pragma unroll
          for (int u = 0; u < kRows / 16; ++u)
            umma_f16(tmem + p.c_dk, sd + 128ull * u, qd + 128ull * u, idesc_d, u != 0 || i != 0);
        }
        if (MODE != kKeys) {
          const uint64_t sd = smem_desc_sw128(s_ds), kd = smem_desc_mn(k_at, p.KT * 128);
#pragma unroll
          for (int u = 0; u < 8; ++u)
            if (u < chunks)
              umma_f16(tmem + p.c_dq, sd + (uint32_t)((u >> 2) * (kRows * 8) + (u & 3) * 2),
                       kd + 128ull * u, idesc_q, u != 0 || (MODE == kQueries && i != 0));
        }
        umma_commit(bd);
      }
      if (p.early && i + 1 < steps) ok = start_scores(i + 1);
    }
    ok = ok && wait_phase(bd, i & 1, &abort_flag, &g_status, kDevTimeoutEpilogue);
    if (loaded < steps) {
      if (one && ok) load_step(loaded);
      ++loaded;
    }
    __syncwarp();
    tc_fence_after();
    if (MODE == kBoth) {
      // dQ of the tile, staged over P and dS.
      const float f = p.a.scale * exp2f((float)-exp_now);
      uint32_t o[kMaxD / 32][16];
#pragma unroll
      for (int u = 0; u < kMaxD / 32; ++u)
        if (half + 2 * u < p.DP / 16) tmem_ld16_issue(lanes + p.c_dq + 16u * (half + 2 * u), o[u]);
      tmem_wait_ld();
#pragma unroll
      for (int u = 0; u < kMaxD / 32; ++u) {
        const int ck = half + 2 * u;
        if (ck < p.DP / 16) {
          uint32_t w[8];
#pragma unroll
          for (int e = 0; e < 8; ++e)
            w[e] = keep &
                   pack2<T>(__uint_as_float(o[u][2 * e]) * f, __uint_as_float(o[u][2 * e + 1]) * f);
          const uint32_t at = s_p + (uint32_t)(ck >> 2) * (kRows * 128);
          st_shared_v4(at + sw128(r, (ck & 3) * 2), w[0], w[1], w[2], w[3]);
          st_shared_v4(at + sw128(r, (ck & 3) * 2 + 1), w[4], w[5], w[6], w[7]);
        }
      }
      fence_async_smem();
      tc_fence_before();
      if (!__syncthreads_and(ok)) {
        ok = false;
        ++i;
        break;
      }
      if (one) {
        for (int d = 0; d < p.DB; ++d)
          tma_store_4d(&mdq, s_p + d * (kRows * 128), d * 64, (t_first + i) * kRows, h, b);
        bulk_commit();
      }
    }
    if (warp == 0 && ok && !p.early && i + 1 < steps) ok = start_scores(i + 1);
    if (kWalkQ) {
      lse = lse_next;
      if (MODE == kKeys) delta = delta_next;
    }
  }
  ok = __syncthreads_and(ok);

  if (ok) {
    __syncwarp();
    tc_fence_after();
    if (MODE != kQueries) {
      // dK and dV: a lane is a key.
      const int keys = min(p.KT, p.a.Nk - kt_fix * p.KT);
      const bool in = !MASK || (r < p.KT && bias[0][r] != -INFINITY);
      const float fv = 1.f / 1024.f, fk = p.a.scale * exp2f((float)-exp_now);
      const long long off =
          (((long long)b * p.a.Nk + kt_fix * p.KT + r) * p.a.H + h) * (long long)p.a.D;
      const long long plane = (long long)p.a.B * p.a.Nk * p.a.H * p.a.D;
      for (int w = 0; w < 2; ++w) {
        const float f = w ? fk : fv;
        for (int u = half; u < p.DP / 16; u += 2) {
          uint32_t o[16];
          __syncwarp();
          tmem_ld16_issue(lanes + (w ? p.c_dk : p.c_dv) + 16u * u, o);
          tmem_wait_ld();
          float d[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) d[e] = in ? __uint_as_float(o[e]) * f : 0.f;
          if (r < keys) {
            if (p.splits > 1) {
              float* to = (w ? p.part_dk : p.part_dv) + split * plane + off + 16 * u;
#pragma unroll
              for (int e = 0; e < 16; e += 4)
                if (16 * u + e < p.a.D)
                  *reinterpret_cast<float4*>(to + e) = make_float4(d[e], d[e + 1], d[e + 2], d[e + 3]);
            } else {
              T* to = static_cast<T*>(w ? p.a.dk : p.a.dv) + off + 16 * u;
#pragma unroll
              for (int e = 0; e < 16; e += 8)
                if (16 * u + e < p.a.D)
                  *reinterpret_cast<uint4*>(to + e) =
                      make_uint4(pack2<T>(d[e], d[e + 1]), pack2<T>(d[e + 2], d[e + 3]),
                                 pack2<T>(d[e + 4], d[e + 5]), pack2<T>(d[e + 6], d[e + 7]));
            }
          }
        }
      }
    } else {
      const int row = t_first * kRows + r;
      const float f = p.a.scale * exp2f((float)-exp_now);
      T* to = static_cast<T*>(p.a.dq) +
              (((long long)b * p.a.Nq + row) * p.a.H + h) * (long long)p.a.D;
      for (int u = half; u < p.DP / 16; u += 2) {
        uint32_t o[16];
        __syncwarp();
        tmem_ld16_issue(lanes + p.c_dq + 16u * u, o);
        tmem_wait_ld();
        float d[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) d[e] = keep ? __uint_as_float(o[e]) * f : 0.f;
        if (row < p.a.Nq) {
#pragma unroll
          for (int e = 0; e < 16; e += 8)
            if (16 * u + e < p.a.D)
              *reinterpret_cast<uint4*>(to + 16 * u + e) =
                  make_uint4(pack2<T>(d[e], d[e + 1]), pack2<T>(d[e + 2], d[e + 3]),
                             pack2<T>(d[e + 4], d[e + 5]), pack2<T>(d[e + 6], d[e + 7]));
        }
      }
    }
  } else if (one) {
    // Let the copies and products that were started end before their memory goes.
    mbar_wait_drain(bf, 0);
    for (int u = 0; u < p.stages && loaded - 1 - u >= 0; ++u)
      mbar_wait_drain(bx + 8u * ((loaded - 1 - u) % p.stages), ((loaded - 1 - u) / p.stages) & 1);
    const uint64_t since = globaltimer();
    while (globaltimer() - since < kDrainLimitNs) {
    }
  }
  if (one) bulk_wait_all();
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512)
                 : "memory");
  }
}

// delta = dO . O, with what the rounding of O left off: O's own rounding would enter every
// dS of its row (BF16, 333 keys: dQ and dK 1.1 times further off).
// `lpr` lanes (a power of two) share a row.
template <typename T>
__global__ void __launch_bounds__(128) row_delta(const __grid_constant__ Args a, float* delta,
                                                 int lpr) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31, sub = lane & (lpr - 1);
  const long long row = ((long long)blockIdx.x * 4 + (threadIdx.x >> 5)) * (32 / lpr) + lane / lpr;
  const bool in = row < (long long)a.B * a.H * a.Nq && sub * 8 < a.D;
  float t = 0.f;
  if (in) {
    const int n = row % a.Nq, h = row / a.Nq % a.H;
    const long long b = row / a.Nq / a.H, off = ((b * a.Nq + n) * a.H + h) * a.D + sub * 8;
    const Pack<T, 8> x = load_pack<T, 8>(static_cast<const T*>(a.out) + off),
                     z = load_pack<T, 8>(static_cast<const T*>(a.low) + off),
                     y = load_pack<T, 8>(static_cast<const T*>(a.dout) + b * a.dos.b + n * a.dos.n +
                                         h * a.dos.h + sub * 8);
#pragma unroll
    for (int e = 0; e < 8; ++e) t = fmaf(to_f32(x.e[e]) + to_f32(z.e[e]), to_f32(y.e[e]), t);
  }
  for (int s = lpr / 2; s > 0; s >>= 1) t += __shfl_xor_sync(~0u, t, s);
  if (in && sub == 0) delta[row] = t;
}

// dK and dV from the query splits' parts, in order.
template <typename T>
__global__ void __launch_bounds__(256) join_parts(const float* __restrict__ dk,
                                                  const float* __restrict__ dv, T* to_k, T* to_v,
                                                  long long n, int splits) {
  pdl_trigger();
  pdl_wait();
  const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  const float* from = blockIdx.y ? dv : dk;
  float4 t = *reinterpret_cast<const float4*>(from + i);
  for (int s = 1; s < splits; ++s) {
    const float4 u = *reinterpret_cast<const float4*>(from + s * n + i);
    t.x += u.x, t.y += u.y, t.z += u.z, t.w += u.w;
  }
  *reinterpret_cast<uint2*>((blockIdx.y ? to_v : to_k) + i) =
      make_uint2(pack2<T>(t.x, t.y), pack2<T>(t.z, t.w));
}

int up(int v, int to) { return (v + to - 1) / to * to; }
size_t align256(size_t n) { return (n + 255) & ~size_t(255); }

constexpr size_t kSmemMax = 224 * 1024;  // beside the static part

size_t smem_of(const BwdParams& p, int mode, int stages) {
  const size_t fix = mode == kQueries ? p.q_bytes : p.k_bytes;
  const size_t walk = mode == kQueries ? p.k_bytes : p.q_bytes;
  return 2 * fix + 2 * stages * walk + (mode == kQueries ? 1 : 2) * 2ull * kRows * 128 + 1024;
}

// Keys of a tile.  Three-block heads: 80 leave shared memory room for P and dS.
int most_keys(int D) { return D > 128 ? 80 : 128; }

void plan(BwdParams* p, int sms) {
  const Args& a = p->a;
  p->DB = (a.D + 63) / 64;
  p->DP = up(a.D, 16);
  const int most = most_keys(a.D);
  p->nkt = (a.Nk + most - 1) / most;
  p->KT = up((a.Nk + p->nkt - 1) / p->nkt, 16);
  p->nkt = (a.Nk + p->KT - 1) / p->KT;
  p->qtiles = (a.Nq + kRows - 1) / kRows;
  p->q_bytes = (uint32_t)p->DB * kRows * 128;
  p->k_bytes = (uint32_t)p->DB * p->KT * 128;
  // Query splits: the number of tiles that the busiest SM works through, and about
  // two tiles' time for every block's start and end.
  const long long units = (long long)a.B * a.H * p->nkt;
  long long best = -1;
  for (int chunk = p->qtiles; chunk >= 1; chunk = chunk > 1 ? (chunk + 1) / 2 : 0) {
    const int splits = (p->qtiles + chunk - 1) / chunk;
    const int even = (p->qtiles + splits - 1) / splits;
    const long long cost = (units * splits + sms - 1) / sms * (even + 2);
    if (best < 0 || cost < best) {
      best = cost;
      p->chunk = even;
      p->splits = (p->qtiles + even - 1) / even;
    }
  }
}

// Tensor memory and stages of one mode.
size_t arrange(BwdParams* p, int mode) {
  const uint32_t two = 2u * p->KT, dp = (uint32_t)p->DP;
  p->stages = smem_of(*p, mode, 2) <= kSmemMax ? 2 : 1;
  if (mode == kBoth) {
    const bool room = two + 3 * dp <= 512;
    const uint32_t at = room ? two : (two > dp ? two : dp);
    p->c_dv = at, p->c_dk = at + dp, p->c_dq = room ? at + 2 * dp : 0;
    p->early = room && p->stages == 2;
  } else {
    p->c_dv = two, p->c_dk = two + dp, p->c_dq = two;
    p->early = p->stages == 2;
  }
  return smem_of(*p, mode, p->stages);
}

template <typename T, bool MASK, int MODE>
cudaError_t run_mode(BwdParams p, const CUtensorMap* m, cudaStream_t s) {
  static std::atomic<unsigned long long> allowed{0};
  const size_t smem = arrange(&p, MODE);
  cudaError_t e = allow_smem(backward_tc<T, MASK, MODE>, &allowed, kSmemMax);
  if (e != cudaSuccess) return e;
  const long long heads = (long long)p.a.B * p.a.H;
  const long long grid = MODE == kQueries ? heads * p.qtiles : heads * p.nkt * p.splits;
  return launch_pdl(kPdlInput, backward_tc<T, MASK, MODE>, dim3((unsigned)grid), dim3(kThreads),
                    smem, s, m[0], m[1], m[2], m[3], m[4], p);
}

template <typename T, bool MASK>
cudaError_t run(BwdParams p, const CUtensorMap* m, float* delta, cudaStream_t s) {
  cudaError_t e;
  if (p.nkt == 1) {
    e = run_mode<T, MASK, kBoth>(p, m, s);
  } else {
    const long long rows = (long long)p.a.B * p.a.H * p.a.Nq;
    const int lpr = p.a.D <= 64 ? 8 : p.a.D <= 128 ? 16 : 32, per = 4 * (32 / lpr);
    e = launch_pdl(kPdlInput, row_delta<T>, dim3((unsigned)((rows + per - 1) / per)), dim3(128), 0, s,
                   p.a, delta, lpr);
    p.a.delta = delta;
    if (e == cudaSuccess) e = run_mode<T, MASK, kKeys>(p, m, s);
    if (e == cudaSuccess) e = run_mode<T, MASK, kQueries>(p, m, s);
  }
  if (e == cudaSuccess && p.splits > 1) {
    const long long n = (long long)p.a.B * p.a.Nk * p.a.H * p.a.D;
    e = launch_pdl(kPdlInput, join_parts<T>, dim3((unsigned)((n / 4 + 255) / 256), 2), dim3(256), 0,
                   s, (const float*)p.part_dk, (const float*)p.part_dv, static_cast<T*>(p.a.dk),
                   static_cast<T*>(p.a.dv), n, p.splits);
  }
  return e;
}

}  // namespace

long long backward_workspace_bytes(int B, int Nq, int Nk, int H, int D) {
  BwdParams p{};
  p.a.B = B, p.a.Nq = Nq, p.a.Nk = Nk, p.a.H = H, p.a.D = D;
  plan(&p, device_sms());
  const size_t n = (size_t)B * Nk * H * D * 4;
  size_t total = p.nkt > 1 ? align256((size_t)B * H * Nq * 4) : 0;
  if (p.splits > 1) total += 2 * align256(n * p.splits);
  return (long long)total;
}

bool backward_reads_output(int Nk, int D) { return Nk > most_keys(D); }

cudaError_t backward_status(int* status) {
  cudaError_t e = cudaMemcpyFromSymbol(status, g_status, sizeof(int));
  const int zero = 0;
  return e == cudaSuccess ? cudaMemcpyToSymbol(g_status, &zero, sizeof(int)) : e;
}

cudaError_t launch_backward(const Args& a, bool bf16, void* ws, cudaStream_t s, const char** why) {
  BwdParams p{};
  p.a = a;
  plan(&p, device_sms());
  unsigned char* at = static_cast<unsigned char*>(ws);
  float* delta = nullptr;
  if (p.nkt > 1) {
    delta = reinterpret_cast<float*>(at);
    at += align256((size_t)a.B * a.H * a.Nq * 4);
  }
  if (p.splits > 1) {
    p.part_dk = reinterpret_cast<float*>(at);
    p.part_dv = reinterpret_cast<float*>(at + align256((size_t)a.B * a.Nk * a.H * a.D * 4 * p.splits));
  }
  CUtensorMap m[5];
  Pick out;
  const Strides dense{(long long)a.Nq * a.H * a.D, (long long)a.H * a.D, a.D};
  if (!encode_tile4(&m[0], &p.qp, a.q, a.qs, a.B, a.Nq, a.H, a.D, kRows, bf16) ||
      !encode_tile4(&m[1], &p.kp, a.k, a.ks, a.B, a.Nk, a.H, a.D, p.KT, bf16) ||
      !encode_tile4(&m[2], &p.vp, a.v, a.vs, a.B, a.Nk, a.H, a.D, p.KT, bf16) ||
      !encode_tile4(&m[3], &p.gp, a.dout, a.dos, a.B, a.Nq, a.H, a.D, kRows, bf16) ||
      !encode_tile4(&m[4], &out, a.dq, dense, a.B, a.Nq, a.H, a.D, kRows, bf16)) {
    *why = "tensor map encode failed";
    return cudaErrorInvalidValue;
  }
  const bool mask = a.mask_kind != kMaskNone;
  if (bf16)
    return mask ? run<__nv_bfloat16, true>(p, m, delta, s)
                : run<__nv_bfloat16, false>(p, m, delta, s);
  return mask ? run<__half, true>(p, m, delta, s) : run<__half, false>(p, m, delta, s);
}

}  // namespace xattn
}  // namespace nova
