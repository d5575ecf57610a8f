// Cross-attention forward on the tensor cores.
//
// A block takes 128 queries of one head at a time.  One warp starts the copies (TMA)
// and the products (tcgen05); four do the softmax, one query (one tensor-memory lane)
// a thread.  They wait for one another at mbarriers only.
//
//   S = Q K^T      both operands as TMA lands them (rows of 64 elements, swizzled)
//   P = 2^(c S + bias - m)   read from and written back to tensor memory, in place
//                            (the product is rounded before m is taken off, so that a
//                            row's largest probability is 2^0 and a single key's is one)
//   O += P V       P from tensor memory; V as it lies, its head index contiguous
//
// The keys come in `nkt` tiles of `KT` (a multiple of 16, at most 128).  With one
// tile (77 text tokens) the blocks share all heads' query tiles evenly, in a row; K and
// V stay in shared memory while the head does, the next queries land as soon as S has
// been formed, and the next S is formed while finished rows leave.  With more, K and V
// run through two stages and O keeps its place, its scale renewed only when a row's
// maximum has risen by more than 2^kLazy.  Too few queries for the SMs against many
// keys: the keys are split over blocks, which leave partial rows in the workspace for a
// second kernel to join.
//
// What bounds it.  8 x 4096 queries x 10 heads x 64, 77 keys, FP16: 25.7 us, 85 MB at
// 3.3 TB/s (51 % of the measured copy bandwidth).  A tile takes 5,900 cycles from its
// scores to its rows, three blocks on an SM: scores 1,000, maximum 850, exponentials
// 1,800, product 1,000, rows 900.  Steps that were kept: the warp of its own (28.8 to 26
// us), waits that read the timer late and descriptors in uniform registers (products
// 800 to 450 cycles to start), a row's scores held in registers (26 to 24.5 us at 2.7
// blocks).  Four blocks with 96 registers spilled (33 us).
#include <cuda_runtime.h>

#include <algorithm>

#include "nova_attention.cuh"

namespace nova {
namespace xattn {

using namespace tc;

namespace {

constexpr int kRows = 128;
constexpr int kThreads = kRows + 32;  // a thread for a row, and a warp that starts the work
constexpr int kBlocks = 3;       // on an SM, by their registers
constexpr int kMostSplits = 64;  // of the keys: two for every lane of the joining warp
constexpr float kLazy = 4.f;
constexpr int kHeld = 80;  // scores that a thread can hold with three blocks on an SM

struct FwdParams {
  Args a;
  Pick qp, kp, vp, op;
  int KT, nkt;       // keys per tile, tiles
  int DB, DP;        // 64-element blocks and padded width of a head
  int qtiles;        // query tiles of a head
  long long total;   // query tiles of all heads, which the blocks share evenly
  int blocks;        // for each key split
  bool walks;        // a block may have more than one
  int splits, per;   // key splits, tiles per split
  int kstages;           // of K and V
  uint32_t tmem_cols, o_col;
  uint32_t q_bytes, k_bytes;  // one stage of Q, of K (= of V)
  float* part_o;    // [splits][B][Nq][H][D]
  float* part_lse;  // [splits][B][H][Nq]
};

__device__ int g_status;

template <typename T, bool MASK, bool ONE>
__global__ void __launch_bounds__(kThreads, kBlocks) forward_tc(const __grid_constant__ CUtensorMap mq,
                                                       const __grid_constant__ CUtensorMap mk,
                                                       const __grid_constant__ CUtensorMap mv,
                                                       const __grid_constant__ CUtensorMap mo,
                                                       const __grid_constant__ FwdParams p) {
  constexpr bool kBf16 = !std::is_same<T, __half>::value;
  extern __shared__ unsigned char raw[];
  // Landed: Q, K and V [2].  Formed: S, O.  Left by the rows' warps: the mask, P, rows.
  __shared__ uint64_t bars[8];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  __shared__ alignas(8) float bias[kRows];
  __shared__ float refs[4];  // largest bias of the sample, a copy for each warp
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(~0u, tid >> 5, 0);  // the same for the warp, and known to be
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
  // Q, the finished rows (over Q where a block has one query tile), K, V.
  const uint32_t sq = base, so = p.walks ? sq + p.q_bytes : sq;
  const uint32_t sk = so + p.q_bytes, sv = sk + p.kstages * p.k_bytes;
  const uint32_t bq = smem_u32(&bars[0]), bkv = bq + 8, bs = bq + 24, bo = bq + 32, bm = bq + 40,
                 bp = bq + 48, br = bq + 56;
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&tmem_slot)),
                 "r"(p.tmem_cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (tid == 32) {
    for (int i = 0; i < 8; ++i) mbar_init(bq + 8u * i, i < 5 ? 1 : kRows / 32);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    abort_flag = 0;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(~0u, tmem_slot, 0);
  pdl_trigger();
  pdl_wait();

  unsigned id = blockIdx.x;
  const int split = id % p.splits;
  id /= p.splits;
  // Query tiles first, first + 1, ... of all heads in a row, and this split's key tiles.
  const int first = (int)((long long)id * p.total / p.blocks);
  const int tiles = (int)((id + 1ll) * p.total / p.blocks) - first;
  const int k0 = split * p.per, nk = min(p.nkt, k0 + p.per) - k0;
  const bool resident = nk == 1;  // K and V stay while the head does
  const int head0 = first / p.qtiles;
  struct Spot {
    int b, h, n;  // sample, head, first query
    int turn;     // heads before this one in the block's walk
  };
  const auto spot = [&](int t) {
    const int g = first + t, head = g / p.qtiles, b = head / p.a.H;
    return Spot{b, head - b * p.a.H, (g - head * p.qtiles) * kRows, head - head0};
  };
  const auto wait = [&](uint32_t bar, uint32_t parity, int code) {
    return wait_phase(bar, parity & 1, &abort_flag, &g_status, code);
  };

  if (warp == kRows / 32) {
    // ---- The warp that starts copies and products ----
    const bool one = elect_one();
    const auto load_q = [&](int t) {
      if (!one) return;
      const Spot at = spot(t);
      mbar_expect_tx(bq, p.q_bytes);
      for (int d = 0; d < p.DB; ++d)
        tma_load_4d(sq + d * (kRows * 128), &mq, d * 64, at.n, at.h * p.qp.h, at.b * p.qp.b, bq);
    };
    // The i-th pair of K and V tiles that the block goes through: its head's key tiles,
    // or one for each head.
    const auto load_kv = [&](int i) {
      if (!one) return;
      const int head = head0 + (resident ? i : 0), h = head % p.a.H, b = head / p.a.H;
      const int j = resident ? 0 : i, stage = i % p.kstages;
      const uint32_t bar = bkv + 8u * stage, at = stage * p.k_bytes;
      mbar_expect_tx(bar, 2 * p.k_bytes);
      for (int d = 0; d < p.DB; ++d)
        tma_load_4d(sk + at + d * (p.KT * 128), &mk, d * 64, (k0 + j) * p.KT, h * p.kp.h,
                    b * p.kp.b, bar);
      for (int d = 0; d < p.DB; ++d)
        tma_load_4d(sv + at + d * (p.KT * 128), &mv, d * 64, (k0 + j) * p.KT, h * p.vp.h,
                    b * p.vp.b, bar);
    };
    const uint32_t idesc_s = instr_desc(kBf16, kRows, p.KT, false, false);
    const uint32_t idesc_o = instr_desc(kBf16, kRows, p.DP, false, true);
    const int nd = p.DP / 16, nc = p.KT / 16;
    const uint64_t qd = smem_desc_sw128(sq);
    // S of the tile in Q and the i-th K.
    const auto scores = [&](int i) {
      const uint64_t kd = smem_desc_sw128(sk + (i % p.kstages) * p.k_bytes);
      tc_fence_after();
      if (one) {
#pragma unroll
        for (int s = 0; s < kMaxD / 16; ++s)
          if (s < nd) umma_f16(tmem, qd + (uint32_t)((s >> 2) * (kRows * 8) + (s & 3) * 2),
                   kd + (uint32_t)((s >> 2) * (p.KT * 8) + (s & 3) * 2), idesc_s, s != 0);
        umma_commit(bs);
      }
    };
    const auto products = [&](int i, int j) {
      const uint64_t vd = smem_desc_mn(sv + (i % p.kstages) * p.k_bytes, p.KT * 128);
      tc_fence_after();
      if (one) {
#pragma unroll
        for (int s = 0; s < 8; ++s)
          if (s < nc)
            umma_f16_ta(tmem + p.o_col, tmem + 8u * s, vd + 128ull * s, idesc_o, s != 0 || j != 0);
        umma_commit(bo);
      }
    };
    const int pairs = resident ? spot(tiles - 1).turn + 1 : nk;
    int qn = 1, kn = min(pairs, p.kstages);  // copies started
    load_q(0);
    for (int j = 0; j < kn; ++j) load_kv(j);
    bool ok = wait(bq, 0, kDevTimeoutProducer) && wait(bkv, 0, kDevTimeoutProducer);
    ok = __all_sync(~0u, ok);
    if (ok) scores(0);
    int step = 0;
    for (int t = 0; t < tiles && ok; ++t) {
      for (int j = 0; j < nk && ok; ++j, ++step) {
        if (j == nk - 1 && t + 1 < tiles) {
          // Nothing reads Q any more once the last scores are there.
          ok = wait(bs, step, kDevTimeoutMma);
          if (ok) load_q(t + 1);
          ++qn;
        }
        ok = ok && wait(bp, step, kDevTimeoutMma);
        // The rows of the last tile have left their place before new ones are written
        // there, which happens behind this product.
        if (one) bulk_wait_read_all();
        if (!(ok = __all_sync(~0u, ok))) break;
        products(resident ? spot(t).turn : j, j);
        if (j + 1 < nk) {
          // Behind the product that reads P, in the same order.
          ok = __all_sync(~0u, wait(bkv + 8u * ((j + 1) % p.kstages), (j + 1) / p.kstages,
                                    kDevTimeoutProducer));
          if (!ok) break;
          scores(j + 1);
          if (kn < nk) {
            ok = __all_sync(~0u, wait(bo, step, kDevTimeoutMma));
            if (!ok) break;
            load_kv(kn++);
          }
        }
      }
      ok = ok && wait(br, t, kDevTimeoutEpilogue);
      if (!(ok = __all_sync(~0u, ok))) break;
      const Spot at = spot(t);
      if (t + 1 < tiles) {
        const int turn = spot(t + 1).turn;
        ok = wait(bq, t + 1, kDevTimeoutProducer);
        if (turn != at.turn) {
          // The next head: the products with the last one's K and V are there.
          if (kn < pairs && ok) load_kv(kn++);
          ok = ok && wait(bkv + 8u * (turn % p.kstages), turn / p.kstages, kDevTimeoutProducer);
        }
        if (!(ok = __all_sync(~0u, ok))) break;
        scores(turn);
      }
      if (one && p.splits == 1) {
        for (int d = 0; d < p.DB; ++d)
          tma_store_4d(&mo, so + d * (kRows * 128), d * 64, at.n, at.h, at.b);
        bulk_commit();
      }
    }
    if (one) {
      if (!ok) {
        // Let the copies and products that were started end before their memory goes.
        mbar_wait_drain(bq, (qn - 1) & 1);
        for (int i = 0; i < p.kstages && kn - 1 - i >= 0; ++i)
          mbar_wait_drain(bkv + 8u * ((kn - 1 - i) % p.kstages), ((kn - 1 - i) / p.kstages) & 1);
        const uint64_t since = globaltimer();
        while (globaltimer() - since < kDrainLimitNs) {
        }
      }
      bulk_wait_all();
    }
  } else {
    // ---- The rows' warps: one query a thread ----
    const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
    const float c = p.a.scale * kLog2e;
    const int chunks = p.KT / 16;
    int step = 0, turn_seen = -1;
    bool ok = true;
    // Who reads lse wants the largest bias: the four warps look for the first sample's
    // together (none of them can have given up yet), for a later one's each by itself.
    const bool wants_ref = MASK && is_additive(p.a) && (p.a.lse || p.splits > 1);
    int b_seen = -1;
    for (int t = 0; t < tiles && ok; ++t) {
      const Spot at = spot(t);
      const int b = at.b, h = at.h;
      if (wants_ref && b != b_seen) {
        float top = warp_most(largest_bias(p.a, b, t ? lane : tid, t ? 32 : kRows));
        if (t == 0) {
          if (lane == 0) refs[warp] = top;
          asm volatile("bar.sync 1, %0;" ::"n"(kRows) : "memory");
          top = fmaxf(fmaxf(refs[0], refs[1]), fmaxf(refs[2], refs[3]));
          asm volatile("bar.sync 1, %0;" ::"n"(kRows) : "memory");
        }
        if (lane == 0) refs[warp] = top;
        b_seen = b;
      }
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < nk; ++j, ++step) {
        const int key0 = (k0 + j) * p.KT, keys = min(p.KT, p.a.Nk - key0);
        if (MASK && (at.turn != turn_seen || !resident)) {
          // The bias of this tile's keys; the rows of V behind a masked key are cleared:
          // P is zero there, and zero times infinity is not.
          float x = -INFINITY;
          const bool in = tid < keys && key_bias(p.a, b, key0 + tid, &x);
          // The scores before have been read by everyone who reads the old bias.
          if (j > 0) ok = wait(bo, step - 1, kDevTimeoutMma);
          bias[tid] = in ? x : -INFINITY;
          const int pair = resident ? at.turn : j, stage = pair % p.kstages;
          turn_seen = at.turn;
          ok = ok && wait(bkv + 8u * stage, pair / p.kstages, kDevTimeoutProducer);
          if (ok && !in && tid < keys) {
            for (int d = 0; d < p.DB; ++d)
              for (int i = 0; i < 8; ++i)
                st_shared_v4(sv + stage * p.k_bytes + d * (p.KT * 128) + sw128(tid, i), 0, 0, 0, 0);
            fence_async_smem();
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(bm);
          ok = ok && wait(bm, pair, kDevTimeoutEpilogue);
        }
        ok = ok && wait(bs, step, kDevTimeoutMma);
        __syncwarp();
        if (!__all_sync(~0u, ok)) {
          ok = false;
          break;
        }
        tc_fence_after();

        // The row's scores twice: the maximum, then P.
        // Tiles of up to kHeld keys stay in registers from one to the other.
        uint32_t r[ONE ? kHeld / 16 : 4][16];
        float top = -INFINITY;
        // Scores e and e + 1 of a piece, in base 2; minus infinity where the key is out.
        const auto score2 = [&](const uint32_t(&x)[16], int col, int e) {
          float2 v = make_float2(__uint_as_float(x[e]), __uint_as_float(x[e + 1]));
          if (MASK) {
            const float2 add = *reinterpret_cast<const float2*>(&bias[col + e]);
            v = __ffma2_rn(v, make_float2(c, c), add);
            if (add.x == -INFINITY) v.x = -INFINITY;
            if (add.y == -INFINITY) v.y = -INFINITY;
          } else {
            v = __fmul2_rn(v, make_float2(c, c));
          }
          return v;
        };
        // A chunk's largest score; the chunk is left as scores in base 2.
        const auto take_top = [&](uint32_t(&x)[16], int col) {
          const bool whole = MASK || col + 16 <= keys;
#pragma unroll
          for (int e = 0; e < 16; e += 2) {
            float2 v = score2(x, col, e);
            if (!whole) {
              if (col + e >= keys) v.x = -INFINITY;
              if (col + e + 1 >= keys) v.y = -INFINITY;
            }
            top = fmaxf(top, fmaxf(v.x, v.y));
            x[e] = __float_as_uint(v.x);
            x[e + 1] = __float_as_uint(v.y);
          }
        };
        // Chunks of 16 two by two, the next two on their way; `use` once for each.
        const auto each_chunk = [&](auto&& use) {
          tmem_ld16_issue(lanes, r[0]);
          if (1 < chunks) tmem_ld16_issue(lanes + 16u, r[1]);
#pragma unroll 1
          for (int i = 0; i < chunks; i += 4) {
            tmem_wait_ld();
            if (i + 2 < chunks) tmem_ld16_issue(lanes + 16u * (i + 2), r[2]);
            if (i + 3 < chunks) tmem_ld16_issue(lanes + 16u * (i + 3), r[3]);
            use(r[0], 16 * i);
            if (i + 1 < chunks) use(r[1], 16 * (i + 1));
            if (i + 2 < chunks) {
              tmem_wait_ld();
              if (i + 4 < chunks) tmem_ld16_issue(lanes + 16u * (i + 4), r[0]);
              if (i + 5 < chunks) tmem_ld16_issue(lanes + 16u * (i + 5), r[1]);
              use(r[2], 16 * (i + 2));
              if (i + 3 < chunks) use(r[3], 16 * (i + 3));
            }
          }
        };
        if constexpr (ONE) {
#pragma unroll
          for (int i = 0; i < kHeld / 16; ++i)
            if (i < chunks) tmem_ld16_issue(lanes + 16u * i, r[i]);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < kHeld / 16; ++i)
            if (i < chunks) take_top(r[i], 16 * i);
        } else {
          each_chunk(take_top);
        }
        // The scale that the row's sums are kept at.
        float factor = 1.f;
        if (j == 0) {
          m = top;
        } else if (top > m + kLazy || m == -INFINITY) {
          const float to = fmaxf(top, m);
          factor = m == -INFINITY ? 1.f : ex2(m - to);  // nothing yet: zeros stay zeros
          m = to;
        }
        if (j > 0) {
          ok = wait(bo, step - 1, kDevTimeoutMma);
          __syncwarp();
          tc_fence_after();
          if (__any_sync(~0u, factor != 1.f)) {
            l *= factor;
#pragma unroll 1
            for (int i = 0; i < p.DP / 16; ++i) {
              uint32_t o[16];
              tmem_ld16_issue(lanes + p.o_col + 16u * i, o);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * factor);
              tmem_st16(lanes + p.o_col + 16u * i, o);
            }
          }
        }
        const float sub = m == -INFINITY ? 0.f : m;

        // P, packed over the scores that have been read.
        const auto put_p = [&](const uint32_t(&x)[16], int col) {
          const bool whole = ONE || MASK || col + 16 <= keys;
          uint32_t o[8];
          float2 sum = make_float2(0.f, 0.f);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float2 v = ONE ? make_float2(__uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1]))
                           : score2(x, col, 2 * e);
            v = __fadd2_rn(v, make_float2(-sub, -sub));
            v = make_float2(ex2(v.x), ex2(v.y));
            if (!whole) {
              if (col + 2 * e >= keys) v.x = 0.f;
              if (col + 2 * e + 1 >= keys) v.y = 0.f;
            }
            sum = __fadd2_rn(sum, v);
            o[e] = pack2<T>(v.x, v.y);
          }
          l += sum.x + sum.y;
          tmem_st8(lanes + (uint32_t)(col / 2), o);
        };
        if constexpr (ONE) {
#pragma unroll
          for (int i = 0; i < kHeld / 16; ++i)
            if (i < chunks) put_p(r[i], 16 * i);
        } else {
          each_chunk(put_p);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bp);
      }
      ok = ok && wait(bo, step - 1, kDevTimeoutEpilogue);
      __syncwarp();
      if (!(ok = __all_sync(~0u, ok))) break;
      tc_fence_after();

      // O / sum.
      const int row = at.n + tid;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const float ref = wants_ref ? refs[warp] : 0.f;
      const float lse = l == 0.f ? -INFINITY : m - ref + log2f(l);
      const long long lrow = ((long long)b * p.a.H + h) * p.a.Nq + row;
      if (p.splits > 1) {
        float* po = p.part_o + ((((long long)split * p.a.B + b) * p.a.Nq + row) * p.a.H + h) * p.a.D;
#pragma unroll 1
        for (int i = 0; i < p.DP / 16; ++i) {
          uint32_t o[16];
          __syncwarp();
          tmem_ld16_issue(lanes + p.o_col + 16u * i, o);
          tmem_wait_ld();
          if (row < p.a.Nq) {
#pragma unroll
            for (int e = 0; e < 16; e += 4)
              if (16 * i + e < p.a.D)
                *reinterpret_cast<float4*>(po + 16 * i + e) =
                    make_float4(__uint_as_float(o[e]) * inv, __uint_as_float(o[e + 1]) * inv,
                                __uint_as_float(o[e + 2]) * inv, __uint_as_float(o[e + 3]) * inv);
          }
        }
        if (row < p.a.Nq) p.part_lse[(long long)split * p.a.B * p.a.H * p.a.Nq + lrow] = lse;
      } else {
        const auto put_rows = [&](const uint32_t(&o)[16], int i) {
          uint32_t w[8];
#pragma unroll
          for (int e = 0; e < 8; ++e)
            w[e] = pack2<T>(__uint_as_float(o[2 * e]) * inv, __uint_as_float(o[2 * e + 1]) * inv);
          const uint32_t at = so + (uint32_t)(i >> 2) * (kRows * 128);
          st_shared_v4(at + sw128(tid, (i & 3) * 2), w[0], w[1], w[2], w[3]);
          st_shared_v4(at + sw128(tid, (i & 3) * 2 + 1), w[4], w[5], w[6], w[7]);
        };
#pragma unroll 1
        for (int i = 0; i < p.DP / 16; i += 2) {
          uint32_t o[2][16];
          __syncwarp();
          tmem_ld16_issue(lanes + p.o_col + 16u * i, o[0]);
          if (i + 1 < p.DP / 16) tmem_ld16_issue(lanes + p.o_col + 16u * (i + 1), o[1]);
          tmem_wait_ld();
          put_rows(o[0], i);
          if (i + 1 < p.DP / 16) put_rows(o[1], i + 1);
        }
        if (p.a.lse && row < p.a.Nq) p.a.lse[lrow] = lse;
        if (p.a.low) {
          T* low = static_cast<T*>(p.a.low) +
                   (((long long)b * p.a.Nq + row) * p.a.H + h) * (long long)p.a.D;
#pragma unroll 1
          for (int i = 0; i < p.DP / 16; ++i) {
            uint32_t o[16];
            __syncwarp();
            tmem_ld16_issue(lanes + p.o_col + 16u * i, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; e += 8)
              if (row < p.a.Nq && 16 * i + e < p.a.D) {
                uint32_t w[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                  const float x = __uint_as_float(o[e + 2 * u]) * inv,
                              y = __uint_as_float(o[e + 2 * u + 1]) * inv;
                  const float2 r = unpack2<T>(pack2<T>(x, y));
                  w[u] = pack2<T>(x - r.x, y - r.y);
                }
                *reinterpret_cast<uint4*>(low + 16 * i + e) = make_uint4(w[0], w[1], w[2], w[3]);
              }
          }
          __syncwarp();
        }
        fence_async_smem();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(br);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(p.tmem_cols)
                 : "memory");
  }
}

// Up to eight queries against many keys: K and V are read once, straight into the
// fragments of mma.m16n8k16, without shared memory; a tile of tcgen05 would be a
// sixteenth full and its steps would follow one another.  A warp takes 16 keys at a
// time.  With g = lane / 4 and t = lane % 4:
//
//   S: a lane's 16 bytes of K (key g of 8, elements 8 t .. 8 t + 7 of 32) are the B
//      fragments of two products.  Which elements of a row meet in which product does
//      not matter to their sum, so Q is taken in the same order.
//   P: the scores of 16 keys lie as the A fragment wants them.
//   O: a lane's 16 bytes of V (keys 2t, 2t+1, 2t+8, 2t+9; elements 8 g .. of 64) give
//      the B fragments of eight products, one for each element, by pairing halves of
//      two keys; the columns of product j are elements j, 8 + j, 16 + j, ...
//
// The loads of a step are on their way together.  Rows of keys that take no part are not
// read.  The keys are split over blocks (`per` keys each) and over a block's warps; the
// warps join in shared memory, up to eight blocks as one cluster through distributed
// shared memory, more through the workspace.
constexpr int kTokenBiases = 1024;  // keys whose biases are staged together
constexpr int kTokenWarps = 4, kTokenQueries = 8, kTokenCluster = 8;
// Steps of 16 keys on their way together, with five blocks' registers on an SM (three for
// wide heads): 4 x 2041 keys x 20 heads in 15.3 us, with a mask 16.6 (two steps: 19.4).
__host__ __device__ constexpr int token_steps(int DB, bool mask) { return DB == 1 && !mask ? 2 : 1; }

__device__ __forceinline__ float peer_float(const float* p, int rank) {
  uint32_t at;
  float v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}

// c += A B, rows 8 .. 15 of A zero.
template <typename T>
__device__ __forceinline__ void mma_rows8(float (&c)[2], uint32_t a0, uint32_t a2, uint32_t b0,
                                          uint32_t b1) {
  float x, y;  // rows 8 .. 15
  if constexpr (std::is_same<T, __half>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
        "{%0, %1, %2, %3}, {%4, %5, %6, %5}, {%7, %8}, {%0, %1, %9, %9};"
        : "+f"(c[0]), "+f"(c[1]), "=f"(x), "=f"(y)
        : "r"(a0), "r"(0), "r"(a2), "r"(b0), "r"(b1), "f"(0.f));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
        "{%0, %1, %2, %3}, {%4, %5, %6, %5}, {%7, %8}, {%0, %1, %9, %9};"
        : "+f"(c[0]), "+f"(c[1]), "=f"(x), "=f"(y)
        : "r"(a0), "r"(0), "r"(a2), "r"(b0), "r"(b1), "f"(0.f));
}

// DB: 64-element blocks of a head.
template <typename T, int DB, bool MASK>
__global__ void __launch_bounds__(kTokenWarps * 32, DB == 1 ? 5 : 3)
    forward_token(const __grid_constant__ FwdParams p) {
  constexpr int S = token_steps(DB, MASK), NQ = kTokenQueries, kKeys = 16 * S;
  __shared__ float po[kTokenWarps][NQ][DB * 64];
  __shared__ float pm[kTokenWarps][NQ], pl[kTokenWarps][NQ];
  __shared__ float biases[MASK ? kTokenBiases : 1];
  __shared__ float refs[kTokenWarps];  // largest biases of the sample, a part for each warp
  __shared__ float row[NQ][DB * 64], top_of[NQ], sum_of[NQ];  // of the block, not divided
  pdl_trigger();
  pdl_wait();
  const Args& a = p.a;
  unsigned id = blockIdx.x;
  const int split = id % p.splits;
  id /= p.splits;
  const int h = id % a.H, b = id / a.H;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int first = split * p.per, last = min(a.Nk, first + p.per);
  const T* kp = static_cast<const T*>(a.k) + b * a.ks.b + h * a.ks.h + t * 8;
  const T* vp = static_cast<const T*>(a.v) + b * a.vs.b + h * a.vs.h + g * 8;
  const float c = a.scale * kLog2e;
  const uint4 none = make_uint4(0, 0, 0, 0);
  const bool cluster = p.splits <= kTokenCluster;
  const bool wants_ref = MASK && is_additive(a) && (a.lse || !cluster);
  if (wants_ref) {
    const float part = warp_most(largest_bias(a, b, threadIdx.x, kTokenWarps * 32));
    if (lane == 0) refs[warp] = part;  // read behind the barriers below
  }

  // Q as K is read: row g, elements 8 t of every 32.
  uint4 q[2 * DB];
#pragma unroll
  for (int i = 0; i < 2 * DB; ++i) {
    q[i] = none;
    if (g < a.Nq && i * 32 + t * 8 < a.D)
      q[i] = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + b * a.qs.b + g * a.qs.n +
                                             h * a.qs.h + i * 32 + t * 8);
  }
  float o[DB * 8][2] = {};
  float m = -INFINITY, l = 0.f;  // of row g; l over this lane's keys
  const int piece = MASK ? kTokenBiases : last - first;
  for (int c0 = first; c0 < last; c0 += piece) {
    const int c1 = min(last, c0 + piece);
    if (MASK) {
      __syncthreads();
      for (int i = threadIdx.x; i < kTokenBiases; i += kTokenWarps * 32) {
        float w = 0.f;
        const bool in = c0 + i < c1 && key_bias(a, b, c0 + i, &w);
        biases[i] = in ? w : -INFINITY;
      }
      __syncthreads();
    }
    for (int k0 = c0 + warp * kKeys; k0 < c1; k0 += kTokenWarps * kKeys) {
      // The biases of this lane's keys 2t, 2t+1, 2t+8, 2t+9 of a step, as its scores are;
      // minus infinity for a key that is out.
      float add[S][4];
      uint4 kr[S][2][2 * DB], vr[S][4][DB];
  #pragma unroll
      for (int s = 0; s < S; ++s) {
  #pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int key = k0 + 16 * s + 8 * u + g;
          const bool in = MASK ? biases[key - c0] != -INFINITY : key < c1;
          const T* at = kp + (long long)key * a.ks.n;
  #pragma unroll
          for (int i = 0; i < 2 * DB; ++i) {
            kr[s][u][i] = none;
            if (in && i * 32 + t * 8 < a.D) kr[s][u][i] = *reinterpret_cast<const uint4*>(at + i * 32);
          }
        }
  #pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = k0 + 16 * s + 2 * t + (e & 1) + (e >> 1) * 8;
          add[s][e] = MASK ? biases[key - c0] : key < c1 ? 0.f : -INFINITY;
          const T* at = vp + (long long)key * a.vs.n;
  #pragma unroll
          for (int i = 0; i < DB; ++i) {
            vr[s][e][i] = none;
            if (add[s][e] != -INFINITY && i * 64 + g * 8 < a.D)
              vr[s][e][i] = *reinterpret_cast<const uint4*>(at + i * 64);
          }
        }
      }
      float x[S][2][2];
      float top = m;
  #pragma unroll
      for (int s = 0; s < S; ++s)
  #pragma unroll
        for (int u = 0; u < 2; ++u) {
          x[s][u][0] = x[s][u][1] = 0.f;
  #pragma unroll
          for (int i = 0; i < 2 * DB; ++i) {
            mma_rows8<T>(x[s][u], q[i].x, q[i].y, kr[s][u][i].x, kr[s][u][i].y);
            mma_rows8<T>(x[s][u], q[i].z, q[i].w, kr[s][u][i].z, kr[s][u][i].w);
          }
  #pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float w = add[s][2 * u + e];
            x[s][u][e] = w == -INFINITY ? -INFINITY : fmaf(x[s][u][e], c, w);
            top = fmaxf(top, x[s][u][e]);
          }
        }
      top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
      top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
      const float base = top == -INFINITY ? 0.f : top;
      const float f = ex2(m - base);
      m = top;
      l *= f;
      if (__any_sync(~0u, f != 1.f)) {
  #pragma unroll
        for (int i = 0; i < DB * 8; ++i) o[i][0] *= f, o[i][1] *= f;
      }
  #pragma unroll
      for (int s = 0; s < S; ++s) {
  #pragma unroll
        for (int u = 0; u < 2; ++u)
  #pragma unroll
          for (int e = 0; e < 2; ++e) {
            x[s][u][e] = add[s][2 * u + e] == -INFINITY ? 0.f : ex2(x[s][u][e] - base);
            l += x[s][u][e];
          }
        const uint32_t a0 = pack2<T>(x[s][0][0], x[s][0][1]), a2 = pack2<T>(x[s][1][0], x[s][1][1]);
  #pragma unroll
        for (int i = 0; i < DB; ++i) {
          const auto pair = [&](uint32_t v0, uint32_t v1, uint32_t v2, uint32_t v3, int e) {
            mma_rows8<T>(o[i * 8 + e], a0, a2, __byte_perm(v0, v1, 0x5410), __byte_perm(v2, v3, 0x5410));
            mma_rows8<T>(o[i * 8 + e + 1], a0, a2, __byte_perm(v0, v1, 0x7632),
                         __byte_perm(v2, v3, 0x7632));
          };
          pair(vr[s][0][i].x, vr[s][1][i].x, vr[s][2][i].x, vr[s][3][i].x, 0);
          pair(vr[s][0][i].y, vr[s][1][i].y, vr[s][2][i].y, vr[s][3][i].y, 2);
          pair(vr[s][0][i].z, vr[s][1][i].z, vr[s][2][i].z, vr[s][3][i].z, 4);
          pair(vr[s][0][i].w, vr[s][1][i].w, vr[s][2][i].w, vr[s][3][i].w, 6);
        }
      }
    }
  }
  l += __shfl_xor_sync(~0u, l, 1);
  l += __shfl_xor_sync(~0u, l, 2);
#pragma unroll
  for (int i = 0; i < DB; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      // Columns 2t and 2t+1 of product e: elements e of the 8-element pieces 2t, 2t+1.
      po[warp][g][i * 64 + 16 * t + e] = o[i * 8 + e][0];
      po[warp][g][i * 64 + 16 * t + 8 + e] = o[i * 8 + e][1];
    }
  if (t == 0) {
    pm[warp][g] = m;
    pl[warp][g] = l;
  }
  __syncthreads();
  // The block's rows: the same sums in the same order in every thread that forms one.
  for (int z = threadIdx.x; z < NQ * DB * 64; z += kTokenWarps * 32) {
    const int i = z / (DB * 64), d = z % (DB * 64);
    float top = -INFINITY, sum = 0.f, acc = 0.f;
#pragma unroll
    for (int w = 0; w < kTokenWarps; ++w) top = fmaxf(top, pm[w][i]);
    const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int w = 0; w < kTokenWarps; ++w) {
      const float f = ex2(pm[w][i] - base);
      sum = fmaf(f, pl[w][i], sum);
      acc = fmaf(f, po[w][i][d], acc);
    }
    row[i][d] = acc;
    if (d == 0) {
      top_of[i] = top;
      sum_of[i] = sum;
    }
  }
  if (cluster) {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  } else {
    __syncthreads();
  }
  // The cluster's rows, a share of them by every block; or this block's for the
  // joining kernel.
  const int ranks = cluster ? p.splits : 1, rank = cluster ? split : 0;
  float ref = wants_ref ? refs[0] : 0.f;
#pragma unroll
  for (int w = 1; w < kTokenWarps; ++w)
    if (wants_ref) ref = fmaxf(ref, refs[w]);
  for (int z = threadIdx.x * ranks + rank; z < a.Nq * DB * 64; z += kTokenWarps * 32 * ranks) {
    const int i = z / (DB * 64), d = z % (DB * 64);
    if (d >= a.D) continue;
    float top = top_of[i], sum = sum_of[i], acc = row[i][d];
    if (cluster) {
      // All peers' values are on their way before the first is used.
      float tops[kTokenCluster], sums[kTokenCluster], accs[kTokenCluster];
#pragma unroll
      for (int r = 0; r < kTokenCluster; ++r) {
        const int peer = min(r, ranks - 1);
        tops[r] = peer_float(&top_of[i], peer);
        sums[r] = peer_float(&sum_of[i], peer);
        accs[r] = peer_float(&row[i][d], peer);
      }
      top = -INFINITY;
#pragma unroll
      for (int r = 0; r < kTokenCluster; ++r) top = fmaxf(top, tops[r]);
      const float base = top == -INFINITY ? 0.f : top;
      sum = acc = 0.f;
#pragma unroll
      for (int r = 0; r < kTokenCluster; ++r) {
        const float f = r < ranks ? ex2(tops[r] - base) : 0.f;
        sum = fmaf(f, r < ranks ? sums[r] : 0.f, sum);
        acc = fmaf(f, r < ranks ? accs[r] : 0.f, acc);
      }
    }
    const float v = sum == 0.f ? 0.f : acc / sum;
    const long long at = ((long long)b * a.H + h) * a.Nq + i;
    const long long off = (((long long)b * a.Nq + i) * a.H + h) * a.D + d;
    const float lse = sum == 0.f ? -INFINITY : top - ref + log2f(sum);
    if (cluster) {
      const T r = from_f32<T>(v);
      static_cast<T*>(a.out)[off] = r;
      if (a.low) static_cast<T*>(a.low)[off] = from_f32<T>(v - to_f32(r));
      if (d == 0 && a.lse) a.lse[at] = lse;
    } else {
      p.part_o[(long long)split * a.B * a.Nq * a.H * a.D + off] = v;
      if (d == 0) p.part_lse[(long long)split * a.B * a.H * a.Nq + at] = lse;
    }
  }
  if (cluster) {
    // No block leaves while another reads its rows.
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
}

// Joins the splits' rows: a warp for a row.
template <typename T>
__global__ void __launch_bounds__(128) join_splits(const __grid_constant__ FwdParams p) {
  pdl_trigger();
  pdl_wait();
  const long long rows = (long long)p.a.B * p.a.H * p.a.Nq;
  const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= rows) return;
  const int lane = threadIdx.x & 31;
  const int n = row % p.a.Nq, h = row / p.a.Nq % p.a.H;
  const long long b = row / p.a.Nq / p.a.H;
  // A lane for a split's weight (two: there are at most 64).
  float w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    w[i] = lane + 32 * i < p.splits ? p.part_lse[(lane + 32 * i) * rows + row] : -INFINITY;
  float top = fmaxf(w[0], w[1]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
  const float sub = top == -INFINITY ? 0.f : top;
  const long long off = ((b * p.a.Nq + n) * p.a.H + h) * p.a.D, plane = rows * p.a.D;
  w[0] = ex2(w[0] - sub);
  w[1] = ex2(w[1] - sub);
  float acc[kMaxD / 32] = {}, sum = 0.f;
#pragma unroll 4
  for (int s = 0; s < p.splits; ++s) {
    const float f = __shfl_sync(~0u, s < 32 ? w[0] : w[1], s & 31);
    sum += f;
#pragma unroll
    for (int i = 0; i < kMaxD / 32; ++i)
      if (lane + 32 * i < p.a.D)
        acc[i] = fmaf(f, p.part_o[s * plane + off + lane + 32 * i], acc[i]);
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int i = 0; i < kMaxD / 32; ++i)
    if (lane + 32 * i < p.a.D) {
      const float v = acc[i] * inv;
      const T r = from_f32<T>(v);
      static_cast<T*>(p.a.out)[off + lane + 32 * i] = r;
      if (p.a.low) static_cast<T*>(p.a.low)[off + lane + 32 * i] = from_f32<T>(v - to_f32(r));
    }
  if (p.a.lse && lane == 0) p.a.lse[row] = sum == 0.f ? -INFINITY : top + log2f(sum);
}

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                   const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                   const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                   CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static const EncodeTiledFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) !=
            cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<EncodeTiledFn>(f);
  }();
  return fn;
}

int up(int v, int to) { return (v + to - 1) / to * to; }

}  // namespace

bool encode_tile4(CUtensorMap* map, Pick* pick, const void* ptr, const Strides& s, int B, int N,
                  int H, int D, int rows, bool bf16) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  pick->h = H > 1 && s.h != 0;
  pick->b = B > 1 && s.b != 0;
  // A dimension of size 1 is never stepped along: any legal stride does.
  const cuuint64_t row = (cuuint64_t)D * 2;
  cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)N, pick->h ? (cuuint64_t)H : 1,
                        pick->b ? (cuuint64_t)B : 1};
  cuuint64_t strides[3] = {N > 1 ? (cuuint64_t)s.n * 2 : row, pick->h ? (cuuint64_t)s.h * 2 : row,
                           pick->b ? (cuuint64_t)s.b * 2 : row};
  cuuint32_t box[4] = {64, (cuuint32_t)rows, 1, 1}, step[4] = {1, 1, 1, 1};
  return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
            const_cast<void*>(ptr), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

namespace {

constexpr size_t kSmemMax = 227 * 1024 - 1024;  // beside the static part

// Few queries, more keys than one tile: the form that reads straight into fragments.
bool is_token(const Args& a) { return a.Nq <= kTokenQueries && a.Nk > 128; }

// Its split: blocks for four times the SMs, of at least one step of every warp; a
// power of two up to a cluster's eight.
void plan_token(FwdParams* p, int sms) {
  const Args& a = p->a;
  const int step = kTokenWarps * 16 * token_steps((a.D + 63) / 64, a.mask_kind != kMaskNone);
  const long long heads = (long long)a.B * a.H;
  long long want = (4ll * sms + heads - 1) / heads;
  const int steps = (a.Nk + step - 1) / step;
  if (want > steps) want = steps;
  if (want > kMostSplits) want = kMostSplits;
  // More blocks than a cluster's where that leaves each of them 512 keys or more: the
  // second kernel takes 3 us.
  if (want > 2 * kTokenCluster && a.Nk / kTokenCluster >= 1024) {
    want = std::min(want, (long long)a.Nk / 512);
    p->per = (int)((steps + want - 1) / want) * step;
    p->splits = (a.Nk + p->per - 1) / p->per;
    return;
  }
  p->splits = 1;
  while (p->splits < kTokenCluster && p->splits < want) p->splits *= 2;
  p->per = (int)((steps + p->splits - 1) / p->splits) * step;
}

template <typename T, int DB>
cudaError_t run_token_d(const FwdParams& p, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((long long)p.a.B * p.a.H * p.splits));
  cfg.blockDim = dim3(kTokenWarps * 32);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled(kPdlInput) ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = p.splits <= kTokenCluster ? p.splits : 1;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return p.a.mask_kind == kMaskNone ? cudaLaunchKernelEx(&cfg, forward_token<T, DB, false>, p)
                                    : cudaLaunchKernelEx(&cfg, forward_token<T, DB, true>, p);
}
template <typename T>
cudaError_t run_token(const FwdParams& p, cudaStream_t s) {
  cudaError_t e = p.a.D <= 64    ? run_token_d<T, 1>(p, s)
                  : p.a.D <= 128 ? run_token_d<T, 2>(p, s)
                                 : run_token_d<T, 3>(p, s);
  if (e == cudaSuccess && p.splits > kTokenCluster) {
    const long long rows = (long long)p.a.B * p.a.H * p.a.Nq;
    e = launch_pdl(kPdlInput, join_splits<T>, dim3((unsigned)((rows + 3) / 4)), dim3(128), 0, s, p);
  }
  return e;
}

// The split of one call over blocks, tiles and stages.
void plan(FwdParams* p, int sms) {
  const Args& a = p->a;
  p->DB = (a.D + 63) / 64;
  // Two stages of K and V beside Q fit shared memory, and S beside O a half of
  // tensor memory, with 128 keys a tile up to 128-wide heads and with 96 above.
  const int most = a.Nk > 128 && p->DB > 2 ? 96 : 128;
  p->nkt = (a.Nk + most - 1) / most;
  p->KT = up((a.Nk + p->nkt - 1) / p->nkt, 16);
  p->nkt = (a.Nk + p->KT - 1) / p->KT;
  p->DP = up(a.D, 16);
  p->qtiles = (a.Nq + kRows - 1) / kRows;
  p->total = (long long)a.B * a.H * p->qtiles;
  p->splits = 1;
  p->per = p->nkt;
  if (p->nkt > 1 && p->total < sms) {
    const long long want = std::min((long long)std::min(p->nkt, kMostSplits), kBlocks * sms / p->total);
    p->per = (int)((p->nkt + want - 1) / want);
    p->splits = (p->nkt + p->per - 1) / p->per;
  }
  p->q_bytes = (uint32_t)p->DB * kRows * 128;
  p->k_bytes = (uint32_t)p->DB * p->KT * 128;
  const bool one = p->per == 1;
  // With one tile O takes the columns that P leaves of S.
  p->o_col = (uint32_t)(one ? up(p->KT / 2, 16) : p->KT);
  const int cols = p->KT > (int)p->o_col + p->DP ? p->KT : (int)p->o_col + p->DP;
  p->tmem_cols = cols <= 32 ? 32 : cols <= 64 ? 64 : cols <= 128 ? 128 : cols <= 256 ? 256 : 512;
  // One tile: the next head's K and V land beside this one's where that costs no block
  // of an SM.
  const auto smem = [&](int stages) {
    return (one ? 2ull : 1ull) * p->q_bytes + 2ull * stages * p->k_bytes + 1024;
  };
  const auto per_sm = [&](int stages) {
    return std::min((long long)(kSmemMax / smem(stages)),
                    std::min((long long)kBlocks, 512ll / p->tmem_cols));
  };
  p->kstages = one && per_sm(2) < per_sm(1) ? 1 : 2;
  long long blocks = one ? std::max(1ll, per_sm(p->kstages)) * sms / p->splits : p->total;
  p->blocks = (int)std::max(1ll, std::min(blocks, p->total));
  p->walks = p->blocks < p->total;
}

size_t smem_bytes(const FwdParams& p) {
  size_t n = (p.walks ? 2ull : 1ull) * p.q_bytes + 2ull * p.kstages * p.k_bytes + 1024;
  // No more blocks on an SM than its tensor memory holds.
  const size_t least = kSmemMax / (512 / p.tmem_cols + 1) + 1;
  return n > least ? n : least;
}

size_t align256(size_t n) { return (n + 255) & ~size_t(255); }

template <typename T, bool MASK, bool ONE>
cudaError_t run(const FwdParams& p, const CUtensorMap* m, cudaStream_t s) {
  static std::atomic<unsigned long long> allowed{0};
  const size_t smem = smem_bytes(p);
  cudaError_t e = allow_smem(forward_tc<T, MASK, ONE>, &allowed, kSmemMax);
  if (e != cudaSuccess) return e;
  const unsigned grid = (unsigned)((long long)p.blocks * p.splits);
  e = launch_pdl(kPdlInput, forward_tc<T, MASK, ONE>, dim3(grid), dim3(kThreads), smem, s, m[0], m[1],
                 m[2], m[3], p);
  if (e == cudaSuccess && p.splits > 1) {
    const long long rows = (long long)p.a.B * p.a.H * p.a.Nq;
    e = launch_pdl(kPdlInput, join_splits<T>, dim3((unsigned)((rows + 3) / 4)), dim3(128), 0, s, p);
  }
  return e;
}

}  // namespace

long long forward_workspace_bytes(int B, int Nq, int Nk, int H, int D) {
  size_t most = 0;
  for (int mask : {kMaskNone, kMaskBool}) {  // the larger of the two splits
    FwdParams p{};
    p.a.B = B, p.a.Nq = Nq, p.a.Nk = Nk, p.a.H = H, p.a.D = D, p.a.mask_kind = mask;
    const bool token = is_token(p.a);
    if (token) plan_token(&p, device_sms());
    else plan(&p, device_sms());
    if (p.splits == 1 || (token && p.splits <= kTokenCluster)) continue;
    const size_t rows = (size_t)B * H * Nq * p.splits;
    most = std::max(most, align256(rows * D * 4) + align256(rows * 4));
  }
  return (long long)most;
}

cudaError_t forward_status(int* status) {
  cudaError_t e = cudaMemcpyFromSymbol(status, g_status, sizeof(int));
  const int zero = 0;
  return e == cudaSuccess ? cudaMemcpyToSymbol(g_status, &zero, sizeof(int)) : e;
}

cudaError_t launch_forward(const Args& a, bool bf16, void* ws, cudaStream_t s, const char** why) {
  FwdParams p{};
  p.a = a;
  const bool token = is_token(a);
  if (token) plan_token(&p, device_sms());
  else plan(&p, device_sms());
  const size_t rows = (size_t)a.B * a.H * a.Nq * p.splits;
  p.part_o = static_cast<float*>(ws);
  p.part_lse = p.splits > 1 ? reinterpret_cast<float*>(static_cast<unsigned char*>(ws) +
                                                       align256(rows * a.D * 4))
                            : nullptr;
  if (token) return bf16 ? run_token<__nv_bfloat16>(p, s) : run_token<__half>(p, s);
  CUtensorMap m[4];
  const Strides dense{(long long)a.Nq * a.H * a.D, (long long)a.H * a.D, a.D};
  if (!encode_tile4(&m[0], &p.qp, a.q, a.qs, a.B, a.Nq, a.H, a.D, kRows, bf16) ||
      !encode_tile4(&m[1], &p.kp, a.k, a.ks, a.B, a.Nk, a.H, a.D, p.KT, bf16) ||
      !encode_tile4(&m[2], &p.vp, a.v, a.vs, a.B, a.Nk, a.H, a.D, p.KT, bf16) ||
      !encode_tile4(&m[3], &p.op, a.out, dense, a.B, a.Nq, a.H, a.D, kRows, bf16)) {
    *why = "tensor map encode failed";
    return cudaErrorInvalidValue;
  }
  const bool mask = a.mask_kind != kMaskNone, one = p.KT <= kHeld;
#define NOVA_XATTN_RUN(T)                                                    \
  (mask ? (one ? run<T, true, true>(p, m, s) : run<T, true, false>(p, m, s)) \
        : (one ? run<T, false, true>(p, m, s) : run<T, false, false>(p, m, s)))
  return bf16 ? NOVA_XATTN_RUN(__nv_bfloat16) : NOVA_XATTN_RUN(__half);
#undef NOVA_XATTN_RUN
}

}  // namespace xattn
}  // namespace nova
