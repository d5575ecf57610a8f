// Shared by the cross-attention kernels: arguments, the masks' meaning, and the
// tensor-core pieces that the convolution's GEMM does not need (4-D tiles,
// operands with the other index contiguous, operands in tensor memory).
#pragma once

#include "nova_tc_ptx.cuh"
#include "nova_unet_ops.h"

namespace nova {
namespace xattn {

using namespace unet;

constexpr int kMaskNone = -1, kMaskBool = 3;  // else the element type of an additive mask
constexpr int kMaxD = 160;
constexpr float kLog2e = 1.4426950408889634f;

struct Strides {
  long long b, n, h;  // elements
};

struct Args {
  const void *q, *k, *v, *dout, *mask;
  const float* lse_in;
  void* out;   // o
  void* low;   // what the rounding of o left off, or null
  float* lse;  // [B][H][Nq], base 2, relative to the sample's largest bias; minus
               // infinity for a query without keys
  void *dq, *dk, *dv;
  const float* delta;  // [B][H][Nq]: sum(p dp)
  Strides qs, ks, vs, dos;
  long long mb, mn;  // mask strides
  int B, Nq, Nk, H, D;
  int mask_kind;
  float scale;
};

// An additive bias in base 2.  Above 2^126 the change of base gives way to a line that
// ends at the largest finite value: finite biases stay finite and in their order, so
// that a row with nothing but lowest values is the uniform row that 32 bits give.
__device__ __forceinline__ float bias2(float m) {
  constexpr float kFar = 8.507059173e37f, kMost = 3.402823466e38f;
  const float far = fabsf(m);
  if (!(far > kFar && far <= kMost)) return m * kLog2e;
  const float t = fmaf(far - kFar, (kMost - kFar * kLog2e) / (kMost - kFar), kFar * kLog2e);
  return copysignf(fminf(t, kMost), m);
}

// Bias of key n in base 2, and whether the key takes part.
__device__ __forceinline__ bool key_bias(const Args& a, int b, int n, float* bias) {
  *bias = 0.f;
  if (a.mask_kind == kMaskNone) return true;
  const long long i = b * a.mb + n * a.mn;
  if (a.mask_kind == kMaskBool) return static_cast<const unsigned char*>(a.mask)[i] != 0;
  const float m = load_param(a.mask, a.mask_kind, i);
  if (m == -INFINITY) return false;
  *bias = bias2(m);
  return true;
}

// The largest additive bias of sample b's keys i, i + step, ..., in base 2; minus
// infinity for none.  What a row's logarithm is taken relative to: beside a bias that
// all keys share (the lowest value, -1e9) the logarithm of the sum would be lost.
// Not inlined: few calls need it, and its code would keep the others' from the
// instruction cache (8 x 1024 queries to 77 keys, forward and gradient: 41.5 us, inlined 43.5).
template <typename T>
__device__ __forceinline__ float most_of(const T* m, long long mn, int keys, int i, int step) {
  float top = -INFINITY;
#pragma unroll 1
  for (int n = i; n < keys; n += 8 * step) {
    T v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const long long at = n + (long long)u * step;
      v[u] = m[(at < keys ? at : n) * mn];
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) top = fmaxf(top, to_f32(v[u]));
  }
  return top;
}
static __device__ __noinline__ float largest_bias(const void* mask, int kind, long long from,
                                                  long long mn, int keys, int i, int step) {
  const float top =
      kind == kF32   ? most_of(static_cast<const float*>(mask) + from, mn, keys, i, step)
      : kind == kF16 ? most_of(static_cast<const __half*>(mask) + from, mn, keys, i, step)
                     : most_of(static_cast<const __nv_bfloat16*>(mask) + from, mn, keys, i, step);
  return bias2(top);
}
__device__ __forceinline__ float largest_bias(const Args& a, int b, int i, int step) {
  return largest_bias(a.mask, a.mask_kind, b * a.mb, a.mn, a.Nk, i, step);
}
__device__ __forceinline__ bool is_additive(const Args& a) {
  return a.mask_kind != kMaskNone && a.mask_kind != kMaskBool;
}
__device__ __forceinline__ float warp_most(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, o));
  return v;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
  if constexpr (std::is_same<T, __half>::value)
    return __half22float2(*reinterpret_cast<const __half2*>(&v));
  else
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
}

// Bounded wait: false when the phase did not complete within kWaitLimitNs or another
// thread of the block gave up.  The timer is read only after many tries: its read
// takes as long as one of the products that are waited for here.
__device__ __forceinline__ bool wait_phase(uint32_t bar, uint32_t parity, volatile int* abort_flag,
                                           int* status, int code) {
  uint64_t since = 0;
  for (uint32_t i = 1;; ++i) {
    if (tc::mbar_try_wait(bar, parity)) return true;
    if ((i & 1023u) == 0) {
      if (*abort_flag) return false;
      const uint64_t now = tc::globaltimer();
      if (since == 0) since = now;
      if (now - since > tc::kWaitLimitNs) {
        *abort_flag = 1;
        atomicCAS(status, 0, code);
        return false;
      }
    }
  }
}

// One lane of a converged warp, in a form that the compiler knows to be one.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(p));
  return p != 0;
}

// A tensor [batch][tokens][heads][D] as TMA sees it: (D, tokens, heads, batch),
// tiles of 64 elements x `rows` tokens, 128-byte rows swizzled.  Elements past D
// and tokens past the end read as zero and are not written.  A dimension that all
// its indices share (stride 0) has size 1 there, and its coordinate is 0.
struct Pick {  // factors of the head and batch coordinates: 1, or 0 for a shared dimension
  int h, b;
};
bool encode_tile4(CUtensorMap* map, Pick* pick, const void* p, const Strides& s, int B, int N,
                  int H, int D, int rows, bool bf16);

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int c0, int c1,
                                            int c2, int c3, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tma_store_4d(const CUtensorMap* map, uint32_t src, int c0, int c1,
                                             int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%1, %2, %3, %4}], [%5];" ::"l"(
          reinterpret_cast<uint64_t>(map)),
      "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(src)
      : "memory");
}

// Descriptor of a swizzled 128-byte-row tile read with its contiguous index as
// the operand's M or N (the rows are the contraction): 64-element column blocks
// `block_bytes` apart, 8-row groups 1024 bytes apart.
__device__ __forceinline__ uint64_t smem_desc_mn(uint32_t addr, uint32_t block_bytes) {
  return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)(block_bytes >> 4) << 16) | (64ull << 32) |
         (1ull << 46) | (2ull << 61);
}

// Instruction descriptor: FP32 accumulator, both operands of one 16-bit type;
// a_mn / b_mn: the operand's contiguous index is its M / N.
__device__ __forceinline__ uint32_t instr_desc(bool bf16, int M, int N, bool a_mn, bool b_mn) {
  const uint32_t t = bf16 ? 1u : 0u;
  return (1u << 4) | (t << 7) | (t << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) |
         ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

// D += A B with A in tensor memory: lane = row, a column holds two elements.
__device__ __forceinline__ void umma_f16_ta(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc,
                                            uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void tmem_ld16_issue(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait_ld() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ void st_shared_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c,
                                             uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c),
               "r"(d)
               : "memory");
}

// Byte offset of 16-byte piece `piece` of row `row` in a swizzled tile.
__device__ __forceinline__ uint32_t sw128(int row, int piece) {
  return (uint32_t)row * 128u + (uint32_t)((piece ^ (row & 7)) << 4);
}

// Forward (nova_attention_fwd.cu): workspace and launch.
long long forward_workspace_bytes(int B, int Nq, int Nk, int H, int D);
cudaError_t launch_forward(const Args& a, bool bf16, void* ws, cudaStream_t s, const char** why);
cudaError_t forward_status(int* status);  // of the current device; clears it

// Gradient (nova_attention_bwd.cu).
long long backward_workspace_bytes(int B, int Nq, int Nk, int H, int D);
cudaError_t launch_backward(const Args& a, bool bf16, void* ws, cudaStream_t s, const char** why);
bool backward_reads_output(int Nk, int D);
cudaError_t backward_status(int* status);

}  // namespace xattn
}  // namespace nova
