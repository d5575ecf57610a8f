// Cross attention of one set of tokens to an encoder's states of another length.
//
//   s = scale q k^T + bias[key],  p = softmax(s) over the keys the mask leaves,  o = p v
//
// and its gradient
//
//   dv = p^T do,  dp = do v^T,  ds = p (dp - sum(p dp)),  dq = scale ds k,  dk = scale ds^T q
//
// q is [B][Nq][H][D], k and v are [B][Nk][H][D] with strides of their own; the
// outputs are dense.  A key that the mask leaves out (false, or a bias of minus
// infinity) is never multiplied, whatever its k and v hold; a query without
// keys gets zeros, and passes no gradient on.
#include <string>

#include "../../include/nova_winograd.h"
#include "nova_attention.cuh"

namespace nova {
namespace xattn {

long long workspace_bytes(int B, int Nq, int Nk, int H, int D, bool grad) {
  return grad ? backward_workspace_bytes(B, Nq, Nk, H, D) : forward_workspace_bytes(B, Nq, Nk, H, D);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int check(const char* what, const Args& a, int dtype, bool grad) {
  auto bad = [&](const char* why) {
    return record_error(NOVA_ERR_INVALID_ARGUMENT, std::string(what) + ": " + why);
  };
  if (a.B < 1 || a.Nq < 1 || a.Nk < 1 || a.H < 1 || a.D < 1) return bad("bad sizes");
  if (a.D % 8 || a.D > kMaxD) return bad("head_dim must be a multiple of 8, at most 160");
  if (dtype != kF16 && dtype != kBF16) return bad("element type must be fp16 or bf16");
  if (a.mask_kind < kMaskNone || a.mask_kind > kMaskBool) return bad("bad mask type");
  if (!a.q || !a.k || !a.v || (a.mask_kind != kMaskNone && !a.mask)) return bad("null pointer");
  if (grad ? !a.dout || !a.lse_in || !a.dq || !a.dk || !a.dv : !a.out) return bad("null pointer");
  auto fine = [](const void* p, const Strides& s) {
    return aligned16(p) && s.b >= 0 && s.n > 0 && s.h >= 0 && s.b % 8 == 0 && s.n % 8 == 0 &&
           s.h % 8 == 0;
  };
  if (!fine(a.q, a.qs) || !fine(a.k, a.ks) || !fine(a.v, a.vs) ||
      (grad && !fine(a.dout, a.dos)))
    return bad("rows must start on 16 bytes and no stride may be negative, none of the tokens zero");
  if (grad ? !aligned16(a.dq) || !aligned16(a.dk) || !aligned16(a.dv)
           : !aligned16(a.out) || !aligned16(a.low))
    return bad("outputs must be 16-byte aligned");
  if (a.mb < 0 || a.mn < 0) return bad("negative mask stride");
  const long long rows = (long long)a.B * a.H * (a.Nq > a.Nk ? a.Nq : a.Nk);
  if (rows > (1ll << 31) - 4096) return bad("more than 2^31 - 4096 rows");
  return NOVA_OK;
}

// The workspace of checked arguments, by the current device: the operands' by then,
// whose SMs the launch plans for.
int check_workspace(const char* what, const Args& a, const void* ws, long long ws_bytes, bool grad) {
  const long long need = workspace_bytes(a.B, a.Nq, a.Nk, a.H, a.D, grad);
  if (need > 0 && (!ws || reinterpret_cast<uintptr_t>(ws) % 256))
    return record_error(NOVA_ERR_INVALID_ARGUMENT,
                        std::string(what) + ": workspace missing or not 256-byte aligned");
  if (ws_bytes < need)
    return record_error(NOVA_ERR_WORKSPACE,
                        std::string(what) + ": workspace needs " + std::to_string(need) + " bytes");
  return NOVA_OK;
}

int done(const char* what, cudaError_t e) {
  if (e == cudaSuccess) return NOVA_OK;
  return record_error(NOVA_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
}

}  // namespace xattn
}  // namespace nova

#define NOVA_EXPORT extern "C" __attribute__((visibility("default")))

NOVA_EXPORT long long nova_cross_attention_workspace_bytes(int batch, int queries, int keys,
                                                           int heads, int head_dim, int grad) {
  if (batch < 1 || queries < 1 || keys < 1 || heads < 1 || head_dim < 8 || head_dim % 8 ||
      head_dim > nova::xattn::kMaxD)
    return -1;
  return nova::xattn::workspace_bytes(batch, queries, keys, heads, head_dim, grad != 0);
}

NOVA_EXPORT int nova_cross_attention_v2(const void* d_q, const void* d_k, const void* d_v,
                                        const void* d_mask, void* d_output, void* d_low, void* d_lse,
                                        void* d_workspace, long long ws_bytes, int batch,
                                        int queries, int keys, int heads, int head_dim,
                                        const long long* strides, int dtype, int mask_type,
                                        float scale, void* stream) try {
  using namespace nova;
  using namespace nova::xattn;
  if (!strides) return record_error(NOVA_ERR_INVALID_ARGUMENT, "cross_attention: null strides");
  Args a{};
  a.q = d_q, a.k = d_k, a.v = d_v, a.mask = d_mask, a.out = d_output;
  a.low = d_low;
  a.lse = static_cast<float*>(d_lse);
  const long long* t = strides;
  a.qs = {t[0], t[1], t[2]}, a.ks = {t[3], t[4], t[5]}, a.vs = {t[6], t[7], t[8]};
  a.mb = t[9], a.mn = t[10];
  a.B = batch, a.Nq = queries, a.Nk = keys, a.H = heads, a.D = head_dim;
  a.mask_kind = mask_type, a.scale = scale;
  if (const int rc = check("cross_attention", a, dtype, false)) return rc;
  const OnDeviceOf device(d_q);
  if (const int rc = check_workspace("cross_attention", a, d_workspace, ws_bytes, false)) return rc;
  if (device.status() != cudaSuccess) return done("cross_attention: q", device.status());
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const char* why = nullptr;
  const cudaError_t e = launch_forward(a, dtype == kBF16, d_workspace, s, &why);
  if (why) return record_error(NOVA_ERR_CUDA, std::string("cross_attention: ") + why);
  return done("cross_attention", e);
} catch (...) {
  return NOVA_ERR_ALLOC;
}

NOVA_EXPORT int nova_cross_attention_grad_v2(
    const void* d_q, const void* d_k, const void* d_v, const void* d_mask, const void* d_output,
    const void* d_low, const void* d_grad_output, const void* d_lse, void* d_grad_q, void* d_grad_k, void* d_grad_v,
    void* d_workspace, long long ws_bytes, int batch, int queries, int keys, int heads,
    int head_dim, const long long* strides, int dtype, int mask_type, float scale,
    void* stream) try {
  using namespace nova;
  using namespace nova::xattn;
  if (!strides) return record_error(NOVA_ERR_INVALID_ARGUMENT, "cross_attention_grad: null strides");
  Args a{};
  a.q = d_q, a.k = d_k, a.v = d_v, a.mask = d_mask, a.dout = d_grad_output;
  a.out = const_cast<void*>(d_output);
  a.low = const_cast<void*>(d_low);
  a.lse_in = static_cast<const float*>(d_lse);
  a.dq = d_grad_q, a.dk = d_grad_k, a.dv = d_grad_v;
  const long long* t = strides;
  a.qs = {t[0], t[1], t[2]}, a.ks = {t[3], t[4], t[5]}, a.vs = {t[6], t[7], t[8]};
  a.mb = t[9], a.mn = t[10];
  a.dos = {t[11], t[12], t[13]};
  a.B = batch, a.Nq = queries, a.Nk = keys, a.H = heads, a.D = head_dim;
  a.mask_kind = mask_type, a.scale = scale;
  if (const int rc = check("cross_attention_grad", a, dtype, true)) return rc;
  if (backward_reads_output(keys, head_dim) &&
      (!a.out || !a.low || !aligned16(a.out) || !aligned16(a.low)))
    return record_error(NOVA_ERR_INVALID_ARGUMENT,
                        "cross_attention_grad: these keys want output and low, 16-byte aligned");
  const OnDeviceOf device(d_q);
  if (const int rc = check_workspace("cross_attention_grad", a, d_workspace, ws_bytes, true))
    return rc;
  if (device.status() != cudaSuccess) return done("cross_attention_grad: q", device.status());
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const char* why = nullptr;
  const cudaError_t e = launch_backward(a, dtype == kBF16, d_workspace, s, &why);
  if (why) return record_error(NOVA_ERR_CUDA, std::string("cross_attention_grad: ") + why);
  return done("cross_attention_grad", e);
} catch (...) {
  return NOVA_ERR_ALLOC;
}

NOVA_EXPORT int nova_cross_attention_status(void) try {
  using namespace nova;
  using namespace nova::xattn;
  cudaError_t e = cudaDeviceSynchronize();
  int fwd = 0, bwd = 0;
  if (e == cudaSuccess) e = forward_status(&fwd);
  if (e == cudaSuccess) e = backward_status(&bwd);
  if (e != cudaSuccess) return done("cross_attention_status", e);
  if (fwd || bwd)
    return record_error(NOVA_ERR_DEVICE_TIMEOUT, "cross_attention: a kernel's wait expired (code " +
                                                     std::to_string(fwd ? fwd : bwd) + ")");
  return NOVA_OK;
} catch (...) {
  return NOVA_ERR_ALLOC;
}
