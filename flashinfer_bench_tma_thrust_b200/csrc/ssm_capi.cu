// ssm_capi.cu — the extern "C" entries of the short convolution and the state space scan
// (include/gdn_b200.h): host-side checks, launch parameters, status codes. Nothing here
// throws, allocates or synchronises.
#include "gdn_b200.h"
#include "ssm_launch.h"

namespace {

bool real_ok(int dt) { return dt == GDN_DTYPE_F32 || dt == GDN_DTYPE_BF16; }
bool index_ok(int dt) { return dt == GDN_DTYPE_I32 || dt == GDN_DTYPE_I64; }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int fill_conv(gdn::ConvParams* p, const void* x, int64_t x_row_stride, const void* weight,
              int weight_dtype, const void* bias, int bias_dtype, const void* state,
              void* new_state, int activation, int32_t sections, const int32_t* widths,
              const int32_t* normed, float eps, void* const* outs, int64_t T, int64_t N,
              int32_t C, int32_t W) {
  if (T < 0 || N < 0) return GDN_ERR_INVALID_ARG;
  // (channel numbers are 32-bit, and the last block's go on for up to 1024 behind C)
  if (C <= 0 || C > INT32_MAX - 2048 || W < 2 || W > gdn::kMaxTaps)
    return GDN_ERR_UNSUPPORTED_SHAPE;
  if (sections < 1 || sections > gdn::kMaxSections || !widths || !normed || !outs)
    return GDN_ERR_INVALID_ARG;
  if (!real_ok(weight_dtype) || (bias && !real_ok(bias_dtype))) return GDN_ERR_UNSUPPORTED_DTYPE;
  if ((activation != 0 && activation != 1) || !(eps >= 0.f)) return GDN_ERR_INVALID_ARG;
  *p = gdn::ConvParams{};
  int64_t at = 0;
  for (int32_t s = 0; s < sections; ++s) {
    if (widths[s] <= 0) return GDN_ERR_UNSUPPORTED_SHAPE;
    // the heads of a normed section are whole warps
    if (normed[s] && (at % 128 || widths[s] % 128)) return GDN_ERR_UNSUPPORTED_SHAPE;
    p->begin[s] = static_cast<int>(at);
    p->normed[s] = normed[s] != 0;
    p->out[s] = static_cast<__nv_bfloat16*>(outs[s]);
    at += widths[s];
    if (at > C) return GDN_ERR_UNSUPPORTED_SHAPE;
    if (T > 0 && !outs[s]) return GDN_ERR_INVALID_ARG;
  }
  if (at != C) return GDN_ERR_UNSUPPORTED_SHAPE;
  for (int32_t s = sections; s <= gdn::kMaxSections; ++s) p->begin[s] = C;
  if (T > 0 && (!x || !weight || x_row_stride < 0)) return GDN_ERR_INVALID_ARG;
  if (N > 0 && !new_state) return GDN_ERR_INVALID_ARG;
  p->x = static_cast<const __nv_bfloat16*>(x);
  p->x_stride = x_row_stride;
  p->weight = weight;
  p->bias = bias;
  p->weight_dtype = weight_dtype;
  p->bias_dtype = bias_dtype;
  p->state = static_cast<const __nv_bfloat16*>(state);
  p->new_state = static_cast<__nv_bfloat16*>(new_state);
  p->T = T;
  p->N = N;
  p->C = C;
  p->W = W;
  p->silu = activation;
  p->eps = eps;
  p->sections = sections;
  return GDN_OK;
}

int fill_ssm(gdn::SsmParams* p, const void* x, const void* dt, int dt_dtype, const void* A_log,
             int A_log_dtype, const void* B, const void* C, const void* D, int D_dtype,
             const void* dt_bias, int dt_bias_dtype, const void* state, void* out,
             void* new_state, int64_t T, int64_t N, int32_t H, int32_t G, int32_t P,
             int32_t Ns) {
  if (T < 0 || N < 0) return GDN_ERR_INVALID_ARG;
  if (H <= 0 || G <= 0 || H % G || P < 1 || P > 256) return GDN_ERR_UNSUPPORTED_SHAPE;
  if (Ns != 16 && Ns != 32 && Ns != 64 && Ns != 128 && Ns != 256) return GDN_ERR_UNSUPPORTED_SHAPE;
  if (!real_ok(dt_dtype) || !real_ok(A_log_dtype) || !real_ok(dt_bias_dtype) ||
      (D && !real_ok(D_dtype)))
    return GDN_ERR_UNSUPPORTED_DTYPE;
  if (N > 0 && (!A_log || !dt_bias || !new_state)) return GDN_ERR_INVALID_ARG;
  if (T > 0 && (!x || !dt || !B || !C || !out)) return GDN_ERR_INVALID_ARG;
  // B, C and the states go through in vectors
  if (!aligned16(B) || !aligned16(C) || !aligned16(state) || !aligned16(new_state))
    return GDN_ERR_INVALID_ARG;
  *p = gdn::SsmParams{};
  p->x = static_cast<const __nv_bfloat16*>(x);
  p->B = static_cast<const __nv_bfloat16*>(B);
  p->C = static_cast<const __nv_bfloat16*>(C);
  p->dt = dt;
  p->A_log = A_log;
  p->dt_bias = dt_bias;
  p->D = D;
  p->dt_dtype = dt_dtype;
  p->A_log_dtype = A_log_dtype;
  p->dt_bias_dtype = dt_bias_dtype;
  p->D_dtype = D_dtype;
  p->state = state;
  p->new_state = new_state;
  p->out = static_cast<__nv_bfloat16*>(out);
  p->T = T;
  p->N = N;
  p->H = H;
  p->G = G;
  p->P = P;
  p->Ns = Ns;
  return GDN_OK;
}

}  // namespace

extern "C" {

int gdn_conv_prefill_fwd(const void* x, int64_t x_row_stride, const void* weight,
                         int weight_dtype, const void* bias, int bias_dtype, const void* state,
                         const void* cu_seqlens, int cu_dtype, int activation, int32_t sections,
                         const int32_t* widths, const int32_t* normed, float eps,
                         void* const* outs, void* new_state, int64_t T, int64_t N, int32_t C,
                         int32_t W, int32_t* status, void* stream) {
  gdn::ConvParams p;
  const int rc = fill_conv(&p, x, x_row_stride, weight, weight_dtype, bias, bias_dtype, state,
                           new_state, activation, sections, widths, normed, eps, outs, T, N, C, W);
  if (rc != GDN_OK) return rc;
  if (!index_ok(cu_dtype)) return GDN_ERR_UNSUPPORTED_DTYPE;
  if (N == 0) return GDN_OK;
  if (!cu_seqlens) return GDN_ERR_INVALID_ARG;
  p.cu_seqlens = cu_seqlens;
  p.cu_dtype = cu_dtype;
  p.status = status;
  return gdn::launch_conv_prefill(p, static_cast<cudaStream_t>(stream));
}

int gdn_conv_decode_fwd(const void* x, int64_t x_row_stride, const void* weight,
                        int weight_dtype, const void* bias, int bias_dtype, const void* state,
                        int activation, int32_t sections, const int32_t* widths,
                        const int32_t* normed, float eps, void* const* outs, void* new_state,
                        int64_t B, int32_t C, int32_t W, void* stream) {
  gdn::ConvParams p;
  const int rc = fill_conv(&p, x, x_row_stride, weight, weight_dtype, bias, bias_dtype, state,
                           new_state, activation, sections, widths, normed, eps, outs, B, B, C, W);
  if (rc != GDN_OK) return rc;
  if (B == 0) return GDN_OK;
  return gdn::launch_conv_decode(p, static_cast<cudaStream_t>(stream));
}

int gdn_ssm_decode_fwd(const void* x, const void* dt, int dt_dtype, const void* A_log,
                       int A_log_dtype, const void* B, const void* C, const void* D, int D_dtype,
                       const void* dt_bias, int dt_bias_dtype, const void* state, int state_dtype,
                       void* out, void* new_state, int64_t batch, int32_t H, int32_t G, int32_t P,
                       int32_t Ns, void* stream) {
  gdn::SsmParams p;
  const int rc = fill_ssm(&p, x, dt, dt_dtype, A_log, A_log_dtype, B, C, D, D_dtype, dt_bias,
                          dt_bias_dtype, state, out, new_state, batch, batch, H, G, P, Ns);
  if (rc != GDN_OK) return rc;
  if (!real_ok(state_dtype)) return GDN_ERR_UNSUPPORTED_DTYPE;
  if (batch == 0) return GDN_OK;
  p.state_bf16 = state_dtype == GDN_DTYPE_BF16;
  return gdn::launch_ssm_decode(p, static_cast<cudaStream_t>(stream));
}

int gdn_ssm_prefill_recurrent_fwd(const void* x, const void* dt, int dt_dtype, const void* A_log,
                                  int A_log_dtype, const void* B, const void* C, const void* D,
                                  int D_dtype, const void* dt_bias, int dt_bias_dtype,
                                  const float* state, const void* cu_seqlens, int cu_dtype,
                                  void* out, float* new_state, int64_t T, int64_t N, int32_t H,
                                  int32_t G, int32_t P, int32_t Ns, int32_t* status,
                                  void* stream) {
  gdn::SsmParams p;
  const int rc = fill_ssm(&p, x, dt, dt_dtype, A_log, A_log_dtype, B, C, D, D_dtype, dt_bias,
                          dt_bias_dtype, state, out, new_state, T, N, H, G, P, Ns);
  if (rc != GDN_OK) return rc;
  if (!index_ok(cu_dtype)) return GDN_ERR_UNSUPPORTED_DTYPE;
  if (N == 0) return GDN_OK;
  if (!cu_seqlens) return GDN_ERR_INVALID_ARG;
  p.cu_seqlens = cu_seqlens;
  p.cu_dtype = cu_dtype;
  p.status = status;
  return gdn::launch_ssm_recurrent(p, static_cast<cudaStream_t>(stream));
}

size_t gdn_ssm_prefill_workspace_size(int64_t T, int64_t N, int32_t H, int32_t G, int32_t P,
                                      int32_t Ns) {
  if (T < 0 || N < 0 || H <= 0 || G <= 0 || H % G || !gdn::ssm_chunked_takes(P, Ns, T, N))
    return 0;
  return gdn::ssm_chunked_workspace(T, N, H, G, P, Ns);
}

int gdn_ssm_prefill_fwd(const void* x, const void* dt, int dt_dtype, const void* A_log,
                        int A_log_dtype, const void* B, const void* C, const void* D,
                        int D_dtype, const void* dt_bias, int dt_bias_dtype, const float* state,
                        const void* cu_seqlens, int cu_dtype, void* out, float* new_state,
                        int64_t T, int64_t N, int32_t H, int32_t G, int32_t P, int32_t Ns,
                        void* workspace, size_t workspace_bytes, int32_t* status, void* stream) {
  gdn::SsmParams p;
  const int rc = fill_ssm(&p, x, dt, dt_dtype, A_log, A_log_dtype, B, C, D, D_dtype, dt_bias,
                          dt_bias_dtype, state, out, new_state, T, N, H, G, P, Ns);
  if (rc != GDN_OK) return rc;
  if (!index_ok(cu_dtype)) return GDN_ERR_UNSUPPORTED_DTYPE;
  if (N == 0) return GDN_OK;
  if (!cu_seqlens) return GDN_ERR_INVALID_ARG;
  p.cu_seqlens = cu_seqlens;
  p.cu_dtype = cu_dtype;
  p.status = status;
  if (!gdn::ssm_chunked_takes(P, Ns, T, N))
    return gdn::launch_ssm_recurrent(p, static_cast<cudaStream_t>(stream));
  // bulk copies read x and write out; token coordinates are 32-bit
  if (!aligned16(x) || !aligned16(out) || !aligned16(workspace)) return GDN_ERR_INVALID_ARG;
  if (T > 0x7fffff00LL) return GDN_ERR_UNSUPPORTED_SHAPE;
  const size_t need = gdn::ssm_chunked_workspace(T, N, H, G, P, Ns);
  if (need && (!workspace || workspace_bytes < need)) return GDN_ERR_WORKSPACE;
  p.workspace = static_cast<float*>(workspace);
  return gdn::launch_ssm_chunked(p, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
