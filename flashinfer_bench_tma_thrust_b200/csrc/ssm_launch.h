// ssm_launch.h — launch parameters of the short convolution and the state space scan,
// filled and checked by ssm_capi.cu, used by the kernels' launchers. A launcher returns 0
// or a GDN_ERR_* code.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace gdn {

constexpr int kMaxSections = 8;
constexpr int kMaxTaps = 4;

struct ConvParams {
  const __nv_bfloat16* x;       // [rows, C], rows x_stride elements apart
  int64_t x_stride;
  const void* weight;           // [C, W]
  const void* bias;             // [C] or null
  int weight_dtype, bias_dtype;
  const __nv_bfloat16* state;   // [N, W-1, C] or null (zeros)
  __nv_bfloat16* new_state;     // [N, W-1, C]
  const void* cu_seqlens;       // prompts only
  int cu_dtype;
  int64_t T, N;                 // tokens; sequences (one token each where cu_seqlens is null)
  int C, W;
  int silu;
  float eps;
  // sections of the channels: section i holds [begin[i], begin[i+1]), its rows are
  // contiguous in out[i]
  int sections;
  int begin[kMaxSections + 1];
  int normed[kMaxSections];
  __nv_bfloat16* out[kMaxSections];
  int* status;                  // see below; may be null
};

struct SsmParams {
  const __nv_bfloat16* x;       // [T, H, P]
  const __nv_bfloat16* B;       // [T, G, Ns]
  const __nv_bfloat16* C;       // [T, G, Ns]
  const void* dt;               // [T, H]
  const void* A_log;            // [H]
  const void* dt_bias;          // [H]
  const void* D;                // [H] or null
  int dt_dtype, A_log_dtype, dt_bias_dtype, D_dtype;
  const void* state;            // [N, H, P, Ns] or null (zeros)
  void* new_state;
  int state_bf16;               // single tokens only: the state's type is bf16
  const void* cu_seqlens;       // prompts only
  int cu_dtype;
  __nv_bfloat16* out;           // [T, H, P]
  int64_t T, N;                 // tokens, sequences (equal for single tokens)
  int H, G, P, Ns;
  float* workspace;             // chunked prompts: states of the segments
  int* status;                  // two words, see below; may be null
};

// The status words (device memory or mapped host memory): [0] becomes 1 where a bounded
// wait gave up, [1] where cu_seqlens held a bound outside [0, T] or a decreasing pair.
// Plain stores to words of their own: no atomics on host memory.
__device__ __forceinline__ void report_wait(int* status) {
  if (status) *reinterpret_cast<volatile int*>(status) = 1;
}
__device__ __forceinline__ void report_bad_bounds(int* status) {
  if (status) *reinterpret_cast<volatile int*>(status + 1) = 1;
}

int launch_conv_prefill(const ConvParams& p, cudaStream_t stream);
int launch_conv_decode(const ConvParams& p, cudaStream_t stream);
int launch_ssm_decode(const SsmParams& p, cudaStream_t stream);
int launch_ssm_recurrent(const SsmParams& p, cudaStream_t stream);
// The chunked kernel: the calls it takes, the workspace bytes of a call (0: none), the call.
bool ssm_chunked_takes(int P, int Ns, int64_t T, int64_t N);
size_t ssm_chunked_workspace(int64_t T, int64_t N, int H, int G, int P, int Ns);
int launch_ssm_chunked(const SsmParams& p, cudaStream_t stream);

}  // namespace gdn
