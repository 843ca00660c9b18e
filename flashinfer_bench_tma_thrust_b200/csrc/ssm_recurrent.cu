// ssm_recurrent.cu — the selective state space scan as a recurrence: one new token per
// sequence (a stream of the state through the SMs), and packed prompts token by token.
//
// Per sequence and head h (group h / (H / G) gives B and C), with S [P, Ns] and rows p:
//     d = softplus(dt + dt_bias), g = exp(-exp(A_log) d)          (GDN's gate, fp32)
//     S'[p, :] = g S[p, :] + (d x_p) B,   y_p = S'[p, :] . C + D x_p
// A row needs only its x_p once g, d and B.C are known:
//     y_p = g (S[p, :] . C) + d x_p (B . C) + D x_p
// so one dot product per row, on the row as it was loaded.
#include <algorithm>

#include "gdn_b200.h"
#include "gdn_common.cuh"
#include "ssm_launch.h"

namespace gdn {
namespace {

// A lane's piece of a state row: kE elements in 16 bytes (4 of fp32, 8 of bf16). kLanes
// lanes hold a row of kLanes * kE * kPieces elements; lane l holds elements
// [(j * kLanes + l) * kE, + kE) of piece j.
template <typename S>
struct Piece;
template <>
struct Piece<float> {
  static constexpr int kE = 4;
  static __device__ __forceinline__ void load(const void* base, int64_t i, float (&v)[4]) {
    const float4 f = ld_stream_f4(static_cast<const float*>(base) + i);
    v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
  }
  static __device__ __forceinline__ void store(void* base, int64_t i, const float (&v)[4]) {
    st_stream_f4(static_cast<float*>(base) + i, make_float4(v[0], v[1], v[2], v[3]));
  }
};
template <>
struct Piece<__nv_bfloat16> {
  static constexpr int kE = 8;
  static __device__ __forceinline__ void load(const void* base, int64_t i, float (&v)[8]) {
    uint32_t u[4];
    asm volatile("ld.global.cs.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3])
                 : "l"(static_cast<const __nv_bfloat16*>(base) + i));
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[2 * k] = __uint_as_float(u[k] << 16);
      v[2 * k + 1] = __uint_as_float(u[k] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ void store(void* base, int64_t i, const float (&v)[8]) {
    uint32_t u[4];  // the state's own type: one rounding per step, the user's choice of it
#pragma unroll
    for (int k = 0; k < 4; ++k)
      asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(u[k]) : "f"(v[2 * k + 1]), "f"(v[2 * k]));
    asm volatile("st.global.cs.v4.u32 [%0], {%1,%2,%3,%4};" ::"l"(
                     static_cast<__nv_bfloat16*>(base) + i),
                 "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3])
                 : "memory");
  }
};

// kE consecutive bf16 values (kE = 4 or 8, aligned to their size) as floats.
template <int kE>
__device__ __forceinline__ void load_bf16(const __nv_bfloat16* p, float (&v)[kE]) {
#pragma unroll
  for (int k = 0; k < kE; k += 4) {
    const float4 f = load_bf16x4(p + k);
    v[k] = f.x; v[k + 1] = f.y; v[k + 2] = f.z; v[k + 3] = f.w;
  }
}

template <int kLanes>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ float bf16_at(const __nv_bfloat16* p) {
  return __uint_as_float(static_cast<uint32_t>(*reinterpret_cast<const unsigned short*>(p)) << 16);
}

// ---------------------------------------------------------------- one token per sequence
// HBM bounds it: the state goes through once (5 flop per 8 bytes). A warp takes kRows * kPer
// rows (at most 32: lane r holds x and y of row r) with all its loads in flight before it
// reduces any of them. Blocks of 4 warps share a head's rows, `splits` blocks a head.
template <typename S, int kLanes, int kPieces, int kRows>
__global__ void __launch_bounds__(128) ssm_decode_kernel(const __grid_constant__ SsmParams p,
                                                        int splits) {
  constexpr int kE = Piece<S>::kE;
  constexpr int kPer = 32 / kLanes;  // rows per load
  constexpr int kWarpRows = kRows * kPer;
  static_assert(kWarpRows <= 32, "");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int l = lane % kLanes, sub = lane / kLanes;
  const int64_t head = blockIdx.x / splits;  // flattened (sequence, head)
  const int split = static_cast<int>(blockIdx.x - head * splits);
  const int64_t n = head / p.H;
  const int h = static_cast<int>(head - n * p.H);
  const int64_t grp = n * p.G + h / (p.H / p.G);
  const int row0 = (split * 4 + warp) * kWarpRows;
  if (row0 >= p.P) return;

  float s[kRows][kPieces][kE];
  const int64_t at0 = (head * p.P + row0 + sub) * p.Ns + l * kE;
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      if (p.state && row0 + i * kPer + sub < p.P) {
        Piece<S>::load(p.state, at0 + i * kPer * p.Ns + j * kLanes * kE, s[i][j]);
      } else {
#pragma unroll
        for (int k = 0; k < kE; ++k) s[i][j][k] = 0.f;
      }
    }
  }
  const bool own = lane < kWarpRows && row0 + lane < p.P;
  const float x_lane = own ? bf16_at(p.x + head * p.P + row0 + lane) : 0.f;
  const float v = load_scalar(p.dt, p.dt_dtype, head) + load_scalar(p.dt_bias, p.dt_bias_dtype, h);
  const float d = softplus_ref(v);
  const float g = expf(-expf(load_scalar(p.A_log, p.A_log_dtype, h)) * d);
  const float skip = p.D ? load_scalar(p.D, p.D_dtype, h) : 0.f;
  float b[kPieces][kE], c[kPieces][kE], bc = 0.f;
#pragma unroll
  for (int j = 0; j < kPieces; ++j) {
    const int64_t at = grp * p.Ns + (j * kLanes + l) * kE;
    load_bf16<kE>(p.B + at, b[j]);
    load_bf16<kE>(p.C + at, c[j]);
#pragma unroll
    for (int k = 0; k < kE; ++k) bc = fmaf(b[j][k], c[j][k], bc);
  }
  bc = row_sum<kLanes>(bc);

  float y = 0.f;
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const float dx = d * __shfl_sync(0xffffffffu, x_lane, i * kPer + sub);
    float dot = 0.f;
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      float w[kE];
#pragma unroll
      for (int k = 0; k < kE; ++k) {
        dot = fmaf(s[i][j][k], c[j][k], dot);
        w[k] = fmaf(g, s[i][j][k], dx * b[j][k]);
      }
      if (row0 + i * kPer + sub < p.P)
        Piece<S>::store(p.new_state, at0 + i * kPer * p.Ns + j * kLanes * kE, w);
    }
    dot = row_sum<kLanes>(dot);
    const float yi = fmaf(g, dot, dx * bc);
    // row i * kPer + (lane % kPer) is in the lanes of that sub
    const float mine = kPer == 1 ? yi : __shfl_sync(0xffffffffu, yi, (lane % kPer) * kLanes);
    if (lane / kPer == i) y = mine;
  }
  if (own) p.out[head * p.P + row0 + lane] = __float2bfloat16_rn(fmaf(skip, x_lane, y));
}

// ---------------------------------------------------------------- prompts, token by token
// A warp keeps kRows * kPer rows of one head's state in registers over the whole sequence;
// the inputs of kStep tokens are loaded together. Any P, and the state sizes that the
// chunked kernel does not take; the independent check of that kernel elsewhere.
constexpr int kStep = 4;

template <int kLanes, int kPieces, int kRows>
__global__ void __launch_bounds__(128) ssm_recurrent_kernel(const __grid_constant__ SsmParams p,
                                                           int tiles) {
  constexpr int kE = 4;
  constexpr int kPer = 32 / kLanes;
  constexpr int kWarpRows = kRows * kPer;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int l = lane % kLanes, sub = lane / kLanes;
  const int64_t head = blockIdx.x / tiles;
  const int tile = static_cast<int>(blockIdx.x - head * tiles);
  const int64_t n = head / p.H;
  const int h = static_cast<int>(head - n * p.H);
  const int grp = h / (p.H / p.G);
  const int row0 = (tile * 4 + warp) * kWarpRows;
  if (row0 >= p.P) return;

  int64_t start = load_index(p.cu_seqlens, p.cu_dtype, n);
  int64_t end = load_index(p.cu_seqlens, p.cu_dtype, n + 1);
  if (p.status && threadIdx.x == 0 && h == 0 && tile == 0 &&
      (start < 0 || end > p.T || end < start))
    report_bad_bounds(p.status);
  start = start < 0 ? 0 : (start > p.T ? p.T : start);
  end = end < 0 ? 0 : (end > p.T ? p.T : end);

  float s[kRows][kPieces][kE];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int r = row0 + i * kPer + sub;
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      if (p.state && r < p.P) {
        Piece<float>::load(p.state, (head * p.P + r) * p.Ns + (j * kLanes + l) * kE, s[i][j]);
      } else {
#pragma unroll
        for (int k = 0; k < kE; ++k) s[i][j][k] = 0.f;
      }
    }
  }
  const float neg_a = -expf(load_scalar(p.A_log, p.A_log_dtype, h));
  const float dtb = load_scalar(p.dt_bias, p.dt_bias_dtype, h);
  const float skip = p.D ? load_scalar(p.D, p.D_dtype, h) : 0.f;

  for (int64_t t0 = start; t0 < end; t0 += kStep) {
    float b[kStep][kPieces][kE], c[kStep][kPieces][kE], x[kStep][kRows], d[kStep], g[kStep];
#pragma unroll
    for (int a = 0; a < kStep; ++a) {
      const int64_t t = min(t0 + a, end - 1);
#pragma unroll
      for (int j = 0; j < kPieces; ++j) {
        const int64_t at = (t * p.G + grp) * p.Ns + (j * kLanes + l) * kE;
        load_bf16<kE>(p.B + at, b[a][j]);
        load_bf16<kE>(p.C + at, c[a][j]);
      }
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const int r = row0 + i * kPer + sub;
        x[a][i] = r < p.P ? bf16_at(p.x + (t * p.H + h) * p.P + r) : 0.f;
      }
      d[a] = load_scalar(p.dt, p.dt_dtype, t * p.H + h);
    }
#pragma unroll
    for (int a = 0; a < kStep; ++a) {
      d[a] = softplus_ref(d[a] + dtb);
      g[a] = expf(neg_a * d[a]);
    }
#pragma unroll
    for (int a = 0; a < kStep; ++a) {
      if (t0 + a >= end) break;
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const float dx = d[a] * x[a][i];
        float dot = 0.f;
#pragma unroll
        for (int j = 0; j < kPieces; ++j) {
#pragma unroll
          for (int k = 0; k < kE; ++k) {
            s[i][j][k] = fmaf(g[a], s[i][j][k], dx * b[a][j][k]);
            dot = fmaf(s[i][j][k], c[a][j][k], dot);
          }
        }
        dot = row_sum<kLanes>(dot);
        const int r = row0 + i * kPer + sub;
        if (l == 0 && r < p.P)
          p.out[((t0 + a) * p.H + h) * p.P + r] = __float2bfloat16_rn(fmaf(skip, x[a][i], dot));
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int r = row0 + i * kPer + sub;
    if (r >= p.P) continue;
#pragma unroll
    for (int j = 0; j < kPieces; ++j)
      Piece<float>::store(p.new_state, (head * p.P + r) * p.Ns + (j * kLanes + l) * kE, s[i][j]);
  }
}

template <typename S, int kLanes, int kPieces, int kRows>
int decode_as(const SsmParams& p, cudaStream_t stream) {
  constexpr int kBlockRows = 4 * kRows * (32 / kLanes);
  const int64_t heads = p.N * p.H;
  const int splits = (p.P + kBlockRows - 1) / kBlockRows;
  if (heads * splits > 0x7fffffffLL) return GDN_ERR_UNSUPPORTED_SHAPE;
  ssm_decode_kernel<S, kLanes, kPieces, kRows>
      <<<static_cast<unsigned>(heads * splits), 128, 0, stream>>>(p, splits);
  return cudaGetLastError() == cudaSuccess ? 0 : GDN_ERR_CUDA;
}

template <int kLanes, int kPieces, int kRows>
int recurrent_as(const SsmParams& p, cudaStream_t stream) {
  constexpr int kTile = 4 * kRows * (32 / kLanes);
  const int tiles = (p.P + kTile - 1) / kTile;
  const int64_t blocks = p.N * p.H * tiles;
  if (blocks > 0x7fffffffLL) return GDN_ERR_UNSUPPORTED_SHAPE;
  ssm_recurrent_kernel<kLanes, kPieces, kRows>
      <<<static_cast<unsigned>(blocks), 128, 0, stream>>>(p, tiles);
  return cudaGetLastError() == cudaSuccess ? 0 : GDN_ERR_CUDA;
}

}  // namespace

int launch_ssm_decode(const SsmParams& p, cudaStream_t stream) {
  if (p.state_bf16) {
    switch (p.Ns) {
      case 16: return decode_as<__nv_bfloat16, 2, 1, 2>(p, stream);
      case 32: return decode_as<__nv_bfloat16, 4, 1, 4>(p, stream);
      case 64: return decode_as<__nv_bfloat16, 8, 1, 4>(p, stream);
      case 128: return decode_as<__nv_bfloat16, 16, 1, 4>(p, stream);
      case 256: return decode_as<__nv_bfloat16, 32, 1, 4>(p, stream);
    }
    return GDN_ERR_UNSUPPORTED_SHAPE;
  }
  switch (p.Ns) {
    case 16: return decode_as<float, 4, 1, 4>(p, stream);
    case 32: return decode_as<float, 8, 1, 8>(p, stream);
    case 64: return decode_as<float, 16, 1, 8>(p, stream);
    case 128: return decode_as<float, 32, 1, 8>(p, stream);
    case 256: return decode_as<float, 32, 2, 4>(p, stream);
  }
  return GDN_ERR_UNSUPPORTED_SHAPE;
}

int launch_ssm_recurrent(const SsmParams& p, cudaStream_t stream) {
  switch (p.Ns) {
    case 16: return recurrent_as<4, 1, 2>(p, stream);
    case 32: return recurrent_as<8, 1, 2>(p, stream);
    case 64: return recurrent_as<16, 1, 4>(p, stream);
    case 128: return recurrent_as<32, 1, 4>(p, stream);
    case 256: return recurrent_as<32, 2, 4>(p, stream);
  }
  return GDN_ERR_UNSUPPORTED_SHAPE;
}

}  // namespace gdn
