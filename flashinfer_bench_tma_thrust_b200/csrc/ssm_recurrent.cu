// ssm_recurrent.cu — the selective state space scan as a recurrence: one new token per
// sequence (a stream of the state through the SMs), and packed prompts token by token.
//
// Per sequence and head h (group h / (H / G) gives B and C), with S [P, Ns] and rows p:
//     d = softplus(dt + dt_bias), g = exp(-exp(A_log) d)          (GDN's gate, fp32)
//     S'[p, :] = g S[p, :] + (d x_p) B,   y_p = S'[p, :] . C + D x_p
// A row needs only its x_p once g, d and B.C are known:
//     y_p = g (S[p, :] . C) + d x_p (B . C) + D x_p
// so one dot product per row, on the row as it was loaded.
#include <type_traits>

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
  static __device__ __forceinline__ void unpack(const uint4& u, float2 (&v)[2]) {
    v[0] = make_float2(__uint_as_float(u.x), __uint_as_float(u.y));
    v[1] = make_float2(__uint_as_float(u.z), __uint_as_float(u.w));
  }
  static __device__ __forceinline__ uint4 pack(const float2 (&v)[2]) {
    return make_uint4(__float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[1].x),
                      __float_as_uint(v[1].y));
  }
};
template <>
struct Piece<__nv_bfloat16> {
  static constexpr int kE = 8;
  static __device__ __forceinline__ void unpack(const uint4& w, float2 (&v)[4]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int k = 0; k < 4; ++k)
      v[k] = make_float2(__uint_as_float(u[k] << 16), __uint_as_float(u[k] & 0xffff0000u));
  }
  static __device__ __forceinline__ uint4 pack(const float2 (&v)[4]) {
    uint32_t u[4];  // the state's own type: one rounding per step, the user's choice of it
#pragma unroll
    for (int k = 0; k < 4; ++k)
      asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(u[k]) : "f"(v[k].y), "f"(v[k].x));
    return make_uint4(u[0], u[1], u[2], u[3]);
  }
};
// Streaming access to the state: each element is touched once per launch.
template <typename S>
__device__ __forceinline__ uint4 load_piece(const void* base, int64_t i) {
  uint4 u;
  asm volatile("ld.global.cs.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w)
               : "l"(static_cast<const S*>(base) + i));
  return u;
}
template <typename S>
__device__ __forceinline__ void store_piece(void* base, int64_t i, const uint4& u) {
  asm volatile("st.global.cs.v4.u32 [%0], {%1,%2,%3,%4};" ::"l"(static_cast<S*>(base) + i),
               "r"(u.x), "r"(u.y), "r"(u.z), "r"(u.w)
               : "memory");
}

// kE consecutive bf16 values (kE = 4 or 8, aligned to their size) as pairs of floats.
template <int kE>
__device__ __forceinline__ void load_bf16(const __nv_bfloat16* p, float2 (&v)[kE / 2]) {
#pragma unroll
  for (int k = 0; k < kE; k += 4) {
    const float4 f = load_bf16x4(p + k);
    v[k / 2] = make_float2(f.x, f.y);
    v[k / 2 + 1] = make_float2(f.z, f.w);
  }
}

template <int kLanes>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Sums of kRows rows over their kLanes lanes; lane l of a row's lanes is left with that of row
// l / (kLanes / kRows). Each exchange halves the rows that a lane still sums: for 4 rows of 16
// lanes 5 shuffles, not 16.
template <int kLanes, int kRows>
__device__ __forceinline__ float row_sums(float (&v)[kRows]) {
  static_assert(kRows <= kLanes, "");
  int o = kLanes / 2;
#pragma unroll
  for (int rows = kRows / 2; rows > 0; rows /= 2, o /= 2) {
    const bool hi = threadIdx.x & o;
#pragma unroll
    for (int i = 0; i < rows; ++i) {
      const float send = hi ? v[i] : v[i + rows], keep = hi ? v[i + rows] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
    }
  }
  float sum = v[0];
#pragma unroll
  for (; o > 0; o /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return sum;
}

__device__ __forceinline__ float bf16_at(const __nv_bfloat16* p) {
  return __uint_as_float(static_cast<uint32_t>(*reinterpret_cast<const unsigned short*>(p)) << 16);
}

// ---------------------------------------------------------------- one token per sequence
// HBM bounds it: the state goes through once (5 flop per 8 bytes): 256 sequences of 32 heads of
// 128 x 128 in fp32 take 162 us in short runs, 6.7 TB/s, and 177 where the power limit holds the
// clocks down; 300 of 80 heads of 64 x 128 in bf16, with twice the rows per byte, 136 us, 5.8 TB/s,
// and 143, near the issue limit. A warp takes batches of
// kRows * kPer rows, of which each lane holds x and y of one; a batch's loads are all in
// flight, and the next batch's too, before it is used. Blocks of 4 warps share a head's rows.
template <typename S, int kLanes, int kPieces, int kRows, bool kLoop>
__global__ void __launch_bounds__(128) ssm_decode_kernel(const __grid_constant__ SsmParams p,
                                                        int splits, int batches) {
  constexpr int kE = Piece<S>::kE, kH = kE / 2;
  constexpr int kPer = 32 / kLanes;  // rows per load
  constexpr int kBatch = kRows * kPer;
  constexpr int kShare = kLanes / kRows;  // lanes that end up with the same row's y
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int l = lane % kLanes, sub = lane / kLanes;
  const int64_t head = blockIdx.x / splits;  // flattened (sequence, head)
  const int split = static_cast<int>(blockIdx.x - head * splits);
  const int64_t n = head / p.H;
  const int h = static_cast<int>(head - n * p.H);
  const int64_t grp = n * p.G + h / (p.H / p.G);
  const int first = (split * 4 + warp) * batches * kBatch;
  const int end = min(first + batches * kBatch, p.P);
  if (first >= end) return;

  // without kLoop (one batch) `next` is the batch itself
  uint4 next[kRows][kPieces];
  auto load = [&](int row0) {
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int r = row0 + i * kPer + sub;
#pragma unroll
      for (int j = 0; j < kPieces; ++j)
        next[i][j] = p.state && r < end
                         ? load_piece<S>(p.state, (head * p.P + r) * p.Ns + (j * kLanes + l) * kE)
                         : make_uint4(0u, 0u, 0u, 0u);
    }
  };
  load(first);
  const float v = load_scalar(p.dt, p.dt_dtype, head) + load_scalar(p.dt_bias, p.dt_bias_dtype, h);
  const float a_log = load_scalar(p.A_log, p.A_log_dtype, h);
  const float skip = p.D ? load_scalar(p.D, p.D_dtype, h) : 0.f;
  float2 b[kPieces][kH], c[kPieces][kH];
#pragma unroll
  for (int j = 0; j < kPieces; ++j) {
    const int64_t at = grp * p.Ns + (j * kLanes + l) * kE;
    load_bf16<kE>(p.B + at, b[j]);
    load_bf16<kE>(p.C + at, c[j]);
  }
  const float d = softplus_ref(v);
  const float g = expf(-expf(a_log) * d);
  float bc = 0.f;
#pragma unroll
  for (int j = 0; j < kPieces; ++j) {
#pragma unroll
    for (int k = 0; k < kH; ++k) bc = fmaf(b[j][k].x, c[j][k].x, fmaf(b[j][k].y, c[j][k].y, bc));
  }
  bc = row_sum<kLanes>(bc);
  const float2 g2 = make_float2(g, g);

#pragma unroll 1
  for (int row0 = first; row0 < end; row0 += kBatch) {
    uint4 s[kRows][kPieces];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
#pragma unroll
      for (int j = 0; j < kPieces; ++j) s[i][j] = next[i][j];
    }
    if (kLoop && row0 + kBatch < end) load(row0 + kBatch);
    const int mine = row0 + l / kShare * kPer + sub;
    const float x_mine = mine < end ? bf16_at(p.x + head * p.P + mine) : 0.f;
    const float dx_mine = d * x_mine;
    float dots[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int r = row0 + i * kPer + sub;
      const float dx = __shfl_sync(0xffffffffu, dx_mine, i * kShare, kLanes);
      const float2 dx2 = make_float2(dx, dx);
      float2 dot = make_float2(0.f, 0.f);
#pragma unroll
      for (int j = 0; j < kPieces; ++j) {
        float2 w[kH];
        Piece<S>::unpack(s[i][j], w);
#pragma unroll
        for (int k = 0; k < kH; ++k) {
          dot = __ffma2_rn(w[k], c[j][k], dot);
          w[k] = __ffma2_rn(g2, w[k], __fmul2_rn(dx2, b[j][k]));
        }
        if (r < end)
          store_piece<S>(p.new_state, (head * p.P + r) * p.Ns + (j * kLanes + l) * kE,
                         Piece<S>::pack(w));
      }
      dots[i] = dot.x + dot.y;
    }
    const float y = fmaf(g, row_sums<kLanes>(dots), dx_mine * bc);
    if (l % kShare == 0 && mine < end)
      p.out[head * p.P + mine] = __float2bfloat16_rn(fmaf(skip, x_mine, y));
    if (!kLoop) break;
  }
}

// ---------------------------------------------------------------- prompts, token by token
// A warp keeps kRows * kPer rows of one head's state in registers over the whole sequence;
// the inputs of kStep tokens are loaded together. Any P, and the state sizes that the
// chunked kernel does not take; the independent check of that kernel elsewhere. Bound by the
// chain of a token's loads, products and reductions, 2 us for four tokens: 64 sequences of 4
// tokens of 32 heads of 128 x 128 113 us, of which the states' way in and out is 85.
constexpr int kStep = 4;

template <int kLanes, int kPieces, int kRows>
__global__ void __launch_bounds__(128) ssm_recurrent_kernel(const __grid_constant__ SsmParams p,
                                                           int tiles) {
  constexpr int kE = 4, kH = 2;
  constexpr int kPer = 32 / kLanes;
  constexpr int kWarpRows = kRows * kPer;
  constexpr int kShare = kLanes / kRows;  // lanes that end up with the same row's y
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

  float2 s[kRows][kPieces][kH];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int r = row0 + i * kPer + sub;
#pragma unroll
    for (int j = 0; j < kPieces; ++j)
      Piece<float>::unpack(
          p.state && r < p.P
              ? load_piece<float>(p.state, (head * p.P + r) * p.Ns + (j * kLanes + l) * kE)
              : make_uint4(0u, 0u, 0u, 0u),
          s[i][j]);
  }
  const float neg_a = -expf(load_scalar(p.A_log, p.A_log_dtype, h));
  const float dtb = load_scalar(p.dt_bias, p.dt_bias_dtype, h);
  const float skip = p.D ? load_scalar(p.D, p.D_dtype, h) : 0.f;

  for (int64_t t0 = start; t0 < end; t0 += kStep) {
    float2 b[kStep][kPieces][kH], c[kStep][kPieces][kH];
    float x[kStep][kRows], d[kStep], g[kStep];
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
      float dots[kRows];
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const float dx = d[a] * x[a][i];
        const float2 dx2 = make_float2(dx, dx), g2 = make_float2(g[a], g[a]);
        float2 dot2 = make_float2(0.f, 0.f);
#pragma unroll
        for (int j = 0; j < kPieces; ++j) {
#pragma unroll
          for (int k = 0; k < kH; ++k) {
            s[i][j][k] = __ffma2_rn(g2, s[i][j][k], __fmul2_rn(dx2, b[a][j][k]));
            dot2 = __ffma2_rn(s[i][j][k], c[a][j][k], dot2);
          }
        }
        dots[i] = dot2.x + dot2.y;
        if (l == 0) dots[i] = fmaf(skip, x[a][i], dots[i]);
      }
      const float y = row_sums<kLanes>(dots);
      const int r = row0 + l / kShare * kPer + sub;
      if (l % kShare == 0 && r < p.P)
        p.out[((t0 + a) * p.H + h) * p.P + r] = __float2bfloat16_rn(y);
    }
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int r = row0 + i * kPer + sub;
    if (r >= p.P) continue;
#pragma unroll
    for (int j = 0; j < kPieces; ++j)
      store_piece<float>(p.new_state, (head * p.P + r) * p.Ns + (j * kLanes + l) * kE,
                         Piece<float>::pack(s[i][j]));
  }
}

template <typename S, int kLanes, int kPieces, int kRows>
int decode_as(const SsmParams& p, cudaStream_t stream) {
  // Batches per warp at most, where the grid stays full. A warp's gates and its B and C cost as
  // much as a batch of bf16 rows (300 x 80 heads of 64 x 128: 1 batch 148 us, 4 batches 134); with
  // fp32 rows HBM has the next block's loads to do meanwhile (256 x 32 heads of 128 x 128: 161 us
  // with 1 batch, 168 with 2).
  constexpr bool kLoops = std::is_same_v<S, __nv_bfloat16>;
  constexpr int kMostBatches = kLoops ? 4 : 1;
  constexpr int kBlockRows = 4 * kRows * (32 / kLanes);
  const int64_t heads = p.N * p.H;
  const int whole = (p.P + kBlockRows - 1) / kBlockRows;  // batches of a whole head
  int batches = 1;
  while (batches < kMostBatches && batches < whole && heads * (whole / (2 * batches)) >= 148 * 16)
    batches *= 2;
  const int splits = (whole + batches - 1) / batches;
  if (heads * splits > 0x7fffffffLL) return GDN_ERR_UNSUPPORTED_SHAPE;
  const unsigned grid = static_cast<unsigned>(heads * splits);
  if (kLoops && batches > 1) {
    ssm_decode_kernel<S, kLanes, kPieces, kRows, kLoops>
        <<<grid, 128, 0, stream>>>(p, splits, batches);
  } else {
    ssm_decode_kernel<S, kLanes, kPieces, kRows, false><<<grid, 128, 0, stream>>>(p, splits, 1);
  }
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
    case 128: return decode_as<float, 32, 1, 4>(p, stream);
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
