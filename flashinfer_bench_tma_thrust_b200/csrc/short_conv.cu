// short_conv.cu — short causal depthwise convolution over packed prompts and for one new
// token per sequence, with silu, split outputs and the L2 norm of 128-channel heads fused
// into the store.
//
// With W taps (2 to 4) and u the inputs of a sequence, its W-1 earlier rows (the state, or
// zeros) in front:
//     c_t[ch] = bias[ch] + sum_k weight[ch][k] u_{t-W+1+k}[ch],   y = silu(c)
// and in a normed section every head of 128 channels is divided by sqrt(sum y^2 + eps).
// 2 W flop stand against 4 bytes of traffic per element, so HBM bounds it: each input is
// read once, a run of tokens per thread keeps the last W-1 rows in registers, and the
// outputs leave in vector stores, each section to its own dense tensor (what the operators
// behind it take) with no pass of its own for split, silu or norm.
//
// A thread owns 8 adjacent channels (16 bytes of a row), so a head is 16 lanes. For prompts its
// rows arrive by asynchronous copies in a ring of its own in shared memory, 12 to 16 rows ahead:
// with rows in flight in registers (4 per thread, 16 warps per SM) HBM's latency was not
// covered. No thread waits for another. Sums are fp32; silu takes ex2.approx and a shared
// approximate reciprocal (relative error below 2^-16, at the exponents of v = -92; the bf16
// rounding of the output is the only other one). 65536 x 6144 take 259 to 271 us in short runs
// (6.2 to 5.9 TB/s) and 299 where the power limit holds the clocks down; 19679 x 8192, half of the
// channels normed, 131 and 138 us: besides HBM (55 % busy) the instructions per row (130 for 8
// channels, 59 % of the issue slots) come near a bound then.
#include <cfloat>
#include <cmath>

#include "gdn_b200.h"
#include "gdn_common.cuh"
#include "ssm_launch.h"

namespace gdn {
namespace {

constexpr int kVec = 8;         // channels per thread
constexpr int kThreads = 128;   // 1024 channels per block
constexpr int kP = kVec / 2;    // pairs of channels
constexpr float kLog2e = 1.4426950408889634f;

// Eight channels of one row as stored.
struct Row {
  uint4 w;
};

__device__ __forceinline__ float2 pair(uint32_t u) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
__device__ __forceinline__ void pairs(const Row& r, float2 (&v)[kP]) {
  v[0] = pair(r.w.x);
  v[1] = pair(r.w.y);
  v[2] = pair(r.w.z);
  v[3] = pair(r.w.w);
}

// Channels [c, c + 8) of a row; with kWide one 16-byte access (the launcher has checked
// alignment and that 8 divides every section), else one access per channel below C.
template <bool kWide>
__device__ __forceinline__ Row load_row(const __nv_bfloat16* row, int c, int C) {
  if (kWide) return Row{*reinterpret_cast<const uint4*>(row + c)};
  const unsigned short* p = reinterpret_cast<const unsigned short*>(row);
  uint32_t u[kP];
#pragma unroll
  for (int i = 0; i < kP; ++i) {
    const uint32_t lo = c + 2 * i < C ? p[c + 2 * i] : 0u;
    const uint32_t hi = c + 2 * i + 1 < C ? p[c + 2 * i + 1] : 0u;
    u[i] = lo | (hi << 16);
  }
  return Row{make_uint4(u[0], u[1], u[2], u[3])};
}

template <bool kWide>
__device__ __forceinline__ void store_row(__nv_bfloat16* row, int c, int C, const Row& r) {
  if (kWide) {
    *reinterpret_cast<uint4*>(row + c) = r.w;
    return;
  }
  unsigned short* p = reinterpret_cast<unsigned short*>(row);
  const uint32_t u[kP] = {r.w.x, r.w.y, r.w.z, r.w.w};
#pragma unroll
  for (int i = 0; i < kVec; ++i)
    if (c + i < C) p[c + i] = static_cast<unsigned short>(u[i >> 1] >> ((i & 1) * 16));
}

// What a thread knows of its channels, in pairs.
template <int W>
struct Taps {
  float2 w[W][kP];
  float2 bias[kP];
};

// kN consecutive fp32 or bf16 parameters from element i on (16-byte aligned) as floats.
template <int kN>
__device__ __forceinline__ void load_params(const void* base, int dtype, int64_t i,
                                            float (&v)[kN]) {
  if (dtype == kBF16) {
    const uint4* p = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(base) + i);
#pragma unroll
    for (int k = 0; k < kN / 8; ++k) {
      float2 f[kP];
      pairs(Row{p[k]}, f);
#pragma unroll
      for (int e = 0; e < kP; ++e) {
        v[8 * k + 2 * e] = f[e].x;
        v[8 * k + 2 * e + 1] = f[e].y;
      }
    }
  } else {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(base) + i);
#pragma unroll
    for (int k = 0; k < kN / 4; ++k) {
      const float4 f = p[k];
      v[4 * k] = f.x;
      v[4 * k + 1] = f.y;
      v[4 * k + 2] = f.z;
      v[4 * k + 3] = f.w;
    }
  }
}

template <int W, bool kWide>
__device__ __forceinline__ Taps<W> load_taps(const ConvParams& p, int c) {
  float w[kVec * W], b[kVec];
#pragma unroll
  for (int i = 0; i < kVec; ++i) b[i] = 0.f;
  if (kWide) {
    load_params(p.weight, p.weight_dtype, static_cast<int64_t>(c) * W, w);
    if (p.bias) load_params(p.bias, p.bias_dtype, c, b);
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const bool in = c + i < p.C;
      if (in && p.bias) b[i] = load_scalar(p.bias, p.bias_dtype, c + i);
#pragma unroll
      for (int k = 0; k < W; ++k)
        w[i * W + k] =
            in ? load_scalar(p.weight, p.weight_dtype, static_cast<int64_t>(c + i) * W + k) : 0.f;
    }
  }
  Taps<W> t;
#pragma unroll
  for (int i = 0; i < kP; ++i) {
    t.bias[i] = make_float2(b[2 * i], b[2 * i + 1]);
#pragma unroll
    for (int k = 0; k < W; ++k) t.w[k][i] = make_float2(w[2 * i * W + k], w[(2 * i + 1) * W + k]);
  }
  return t;
}

// Where a thread's channels go: its section (kWide: all 8 channels lie in one).
struct Place {
  __nv_bfloat16* out;
  int64_t width;
  int at, normed;
};
__device__ __forceinline__ Place place_of(const ConvParams& p, int c) {
  int s = 0;
#pragma unroll 1
  while (s + 1 < p.sections && c >= p.begin[s + 1]) ++s;
  return Place{p.out[s], p.begin[s + 1] - p.begin[s], c - p.begin[s], p.normed[s]};
}

// silu, v / (1 + e^-v), of two values with three MUFU operations instead of four: one reciprocal
// of the product of the denominators, which fp32 holds for v from kFar up. A NaN is kept by the
// factor v but not by the exponent, which both values share.
constexpr float kFar = -43.5f;
__device__ __forceinline__ float2 silu2(float2 v) {
  const float2 z = __fmul2_rn(v, make_float2(-kLog2e, -kLog2e));
  float2 e;
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(fminf(z.x, 63.f)));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(fminf(z.y, 63.f)));
  const float2 a = __fadd2_rn(e, make_float2(1.f, 1.f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(a.x * a.y));
  return __fmul2_rn(v, __fmul2_rn(make_float2(a.y, a.x), make_float2(r, r)));
}
// What silu2 makes silu(v) of where v is below kFar. There silu(v) is v e^v to the last bit, and
// silu2 halves a value as small as 2 v e^v. Two factors, since e^v leaves the normal numbers (at
// -87) before v e^v does (at -92). -infinity gives zero.
__device__ __forceinline__ float from_far(float v) {
  v = fmaxf(v, -120.f);  // (zero from -108 down)
  float h;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(h) : "f"(v * (0.5f * kLog2e)));
  return (v + v) * h * h;
}
// silu of rows of eight values. Values below kFar are rare: a minimum over all rows finds them.
// (With a branch per row the rows' instructions do not mix: 12 % more time. The minimum costs
// 0.6 %, and the pass over such values up to a quarter where most rows have one.)
template <int kTok>
__device__ __forceinline__ void silu_rows(float2 (&y)[kTok][kP]) {
  float low = 0.f;
#pragma unroll
  for (int t = 0; t < kTok; ++t) {
#pragma unroll
    for (int i = 0; i < kP; ++i) low = fminf(low, fminf(y[t][i].x, y[t][i].y));
  }
  if (low < kFar) {
#pragma unroll
    for (int t = 0; t < kTok; ++t) {
#pragma unroll
      for (int i = 0; i < kP; ++i) {
        if (y[t][i].x < kFar) y[t][i].x = from_far(y[t][i].x);
        if (y[t][i].y < kFar) y[t][i].y = from_far(y[t][i].y);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < kTok; ++t) {
#pragma unroll
    for (int i = 0; i < kP; ++i) y[t][i] = silu2(y[t][i]);
  }
}

// The W-1 rows before the current one, as floats.
template <int W>
struct Window {
  float2 v[W - 1][kP];
  __device__ __forceinline__ void set(int r, const Row& row) {
    pairs(row, v[r]);
  }
};

// Sums of kTok values per lane over 16 lanes, each in every lane. Two values: an exchange that
// leaves one value per lane, three more steps on it, and two broadcasts, 6 shuffles for 8. The
// order of the sums is the same for one value: bits do not depend on how tokens fall into rows.
template <int kTok>
__device__ __forceinline__ void head_sums(float (&q)[kTok]) {
  const uint32_t lanes = 0xffffu << (threadIdx.x & 16);
  if constexpr (kTok == 2) {
    const bool hi = threadIdx.x & 1;
    float s = (hi ? q[1] : q[0]) + __shfl_xor_sync(lanes, hi ? q[0] : q[1], 1);
#pragma unroll
    for (int o = 2; o < 16; o <<= 1) s += __shfl_xor_sync(lanes, s, o);
    q[0] = __shfl_sync(lanes, s, 0, 16);
    q[1] = __shfl_sync(lanes, s, 1, 16);
  } else {
#pragma unroll
    for (int t = 0; t < kTok; ++t) {
#pragma unroll
      for (int o = 1; o < 16; o <<= 1) q[t] += __shfl_xor_sync(lanes, q[t], o);
    }
  }
}

// A thread's part of its head's sum of squares.
__device__ __forceinline__ float square_sum(const float2 (&y)[kP]) {
  float2 q = __fmul2_rn(y[0], y[0]);
#pragma unroll
  for (int i = 1; i < kP; ++i) q = __ffma2_rn(y[i], y[i], q);
  return q.x + q.y;
}

// The norm of a head whose sum of squares (with eps) is not between kLeastSum and FLT_MAX: squares
// that fp32 cannot hold are missing in it or have made it infinite. The head, and eps with it, is
// scaled by a power of two that brings its largest value (or the root of eps) next to one, and is
// left so; returns what it is then multiplied by. Zeros without eps (0 / 0), infinities and NaN:
// as they were.
constexpr float kLeastSum = 0x1p-80f;  // a square below 2^-126 is nothing to it
__device__ __forceinline__ float norm_far(float2 (&y)[kP], float eps, float r) {
  const uint32_t lanes = 0xffffu << (threadIdx.x & 16);
  float m = sqrtf(eps);
#pragma unroll
  for (int i = 0; i < kP; ++i) m = fmaxf(m, fmaxf(fabsf(y[i].x), fabsf(y[i].y)));
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) m = fmaxf(m, __shfl_xor_sync(lanes, m, o));
  if (m == 0.f || m > FLT_MAX) return r;
  const float s = __uint_as_float((254u - min(__float_as_uint(m) >> 23, 253u)) << 23);
#pragma unroll
  for (int i = 0; i < kP; ++i) y[i] = __fmul2_rn(y[i], make_float2(s, s));
  float q[1] = {square_sum(y)};
  head_sums(q);
  return rsqrtf(fmaf(eps * s, s, q[0]));
}

// kTok output rows from row `at` on (kWide: at `out`): the taps over the window and `rows`
// (which enter the window one by one), activation, norm of the head (16 lanes), store. All lanes
// of the warp call it; `live` says whether this thread's channels exist. Without kCareful a
// head whose sum of squares is out of range sets `far`, and its row is not right. (Branches to
// norm_far between the rows cost 3 % of the time, registers included; such heads are freaks.)
template <int W, bool kWide, bool kCareful, int kTok>
__device__ __forceinline__ void output_rows(const ConvParams& p, const Taps<W>& taps,
                                            const Place& pl, int c, int64_t at,
                                            __nv_bfloat16* out, Window<W>& win,
                                            const Row (&rows)[kTok], bool live, bool& far) {
  float2 y[kTok][kP];
#pragma unroll
  for (int t = 0; t < kTok; ++t) {
    float2 in[kP];
    pairs(rows[t], in);
#pragma unroll
    for (int i = 0; i < kP; ++i) {
      const float2 cur = in[i];
      float2 s = taps.bias[i];
#pragma unroll
      for (int k = 0; k < W - 1; ++k) s = __ffma2_rn(taps.w[k][i], win.v[k][i], s);
      y[t][i] = __ffma2_rn(taps.w[W - 1][i], cur, s);
#pragma unroll
      for (int k = 0; k + 1 < W - 1; ++k) win.v[k][i] = win.v[k + 1][i];
      win.v[W - 2][i] = cur;
    }
  }
  if (p.silu) silu_rows(y);
  if (pl.normed) {  // the same for the 16 lanes of a head
    float q[kTok];
#pragma unroll
    for (int t = 0; t < kTok; ++t) q[t] = square_sum(y[t]);
    head_sums(q);
#pragma unroll
    for (int t = 0; t < kTok; ++t) {
      const float sum = q[t] + p.eps;
      float r = rsqrtf(sum);
      if (!(sum >= kLeastSum && sum <= FLT_MAX)) {
        if (kCareful) {
          r = norm_far(y[t], p.eps, r);
        } else {
          far = true;
        }
      }
#pragma unroll
      for (int i = 0; i < kP; ++i) y[t][i] = __fmul2_rn(y[t][i], make_float2(r, r));
    }
  }
  if (!live) return;
#pragma unroll
  for (int t = 0; t < kTok; ++t) {
    uint32_t u[kP];
#pragma unroll
    for (int i = 0; i < kP; ++i)
      asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(u[i]) : "f"(y[t][i].y), "f"(y[t][i].x));
    if (kWide) {
      *reinterpret_cast<uint4*>(out) = make_uint4(u[0], u[1], u[2], u[3]);
      out += pl.width;
    } else {
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        if (c + i >= p.C) break;
        const Place q = place_of(p, c + i);
        reinterpret_cast<unsigned short*>(q.out)[(at + t) * q.width + q.at] =
            static_cast<unsigned short>(u[i >> 1] >> ((i & 1) * 16));
      }
    }
  }
}

// How many i in [1, N] have cu[i] <= t: the sequence that token t lies in (N: none). A
// 32-way search by the whole warp: one round for up to 32 sequences, two up to 1024.
__device__ __forceinline__ int64_t find_sequence(const void* cu, int dtype, int64_t N, int64_t t) {
  const int lane = threadIdx.x & 31;
  int64_t lo = 0, hi = N;
  while (hi > lo) {
    const int64_t step = (hi - lo + 31) / 32;
    const int64_t i = lo + (lane + 1) * step - 1;
    const bool le = i < hi && load_index(cu, dtype, i + 1) <= t;
    lo += __popc(__ballot_sync(0xffffffffu, le)) * step;
    hi = min(hi, lo + step - 1);
  }
  return lo;
}

__device__ __forceinline__ int64_t bound(const ConvParams& p, int64_t i) {
  const int64_t v = load_index(p.cu_seqlens, p.cu_dtype, i);
  return v < 0 ? 0 : (v > p.T ? p.T : v);
}

// Prompts. Blocks [0, tiles) of grid.y take `run` tokens each; the N behind them write one
// sequence's new state (its last W-1 inputs, from the state where it is shorter).
constexpr int kAhead = 4, kSlots = 4;  // rows per batch, batches in the ring

__device__ __forceinline__ void copy16_async(uint4* to, const __nv_bfloat16* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                   static_cast<uint32_t>(__cvta_generic_to_shared(to))),
               "l"(from)
               : "memory");
}

// A thread's way through the tokens of a tile, over the sequences' bounds.
template <int W, bool kWide>
struct Walk {
  const ConvParams& p;
  const int c;
  int64_t n, start, end;  // the sequence; none left (n = N): nothing is written
  Window<W> win;
  __device__ __forceinline__ Walk(const ConvParams& p_, int c_) : p(p_), c(c_) {}
  __device__ __forceinline__ void bounds() {
    start = end = p.T;
    if (n < p.N) {
      start = bound(p, n);
      end = bound(p, n + 1);
    }
  }
  __device__ __forceinline__ void begin(int64_t t0) {  // by the whole warp
    n = find_sequence(p.cu_seqlens, p.cu_dtype, p.N, t0);
    bounds();
#pragma unroll
    for (int r = 0; r < W - 1; ++r) win.set(r, Row{make_uint4(0u, 0u, 0u, 0u)});
    if (n < p.N && start < t0) {  // the tile begins inside a sequence
#pragma unroll
      for (int r = 0; r < W - 1; ++r) {
        const int64_t u = t0 - (W - 1) + r;
        if (u >= start) {
          win.set(r, load_row<kWide>(p.x + u * p.x_stride, c, p.C));
        } else if (p.state) {
          win.set(r,
                  load_row<kWide>(p.state + (n * (W - 1) + (u - start) + (W - 1)) * p.C, c, p.C));
        }
      }
    }
  }
  // Whether token t, the one behind the last that was asked for, lies in a sequence; the window is
  // then that of t.
  __device__ __forceinline__ bool next(int64_t t) {
    while (t >= end && n < p.N) {  // into the next sequence that has tokens
      ++n;
      bounds();
    }
    if (n >= p.N || t < start) return false;
    if (t == start) {
#pragma unroll
      for (int r = 0; r < W - 1; ++r)
        win.set(r, p.state ? load_row<kWide>(p.state + (n * (W - 1) + r) * p.C, c, p.C)
                           : Row{make_uint4(0u, 0u, 0u, 0u)});
    }
    return true;
  }
};

// A tile's tokens with care, by the whole warp (the norms need whole heads). A function of its own:
// in line it cost the first pass registers, and with them 9 %.
template <int W, bool kWide>
__device__ __noinline__ void tile_again(const ConvParams& p, int c, int64_t t0, int64_t t1) {
  const bool live = c < p.C;
  const int cl = live ? c : 0;
  const Taps<W> taps = load_taps<W, kWide>(p, cl);
  Place pl = place_of(p, cl);
  if (!live) pl.normed = 0;
  Walk<W, kWide> walk(p, cl);
  walk.begin(t0);
  bool far = false;
#pragma unroll 1
  for (int64_t t = t0; t < t1; ++t) {
    if (!walk.next(t)) continue;
    const Row row[1] = {load_row<kWide>(p.x + t * p.x_stride, cl, p.C)};
    output_rows<W, kWide, true, 1>(p, taps, pl, cl, t, pl.out + t * pl.width + pl.at, walk.win, row,
                                   live, far);
  }
}

template <int W, bool kWide>
__global__ void __launch_bounds__(kThreads, W == 2 ? 5 : 4)  // blocks per SM, as without tile_again
conv_prefill_kernel(const __grid_constant__ ConvParams p, int64_t tiles, int run) {
  const int c = (blockIdx.x * kThreads + threadIdx.x) * kVec;
  const bool live = c < p.C;
  const int64_t by = blockIdx.y + static_cast<int64_t>(blockIdx.z) * gridDim.y;
  if (by >= tiles + p.N) return;
  if (by >= tiles) {
    const int64_t n = by - tiles;
    const int64_t start = bound(p, n), end = bound(p, n + 1);
    const int64_t len = end > start ? end - start : 0;
    if (c == 0) {
      const int64_t lo = load_index(p.cu_seqlens, p.cu_dtype, n);
      const int64_t hi = load_index(p.cu_seqlens, p.cu_dtype, n + 1);
      if (lo < 0 || hi > p.T || hi < lo) report_bad_bounds(p.status);
    }
    if (!live) return;
#pragma unroll
    for (int r = 0; r < W - 1; ++r) {
      Row v{make_uint4(0u, 0u, 0u, 0u)};
      const int64_t at = len + r;  // row of [state; inputs]
      if (at >= W - 1) {
        v = load_row<kWide>(p.x + (start + at - (W - 1)) * p.x_stride, c, p.C);
      } else if (p.state) {
        v = load_row<kWide>(p.state + (n * (W - 1) + at) * p.C, c, p.C);
      }
      store_row<kWide>(p.new_state + (n * (W - 1) + r) * p.C, c, p.C, v);
    }
    return;
  }
  const int64_t t0 = by * run;
  const int64_t t1 = min(t0 + run, p.T);
  const int cl = live ? c : 0;
  // The ring: batch b of kAhead rows in slot b % kSlots, at this thread's own place. Asked for
  // before anything else: x needs no bounds.
  __shared__ uint4 ring[kSlots][kAhead][kThreads];
  const int batches = static_cast<int>((t1 - t0 + kAhead - 1) / kAhead);
  const __nv_bfloat16* from = p.x + t0 * p.x_stride + cl;
  auto fetch = [&](int b) {
    if (kWide && b < batches) {
      uint4* const to = &ring[b % kSlots][0][threadIdx.x];
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        if (t0 + b * kAhead + a < t1) copy16_async(to + a * kThreads, from);
        from += p.x_stride;
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  auto fetched = [&](int b, int a) {
    return kWide ? Row{ring[b % kSlots][a][threadIdx.x]}
                 : load_row<kWide>(p.x + (t0 + b * kAhead + a) * p.x_stride, cl, p.C);
  };
#pragma unroll 1
  for (int b = 0; b < kSlots - 1; ++b) fetch(b);
  const Taps<W> taps = load_taps<W, kWide>(p, cl);
  Place pl = place_of(p, cl);
  if (!live) pl.normed = 0;  // (a normed section is whole warps)
  Walk<W, kWide> walk(p, cl);
  walk.begin(t0);
  bool far = false;
  __nv_bfloat16* to = pl.out + t0 * pl.width + pl.at;  // kWide: the batch's first output row
#pragma unroll 1
  for (int b = 0; b < batches; ++b, to += kAhead * pl.width) {
    const int64_t tb = t0 + b * kAhead;
    fetch(b + kSlots - 1);  // its slot's rows are in registers or behind
    asm volatile("cp.async.wait_group %0;" ::"n"(kSlots - 1) : "memory");
    if (walk.n < p.N && walk.start < tb && tb + kAhead <= min(walk.end, t1)) {
      // all of the batch and the rows before it lie in one sequence
#pragma unroll
      for (int a = 0; a < kAhead; a += 2) {  // two rows at a time: more take too many registers
        const Row rows[2] = {fetched(b, a), fetched(b, a + 1)};
        output_rows<W, kWide, false, 2>(p, taps, pl, cl, tb + a, to + a * pl.width, walk.win, rows,
                                        live, far);
      }
      continue;
    }
#pragma unroll 1
    for (int a = 0; a < kAhead; ++a) {
      const int64_t t = tb + a;
      if (t >= t1) break;
      if (!walk.next(t)) continue;
      const Row row[1] = {fetched(b, a)};
      output_rows<W, kWide, false, 1>(p, taps, pl, cl, t, to + a * pl.width, walk.win, row, live,
                                      far);
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  if (__any_sync(0xffffffffu, far)) tile_again<W, kWide>(p, c, t0, t1);
}

// One token per sequence, bound by HBM (1024 sequences of 8192 channels with 4 taps 26.7 us, in
// short and long runs, 5.0 TB/s with the launch): each thread reads its 8 channels of the W-1
// state rows and of x, and writes the rows moved up by one, so the new state may be the old one's
// memory.
template <int W>
constexpr int kDecodeBlocks = W == 4 ? 4 : (W == 3 ? 5 : 7);  // per SM, by the registers

template <int W, bool kWide>
__global__ void __launch_bounds__(kThreads, kDecodeBlocks<W>)
conv_decode_kernel(const __grid_constant__ ConvParams p, int per_thread) {
  const int c = (blockIdx.x * kThreads + threadIdx.x) * kVec;
  const bool live = c < p.C;
  const int64_t by = blockIdx.y + static_cast<int64_t>(blockIdx.z) * gridDim.y;
  const int64_t n0 = by * per_thread, n1 = min(n0 + per_thread, p.N);
  if (n0 >= p.N) return;
  const int cl = live ? c : 0;
  auto load = [&](int64_t n, Row(&rows)[W]) {
#pragma unroll
    for (int r = 0; r < W - 1; ++r)
      rows[r] = p.state ? load_row<kWide>(p.state + (n * (W - 1) + r) * p.C, cl, p.C)
                        : Row{make_uint4(0u, 0u, 0u, 0u)};
    rows[W - 1] = load_row<kWide>(p.x + n * p.x_stride, cl, p.C);
  };
  Row next[W];
  load(n0, next);
  const Taps<W> taps = load_taps<W, kWide>(p, cl);
  Place pl = place_of(p, cl);
  if (!live) pl.normed = 0;
  bool far = false;  // (with care at once: bound by memory, it costs nothing here)
  for (int64_t n = n0; n < n1; ++n) {
    Row rows[W];
#pragma unroll
    for (int r = 0; r < W; ++r) rows[r] = next[r];
    if (n + 1 < n1) load(n + 1, next);
    if (live) {
#pragma unroll
      for (int r = 0; r < W - 1; ++r)
        store_row<kWide>(p.new_state + (n * (W - 1) + r) * p.C, c, p.C, rows[r + 1]);
    }
    Window<W> win;
#pragma unroll
    for (int r = 0; r < W - 1; ++r) win.set(r, rows[r]);
    const Row row[1] = {rows[W - 1]};
    output_rows<W, kWide, true, 1>(p, taps, pl, cl, n, pl.out + n * pl.width + pl.at, win, row,
                                   live, far);
  }
}

bool wide_ok(const ConvParams& p) {
  auto al = [](const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15u) == 0; };
  if (!al(p.x) || p.x_stride % kVec || p.C % kVec || !al(p.new_state) ||
      (p.state && !al(p.state)) || !al(p.weight) || (p.bias && !al(p.bias)))
    return false;
  for (int s = 0; s < p.sections; ++s)
    if (p.begin[s + 1] % kVec || !al(p.out[s])) return false;
  return true;
}

// grid.y holds at most 65535 rows; more go to grid.z.
dim3 rows_grid(unsigned bx, int64_t rows) {
  const int64_t y = rows < 32768 ? rows : 32768;
  return dim3(bx, static_cast<unsigned>(y), static_cast<unsigned>((rows + y - 1) / y));
}

template <int W>
int prefill_w(const ConvParams& p, cudaStream_t stream) {
  const unsigned bx = (p.C + kThreads * kVec - 1) / (kThreads * kVec);
  // Four blocks per SM run at a time. While one round of them covers the tokens in runs of 48 or
  // less, it does: 8192 channels, in a graph, 7 tokens 3.6 us in runs of 1 and 5.7 of 8; 1000 11.0
  // in runs of 16, 12.3 of 8; 3000 26.9 of 44, 28.7 of 48, 32.1 of 8. Beyond, a run costs its rows
  // and as long as 10 more (bounds, taps, W-1 rows again), and the last round is half empty: with
  // `round` tokens to a round of runs of one, (round / run + 1/2) (run + 10) is least at
  // sqrt(20 round). 5000 tokens 43.0 us in runs of 32, 44.7 of 48, 47.0 of 64; 19679 130.3 of 64,
  // 135 of 32 or 128; 65536 x 6144 259 of 112 (the rule's), 266 of 72, 265 of 128, 264 of 144.
  const int64_t round = (bx * p.T + 148 * 4 - 1) / (148 * 4);
  const int run = round <= 2    ? static_cast<int>(round < 1 ? 1 : round)
                  : round <= 48 ? static_cast<int>(round + 3) / 4 * 4
                                : static_cast<int>(std::sqrt(20.0 * round) / 8 + 0.5) * 8;
  const int64_t tiles = (p.T + run - 1) / run;
  const int64_t rows = tiles + p.N;
  if (rows > (int64_t{1} << 30)) return GDN_ERR_UNSUPPORTED_SHAPE;
  const dim3 grid = rows_grid(bx, rows);
  if (wide_ok(p)) {
    conv_prefill_kernel<W, true><<<grid, kThreads, 0, stream>>>(p, tiles, run);
  } else {
    conv_prefill_kernel<W, false><<<grid, kThreads, 0, stream>>>(p, tiles, run);
  }
  return cudaGetLastError() == cudaSuccess ? 0 : GDN_ERR_CUDA;
}

template <int W>
int decode_w(const ConvParams& p, cudaStream_t stream) {
  const unsigned bx = (p.C + kThreads * kVec - 1) / (kThreads * kVec);
  if (p.N > (int64_t{1} << 30)) return GDN_ERR_UNSUPPORTED_SHAPE;
  // One round of blocks: a thread's sequences share the load of its taps, and each one's rows are
  // under way while it has the one before in hand (1024 x 8192: 14 in one round 26.7 us, 4 in three
  // and a half 28.8, 1 each 32.3).
  const int64_t round = 148 * kDecodeBlocks<W>;
  const int per_thread = static_cast<int>((bx * p.N + round - 1) / round);
  const dim3 grid = rows_grid(bx, (p.N + per_thread - 1) / per_thread);
  if (wide_ok(p)) {
    conv_decode_kernel<W, true><<<grid, kThreads, 0, stream>>>(p, per_thread);
  } else {
    conv_decode_kernel<W, false><<<grid, kThreads, 0, stream>>>(p, per_thread);
  }
  return cudaGetLastError() == cudaSuccess ? 0 : GDN_ERR_CUDA;
}

}  // namespace

int launch_conv_prefill(const ConvParams& p, cudaStream_t stream) {
  if (p.W == 2) return prefill_w<2>(p, stream);
  if (p.W == 3) return prefill_w<3>(p, stream);
  return prefill_w<4>(p, stream);
}

int launch_conv_decode(const ConvParams& p, cudaStream_t stream) {
  if (p.W == 2) return decode_w<2>(p, stream);
  if (p.W == 3) return decode_w<3>(p, stream);
  return decode_w<4>(p, stream);
}

}  // namespace gdn
