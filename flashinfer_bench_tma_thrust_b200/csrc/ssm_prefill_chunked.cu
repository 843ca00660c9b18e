// ssm_prefill_chunked.cu — the state space scan over packed prompts on the tensor cores
// (head sizes and state sizes of 64 and 128).
//
// Chunks of L = 128 tokens. With G_t the in-chunk cumulative log decay (log2 units), d_t the
// step and S the state entering the chunk, per head
//     y_i   = e^{G_i} (C_i S^T) + sum_{j <= i} (C_i . B_j) e^{G_i - G_j} d_j x_j + D x_i
//     S'    = e^{G_L} S + sum_j (e^{G_L - G_j} d_j x_j) (outer) B_j
// What a chunk adds to the state does not depend on S, so the chunks of a sequence are
// chained by one multiply-add of the state only, and everything else overlaps.
//
// One block per (column block, segment): 128 columns of x, that is one head of 128 or two
// heads of 64 of one group (they share C B^T), over the chunks of one segment of a sequence.
// Three products per chunk on tcgen05, accumulators in TMEM (512 columns):
//     [CB, Y] [token, token | column]  = C [B; S]^T   S rounded to bf16, in shared memory
//                                                     behind B: one operand of 256 rows
//     dS      [column, n]              = (f x)^T B    f x transposed into TMEM as three bf16
//                                                     terms, by quarters of 32 tokens
//     Y                               += M x          M = CB masked and decayed, bf16 in TMEM
// Between the first and the last the block multiplies Y by e^{G_i} in TMEM. The state stays
// in fp32 registers (thread = column, half of n) for the whole segment.
//
// Roundings: x, B and C are exact bf16 operands, and so are the three terms of f x, whose sum
// is the fp32 product (the state, an fp32 result, is off by 3e-7; two terms left 2e-6). S and M
// are rounded once to bf16 as operands (a second term of S has no room in shared memory, one of M
// would double its product): they reach only y, which is rounded to bf16 itself. Relative to 64
// bits y is off by 0.0017 to 0.0022, of which its own rounding is 0.0017; most where a first state
// makes up most of y.
//
// Segments. With few (sequence, column block) chains the sequences are cut into segments of a
// multiple of 128 tokens. A first kernel (the same code, second product only) computes what
// each segment, or each part of one, adds to the state and what it leaves of it; each block of
// the second kernel then folds those of the segments before its own into its first state.
//
// Warps: 0-7 the output (M, the scaling of Y, y, and a chunk's first quarter of f x), 8-15 the
// state (the other quarters, S), which run at their own pace and so cover each other's waits; 16
// issues the products, each as soon as its operands are there, 17 the bulk copies, 18 and 19
// the gates (one head each, up to four chunks ahead). Every wait is bounded; a block that gives
// up reports it and runs on without waiting, so no barrier is left short of its threads.
//
// What bounds it: the chain of one chunk (product, M, M x, y, the next product) through single
// buffers of C B^T and Y, some 6400 cycles of which the tensor cores work half. No unit is at its
// limit: with heads and states of 128 the busy SMs issue in 62 % of the cycles, the tensor pipe is
// at 47 %, shared memory's banks move 3900 lines of 128 bytes per chunk (1800 of them for the
// roles' own loads and stores), HBM is at 35 %; the longest stall is for loads from TMEM, then
// fixed latencies. In long runs the power limit holds the clocks down besides. 4 x 32768 tokens of
// 32 heads take 1030 us in short runs and 1110 in long ones (3.1 and 2.9 TB/s of the bytes that
// have to move), one sequence of 32768 of 64 heads of 64 367 us in a graph and 430 in long runs, of
// which the segments' states take a quarter, and one chunk, mostly latency, 10.4 us. Two chunks per
// SM at a time would need twice the shared memory.
#include <algorithm>
#include <cfloat>
#include <cmath>

#include "gdn_b200.h"
#include "gdn_chunk_common.cuh"
#include "ssm_launch.h"

namespace gdn {
namespace {

using namespace sm100;
using chunk::kLog2e;
using chunk::named_bar_sync;

constexpr int kL = 128;             // tokens per chunk
constexpr int kBlock = 16384;       // a [128 rows x 64 columns] bf16 tile
constexpr int kMaxBars = 48;

// Registers per thread of the output kernel: 96 at launch (640 threads), then shared out anew
// between the output's, the state's and the other warps: 256 x 96 + 256 x 104 + 128 x 80 is
// what 640 x 96 were. Spills are what this avoids: the shared memory leaves L1 next to nothing,
// and a few local accesses per chunk cost more than a product.
constexpr int kLaunchRegs = 96, kOutRegs = kLaunchRegs, kStateRegs = 104, kMiscRegs = 80;
static_assert(256 * kOutRegs + 256 * kStateRegs + 128 * kMiscRegs <= 640 * kLaunchRegs, "");

template <int kRegs>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
}
template <int kRegs>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs));
}

// Shared memory by 32-bit address.
__device__ __forceinline__ float lds(uint32_t a) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ void sts(uint32_t a, float v) {
  asm volatile("st.shared.f32 [%0], %1;" ::"r"(a), "f"(v) : "memory");
}
__device__ __forceinline__ void sts4(uint32_t a, float x, float y, float z, float w) {
  asm volatile("st.shared.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(a), "f"(x), "f"(y), "f"(z), "f"(w)
               : "memory");
}
__device__ __forceinline__ float2 lds2(uint32_t a) {
  float2 v;
  asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a));
  return v;
}
__device__ __forceinline__ float4 lds4(uint32_t a) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(a));
  return v;
}
__device__ __forceinline__ float2 sub2(float2 a, float2 b) {
  return __fadd2_rn(a, make_float2(-b.x, -b.y));
}
__device__ __forceinline__ uint4 lds4u(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(a)
               : "memory");
  return v;
}
__device__ __forceinline__ void sts4u(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w)
               : "memory");
}
__device__ __forceinline__ void sts_u16(uint32_t a, unsigned short v) {
  asm volatile("st.shared.u16 [%0], %1;" ::"r"(a), "h"(v) : "memory");
}
__device__ __forceinline__ uint32_t lds_u16(uint32_t a) {
  unsigned short v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(a) : "memory");
  return v;
}
// Offset of row `row`'s 16-byte chunk 0 in a swizzled tile; chunk k is at this XOR 16 k.
__device__ __forceinline__ uint32_t row_base(uint32_t row) {
  return row * 128u + ((row & 7u) << 4);
}

// TMEM columns
constexpr uint32_t kTG = 0;         // C B^T; then M, 8 of every 16 columns per head
constexpr uint32_t kTY = 128;
constexpr uint32_t kTD = 256;       // dS
constexpr uint32_t kTF = 384;       // f x: 48 columns per place (the states kernel: from 0 on)
constexpr int kTerms = 3;           // bf16 terms of f x

// Of one head and chunk; read by offset (the order is kCum to kTot).
struct Gates {
  float cum[kL];                    // G from the start of the token's block of 32
  float dec[kL];                    // e^G
  float u[kL];                      // d_j e^{G_r - G_j}, r the end of j's block of 32
  float f[kL];                      // d_j e^{G_L - G_j}
  float h[kL];                      // log2 d_j - G_j, for pairs within a block
  float tot[4];                     // G over each block of 32
};
constexpr uint32_t kCum = 0, kDec = 512, kU = 1024, kF = 1536, kH = 2048, kTot = 2560;
constexpr uint32_t kGatesBytes = sizeof(Gates);
static_assert(kGatesBytes == kTot + 16 && kGatesBytes % 16 == 0, "");

// Chunks whose gates there is room for. The gates' warp takes some 3000 cycles a chunk, in a chain
// of short dependent steps: with two stages it was in the loop of the others' waits.
constexpr int kGateStages = 4;

struct Maps {
  CUtensorMap x, b, c, out;         // bf16 {64, T, columns / 64}, box {64, 128, blocks}
  // fp32 states {32, rows of all heads, Ns / 32}, box {32, P, Ns / 32}: the first states, what
  // the segments add, and where the kernel's last states go
  CUtensorMap first, add, last;
};

struct Segments {
  int64_t slots;                    // grid: slots x column blocks
  int len;                          // tokens per segment; 0: one per sequence
  int parts, part;                  // the states kernel: blocks per segment, tokens of each
  float* add;                       // [slots, parts, H, P, Ns] (through the maps)
  float* left;                      // [slots, parts, H]
};

template <int P, int NS, bool kStates>
struct Cfg {
  static constexpr int kHeads = 128 / P;
  static constexpr int kNB = NS / 64;
  // Stages: x stays until its y has left through the same memory; B and C are read early.
  static constexpr int kXStages = 3, kBStages = kStates ? 3 : 1;
  // f x is written by 32 tokens, into places in turn.
  static constexpr int kPlaces = kStates ? 4 : 2;
  static constexpr int kOutWarps = kStates ? 0 : 8, kStateWarps = kStates ? 16 : 8;
  static constexpr int kFxWarps = 8;  // that write one quarter of a chunk's f x
  static constexpr int kThreads = 32 * (kOutWarps + kStateWarps + 4);
  static constexpr uint32_t kXBytes = 2 * kBlock, kBBytes = kNB * kBlock;
  static constexpr uint32_t kX = 0;
  static constexpr uint32_t kB = kX + kXStages * kXBytes;
  // Output kernel: behind each 64-wide block of B the same block of the state, 128 rows of each,
  // so that both are one operand of 256 rows.
  static constexpr uint32_t kBStep = kStates ? kBlock : 2 * kBlock;
  static constexpr uint32_t kS = kB + kBlock;
  static constexpr uint32_t kC = kB + kBStages * kNB * kBStep;
  static constexpr uint32_t kGates = kC + (kStates ? 0 : kBBytes);
  static constexpr uint32_t kBars = kGates + kGateStages * kHeads * sizeof(Gates);
  static constexpr uint32_t kBytes = kBars + 8 * kMaxBars + 1024;  // and the alignment
};

enum Bar {
  kFullX = 0,                          // [3] one per stage
  kFullB = kFullX + 3,                 // [3]
  kFullC = kFullB + 3,
  kGatesFull = kFullC + 1,             // [kGateStages]
  kGatesFree = kGatesFull + kGateStages,
  kCB = kGatesFree + kGateStages,      // products done: C [B; S]^T
  kDS = kCB + 1,                       //   dS [3, by stage of B]
  kYM = kDS + 3,                       //   M x
  kFx = kYM + 1,                       // f x written [4, by place]
  kFxFree = kFx + 4,                   // f x read by its products [4, by quarter of a chunk]
  kMy = kFxFree + 4,                   // M and the scaled Y written
  kState = kMy + 1,                    // S written, dS read [2]
  kYFree = kState + 2,                 // Y read out
  kStaged = kYFree + 1,                // y in shared memory [3]
  kZeroed = kStaged + 3,
  kChecked = kZeroed + 1,              // nothing in x that is not finite, or no more
  kFullState = kChecked + 1,           // a state in the second and third stage of x
  kStateRead = kFullState + 1,
  kBarCount = kStateRead + 1,
};
static_assert(kBarCount <= kMaxBars, "");

__device__ __forceinline__ int64_t clamp_to(int64_t v, int64_t T) {
  return v < 0 ? 0 : (v > T ? T : v);
}
__device__ __forceinline__ int64_t clamp_bound(const SsmParams& p, int64_t i) {
  return clamp_to(load_index(p.cu_seqlens, p.cu_dtype, i), p.T);
}

// Segment `slot` in the order of the sequences: (sequence, segment of it) and the sequence's
// bounds as they stand in cu_seqlens. Whole warp.
__device__ __forceinline__ void find_segment(const SsmParams& p, const Segments& sg, int64_t slot,
                                             int64_t& n, int64_t& seg, int64_t& lo, int64_t& hi) {
  const int lane = threadIdx.x & 31;
  seg = 0;
  if (sg.len == 0) {
    // One segment per sequence; up to 32 sequences go longest first, so that the longest do
    // not start last.
    n = slot;
    if (p.N > 32) {
      lo = load_index(p.cu_seqlens, p.cu_dtype, n);
      hi = load_index(p.cu_seqlens, p.cu_dtype, n + 1);
      return;
    }
    int64_t a = 0, b = 0, len = -1;
    if (lane < p.N) {
      a = load_index(p.cu_seqlens, p.cu_dtype, lane);
      b = load_index(p.cu_seqlens, p.cu_dtype, lane + 1);
      len = max(clamp_to(b, p.T) - clamp_to(a, p.T), int64_t{0});
    }
    int rank = 0;
    for (int k = 0; k < static_cast<int>(p.N); ++k) {
      const int64_t other = __shfl_sync(0xffffffffu, len, k);
      rank += other > len || (other == len && k < lane);
    }
    n = __ffs(__ballot_sync(0xffffffffu, lane < p.N && rank == slot)) - 1;
    lo = __shfl_sync(0xffffffffu, a, static_cast<int>(n));
    hi = __shfl_sync(0xffffffffu, b, static_cast<int>(n));
    return;
  }
  lo = hi = 0;
  int64_t before = 0;
  for (int64_t n0 = 0; n0 < p.N; n0 += 32) {
    int64_t cnt = 0;
    if (n0 + lane < p.N) {
      const int64_t len = clamp_bound(p, n0 + lane + 1) - clamp_bound(p, n0 + lane);
      cnt = len > sg.len ? (len + sg.len - 1) / sg.len : 1;
    }
    int64_t incl = cnt;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    const uint32_t past = __ballot_sync(0xffffffffu, before + incl > slot);
    if (past) {
      const int src = __ffs(past) - 1;
      n = n0 + src;
      seg = slot - before - __shfl_sync(0xffffffffu, incl - cnt, src);
      lo = load_index(p.cu_seqlens, p.cu_dtype, n);
      hi = load_index(p.cu_seqlens, p.cu_dtype, n + 1);
      return;
    }
    before += __shfl_sync(0xffffffffu, incl, 31);
  }
  n = p.N;
}

__device__ __forceinline__ float lg2(float x) {  // log2 0 = -inf
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// softplus(v) = max(v, 0) + log(1 + u), u = e^-|v|, with log(1 + u) = 2 atanh(s) by its series in
// s = u / (2 + u) <= 1/3: a tenth of the instructions of log1pf(expf(v)), which with one or two
// warps on all of a chunk's gates set the pace of the kernel. The first term left out is below
// 2^-28 of the sum; u has ex2.approx's 2 ulp and, through the exponent's rest, no more.
__device__ __forceinline__ float softplus(float v) {
  const float x = -fminf(fabsf(v), 200.f);  // (e^-200 is zero; an infinite v leaves no NaN)
  const float z = x * kLog2e;
  const float rest = fmaf(x, kLog2e, -z);  // what rounding z left
  const float e = ex2(z);
  const float u = fmaf(e * 0.6931472f, rest, e);
  const float s = __fdividef(u, 2.f + u), q = s * s;
  float p = 1.f / 15.f;
  p = fmaf(p, q, 1.f / 13.f);
  p = fmaf(p, q, 1.f / 11.f);
  p = fmaf(p, q, 1.f / 9.f);
  p = fmaf(p, q, 1.f / 7.f);
  p = fmaf(p, q, 1.f / 5.f);
  p = fmaf(p, q, 1.f / 3.f);
  const float t = s + s;
  return fmaxf(v, 0.f) + fmaf(t, p * q, t) + (v != v ? v : 0.f);  // (fmaxf drops a NaN)
}

// Gates of a chunk's first `valid` tokens (the others: d = 0, no decay) of one head, four tokens
// per lane (a block of 32: eight lanes). All sums run over terms of one sign, so none cancels.
__device__ __forceinline__ void write_gates(uint32_t g, const float (&raw)[4], float neg_a,
                                            float dtb, int valid, int lane) {
  float d[4], lg[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const bool in = lane * 4 + k < valid;
    d[k] = in ? softplus(raw[k] + dtb) : 0.f;
    const float l = in ? neg_a * d[k] * kLog2e : 0.f;
    // 2^-127 is zero to ex2: a stronger decay changes nothing, and the sums stay small. A NaN
    // stays one.
    lg[k] = l < -127.f ? -127.f : l;
  }
  float pre = (lg[0] + lg[1]) + (lg[2] + lg[3]), suf = pre;  // over the block, to and from here
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    const float a = __shfl_up_sync(0xffffffffu, pre, o, 8);
    const float b = __shfl_down_sync(0xffffffffu, suf, o, 8);
    if ((lane & 7) >= o) pre += a;
    if ((lane & 7) + o < 8) suf += b;
  }
  float before = __shfl_up_sync(0xffffffffu, pre, 1, 8);
  float behind = __shfl_down_sync(0xffffffffu, suf, 1, 8);
  if ((lane & 7) == 0) before = 0.f;
  if ((lane & 7) == 7) behind = 0.f;
  const float b0 = __shfl_sync(0xffffffffu, pre, 7), b1 = __shfl_sync(0xffffffffu, pre, 15);
  const float b2 = __shfl_sync(0xffffffffu, pre, 23), b3 = __shfl_sync(0xffffffffu, pre, 31);
  const int blk = lane >> 3;
  const float head = blk == 0 ? 0.f : (blk == 1 ? b0 : (blk == 2 ? b0 + b1 : b0 + b1 + b2));
  const float tail = blk == 3 ? 0.f : (blk == 2 ? b3 : (blk == 1 ? b2 + b3 : b1 + b2 + b3));
  float c[4], w[4];  // from the block's start, inclusive; to its end, exclusive
  c[0] = before + lg[0];
  c[1] = c[0] + lg[1];
  c[2] = c[1] + lg[2];
  c[3] = c[2] + lg[3];
  w[3] = behind;
  w[2] = w[3] + lg[3];
  w[1] = w[2] + lg[2];
  w[0] = w[1] + lg[1];
  const uint32_t at = g + 16 * lane;
  sts4(at + kCum, c[0], c[1], c[2], c[3]);
  sts4(at + kH, lg2(d[0]) - c[0], lg2(d[1]) - c[1], lg2(d[2]) - c[2], lg2(d[3]) - c[3]);
  sts4(at + kDec, ex2(head + c[0]), ex2(head + c[1]), ex2(head + c[2]), ex2(head + c[3]));
  sts4(at + kU, d[0] * ex2(w[0]), d[1] * ex2(w[1]), d[2] * ex2(w[2]), d[3] * ex2(w[3]));
  sts4(at + kF, d[0] * ex2(w[0] + tail), d[1] * ex2(w[1] + tail), d[2] * ex2(w[2] + tail),
       d[3] * ex2(w[3] + tail));
  if ((lane & 7) == 7) sts(g + kTot + 4 * blk, pre);
}

template <int P, int NS, bool kStates>
__global__ void __launch_bounds__(Cfg<P, NS, kStates>::kThreads, 1)
ssm_chunk_kernel(const __grid_constant__ SsmParams p, const __grid_constant__ Maps maps,
                 const __grid_constant__ Segments sg, int col_blocks) {
  using K = Cfg<P, NS, kStates>;
  constexpr int kHeads = K::kHeads;
  extern __shared__ uint8_t raw_smem[];
  uint8_t* const sm = align_smem<1024>(raw_smem);
  __shared__ int64_t s_where[4];
  __shared__ uint32_t s_tmem;
  // Per stage of x and column: the token of the segment from which on an infinity or NaN in x leaves
  // y not finite (-1: none); whether there is any.
  __shared__ int s_poison[kStates ? 1 : K::kXStages * 128];
  __shared__ volatile int s_poisoned;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kOutWarps = K::kOutWarps;                   // first, then the state's
  constexpr int kMisc = kOutWarps + K::kStateWarps;
  uint64_t* const bars = reinterpret_cast<uint64_t*>(sm + K::kBars);

  if (!kStates && threadIdx.x >= 64 && threadIdx.x < 64 + K::kXStages * 128)
    s_poison[threadIdx.x - 64] = -1;
  const int64_t piece = blockIdx.x / col_blocks;  // a slot, or one of its parts
  const int cb = static_cast<int>(blockIdx.x - piece * col_blocks);
  const int64_t slot = kStates ? piece / sg.parts : piece;
  if (warp == 0) {
    int64_t n, seg, lo, hi;
    find_segment(p, sg, slot, n, seg, lo, hi);
    if (lane == 0) {
      s_where[0] = n;
      s_where[1] = seg;
      s_where[2] = clamp_to(lo, p.T);
      s_where[3] = max(clamp_to(hi, p.T), clamp_to(lo, p.T));
      if (cb == 0 && seg == 0 && n < p.N && (lo < 0 || hi > p.T || hi < lo))
        report_bad_bounds(p.status);
    }
  } else if (threadIdx.x == 32) {
    s_poisoned = 0;
    for (int i = 0; i < 3; ++i) {
      mbar_init(bars + kFullX + i, 1);
      mbar_init(bars + kFullB + i, 1);
      mbar_init(bars + kDS + i, 1);
      mbar_init(bars + kStaged + i, 8);
    }
    mbar_init(bars + kFullC, 1);
    for (int i = 0; i < kGateStages; ++i) {
      mbar_init(bars + kGatesFull + i, kHeads);
      mbar_init(bars + kGatesFree + i, kOutWarps + K::kStateWarps);
    }
    for (int i = 0; i < 2; ++i) mbar_init(bars + kState + i, K::kStateWarps);
    for (int i = 0; i < 4; ++i) {
      mbar_init(bars + kFx + i, K::kFxWarps);
      mbar_init(bars + kFxFree + i, 1);
    }
    for (int i : {kCB, kYM}) mbar_init(bars + i, 1);
    for (int i : {kMy, kYFree}) mbar_init(bars + i, 8);
    mbar_init(bars + kZeroed, K::kStateWarps);
    mbar_init(bars + kChecked, 4);  // (the state's warps with value 0 of each column)
    mbar_init(bars + kFullState, 1);
    mbar_init(bars + kStateRead, K::kStateWarps);
    fence_mbar_init();
  } else if (warp == kMisc) {
    tmem_alloc(&s_tmem, 512);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const int64_t n = s_where[0], seg = s_where[1], s_begin = s_where[2], s_end = s_where[3];
  const int64_t seg_begin = sg.len ? s_begin + seg * sg.len : s_begin;
  const int64_t seg_end = sg.len ? min(seg_begin + sg.len, s_end) : s_end;
  const bool last = seg_end >= s_end;
  if (n >= p.N || (kStates && last)) {  // (the second kernel computes a sequence's last state)
    if (warp == kMisc) tmem_dealloc(s_tmem, 512);
    return;
  }

  const int64_t t_begin = kStates ? seg_begin + (piece - slot * sg.parts) * sg.part : seg_begin;
  const int64_t t_end = kStates ? min(t_begin + sg.part, seg_end) : seg_end;

  const int rep = p.H / p.G;                                  // heads of a group
  const int per_group = (rep + kHeads - 1) / kHeads;
  const int grp = cb / per_group;
  const int h0 = grp * rep + (cb - grp * per_group) * kHeads;  // first head of the block
  const int heads = min(kHeads, (grp + 1) * rep - h0);
  const int tokens = static_cast<int>(t_end - t_begin);
  const int chunks = (tokens + kL - 1) / kL;
  const int tail = tokens - (chunks - 1) * kL;                // of the last chunk
  const int tok0 = static_cast<int>(t_begin);

  const uint32_t tm = s_tmem, sm_u = smem_u32(sm), gates_u = sm_u + K::kGates,
                 bars_u = sm_u + K::kBars;
  Waiter wait, finally;  // the second for what a block that gave up still has to wait for
  const int q = warp & 3;                      // TMEM lane quarter
  const uint32_t lanes = tm + (static_cast<uint32_t>(32 * q) << 16);
  const int row = 32 * q + lane;               // token of a chunk / column of the block
  auto arrive = [&](int bar) {
    __syncwarp();
    if (lane == 0) mbar_arrive(bars + bar);
  };

  const int part = (warp >> 2) & 1;            // of the two warps of a quarter in each role
  const int row_head = kHeads == 2 ? q >> 1 : 0;  // head of column `row`
  // (f x)^T of tokens 32 t to 32 t + 31 of chunk c into TMEM (this warp: 16 of them, of columns
  // 32 q to 32 q + 31): transposed by ldmatrix, scaled, split and stored as the fragments come.
  // Lane l gives ldmatrix token l % 8 + 8 (l / 16) of the 16, columns 8 ((l / 8) % 2) on.
  const uint32_t x_lane = 2048 * part + (row_base(8 * (lane >> 4) + (lane & 7)) ^
                                         (16 * ((q & 1) * 4 + ((lane >> 3) & 1))));
  auto write_fx = [&](int c, int t) {
    const int k = 4 * c + t, place = k % K::kPlaces;
    const uint32_t f = gates_u + (c % kGateStages * kHeads + row_head) * kGatesBytes + kF +
                       4 * (32 * t + 16 * part) + 8 * (lane & 3);
    const float2 f0 = lds2(f), f1 = lds2(f + 32);
    const uint32_t xa = sm_u + K::kX + (c % K::kXStages) * K::kXBytes + (q >> 1) * kBlock +
                        128 * 32 * t + x_lane;
    uint32_t u[2][4];  // [columns 0-15, 16-31]: tokens 0-7 of columns 0-7, 8-15; tokens 8-15
    ldmatrix_x4_trans(xa, u[0]);
    ldmatrix_x4_trans(xa ^ 32, u[1]);
    // The place's last use, `last`, was another quarter. A barrier per quarter, not per place: each
    // role has waited for its quarter's earlier phases itself, and its own f x comes before the next.
    // (A place has two phases per chunk here, of which a role would look at every other: it could
    // take the end of the phase before the last for that of the last.)
    if (const int last = k - K::kPlaces; last >= 0) {
      wait(bars_u + 8 * (kFxFree + last % 4), (last / 4) & 1);
      tc_fence_after();
    }
    const uint32_t at = lanes + (kStates ? 0 : kTF) + 16 * kTerms * place + 8 * part;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t w[kTerms][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // 24 bits in three bf16 terms of 8 by truncation: their sum is x f to the last bit
        float2 v = mul2(make_float2(__uint_as_float(u[h][i] << 16),
                                    __uint_as_float(u[h][i] & 0xffff0000u)),
                        i < 2 ? f0 : f1);
#pragma unroll
        for (int r = 0; r < kTerms; ++r) {
          const uint32_t a = __float_as_uint(v.x), b = __float_as_uint(v.y);
          w[r][i] = __byte_perm(a, b, 0x7632);
          if (r + 1 < kTerms)
            v = sub2(v, make_float2(__uint_as_float(a & 0xffff0000u),
                                    __uint_as_float(b & 0xffff0000u)));
        }
      }
#pragma unroll
      for (int r = 0; r < kTerms; ++r)
        tmem_st_frag(at + 16 * r + (static_cast<uint32_t>(16 * h) << 16), w[r]);
    }
    tmem_st_wait();
    tc_fence_before();
    arrive(kFx + place);
  };

  if (warp < kOutWarps) {
    // ---------------------------------------------------------------- output: token per thread
    const int half = part;
    const int col_head = kHeads == 2 ? half : 0;  // head of columns 64 half to 64 half + 63
    const float skip = p.D && col_head < heads ? load_scalar(p.D, p.D_dtype, h0 + col_head) : 0.f;
    // f x of a chunk's first quarter is this role's: it is written while M x runs, and keeps the
    // state's warps, which have the longer way, from waiting on their own products.
    auto first_fx = [&](int c) {
      wait(bars_u + 8 * (kFullX + c % K::kXStages), (c / K::kXStages) & 1);
      if (c == chunks - 1 && tail < kL) wait(bars_u + 8 * (kZeroed), 0);
      wait(bars_u + 8 * (kGatesFull + c % kGateStages), (c / kGateStages) & 1);
      write_fx(c, 0);
    };
    // (turn -1 only writes the first chunk's)
#pragma unroll 1
    for (int c = -1; c < chunks; ++c) {
      if (c >= 0) {
        const int gs = c % kGateStages;
        const uint32_t ga = gates_u + gs * kHeads * kGatesBytes;
        wait(bars_u + 8 * (kGatesFull + gs), (c / kGateStages) & 1);
        wait(bars_u + 8 * (kCB), c & 1);
        tc_fence_after();
        // ---- M over C B^T, 16 columns at a time: those of head h go to 8 columns of the same
        // 16, so a warp overwrites nothing that another has yet to read. The two warps of a
        // quarter take every other 16 (each has one piece on the diagonal).
#pragma unroll 1
        for (int k = 0; k < 4; ++k) {  // piece k: columns 32 k + 16 half on, in block k of 32
          float g[16];
          const int j0 = 32 * k + 16 * half;
          const uint32_t at = lanes + kTG + j0;
          if (k <= q) {
            tmem_ld16(at, g);
            tmem_ld_wait();
          }
          {
            uint32_t m[kHeads][8];
            if (k < q) {
              // e^{G_i - G_j} d_j = e^{G_i - G_r} (e^{G_r - G_j} d_j), r the end of j's block,
              // between j and i: both exponents are at most 0, and one exponential per row is left
              float ex[kHeads];
              float4 u[kHeads][4];
#pragma unroll
              for (int hh = 0; hh < kHeads; ++hh) {  // all loads before the first use
                const uint32_t gh = ga + hh * kGatesBytes;
                ex[hh] = lds(gh + kCum + 4 * row);
                if (k + 1 < q) ex[hh] += lds(gh + kTot + 4 * (k + 1));
                if (k + 2 < q) ex[hh] += lds(gh + kTot + 4 * (k + 2));
#pragma unroll
                for (int j = 0; j < 4; ++j) u[hh][j] = lds4(gh + kU + 4 * (j0 + 4 * j));
              }
#pragma unroll
              for (int hh = 0; hh < kHeads; ++hh) {
                const float e = ex2(ex[hh]);
                const float2 a = make_float2(e, e);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  const float4 v = u[hh][j];
                  const float2 v0 = mul2(mul2(make_float2(v.x, v.y), a),
                                         make_float2(g[4 * j], g[4 * j + 1]));
                  const float2 v1 = mul2(mul2(make_float2(v.z, v.w), a),
                                         make_float2(g[4 * j + 2], g[4 * j + 3]));
                  m[hh][2 * j] = pack2_rn(v0.x, v0.y);
                  m[hh][2 * j + 1] = pack2_rn(v1.x, v1.y);
                }
              }
            } else if (k == q) {
              const int i = row - j0;  // columns j <= i are on or below the diagonal
              float own[kHeads];
              float4 x[kHeads][4];
#pragma unroll
              for (int hh = 0; hh < kHeads; ++hh) {
                const uint32_t gh = ga + hh * kGatesBytes;
                own[hh] = lds(gh + kCum + 4 * row);
#pragma unroll
                for (int j = 0; j < 4; ++j) x[hh][j] = lds4(gh + kH + 4 * (j0 + 4 * j));
              }
#pragma unroll
              for (int hh = 0; hh < kHeads; ++hh) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  const float4 v = x[hh][j];
                  const float* const gj = g + 4 * j;
                  const float v0 = 4 * j <= i ? gj[0] * ex2(own[hh] + v.x) : 0.f;
                  const float v1 = 4 * j + 1 <= i ? gj[1] * ex2(own[hh] + v.y) : 0.f;
                  const float v2 = 4 * j + 2 <= i ? gj[2] * ex2(own[hh] + v.z) : 0.f;
                  const float v3 = 4 * j + 3 <= i ? gj[3] * ex2(own[hh] + v.w) : 0.f;
                  m[hh][2 * j] = pack2_rn(v0, v1);
                  m[hh][2 * j + 1] = pack2_rn(v2, v3);
                }
              }
            } else {
#pragma unroll
              for (int hh = 0; hh < kHeads; ++hh) {
#pragma unroll
                for (int j = 0; j < 8; ++j) m[hh][j] = 0u;
              }
            }
#pragma unroll
            for (int hh = 0; hh < kHeads; ++hh) tmem_st8(at + 8 * hh, m[hh]);
          }
        }
        // ---- Y = e^{G_i} (C S^T), in place
        {
          const float e = lds(ga + col_head * kGatesBytes + kDec + 4 * row);
          const float2 e2 = make_float2(e, e);
#pragma unroll 1
          for (int k = 0; k < 2; ++k) {
            const uint32_t ty = lanes + kTY + 64 * half + 32 * k;
            float y[32];
            tmem_ld32(ty, y);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              const float2 v = mul2(make_float2(y[i], y[i + 1]), e2);
              y[i] = v.x;
              y[i + 1] = v.y;
            }
            tmem_st32(ty, y);
          }
        }
        tmem_st_wait();
        tc_fence_before();
        arrive(kMy);
        arrive(kGatesFree + gs);
      }
      if (c + 1 < chunks) first_fx(c + 1);
      if (c >= 0) {
        // ---- y: out of TMEM, D x added, over the chunk's x in shared memory
        const int st = c % K::kXStages;
        const uint32_t xrow = sm_u + K::kX + st * K::kXBytes + half * kBlock + row_base(row);
        wait(bars_u + 8 * (kYM), c & 1);
        // (dS, and with it all that reads x, is done too, so that y may replace it. Ahead of kYFree:
        // without that the next chunk's dS does not end, and kChecked cannot run ahead.)
        wait(bars_u + 8 * (kChecked), c & 1);
        tc_fence_after();
        {
          float y[2][32];
          tmem_ld32(lanes + kTY + 64 * half, y[0]);
          tmem_ld32(lanes + kTY + 64 * half + 32, y[1]);
          tmem_ld_wait();
          tc_fence_before();
          arrive(kYFree);  // the next chunk's first product may start
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const uint32_t at = xrow ^ (16 * k);
            const uint4 xv = p.D ? lds4u(at) : make_uint4(0u, 0u, 0u, 0u);
            const uint32_t u[4] = {xv.x, xv.y, xv.z, xv.w};
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 v = fma2(make_float2(skip, skip),
                                    make_float2(__uint_as_float(u[e] << 16),
                                                __uint_as_float(u[e] & 0xffff0000u)),
                                    make_float2(y[k >> 2][8 * (k & 3) + 2 * e],
                                                y[k >> 2][8 * (k & 3) + 2 * e + 1]));
              w[e] = pack2_rn(v.x, v.y);
            }
            sts4u(at, w[0], w[1], w[2], w[3]);
          }
        }
        if (s_poisoned) {
#pragma unroll 1
          for (int k = 0; k < 64; ++k) {  // of this token's columns
            const int first = s_poison[st * 128 + 64 * half + k];
            if ((first >> 7) == c && row >= (first & 127))
              sts_u16((xrow ^ (16 * (k >> 3))) + 2 * (k & 7), 0x7fff);
          }
        }
        if (c < chunks - 1 || tail == kL) {
          fence_async_smem();
          arrive(kStaged + st);  // a bulk store takes the whole tile
        } else {
          // only the sequence's rows: 16 lanes write the 256 bytes of one
          named_bar_sync(1, 256);
          uint8_t* const xt = sm + K::kX + st * K::kXBytes;
          const int l = lane & 15, blk = l >> 3;
          const int64_t base = (static_cast<int64_t>(tok0) + c * kL) * p.H + h0;
          if (kHeads == 1 || blk < heads) {
            for (int r = warp * 2 + (lane >> 4); r < tail; r += 16) {
              const uint4 v =
                  *reinterpret_cast<const uint4*>(xt + blk * kBlock + sw128_chunk(r, l & 7));
              const int64_t at = (base + static_cast<int64_t>(r) * p.H) * P + l * 8;
              *reinterpret_cast<uint4*>(p.out + at) = v;
            }
          }
        }
      }
    }
  } else if (warp < kMisc) {
    if (!kStates) regs_inc<kStateRegs>();
    // ---------------------------------------------------------------- state: column per thread
    constexpr int kNC = NS * 4 / K::kStateWarps;  // state columns per thread, from kNC * sp on
    const int sp = (warp - kOutWarps) >> 2;
    const bool mine = row_head < heads;
    float S[kNC];
#pragma unroll
    for (int i = 0; i < kNC; ++i) S[i] = 0.f;
    float left = 1.f;

    // fp32 states pass through shared memory, by bulk copies in swizzled rows of 32 values: read
    // or written by threads that each own a row, memory would see 16 bytes of every 512 at a
    // time (4 us for 64 KB and the other loads behind it, against 1).
    const uint32_t s_tile = row_head * (P * NS * 4) + row_base(row % P);
    auto s_at = [&](uint32_t base, int i) {  // of S[i], i a multiple of 4
      const int at = kNC * sp + i;
      return base + (at >> 5) * (P * 128) + (s_tile ^ (16 * ((at >> 2) & 7)));
    };
    if (!kStates) {
      const int items = (p.state ? 1 : 0) + static_cast<int>(seg) * sg.parts;
      const int64_t r0 = slot * sg.parts - items;
      for (int k = 0; k < items; ++k) {
        // the sequence's first state, then the parts of its segments before this one
        const int64_t r = r0 + k;
        const float g = p.state && k == 0 ? 0.f : (mine ? sg.left[r * p.H + h0 + row_head] : 0.f);
        wait(bars_u + 8 * (kFullState), k & 1);
        if (mine) {
#pragma unroll
          for (int i = 0; i < kNC; i += 4) {
            const float4 v = lds4(s_at(sm_u + K::kX + K::kXBytes, i));
            S[i] = fmaf(g, S[i], v.x);
            S[i + 1] = fmaf(g, S[i + 1], v.y);
            S[i + 2] = fmaf(g, S[i + 2], v.z);
            S[i + 3] = fmaf(g, S[i + 3], v.w);
          }
        }
        arrive(kStateRead);
      }
    }

    // The state as the operand of the next chunk's C S^T: row = column of the block, n
    // contiguous (K-major).
    const uint32_t s_row = sm_u + K::kS + (kNC * sp >> 6) * K::kBStep + row_base(row);
    auto arrive_state = [&]() {
#pragma unroll
      for (int k = 0; k < kNC / 8; ++k)
        sts4u(s_row ^ (16 * (((kNC * sp >> 3) + k) & 7)), pack2_rn(S[8 * k], S[8 * k + 1]),
              pack2_rn(S[8 * k + 2], S[8 * k + 3]), pack2_rn(S[8 * k + 4], S[8 * k + 5]),
              pack2_rn(S[8 * k + 6], S[8 * k + 7]));
      fence_async_smem();
      arrive(kState);
    };

    auto begin_fx = [&](int c) {
      const int st = c % K::kXStages;
      uint8_t* const xt = sm + K::kX + st * K::kXBytes;
      wait(bars_u + 8 * (kFullX + st), (c / K::kXStages) & 1);
      if (c == chunks - 1 && tail < kL) {
        // Rows behind the sequence hold other tokens or nothing: zeros, so that neither they
        // nor a NaN among them enters a product.
        uint8_t* const bt = sm + K::kB + (c % K::kBStages) * K::kBBytes;
        wait(bars_u + 8 * (kFullB + c % K::kBStages), (c / K::kBStages) & 1);
        for (int i = threadIdx.x - kOutWarps * 32; i < (kL - tail) * 8; i += K::kStateWarps * 32) {
          const uint32_t off = (tail + (i >> 3)) * 128 + (i & 7) * 16;
          const uint4 z = make_uint4(0u, 0u, 0u, 0u);
          *reinterpret_cast<uint4*>(xt + off) = z;
          *reinterpret_cast<uint4*>(xt + kBlock + off) = z;
#pragma unroll
          for (int b = 0; b < K::kNB; ++b) *reinterpret_cast<uint4*>(bt + b * K::kBStep + off) = z;
        }
        fence_async_smem();
        named_bar_sync(2, K::kStateWarps * 32);
        arrive(kZeroed);
      }
      wait(bars_u + 8 * (kGatesFull + c % kGateStages), (c / kGateStages) & 1);
    };
    // The state behind chunk c, from what the chunk adds.
    auto update_state = [&](int c) {
      wait(bars_u + 8 * (kDS + c % K::kBStages), (c / K::kBStages) & 1);
      tc_fence_after();
      const float g =
          lds(gates_u + (c % kGateStages * kHeads + row_head) * kGatesBytes + kDec + 4 * (kL - 1));
      const float2 g2 = make_float2(g, g);
      const uint32_t td = lanes + kTD + (kStates ? 128 * (c & 1) : 0) + kNC * sp;
#pragma unroll
      for (int i0 = 0; i0 < kNC; i0 += 16) {
        float v[16];
        tmem_ld16(td + i0, v);
        tmem_ld_wait();
        const bool finite = fabsf(S[0]) <= FLT_MAX;
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const float2 s = fma2(g2, make_float2(S[i0 + i], S[i0 + i + 1]),
                                make_float2(v[i], v[i + 1]));
          S[i0 + i] = s.x;
          S[i0 + i + 1] = s.y;
        }
        if (!kStates && i0 == 0 && sp == 0) {
          // An infinity or NaN in x leaves none of its column's state finite, and one value shows it.
          // In M x it would reach the tokens before it too (0 x NaN): it gives way to a zero first,
          // and y becomes NaN from its token on. (Looking at x itself, with 8 instructions in each of
          // its readers, took 4 % of the time of 4 x 32768 tokens, this takes 2 %.)
          if (finite && !(fabsf(S[0]) <= FLT_MAX)) {
            const uint32_t xt = sm_u + K::kX + (c % K::kXStages) * K::kXBytes + (q >> 1) * kBlock;
            int first = kL;
#pragma unroll 1
            for (int j = kL - 1; j >= 0; --j) {
              const uint32_t at = xt + sw128_offset(j, row & 63);
              if ((lds_u16(at) & 0x7f80u) != 0x7f80u) continue;
              sts_u16(at, 0);
              first = j;
            }
            if (first < kL) {
              s_poison[c % K::kXStages * 128 + row] = c * kL + first;
              s_poisoned = 1;
              fence_async_smem();
            }
          }
          arrive(kChecked);
        }
      }
      if (kStates) left *= g;
      tc_fence_before();
      arrive(kGatesFree + c % kGateStages);
    };

    // Turn i of the loop writes one quarter of f x (the output kernel: its other warps write each
    // chunk's first) and, with a chunk's first turn, updates the state with the chunk before;
    // one more turn updates it with the last chunk. (One loop: each part of the code exists once.)
    if (chunks > 0) {
      // the states kernel's two times 8 warps take every other quarter
      const int t0 = kStates ? warp >> 3 : 1;
      constexpr int kStep = kStates ? 2 : 1, kTurns = kStates ? 2 : 3;
      if (!kStates) arrive_state();
      int c = 0, t = t0;
#pragma unroll 1
      for (int i = 0; i <= kTurns * chunks; ++i) {
        const bool first = t == t0;
        if (first && c < chunks) begin_fx(c);
        if (kStates && c < chunks) write_fx(c, t);  // while the last chunk's products still run
        if (first && c > 0) {
          update_state(c - 1);
          // C S^T has read the state it replaces: it came before dS's end
          if (!kStates && c < chunks) arrive_state();
          if (kStates) arrive(kState + ((c - 1) & 1));
        }
        if (!kStates && c < chunks) write_fx(c, t);
        if ((t += kStep) >= 4) {
          t = t0;
          ++c;
        }
      }
    }
    if (kStates && mine && sp == 0 && row % P == 0) sg.left[piece * p.H + h0 + row_head] = left;
    if (kStates || last) {
      // over B and the state's operand: the last dS is done, and with it all that reads them
#pragma unroll
      for (int i = 0; i < kNC; i += 4)
        sts4(s_at(sm_u + K::kB, i), S[i], S[i + 1], S[i + 2], S[i + 3]);
      fence_async_smem();
      named_bar_sync(2, K::kStateWarps * 32);
      if (warp == kOutWarps && lane == 0) {
        const int64_t to = ((kStates ? piece : n) * p.H + h0) * static_cast<int64_t>(P);
        for (int hh = 0; hh < heads; ++hh)
          tma_store_3d(&maps.last, sm + K::kB + hh * (P * NS * 4), 0, static_cast<int>(to) + hh * P,
                       0);
        bulk_commit();
        bulk_wait_all();
      }
      __syncwarp();
    }
  } else {
    if (!kStates) regs_dec<kMiscRegs>();
    if (warp == kMisc) {
      // ---------------------------------------------------------------- products
      constexpr uint32_t kIdCB = idesc_bf16(128, 256, false, false);
      constexpr uint32_t kIdDS = idesc_bf16(128, NS, false, true);
      constexpr uint32_t kIdYM = idesc_bf16(128, P, false, true);
      // Descriptors differ in their start address alone: built where they are used, from bases
      // that look new in every chunk, or all of them would be kept in registers.
      const uint64_t d_k = desc_kmajor(0), d_x = desc_mnmajor(0, kBlock),
                     d_b = desc_mnmajor(0, K::kBStep);
      auto fresh = [](uint32_t v) {
        uint32_t r;
        asm volatile("mov.u32 %0, %1;" : "=r"(r) : "r"(v));
        return r;
      };
      auto desc = [](uint64_t kind, uint32_t base, uint32_t off) {
        return kind | static_cast<uint64_t>((base + off) >> 4);
      };
      auto kstep = [](int s, uint32_t block) {
        return static_cast<uint32_t>((s >> 2) * block + (s & 3) * 32);
      };
      for (int c = 0; c < chunks; ++c) {
        const int st = c % K::kBStages, par = (c / K::kBStages) & 1;
        const uint32_t xb = sm_u + K::kX + (c % K::kXStages) * K::kXBytes;
        const uint32_t bb = sm_u + K::kB + st * K::kBBytes;
        const bool zeroed = c == chunks - 1 && tail < kL;
        // dS by quarter t of the chunk's tokens, whose f x is in its place
        auto issue_ds = [&](uint32_t td, int t) {
          const int place = (4 * c + t) % K::kPlaces;
          const uint32_t tf = tm + (kStates ? 0 : kTF) + 16 * kTerms * place;
          const uint32_t b0 = fresh(bb + t * 4096);
          tc_fence_after();
#pragma unroll
          for (int r = 0; r < kTerms; ++r) {
#pragma unroll
            for (int s = 0; s < 2; ++s)
              mma_bf16_ts_w(td, tf + 16 * r + 8 * s, desc(d_b, b0, s * 2048), kIdDS,
                            t > 0 || r > 0 || s > 0);
          }
          mma_commit_w(bars + kFxFree + t);
          if (t == 3) mma_commit_w(bars + kDS + st);
        };
        auto fx_bar = [&](int t) { return bars_u + 8 * (kFx + (4 * c + t) % K::kPlaces); };
        auto fx_par = [&](int t) { return static_cast<uint32_t>(((4 * c + t) / K::kPlaces) & 1); };
        if (kStates) {
          wait(bars_u + 8 * (kFullB + st), par);
          if (c >= 2) wait(bars_u + 8 * (kState + (c & 1)), ((c >> 1) - 1) & 1);
#pragma unroll 1
          for (int t = 0; t < 4; ++t) {
            wait(fx_bar(t), fx_par(t));
            issue_ds(tm + kTD + 128 * (c & 1), t);
          }
          continue;
        }
        // The chunk's products, each as soon as its operands are there and its place is free. What
        // the order has to keep: B's stage and the state's operand are free with the last quarter
        // of dS, so C [B; S]^T comes before that.
        bool cb = false, ym = false, b_in = false, state_in = false;
        bool force = !wait.ok();  // a block that gave up does not wait
        int t = 0;
        uint32_t polls = 1u << 23;  // of some 100 cycles
        auto ready = [&](int bar, uint32_t parity) {
          return force || mbar_test_wait(bars_u + 8 * bar, parity);
        };
#pragma unroll 1
        while (!ym || t < 4) {
          b_in = b_in || ready(kFullB + st, par);
          state_in = state_in || ready(kState, c & 1);
          if (b_in && state_in && t < (cb ? 4 : 3) &&
              ready(kFx + (4 * c + t) % K::kPlaces, ((4 * c + t) / K::kPlaces) & 1)) {
            issue_ds(tm + kTD, t);
            ++t;
          }
          if (!cb) {  // over the places of the last chunk's M and Y
            if (b_in && state_in && ready(kFullC, c & 1) && (!zeroed || ready(kZeroed, 0)) &&
                (c == 0 || ready(kYFree, (c - 1) & 1))) {
              cb = true;
              tc_fence_after();
              const uint32_t b0 = fresh(bb), c0 = fresh(sm_u + K::kC);
#pragma unroll 4
              for (int s = 0; s < NS / 16; ++s)
                mma_bf16_w(tm + kTG, desc(d_k, c0, kstep(s, kBlock)),
                           desc(d_k, b0, kstep(s, K::kBStep)), kIdCB, s > 0);
              mma_commit_w(bars + kCB);
            }
          } else if (!ym && ready(kMy, c & 1) && ready(kChecked, c & 1)) {
            // (behind all of the chunk's f x, whose writers take infinities and NaN out of x: they
            // are done long before M, so this waits for nothing)
            ym = true;
            tc_fence_after();
#pragma unroll 1
            for (int hh = 0; hh < kHeads; ++hh) {
              const uint32_t x0 = fresh(xb + hh * kBlock);
#pragma unroll 4
              for (int s = 0; s < 8; ++s)
                mma_bf16_ts_w(tm + kTY + hh * 64, tm + kTG + 16 * s + 8 * hh,
                              desc(d_x, x0, s * 2048), kIdYM, 1);
            }
            mma_commit_w(bars + kYM);
          }
          if (!force && --polls == 0) {
            force = true;
            wait.left = 0;
          }
        }
      }
      // the block's TMEM may go once the last product is done
      if (chunks > 0) {
        const int c = chunks - 1;
        if (kStates) {
          finally(bars_u + 8 * (kDS + c % K::kBStages), (c / K::kBStages) & 1);
        } else {
          finally(bars_u + 8 * (kYM), c & 1);
        }
      }
    } else if (warp == kMisc + 1) {
      // ---------------------------------------------------------------- bulk copies
      if (lane == 0) {
        const int xc = (h0 * P) / 64, bc = grp * K::kNB;
        auto load_x = [&](int c) {
          const int st = c % K::kXStages;
          mbar_arrive_expect_tx(bars + kFullX + st, K::kXBytes);
          tma_load_3d(sm + K::kX + st * K::kXBytes, &maps.x, bars + kFullX + st, 0, tok0 + c * kL,
                      xc);
        };
        auto load_b = [&](int c) {
          const int st = c % K::kBStages;
          mbar_arrive_expect_tx(bars + kFullB + st, K::kBBytes);
          for (int b = 0; b < K::kNB; ++b)
            tma_load_3d(sm + K::kB + st * K::kBBytes + b * K::kBStep, &maps.b, bars + kFullB + st,
                        0, tok0 + c * kL, bc + b);
        };
        auto load_c = [&](int c) {
          mbar_arrive_expect_tx(bars + kFullC, K::kBBytes);
          tma_load_3d(sm + K::kC, &maps.c, bars + kFullC, 0, tok0 + c * kL, bc);
        };
        if (chunks > 0) {
          load_b(0);
          if (!kStates) load_c(0);
          load_x(0);
        }
        if (!kStates) {  // states, one after the other in the other stages of x
          const int items = (p.state ? 1 : 0) + static_cast<int>(seg) * sg.parts;
          for (int k = 0; k < items; ++k) {
            if (k > 0) wait(bars_u + 8 * (kStateRead), (k - 1) & 1);
            const bool first = p.state && k == 0;
            const int64_t from =
                ((first ? n : slot * sg.parts - items + k) * p.H + h0) * static_cast<int64_t>(P);
            mbar_arrive_expect_tx(bars + kFullState, heads * P * NS * 4);
            for (int hh = 0; hh < heads; ++hh)
              tma_load_3d(sm + K::kX + K::kXBytes + hh * (P * NS * 4),
                          first ? &maps.first : &maps.add, bars + kFullState, 0,
                          static_cast<int>(from) + hh * P, 0);
          }
          if (items > 0) wait(bars_u + 8 * (kStateRead), (items - 1) & 1);
        }
        for (int c = 1; c < K::kXStages && c < chunks; ++c) {
          if (c < K::kBStages) load_b(c);
          load_x(c);
        }
        for (int c = 0; c < chunks; ++c) {
          if (!kStates && c + 2 < chunks) {
            // B and C have one stage: bring the next but one chunk's into L2, so that the copy
            // that has to wait for the stage takes only L2's latency
            for (int b = 0; b < K::kNB; ++b)
              tma_prefetch_3d(&maps.b, 0, tok0 + (c + 2) * kL, bc + b);
            tma_prefetch_3d(&maps.c, 0, tok0 + (c + 2) * kL, bc);
          }
          if (!kStates && c + 1 < chunks) {
            wait(bars_u + 8 * (kCB), c & 1);
            load_c(c + 1);
          }
          if (c + K::kBStages < chunks) {
            wait(bars_u + 8 * (kDS + c % K::kBStages), (c / K::kBStages) & 1);
            load_b(c + K::kBStages);
            if (kStates) load_x(c + K::kXStages);  // x was read before the product
          }
          if (!kStates && (c < chunks - 1 || tail == kL)) {
            const int st = c % K::kXStages;
            wait(bars_u + 8 * (kStaged + st), (c / K::kXStages) & 1);
            const uint8_t* xt = sm + K::kX + st * K::kXBytes;
            for (int b = 0; b < 2; ++b)
              if (kHeads == 1 || b < heads)
                tma_store_3d(&maps.out, xt + b * kBlock, 0, tok0 + c * kL, xc + b);
            bulk_commit();
            if (c + K::kXStages < chunks) {
              bulk_wait_read();
              load_x(c + K::kXStages);
            }
          }
        }
        if (!kStates) bulk_wait_all();
        if (!wait.ok() && chunks > 0) {
          // copies still in flight land in this block's shared memory: let them
          const int c = chunks - 1;
          finally(bars_u + 8 * (kFullX + c % K::kXStages), (c / K::kXStages) & 1);
          finally(bars_u + 8 * (kFullB + c % K::kBStages), (c / K::kBStages) & 1);
          if (!kStates) finally(bars_u + 8 * (kFullC), c & 1);
        }
      }
      __syncwarp();
    } else if (warp - kMisc - 2 < kHeads) {
      // ---------------------------------------------------------------- gates of one head
      const int hh = warp - kMisc - 2;
      const bool present = hh < heads;
      const int h = h0 + (present ? hh : 0);
      const float neg_a = -expf(load_scalar(p.A_log, p.A_log_dtype, h));
      const float dtb = load_scalar(p.dt_bias, p.dt_bias_dtype, h);
      // dt of a chunk as stored, asked for a chunk ahead: nothing may use a value before its chunk
      // (a conversion here would wait for each of the four in turn, 800 cycles each)
      const bool half = p.dt_dtype == kBF16;
      auto load = [&](int c, uint32_t (&raw)[4]) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int t = min(c * kL + 4 * lane + k, tokens - 1);
          const int64_t at = (static_cast<int64_t>(tok0) + t) * p.H + h;
          raw[k] = half ? static_cast<const unsigned short*>(p.dt)[at]
                        : static_cast<const uint32_t*>(p.dt)[at];
        }
      };
      uint32_t raw[4];
      if (chunks > 0) load(0, raw);
#pragma unroll 1
      for (int c = 0; c < chunks; ++c) {
        const int gs = c % kGateStages;
        float dt[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) dt[k] = __uint_as_float(half ? raw[k] << 16 : raw[k]);
        if (c + 1 < chunks) load(c + 1, raw);
        if (c >= kGateStages)
          wait(bars_u + 8 * (kGatesFree + gs), (c / kGateStages - 1) & 1);
        write_gates(gates_u + (gs * kHeads + hh) * kGatesBytes, dt, neg_a,
                    dtb, present ? tokens - c * kL : 0, lane);
        __syncwarp();
        if (lane == 0) mbar_arrive(bars + kGatesFull + gs);
      }
    }
  }
  if (!wait.ok()) report_wait(p.status);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kMisc) tmem_dealloc(tm, 512);
}

bool encode(CUtensorMap* map, const void* base, int64_t T, int64_t cols, uint32_t blocks) {
  chunk::EncodeTiledFn enc = chunk::get_encode_fn();
  if (!enc) return false;
  const cuuint64_t dims[3] = {64, static_cast<cuuint64_t>(T), static_cast<cuuint64_t>(cols / 64)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(cols) * 2, 128};
  const cuuint32_t box[3] = {64, kL, blocks};
  const cuuint32_t estr[3] = {1, 1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box,
             estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool encode_state(CUtensorMap* map, const void* base, int64_t rows, int P, int Ns) {
  chunk::EncodeTiledFn enc = chunk::get_encode_fn();
  if (!enc) return false;
  const cuuint64_t dims[3] = {32, static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(Ns / 32)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(Ns) * 4, 128};
  const cuuint32_t box[3] = {32, static_cast<cuuint32_t>(P), static_cast<cuuint32_t>(Ns / 32)};
  const cuuint32_t estr[3] = {1, 1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, const_cast<void*>(base), dims, strides, box,
             estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int column_blocks(int H, int G, int P) {
  const int heads = 128 / P;
  return G * ((H / G + heads - 1) / heads);
}

// How the sequences are cut, with slots that cover any lengths. Without segments: one slot each.
// In us, with heads and states of 128: a chunk takes 3.4, one of the states' kernel 2.0, that
// kernel's start 9 and each segment that is folded into a first state 1.1. The host does not know
// the lengths: the longest sequence of several is taken as half as long again as their mean.
// 32 heads, whole / in segments, in a graph: 1000 tokens 34.9 / 28.6, 1900 60 / 40, 3000 91 / 53,
// 8192 226 / 105; one head, in segments of 1024 / by this rule: 2000 tokens 55 / 31, 8192 60 / 49,
// 131072 210 / 165. (Four sequences of 300, 400, 2000 and 900 with 16 heads gain nothing: 63.5.)
Segments plan(int64_t T, int64_t N, int H, int G, int P) {
  constexpr int kSms = 148;
  constexpr double kChunk = 3.4, kState = 2.0, kStart = 9, kFold = 1.1;
  Segments sg{};
  sg.slots = N;
  sg.parts = 1;
  const int cols = column_blocks(H, G, P);
  const int64_t fit = kSms / cols;  // segments that run at the same time
  if (N == 0 || fit <= N) return sg;
  const double longest = static_cast<double>(N == 1 ? T : 3 * T / (2 * N)) / kL;  // in chunks
  // as many as fit, but not so many that the folding takes longer than it saves
  double l = static_cast<double>((T + fit - N) / (fit - N + 1)) / kL;
  l = std::ceil(std::max({l, 2.0, std::sqrt(longest * kFold / (kChunk + kState))}));
  if (kChunk * longest <= (kChunk + kState) * l + kStart + kFold * longest / l) return sg;
  sg.len = static_cast<int>(l) * kL;
  sg.slots = T / sg.len + N;
  // A sequence's last segment has no part in the states kernel, and a part takes less than half
  // of a segment's time: several to a segment may fill the SMs better (32 column blocks: 32768
  // tokens, 3 segments with states, 418 us in all in a graph, in 3 parts each 367).
  const double busy = std::max(1.0, static_cast<double>((T - 1) / sg.len - (N - 1) / 2)) * cols;
  double best = 0;
  for (int parts = 1; parts <= 4; ++parts) {
    const double part = std::ceil(l / parts);
    if (part * (parts - 1) >= l) break;
    const double time = std::ceil(busy * parts / kSms) * (kStart + kState * part) +
                        kFold * parts * longest / l;
    if (parts == 1 || time < best) {
      best = time;
      sg.parts = parts;
      sg.part = static_cast<int>(part) * kL;
    }
  }
  return sg;
}

template <int P, int NS>
int launch_as(const SsmParams& p, cudaStream_t stream) {
  Segments sg = plan(p.T, p.N, p.H, p.G, p.P);
  const int64_t pieces = sg.slots * sg.parts;
  const int cols = column_blocks(p.H, p.G, p.P);
  if (pieces * cols > 0x7fffffffLL) return GDN_ERR_UNSUPPORTED_SHAPE;
  Maps maps;
  const int64_t hp = static_cast<int64_t>(p.H) * P, gn = static_cast<int64_t>(p.G) * NS;
  if (!encode(&maps.x, p.x, p.T, hp, 2) || !encode(&maps.b, p.B, p.T, gn, 1) ||
      !encode(&maps.c, p.C, p.T, gn, NS / 64) || !encode(&maps.out, p.out, p.T, hp, 1))
    return GDN_ERR_CUDA;
  // (row coordinates are 32-bit)
  if (p.N * hp > 0x7fffffffLL || pieces * hp > 0x7fffffffLL) return GDN_ERR_UNSUPPORTED_SHAPE;
  const void* const first = p.state ? p.state : p.new_state;
  if (!encode_state(&maps.first, first, p.N * hp, P, NS)) return GDN_ERR_CUDA;
  maps.add = maps.last = maps.first;
  const unsigned grid = static_cast<unsigned>(sg.slots * cols);
  if (sg.len) {
    if (!p.workspace) return GDN_ERR_WORKSPACE;
    sg.add = p.workspace;
    sg.left = p.workspace + pieces * hp * NS;
    if (!encode_state(&maps.add, sg.add, pieces * hp, P, NS)) return GDN_ERR_CUDA;
    maps.last = maps.add;
    using K = Cfg<P, NS, true>;
    auto fn = ssm_chunk_kernel<P, NS, true>;
    if (cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, K::kBytes) !=
        cudaSuccess)
      return GDN_ERR_CUDA;
    fn<<<grid * sg.parts, K::kThreads, K::kBytes, stream>>>(p, maps, sg, cols);
    if (cudaGetLastError() != cudaSuccess) return GDN_ERR_CUDA;
  }
  if (!encode_state(&maps.last, p.new_state, p.N * hp, P, NS)) return GDN_ERR_CUDA;
  using K = Cfg<P, NS, false>;
  auto fn = ssm_chunk_kernel<P, NS, false>;
  // the new shares wait for registers that the launch has to have brought
  static const bool regs_ok = [&] {
    cudaFuncAttributes at;
    return cudaFuncGetAttributes(&at, fn) == cudaSuccess && at.numRegs == kLaunchRegs;
  }();
  if (!regs_ok) return GDN_ERR_CUDA;
  if (cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, K::kBytes) !=
      cudaSuccess)
    return GDN_ERR_CUDA;
  fn<<<grid, K::kThreads, K::kBytes, stream>>>(p, maps, sg, cols);
  return cudaGetLastError() == cudaSuccess ? 0 : GDN_ERR_CUDA;
}

}  // namespace

// Few tokens per sequence go token by token: with 32 heads of 128 and states of 128, us token by
// token against chunked: one sequence of 8 tokens 6.4 / 10.5, of 16 10.4 / 10.5; 8 sequences of
// 4 15.7 / 20.4, of 6 23.1 / 20.4; 64 of 4 113 / 140, of 6 166 / 140.
bool ssm_chunked_takes(int P, int Ns, int64_t T, int64_t N) {
  return (P == 64 || P == 128) && (Ns == 64 || Ns == 128) && T > 4 * N + 8;
}

size_t ssm_chunked_workspace(int64_t T, int64_t N, int H, int G, int P, int Ns) {
  const Segments sg = plan(T, N, H, G, P);
  return sg.len ? static_cast<size_t>(sg.slots * sg.parts) * H *
                      (static_cast<size_t>(P) * Ns + 1) * sizeof(float)
                : 0;
}

int launch_ssm_chunked(const SsmParams& p, cudaStream_t stream) {
  if (p.P == 64) {
    return p.Ns == 64 ? launch_as<64, 64>(p, stream) : launch_as<64, 128>(p, stream);
  }
  return p.Ns == 64 ? launch_as<128, 64>(p, stream) : launch_as<128, 128>(p, stream);
}

}  // namespace gdn
