// linear_act.cu — y = act(x w^T + bias) + residual with one rounding at the end, for any number of rows.
//
//   x [m, k], w [n, k] (nn.Linear), both bf16 or both fp16; bias [n] of their type; residual [m, n] of their type or
//   fp32; y [m, n] of their type or fp32. act: none, ReLU, GELU (erf or tanh), x * sigmoid(1.702 x), SiLU, on the fp32
//   accumulator.
//
// Two kernels, both on tcgen05 with operands by TMA (128-byte swizzle) and fp32 accumulators in TMEM:
//
//  * few_kernel, for up to some hundreds of rows: the weight is the tensor cores' M operand and the tokens are N. A tile
//    is 128 output features by BT = 16 .. 128 tokens, so a single token costs one 16-column MMA per 16 of K instead of a
//    128-row tile of padding, and the kernel is what a few rows need to be: a stream of the weight through shared memory.
//    Where the tiles are fewer than the CTAs that fit the GPU, a cluster of up to eight CTAs shares one: each takes a
//    run of K, leaves its fp32 partial tile in shared memory, and finishes an equal share of the tile's tokens by adding
//    the partials of all of them over distributed shared memory in rank order (no workspace, no atomics; the same call
//    always gives the same bits).
//  * many_kernel, for the rest: 256 tokens x 256 features per CTA pair (tcgen05.mma.cta_group::2), persistent over tiles.
//
// Precision: the tensor core adds into its accumulator with less care than an fp32 add, it truncates (over K = 12288 the
// error grew to 1.4e-5 of the result's norm), so an accumulator takes 1024 of K at most; the epilogue warps then add it to
// fp32 registers, which are the sum proper, while the other TMEM buffer takes the next 1024. That costs 2 % of the time at
// most (every 512 cost 10 %) and holds the error of an fp32 output at 1.0e-6 (bf16) and 1.25e-6 (fp16) of its norm for any
// K (4608 x 12288 x 3072 onto its fp32 residual: 6.7e-7, elementary fp32 operations 8.3e-7). Within 1024 of K the
// accumulator's truncation is what there is.
//
// Measured on the device: 28 x 3072 x 18432 (m x k x n) 24.6 us, 4.6 TB/s of weight, which a kernel that only loads the
// weight by TMA also takes; 4608 x 12288 x 3072 onto an fp32 residual 231 us, 1505 TFLOP/s, in a single call and 243 to 290
// us back to back under the power cap; 512 x 12288 x 3072 49 us; one row, 256 to 3072 features, 4.8 us back to back.
#include <atomic>
#include <type_traits>

#include "gemm_common.cuh"

namespace fb {
namespace lact {

using gemm::BK;

struct Args {
  CUtensorMap tma_w, tma_x;
  const void* bias;
  const void* residual;
  void* out;
  int64_t ld_res, ld_out;
  int m, n, num_kb;
  int splits, tiles_f, tiles_t, group;
  int half;      // operands and 16-bit outputs are fp16 (else bf16)
  int res_f32, out_f32;
  int vec;       // four consecutive outputs (and residuals, biases) are aligned vectors
  uint32_t idesc;
  int* status;
};

// The kernels are instances per activation: with all of them behind a switch in every unrolled place, the code of an
// epilogue outgrew the instruction caches (a 256 x 256 tile took 80 us).
//
// The erf of GELU is Abramowitz and Stegun's 7.1.26 for erfc(|x|), x = z / sqrt 2, off by at most 1.5e-7: y = z h for
// z < 0 and z - z h otherwise, h = erfc(|x|) / 2. A value is off by 3.4e-7 at most, of standard normal inputs 8.4e-8 of the
// norm (6.1e-8 with an fp32 erf), which only an fp32 output shows. Small negative values keep their size, unlike those of
// 1 + erf in fp32, but not every bit: off by 5e-5 of themselves at z = -3 (1 + erf: 1.4e-6), 5e-4 at -4 (3e-4), 4e-3 at -6
// and 2 % at -10 (all). With CUDA's erff the epilogue of a 256 x 256 tile at K = 3072 took longer than its products. The
// sigmoids divide by 1 + exp with the hardware's exp2 and division, (2 + 1.2 |z|) 2^-23 and 2^-22 relative, for the same
// reason; tanh(u) = 2 sigmoid(2u) - 1.
__device__ __forceinline__ float rcp_approx(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float exp2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
template <int ACT>
__device__ __forceinline__ float activate(float z) {
  if constexpr (ACT == FB_ACT_RELU) return z < 0.f ? 0.f : z;  // keeps a NaN
  if constexpr (ACT == FB_ACT_GELU) {
    // |z|, up to 30 where z > 0: nothing is left of erfc there, and +inf * 0 stays out. -inf gives NaN as z/2 * (1 + erf) does
    // (a clamp of |z| would give 0; 8192 x 512 x 4096, bound by the epilogue, 71.6 us with that, 72.8 with this).
    const float s = fmaxf(-z, fminf(z, 30.f));
    const float t = rcp_approx(fmaf(0.3275911f * 0.70710678f, s, 1.0f));
    float h = fmaf(t, 0.5f * 1.061405429f, 0.5f * -1.453152027f);
    h = fmaf(h, t, 0.5f * 1.421413741f);
    h = fmaf(h, t, 0.5f * -0.284496736f);
    h = fmaf(h, t, 0.5f * 0.254829592f);
    const float q = 0.84932180f * z;  // sqrt(log2(e) / 2)
    return fmaf(-s, h * t * exp2_approx(-q * q), fmaxf(z, 0.f));
  }
  if constexpr (ACT == FB_ACT_GELU_TANH) {
    const float u = 0.7978845608028654f * fmaf(0.044715f * z * z, z, z);  // sqrt(2 / pi) (z + 0.044715 z^3)
    return __fdividef(z, 1.0f + __expf(-2.0f * u));
  }
  if constexpr (ACT == FB_ACT_QUICK_GELU) return __fdividef(z, 1.0f + __expf(-1.702f * z));
  if constexpr (ACT == FB_ACT_SILU) return __fdividef(z, 1.0f + __expf(-z));
  return z;
}

// 16-bit value of the operands' type widened to fp32, and back.
template <bool HALF>
__device__ __forceinline__ float widen(uint32_t v) {
  return HALF ? __half2float(__ushort_as_half(static_cast<uint16_t>(v))) : __uint_as_float(v << 16);
}
template <bool HALF>
__device__ __forceinline__ float4 widen4(uint2 u) {
  if constexpr (HALF) {
    const float2 lo = __half22float2(*reinterpret_cast<const __half2*>(&u.x));
    const float2 hi = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
    return make_float4(lo.x, lo.y, hi.x, hi.y);
  } else {
    return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xFFFF0000u), __uint_as_float(u.y << 16),
                       __uint_as_float(u.y & 0xFFFF0000u));
  }
}
template <bool HALF>
__device__ __forceinline__ uint2 narrow4(float4 v) {
  if constexpr (HALF) {
    const __half2 lo = __floats2half2_rn(v.x, v.y), hi = __floats2half2_rn(v.z, v.w);
    return make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
  } else {
    return make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
  }
}
template <bool HALF>
__device__ __forceinline__ uint16_t narrow(float v) {
  return HALF ? __half_as_ushort(__float2half_rn(v)) : __bfloat16_as_ushort(__float2bfloat16_rn(v));
}

__device__ __forceinline__ float4 ld_shared_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

__device__ __forceinline__ float4 ld_shared_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}

// Four consecutive features n0 .. n0 + 3 as aligned vectors, for N tokens at a time: token + i * step, of which those
// below `end` exist. What a call's types decide is decided once for all of them: a branch in every step costs more than
// the step.
__device__ __forceinline__ float4 bias4(const Args& a, int n0) {
  if (a.bias == nullptr) return make_float4(0.f, 0.f, 0.f, 0.f);
  const uint2 u = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(a.bias) + n0));
  return a.half ? widen4<true>(u) : widen4<false>(u);
}
template <int N>
__device__ __forceinline__ void residuals(const Args& a, int token, int step, int end, int n0, float4 (&r)[N]) {
  const int64_t at = token * a.ld_res + n0, by = step * a.ld_res;
  if (a.residual == nullptr) {
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  } else if (a.res_f32) {
    const float* p = static_cast<const float*>(a.residual) + at;
#pragma unroll
    for (int i = 0; i < N; ++i, p += by)
      if (token + i * step < end) r[i] = *reinterpret_cast<const float4*>(p);
  } else {
    const uint16_t* p = static_cast<const uint16_t*>(a.residual) + at;
    uint2 u[N];
#pragma unroll
    for (int i = 0; i < N; ++i, p += by)
      if (token + i * step < end) u[i] = *reinterpret_cast<const uint2*>(p);
    if (a.half) {
#pragma unroll
      for (int i = 0; i < N; ++i) r[i] = widen4<true>(u[i]);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) r[i] = widen4<false>(u[i]);
    }
  }
}
// z: the sums, overwritten
template <int ACT, int N>
__device__ __forceinline__ void finish(const Args& a, int token, int step, int end, int n0, float4 b, const float4 (&r)[N], float4 (&z)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    z[i].x = activate<ACT>(z[i].x + b.x) + r[i].x;
    z[i].y = activate<ACT>(z[i].y + b.y) + r[i].y;
    z[i].z = activate<ACT>(z[i].z + b.z) + r[i].z;
    z[i].w = activate<ACT>(z[i].w + b.w) + r[i].w;
  }
  const int64_t at = token * a.ld_out + n0, by = step * a.ld_out;
  if (a.out_f32) {
    float* p = static_cast<float*>(a.out) + at;
#pragma unroll
    for (int i = 0; i < N; ++i, p += by)
      if (token + i * step < end) *reinterpret_cast<float4*>(p) = z[i];
  } else {
    uint16_t* p = static_cast<uint16_t*>(a.out) + at;
    if (a.half) {
#pragma unroll
      for (int i = 0; i < N; ++i, p += by)
        if (token + i * step < end) *reinterpret_cast<uint2*>(p) = narrow4<true>(z[i]);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i, p += by)
        if (token + i * step < end) *reinterpret_cast<uint2*>(p) = narrow4<false>(z[i]);
    }
  }
}
// One feature of one token, any alignment.
__device__ __forceinline__ float bias1(const Args& a, int n) {
  if (a.bias == nullptr) return 0.f;
  const uint16_t v = __ldg(static_cast<const uint16_t*>(a.bias) + n);
  return a.half ? widen<true>(v) : widen<false>(v);
}
// N values of any alignment: where(i) = token * stride + feature, live(i): it exists.
template <int N, typename Where, typename Live>
__device__ __forceinline__ void residuals1(const Args& a, Where where, Live live, float (&r)[N]) {
  if (a.residual == nullptr) {
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = 0.f;
  } else if (a.res_f32) {
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = live(i) ? static_cast<const float*>(a.residual)[where(i, a.ld_res)] : 0.f;
  } else {
    uint16_t u[N];
#pragma unroll
    for (int i = 0; i < N; ++i) u[i] = live(i) ? static_cast<const uint16_t*>(a.residual)[where(i, a.ld_res)] : 0;
    if (a.half) {
#pragma unroll
      for (int i = 0; i < N; ++i) r[i] = widen<true>(u[i]);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) r[i] = widen<false>(u[i]);
    }
  }
}
// z: the sums with their bias, overwritten
template <int ACT, int N, typename Where, typename Live>
__device__ __forceinline__ void finish1(const Args& a, Where where, Live live, const float (&r)[N], float (&z)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) z[i] = activate<ACT>(z[i]) + r[i];
  if (a.out_f32) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (live(i)) static_cast<float*>(a.out)[where(i, a.ld_out)] = z[i];
  } else if (a.half) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (live(i)) static_cast<uint16_t*>(a.out)[where(i, a.ld_out)] = narrow<true>(z[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (live(i)) static_cast<uint16_t*>(a.out)[where(i, a.ld_out)] = narrow<false>(z[i]);
  }
}

// The bias of a lane's four features of the 128 from f0: f0 + 4 lane + 0 .. 3 (whole), or f0 + lane + 32 * 0 .. 3.
__device__ __forceinline__ float4 lane_bias(const Args& a, int f0, bool whole, int lane) {
  if (whole) return bias4(a, f0 + 4 * lane);
  float b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) b[i] = f0 + lane + 32 * i < a.n ? bias1(a, f0 + lane + 32 * i) : 0.f;
  return make_float4(b[0], b[1], b[2], b[3]);
}

// Finishes tokens j0 + warp, + WARPS, .. below j1 of a tile (token j of the tile is row t0 + j of the output) for the 128
// features from f0 whose sums lie in shared memory as fp32 rows of ROW floats from `base` on, features from column `col`:
// in this CTA's (splits == 1), or as partial sums at the same place of the cluster's CTAs first_rank + s * rank_step, added
// in order of s. SWIZZLE: the 16-byte unit u of row j is at place u ^ (j % 8). Two tokens per warp at a time: a lane
// finishes four consecutive features of each (whole: aligned vectors), or features lane, lane + 32, .. .
template <int ACT, int WARPS, int ROW, bool SWIZZLE>
__device__ __forceinline__ void finish_share(const Args& a, uint32_t base, int col, int rows, int t0, int j0, int j1, int f0, bool whole,
                                             float4 b, int warp, int lane, int splits, int first_rank, int rank_step) {
  constexpr int U = 2;
  if (whole) {
    const int n0 = f0 + 4 * lane;
#pragma unroll 1
    for (int j = j0 + warp; j < j1; j += U * WARPS) {
      float4 r[U], z[U];
      residuals<U>(a, t0 + j, WARPS, t0 + j1, n0, r);
#pragma unroll
      for (int u = 0; u < U; ++u) z[u] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (int s = 0; s < splits; ++s) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int ju = min(j + u * WARPS, rows - 1);  // past the share: read, not written
          const uint32_t at = base + ju * ROW * 4 + (((col >> 2) + lane) ^ (SWIZZLE ? ju & 7 : 0)) * 16;
          const float4 p = splits > 1 ? ld_shared_cluster_f4(mapa_shared(at, first_rank + s * rank_step)) : ld_shared_f4(at);
          z[u].x += p.x, z[u].y += p.y, z[u].z += p.z, z[u].w += p.w;
        }
      }
      finish<ACT, U>(a, t0 + j, WARPS, t0 + j1, n0, b, r, z);
    }
  } else {
    const float bs[4] = {b.x, b.y, b.z, b.w};
#pragma unroll 1
    for (int j = j0 + warp; j < j1; j += U * WARPS) {
      // value i: token j + (i / 4) * WARPS, feature f0 + lane + 32 (i % 4)
      auto exists = [&](int i) { return j + (i >> 2) * WARPS < j1 && f0 + lane + 32 * (i & 3) < a.n; };
      auto where = [&](int i, int64_t ld) {
        return static_cast<int64_t>(t0 + j + (i >> 2) * WARPS) * ld + f0 + lane + 32 * (i & 3);
      };
      float r[4 * U], z[4 * U];
      residuals1<4 * U>(a, where, exists, r);
#pragma unroll
      for (int i = 0; i < 4 * U; ++i) z[i] = bs[i & 3];
#pragma unroll 2
      for (int s = 0; s < splits; ++s) {
#pragma unroll
        for (int i = 0; i < 4 * U; ++i) {
          const int ju = min(j + (i >> 2) * WARPS, rows - 1), c = col + lane + 32 * (i & 3);
          const uint32_t at = base + ju * ROW * 4 + ((c >> 2) ^ (SWIZZLE ? ju & 7 : 0)) * 16 + (c & 3) * 4;
          float p;
          if (splits > 1) {
            asm volatile("ld.shared::cluster.f32 %0, [%1];"
                         : "=f"(p)
                         : "r"(mapa_shared(at, first_rank + s * rank_step))
                         : "memory");
          } else {
            asm volatile("ld.shared.f32 %0, [%1];" : "=f"(p) : "r"(at) : "memory");
          }
          z[i] += p;
        }
      }
      finish1<ACT, 4 * U>(a, where, exists, r, z);
    }
  }
}

// Adds NC accumulator columns at `taddr` (this warp's 32 lanes) to v; the first time they are the sum.
template <int NC, int CW>
__device__ __forceinline__ void promote(uint32_t taddr, bool first, float (&v)[NC]) {
#pragma unroll
  for (int c = 0; c < NC; c += CW) {
    uint32_t r[CW];
    if constexpr (CW == 16) {
      tmem_ld_32x32b_x16(taddr + c, r);
    } else {
      tmem_ld_32x32b_x32(taddr + c, r);
    }
    tmem_ld_wait();
    if (first) {
#pragma unroll
      for (int j = 0; j < CW; ++j) v[c + j] = __uint_as_float(r[j]);
    } else {
#pragma unroll
      for (int j = 0; j < CW; ++j) v[c + j] += __uint_as_float(r[j]);
    }
  }
}

// ---------------------------------------------------------------------------------------------- few rows

constexpr int kFeat = 128;       // output features of a tile
constexpr int kChunkBlocks = 16;  // K blocks of 64 that one accumulator takes

// warp 0 loads, warp 1 issues the MMAs, the others promote the accumulator (TMEM lane = feature, column = token; at 128
// tokens two warps share a lane quarter, so that a thread holds at most 64 sums); all of them write the outputs.
template <int BT>
struct Few {
  static constexpr int kEpiWarps = BT == 128 ? 8 : 4;
  static constexpr int kWarps = 2 + kEpiWarps, kThreads = 32 * kWarps;
  static constexpr int kCols = BT / (kEpiWarps / 4);  // token columns of a thread
  // Two CTAs per SM: while one fills its pipeline or writes its outputs, the other streams.
  static constexpr int kStages = BT == 16 ? 6 : BT == 32 ? 5 : BT == 64 ? 4 : 3;
  static constexpr int kWBytes = kFeat * BK * 2;
  static constexpr int kXBytes = BT * BK * 2;
  static constexpr int kStageBytes = kWBytes + kXBytes;
  static constexpr int kSmemBytes = kStages * kStageBytes + 256 + 1024;
  static constexpr int kTmemCols = BT < 32 ? 32 : 2 * BT;  // two accumulators
  static_assert(kStages * kStageBytes >= BT * kFeat * 4, "the fp32 tile takes the operand stages' place");
};

template <int BT, int ACT>
__global__ void __launch_bounds__(Few<BT>::kThreads, 2) few_kernel(const __grid_constant__ Args a) {
  using C = Few<BT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sW = smem;
  uint8_t* sX = smem + C::kStages * C::kWBytes;
  float* tile = reinterpret_cast<float*>(smem);  // [BT][128] fp32, once every stage has been consumed
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kStages * C::kStageBytes);
  uint64_t* empty = full + C::kStages;
  uint64_t* acc_full = empty + C::kStages;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* drain = acc_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = warp_id(), lane = lane_id();
  const int rank = a.splits > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int t = blockIdx.x / a.splits;
  const int f0 = (t % a.tiles_f) * kFeat, t0 = (t / a.tiles_f) * BT;
  const int kb0 = static_cast<int>(static_cast<int64_t>(a.num_kb) * rank / a.splits);
  const int kb1 = static_cast<int>(static_cast<int64_t>(a.num_kb) * (rank + 1) / a.splits);

  auto load = [&](int stage, int kb) {
    mbar_arrive_expect_tx(&full[stage], C::kStageBytes);
    tma_load_2d(&a.tma_w, &full[stage], sW + stage * C::kWBytes, kb * BK, f0);
    tma_load_2d(&a.tma_x, &full[stage], sX + stage * C::kXBytes, kb * BK, t0);
  };
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], C::kEpiWarps);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
    // this thread's barriers are ready: the first loads do not wait for the rest of the set-up
    for (int s = 0; s < C::kStages && kb0 + s < kb1; ++s) load(s, kb0 + s);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::kTmemCols);
    tmem_relinquish();
  }
  // This CTA's share of the tile's tokens. Its bias and residuals are fetched now, not when the sums are there.
  const int live = min(BT, a.m - t0);
  const int j0 = live * rank / a.splits, j1 = live * (rank + 1) / a.splits;
  const bool whole = a.vec && f0 + kFeat <= a.n;  // every lane's four consecutive features are aligned vectors
  if (a.residual != nullptr) {
    const int line = a.res_f32 ? 32 : 64, lines = kFeat / line;  // features in 128 bytes
    for (int i = threadIdx.x; i < (j1 - j0) * lines; i += C::kThreads) {
      const int n = f0 + (i % lines) * line;
      const int64_t at = static_cast<int64_t>(t0 + j0 + i / lines) * a.ld_res + n;
      if (n < a.n)
        asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const uint8_t*>(a.residual) + (a.res_f32 ? 4 : 2) * at));
    }
  }
  const float4 b = lane_bias(a, f0, whole, lane);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 1, issued[C::kStages];
      for (int s = 0; s < C::kStages; ++s) issued[s] = kb0 + s < kb1 ? 0u : 0xFFFFFFFFu;
      bool ok = true;
      for (int kb = kb0 + C::kStages; kb < kb1; ++kb) {
        if (!mbar_wait(&empty[stage], phase ^ 1u, abort_flag, a.status, FB_DEV_TIMEOUT_MMA)) {
          ok = false;
          break;
        }
        load(stage, kb);
        issued[stage] = phase;
        if (++stage == C::kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (!ok) {
        for (int s = 0; s < C::kStages; ++s)
          if (issued[s] != 0xFFFFFFFFu) mbar_wait_quiet(&full[s], issued[s], kWaitBudgetNs);
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int kc = kb0; ok && kc < kb1; kc += kChunkBlocks) {
        if (!mbar_wait(&acc_empty[acc], acc_phase ^ 1u, abort_flag, a.status, FB_DEV_TIMEOUT_EPI)) break;
        tc_fence_after_sync();
        for (int kb = kc; kb < min(kc + kChunkBlocks, kb1); ++kb) {
          if (!mbar_wait(&full[stage], phase, abort_flag, a.status, FB_DEV_TIMEOUT_TMA)) {
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t w0 = smem_u32(sW + stage * C::kWBytes), x0 = smem_u32(sX + stage * C::kXBytes);
#pragma unroll
          for (int k = 0; k < BK / 16; ++k)
            umma_bf16_ss(tmem_base + acc * BT, sdesc_kmajor_sw128(w0 + 32 * k), sdesc_kmajor_sw128(x0 + 32 * k), a.idesc,
                         (kb > kc || k > 0) ? 1u : 0u);
          umma_commit(&empty[stage]);
          if (++stage == C::kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        umma_commit(&acc_full[acc]);
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1u;
      }
      umma_commit(drain);  // every MMA issued by this thread is over before TMEM is released
      mbar_wait_quiet(drain, 0, kWaitBudgetNs);
    }
  } else {
    const int quarter = warp & 3;  // the TMEM lanes a warp may read are fixed by warp % 4
    const int col0 = ((warp - 2) >> 2) * C::kCols;
    float v[C::kCols];
#pragma unroll
    for (int j = 0; j < C::kCols; ++j) v[j] = 0.f;  // the sum over no K at all
    int acc = 0;
    uint32_t acc_phase = 0;
    for (int kc = kb0; kc < kb1; kc += kChunkBlocks) {
      if (!mbar_wait(&acc_full[acc], acc_phase, abort_flag, a.status, FB_DEV_TIMEOUT_MMA)) break;
      tc_fence_after_sync();
      promote<C::kCols, C::kCols == 32 ? 32 : 16>(tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + acc * BT + col0, kc == kb0, v);
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[acc]);
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1u;
    }
    // The last accumulator was complete, so the tensor core has read every stage: the tile takes their place.
    const int f = quarter * 32 + lane;
#pragma unroll
    for (int j = 0; j < C::kCols; ++j) tile[(col0 + j) * kFeat + f] = v[j];
  }
  __syncwarp();
  tc_fence_before_sync();
  if (a.splits > 1) {
    cluster_sync_all();
  } else {
    __syncthreads();
  }

  finish_share<ACT, C::kWarps, kFeat, false>(a, smem_u32(tile), 0, BT, t0, j0, j1, f0, whole, b, warp, lane, a.splits, 0, 1);
  __syncwarp();
  if (a.splits > 1) {
    cluster_sync_all();  // nobody reads this CTA's tile any more: it may exit
  } else {
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, C::kTmemCols);
  }
}

// ---------------------------------------------------------------------------------------------- many rows

// A cluster of two CTAs per 256 x 256 tile: each loads its own 128 token rows and 128 of the 256 weight rows, the leader
// issues M = 256, N = 256 MMAs that read both, and each CTA's TMEM gets its 128 rows (256 columns, two accumulators).
// An operand stage is 128 of K (two 64-wide boxes of each operand, 64 KB per CTA), an accumulator takes eight stages.
// Eight epilogue warps, two per TMEM lane quarter, hold the 128 sums of their half row in registers; a finished tile
// goes through 4 KB of shared memory per warp, 32 x 32 values at a time, so that residuals and outputs are contiguous
// accesses, while the tensor core already works on the next tile.
//
// SPLIT, for fewer tiles than pairs: a cluster of `splits` pairs shares one tile, each pair a run of K. The sums go to shared
// memory (128 KB, in the place of the operand stages), and every CTA finishes an equal share of its 128 rows by adding the
// partial sums of the CTAs that hold the same rows. (Against few_kernel's 128 x 128 tiles this halves the operand bytes that
// an SM has to take in per product: at 512 x 3072 those bytes, not the products, set few_kernel's time.)
namespace many {
constexpr int kTile = 256;
constexpr int kMaxSplits = 4;
constexpr int kEpiWarps = 8;
constexpr int kCols = 4 * kTile / kEpiWarps;  // sums of a thread
// Three warpgroups: loads and MMAs (two of its warps idle), and the two of the epilogue, which take the registers that
// the first gives back. 128 x 40 + 256 x 232 = 384 x 168, what the block is launched with.
constexpr int kThreads = 128 + 32 * kEpiWarps;
constexpr int kLeanRegs = 40, kEpiRegs = 232, kLaunchRegs = 168;
static_assert(128 * kLeanRegs + 256 * kEpiRegs == (128 + 32 * kEpiWarps) * kLaunchRegs, "the split is what the launch allots");
constexpr int kSub = 2;
constexpr int kStages = 3;
constexpr int kChunkStages = 8;
constexpr int kBoxBytes = 128 * BK * 2;
constexpr int kOpBytes = kSub * kBoxBytes;
constexpr int kStageBytes = 2 * kOpBytes;
constexpr int kPatchBytes = 32 * 32 * 4;
constexpr int kSmemBytes = kStages * kStageBytes + kEpiWarps * kPatchBytes + 256 + 1024;
constexpr uint32_t kTmemCols = 512;

// Arrives on the barrier at shared-memory offset `bar` of both CTAs of the pair whose leader has cluster rank `lead` when
// every MMA issued so far by this thread is complete. (It signals barriers; it loads nothing.)
__device__ __forceinline__ void commit_pair(uint32_t bar, int lead) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
      "h"(static_cast<unsigned short>(3 << lead))
      : "memory");
}

// Token tiles in groups of a.group, tokens fastest inside a group: the tiles that run at once share rows of both operands.
__device__ __forceinline__ void place(const Args& a, int tile, int& mb, int& nb) {
  const int per_group = a.group * a.tiles_f;
  const int g = tile / per_group;
  const int first = g * a.group;
  const int gm = min(a.tiles_t - first, a.group);
  const int in_group = tile - g * per_group;
  mb = first + in_group % gm;
  nb = in_group / gm;
}

template <int ACT, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1) many_kernel(const __grid_constant__ Args a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sX = smem;
  uint8_t* sW = smem + kStages * kOpBytes;
  uint8_t* sP = sW + kStages * kOpBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(sP + kEpiWarps * kPatchBytes);
  uint64_t* empty = full + kStages;
  uint64_t* acc_full = empty + kStages;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* drain = acc_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = warp_id(), lane = lane_id();
  const int cta = static_cast<int>(cluster_ctarank());
  const int rank = cta & 1, lead = cta & ~1, split = SPLIT ? cta >> 1 : 0;  // in the pair, its leader, which run of K
  const bool leader = rank == 0;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 2 * kEpiWarps);  // the epilogue warps of both CTAs
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&a.tma_w);
    tma_prefetch_desc(&a.tma_x);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, kTmemCols);
    tmem_relinquish_pair();
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();  // both CTAs' barriers exist before either signals the other
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  const int tiles = a.tiles_f * a.tiles_t;
  const int pair = SPLIT ? blockIdx.x / (2 * a.splits) : blockIdx.x >> 1, npairs = SPLIT ? tiles : gridDim.x >> 1;
  const int stages_all = (a.num_kb + kSub - 1) / kSub;  // a K tail past the end is zero-filled by TMA
  const int ks0 = SPLIT ? stages_all * split / a.splits : 0, ks1 = SPLIT ? stages_all * (split + 1) / a.splits : stages_all;

  if (warp < 4) {
    reg_dealloc<kLeanRegs>();
    if (warp == 0 && lane == 0) {
      int stage = 0;
      uint32_t phase = 0, issued[kStages];
      for (int s = 0; s < kStages; ++s) issued[s] = 0xFFFFFFFFu;
      bool ok = true;
      for (int tile = pair; ok && tile < tiles; tile += npairs) {
        int mb, nb;
        place(a, tile, mb, nb);
        for (int ks = ks0; ks < ks1; ++ks) {
          if (!mbar_wait(&empty[stage], phase ^ 1u, abort_flag, a.status, FB_DEV_TIMEOUT_MMA)) {
            ok = false;
            break;
          }
          const uint32_t bar = mapa_shared(smem_u32(&full[stage]), lead);
          if (leader) mbar_arrive_expect_tx(&full[stage], 2 * kStageBytes);
#pragma unroll
          for (int h = 0; h < kSub; ++h) {
            const int kx = (ks * kSub + h) * BK;
            tma_load_2d_pair(&a.tma_x, bar, sX + stage * kOpBytes + h * kBoxBytes, kx, mb * kTile + 128 * rank);
            tma_load_2d_pair(&a.tma_w, bar, sW + stage * kOpBytes + h * kBoxBytes, kx, nb * kTile + 128 * rank);
          }
          issued[stage] = phase;
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (!ok && leader) {
        // every load of both CTAs completes on the leader's full barriers: let them land (bounded)
        for (int s = 0; s < kStages; ++s)
          if (issued[s] != 0xFFFFFFFFu) mbar_wait_quiet(&full[s], issued[s], kWaitBudgetNs);
      }
    } else if (warp == 1 && lane == 0 && leader) {
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int tile = pair; ok && tile < tiles; tile += npairs) {
        for (int kc = ks0; ok && kc < ks1; kc += kChunkStages) {
          if (!mbar_wait(&acc_empty[acc], acc_phase ^ 1u, abort_flag, a.status, FB_DEV_TIMEOUT_EPI)) {
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * kTile);
          for (int ks = kc; ks < min(kc + kChunkStages, ks1); ++ks) {
            if (!mbar_wait(&full[stage], phase, abort_flag, a.status, FB_DEV_TIMEOUT_TMA)) {
              ok = false;
              break;
            }
            tc_fence_after_sync();
            const uint32_t x0 = smem_u32(sX + stage * kOpBytes), w0 = smem_u32(sW + stage * kOpBytes);
#pragma unroll
            for (int h = 0; h < kSub; ++h) {
#pragma unroll
              for (int k = 0; k < BK / 16; ++k)
                umma_bf16_ss_pair(d_tmem, sdesc_kmajor_sw128(x0 + h * kBoxBytes + 32 * k),
                                  sdesc_kmajor_sw128(w0 + h * kBoxBytes + 32 * k), a.idesc,
                                  (ks > kc || h > 0 || k > 0) ? 1u : 0u);
            }
            commit_pair(smem_u32(&empty[stage]), lead);
            if (++stage == kStages) {
              stage = 0;
              phase ^= 1u;
            }
          }
          if (!ok) break;
          commit_pair(smem_u32(&acc_full[acc]), lead);
          acc ^= 1;
          if (acc == 0) acc_phase ^= 1u;
        }
      }
      umma_commit_pair(mapa_shared(smem_u32(drain), lead));
      mbar_wait_quiet(drain, 0, kWaitBudgetNs);
    }
    if constexpr (SPLIT) {
      __syncwarp();
      cluster_sync_all();  // the partial sums are in shared memory; the barrier before the exit: they have been read
    }
  } else {
    reg_alloc<kEpiRegs>();
    const int quarter = warp & 3;  // the TMEM lanes a warp may read are fixed by warp % 4
    const int part = (warp - 4) >> 2;
    uint8_t* patch = sP + (warp - 4) * kPatchBytes;
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    for (int tile = pair; ok && tile < tiles; tile += npairs) {
      int mb, nb;
      place(a, tile, mb, nb);
      const int row0 = mb * kTile + 128 * rank + quarter * 32, col0 = nb * kTile + part * kCols;
      if (a.residual != nullptr && row0 + lane < a.m) {  // the row's residuals: in L2 by the time the sums are there
        const int line = a.res_f32 ? 32 : 64;
        for (int n = col0; n < min(col0 + kCols, a.n); n += line) {
          const int64_t at = static_cast<int64_t>(row0 + lane) * a.ld_res + n;
          asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const uint8_t*>(a.residual) + (a.res_f32 ? 4 : 2) * at));
        }
      }
      uint2 b[kCols / 32];  // the bias of this lane's four features of each step below
#pragma unroll
      for (int c = 0; c < kCols / 32; ++c) {
        const int n = col0 + 32 * c + 4 * (lane & 7);
        b[c] = a.vec && a.bias != nullptr && n + 4 <= a.n
                   ? __ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(a.bias) + n))
                   : make_uint2(0u, 0u);
      }
      float v[kCols];
#pragma unroll
      for (int j = 0; j < kCols; ++j) v[j] = 0.f;  // the sum over no K at all
      for (int kc = ks0; kc < ks1; kc += kChunkStages) {
        if (!mbar_wait(&acc_full[acc], acc_phase, abort_flag, a.status, FB_DEV_TIMEOUT_MMA)) {
          ok = false;
          break;
        }
        tc_fence_after_sync();
        promote<kCols, 32>(tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + acc * kTile + part * kCols, kc == ks0, v);
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive_remote(mapa_shared(smem_u32(&acc_empty[acc]), lead));
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1u;
      }
      if constexpr (SPLIT) {
        // [128 rows][256 columns]; the tensor core has read every stage. After a wait that gave up the values do not matter.
        float* sums = reinterpret_cast<float*>(smem);
        const int row = quarter * 32 + lane;
#pragma unroll
        for (int w = 0; w < kCols / 4; ++w)
          *reinterpret_cast<float4*>(sums + row * kTile + (((part * kCols / 4 + w) ^ (row & 7)) << 2)) =
              make_float4(v[4 * w], v[4 * w + 1], v[4 * w + 2], v[4 * w + 3]);
        __syncwarp();
        cluster_sync_all();
        const int first = mb * kTile + 128 * rank, live = max(0, min(128, a.m - first));
        for (int f0 = nb * kTile; f0 < min((nb + 1) * kTile, a.n); f0 += 128) {
          const bool whole = a.vec && f0 + 128 <= a.n;
          finish_share<ACT, kEpiWarps, kTile, true>(a, smem_u32(sums), f0 - nb * kTile, 128, first, live * split / a.splits,
                                                    live * (split + 1) / a.splits, f0, whole, lane_bias(a, f0, whole, lane),
                                                    warp - 4, lane, a.splits, rank, 2);
        }
        break;
      }
      if (!ok) break;
      if (row0 >= a.m) continue;
      // 32 columns at a time through the patch: row = lane, the 16-byte unit u of a row at place u ^ (row % 8)
#pragma unroll 1
      for (int c = 0; c < kCols / 32; ++c) {
        const int n0 = col0 + 32 * c;
        if (n0 >= a.n) break;
        const bool whole = a.vec && n0 + 32 <= a.n;  // every lane's four consecutive features are aligned vectors
        // eight lanes per row, four features each
        const int u = lane & 7, first = lane >> 3, n = n0 + 4 * u;
        float4 r[8];
        if (whole) residuals<8>(a, row0 + first, 4, a.m, n, r);
        __syncwarp();
#pragma unroll
        for (int k = 0; k < kCols / 32; ++k) {
          if (c == k) {
#pragma unroll
            for (int w = 0; w < 8; ++w)
              *reinterpret_cast<float4*>(patch + lane * 128 + ((w ^ (lane & 7)) << 4)) =
                  make_float4(v[32 * k + 4 * w], v[32 * k + 4 * w + 1], v[32 * k + 4 * w + 2], v[32 * k + 4 * w + 3]);
          }
        }
        __syncwarp();
        if (whole) {
          float4 z[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int row = first + 4 * i;
            z[i] = *reinterpret_cast<const float4*>(patch + row * 128 + ((u ^ (row & 7)) << 4));
          }
          const uint2 bc = c == 0 ? b[0] : c == 1 ? b[1] : c == 2 ? b[2] : b[3];
          finish<ACT, 8>(a, row0 + first, 4, a.m, n, a.half ? widen4<true>(bc) : widen4<false>(bc), r, z);
        } else {
          const int n1 = n0 + lane;
          const float b1 = n1 < a.n ? bias1(a, n1) : 0.f;
#pragma unroll 1
          for (int h = 0; h < 32; h += 8) {
            auto is = [&](int i) { return row0 + h + i < a.m && n1 < a.n; };
            auto where = [&](int i, int64_t ld) { return static_cast<int64_t>(row0 + h + i) * ld + n1; };
            float r1[8], z1[8];
            residuals1<8>(a, where, is, r1);
#pragma unroll
            for (int i = 0; i < 8; ++i)
              z1[i] = *reinterpret_cast<const float*>(patch + (h + i) * 128 + (((lane >> 2) ^ ((h + i) & 7)) << 4) + 4 * (lane & 3)) + b1;
            finish1<ACT, 8>(a, where, is, r1, z1);
          }
        }
      }
    }
  }
  __syncwarp();
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();  // the peer no longer signals this CTA; nobody reads this CTA's TMEM, or its partial sums
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem_base, kTmemCols);
  }
}
}  // namespace many

// Rows of a 16-bit matrix whose start or stride is not a multiple of 16 bytes, copied to rows of `ldo` elements (a
// multiple of 8): what TMA can read. The columns past k are never read (the tensor map ends at k). Eight elements per
// thread, one 16-byte store: inside a row from the four or five aligned words that hold them, near its ends one by one
// (a word there may reach out of the matrix).
__global__ void __launch_bounds__(256) align_rows_kernel(const uint16_t* __restrict__ in, int64_t ld, int64_t rows, int k,
                                                         uint16_t* __restrict__ out, int64_t ldo) {
  const int64_t per_row = ldo / 8, all = rows * per_row;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < all; i += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t row = i / per_row;
    const int c = static_cast<int>(i - row * per_row) * 8;
    const uint16_t* s = in + row * ld + c;
    uint32_t w[4];
    if (c >= 8 && c + 9 <= k) {
      if (reinterpret_cast<uintptr_t>(s) & 2u) {
        const uint32_t* p = reinterpret_cast<const uint32_t*>(s - 1);
        uint32_t v[5];
#pragma unroll
        for (int j = 0; j < 5; ++j) v[j] = __ldg(p + j);
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = __funnelshift_r(v[j], v[j + 1], 16);
      } else {
        const uint32_t* p = reinterpret_cast<const uint32_t*>(s);
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = __ldg(p + j);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t lo = c + 2 * j < k ? __ldg(s + 2 * j) : 0, hi = c + 2 * j + 1 < k ? __ldg(s + 2 * j + 1) : 0;
        w[j] = lo | hi << 16;
      }
    }
    *reinterpret_cast<uint4*>(out + row * ldo + c) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

template <typename K>
static cudaError_t launch(K kernel, const Args& a, int ctas, int cluster, int threads, int smem, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas, 1, 1);
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, a);
}
template <int ACT>
static cudaError_t go_few(const Args& a, int bt, int ctas, cudaStream_t st) {
  switch (bt) {
    case 16: return launch(few_kernel<16, ACT>, a, ctas, a.splits, Few<16>::kThreads, Few<16>::kSmemBytes, st);
    case 32: return launch(few_kernel<32, ACT>, a, ctas, a.splits, Few<32>::kThreads, Few<32>::kSmemBytes, st);
    case 64: return launch(few_kernel<64, ACT>, a, ctas, a.splits, Few<64>::kThreads, Few<64>::kSmemBytes, st);
    default: return launch(few_kernel<128, ACT>, a, ctas, a.splits, Few<128>::kThreads, Few<128>::kSmemBytes, st);
  }
}
// f(std::integral_constant<int, ACT>) for the activation of the call.
template <typename F>
static cudaError_t with_act(int act, F f) {
  switch (act) {
    case FB_ACT_RELU: return f(std::integral_constant<int, FB_ACT_RELU>());
    case FB_ACT_GELU: return f(std::integral_constant<int, FB_ACT_GELU>());
    case FB_ACT_GELU_TANH: return f(std::integral_constant<int, FB_ACT_GELU_TANH>());
    case FB_ACT_QUICK_GELU: return f(std::integral_constant<int, FB_ACT_QUICK_GELU>());
    case FB_ACT_SILU: return f(std::integral_constant<int, FB_ACT_SILU>());
    default: return f(std::integral_constant<int, FB_ACT_NONE>());
  }
}

static int encode_rows(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int64_t ld, int box_rows, bool half,
                       std::string& err) {
  EncodeTiledFn enc = encode_fn();
  if (!enc) {
    err = "cuTensorMapEncodeTiled unavailable (fb_init not run?)";
    return FB_ERR_INIT;
  }
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld) * 2};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(BK), static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t estr[2] = {1, 1};
  const CUresult r = enc(map, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
                         const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    err = "cuTensorMapEncodeTiled failed (" + std::to_string(static_cast<int>(r)) + ")";
    return FB_ERR_CUDA;
  }
  return FB_OK;
}

// Clusters of 2 s CTAs of many_kernel that run at once (a cluster stays inside one group of SMs, so fewer than the SMs
// alone would hold); asked of the driver once, in linear_act_setup.
static std::atomic<int> g_clusters[many::kMaxSplits + 1];

static int64_t up8(int64_t k) { return (k + 7) / 8 * 8; }
// A matrix's row stride as TMA sees it: a single row has none, so any will do.
static int64_t row_stride(int64_t ld, int rows, int k) { return rows == 1 ? up8(k) : ld; }
static bool tma_rows(const void* p, int64_t ld, int rows, int k) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && row_stride(ld, rows, k) % 8 == 0;
}
static int64_t copy_bytes(int rows, int k) { return 2 * static_cast<int64_t>(rows) * up8(k); }  // a multiple of 16

}  // namespace lact

std::string linear_act_setup() {
  using namespace lact;
  cudaError_t e = cudaSuccess;
  bool split_ok = true;
  auto raise = [&](auto kernel, int bytes) {
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  };
  for (int act = FB_ACT_NONE; act <= FB_ACT_SILU; ++act) {
    with_act(act, [&](auto c) {
      constexpr int ACT = decltype(c)::value;
      raise(few_kernel<16, ACT>, Few<16>::kSmemBytes);
      raise(few_kernel<32, ACT>, Few<32>::kSmemBytes);
      raise(few_kernel<64, ACT>, Few<64>::kSmemBytes);
      raise(few_kernel<128, ACT>, Few<128>::kSmemBytes);
      raise(many::many_kernel<ACT, false>, many::kSmemBytes);
      raise(many::many_kernel<ACT, true>, many::kSmemBytes);
      for (const void* k : {reinterpret_cast<const void*>(many::many_kernel<ACT, false>),
                            reinterpret_cast<const void*>(many::many_kernel<ACT, true>)}) {
        cudaFuncAttributes at;
        if (e == cudaSuccess) e = cudaFuncGetAttributes(&at, k);
        if (e == cudaSuccess && at.numRegs != many::kLaunchRegs) split_ok = false;
      }
      return cudaSuccess;
    });
  }
  // The register split takes more than a launch with fewer registers per thread would have: setmaxnreg.inc would wait
  // for good. So a build that compiled to another number is refused here.
  if (!split_ok) return "linear_act: many_kernel is not compiled to " + std::to_string(many::kLaunchRegs) + " registers";
  for (int s = 2; e == cudaSuccess && s <= many::kMaxSplits; ++s) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * s * 74, 1, 1);
    cfg.blockDim = dim3(many::kThreads, 1, 1);
    cfg.dynamicSmemBytes = many::kSmemBytes;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2 * s;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    e = cudaOccupancyMaxActiveClusters(&n, many::many_kernel<FB_ACT_NONE, true>, &cfg);
    g_clusters[s].store(n, std::memory_order_relaxed);
  }
  return e == cudaSuccess ? std::string() : std::string("cudaFuncSetAttribute(linear_act): ") + cudaGetErrorString(e);
}

int64_t linear_act_work_bytes(const fb_linear_act_args& p) {
  int64_t n = 0;
  if (p.m > 0 && p.n > 0 && p.k > 0) {
    if (!lact::tma_rows(p.x, p.ldx, p.m, p.k)) n += lact::copy_bytes(p.m, p.k);
    if (!lact::tma_rows(p.w, p.ldw, p.n, p.k)) n += lact::copy_bytes(p.n, p.k);
  }
  return n;
}

int launch_linear_act(const fb_linear_act_args& p, cudaStream_t st, std::string& err) {
  using namespace lact;
  auto bad = [&](int code, const char* what) {
    err = std::string("fb_linear_act: ") + what;
    return code;
  };
  if (p.m < 0 || p.n < 1 || p.k < 0) return bad(FB_ERR_ARG, "need m >= 0, n >= 1, k >= 0");
  if (p.m > (1 << 30) || p.n > (1 << 30) || p.k > (1 << 30)) return bad(FB_ERR_UNSUPPORTED, "m, n and k are at most 2^30");
  if (p.dtype != FB_BF16 && p.dtype != FB_F16) return bad(FB_ERR_UNSUPPORTED, "x and w must be FB_BF16 or FB_F16");
  if (p.out_dtype != p.dtype && p.out_dtype != FB_F32) return bad(FB_ERR_UNSUPPORTED, "out is of x's type or FB_F32");
  if (p.residual && p.residual_dtype != p.dtype && p.residual_dtype != FB_F32)
    return bad(FB_ERR_UNSUPPORTED, "residual is of x's type or FB_F32");
  if (p.act < FB_ACT_NONE || p.act > FB_ACT_SILU) return bad(FB_ERR_ARG, "unknown activation");
  if (p.m == 0) return FB_OK;
  if (!p.out || (p.k > 0 && (!p.x || !p.w))) return bad(FB_ERR_ARG, "null pointer");
  if ((p.k > 0 && (p.ldx < p.k || p.ldw < p.k)) || p.ld_out < p.n || (p.residual && p.ld_residual < p.n))
    return bad(FB_ERR_ARG, "a row stride is shorter than the row");
  auto align = [](const void* q, int n) { return reinterpret_cast<uintptr_t>(q) % n == 0; };
  const int osz = p.out_dtype == FB_F32 ? 4 : 2, rsz = p.residual_dtype == FB_F32 ? 4 : 2;
  if (!align(p.x, 2) || !align(p.w, 2) || !align(p.bias, 2) || !align(p.out, osz) || (p.residual && !align(p.residual, rsz)))
    return bad(FB_ERR_ALIGN, "a pointer is not aligned to its elements");
  std::string derr;
  DeviceState* dev = device_for(Operator::kLinearAct, derr);
  if (!dev) {
    err = derr;
    return FB_ERR_INIT;
  }
  Args a;
  memset(&a, 0, sizeof(a));
  const bool half = p.dtype == FB_F16;
  a.vec = align(p.out, 4 * osz) && p.ld_out % 4 == 0 && align(p.bias, 8) &&
          (!p.residual || (align(p.residual, 4 * rsz) && p.ld_residual % 4 == 0));
  a.num_kb = (p.k + BK - 1) / BK;
  const int64_t tiles_many = ((p.m + 255ll) / 256) * ((p.n + 255ll) / 256);
  // many_kernel's larger tiles pay once there is work for them; below, few_kernel is done sooner (no second CTA to meet, a
  // smaller tile to fill and write). Measured, few against many, each call with a cold L2: 256 x 3072 x 3072 (m x k x n)
  // 14.7 / 16.6 us, 2048 x 1024 x 1024 12.4 / 14.5, 1024 x 1024 x 4096 14.5 / 14.5, 1024 x 3072 x 3072 26.8 / 24.8,
  // 8192 x 1024 x 1024 26.8 / 20.7, 4608 x 3072 x 3072 82 / 60; up to 128 rows few_kernel's one token tile is never worse.
  // With many tiles and little K it is the epilogue that counts, which many_kernel overlaps (2000 x 100 x 17000 79 / 70;
  // with outputs written one by one, 17001, it is the slower of the two, 126 / 182).
  // Without depth (k = 0) there are no tensor maps, which many_kernel would prefetch: few_kernel then touches none.
  const bool many_rows =
      p.k > 0 && p.m > 128 && (static_cast<double>(p.m) * p.n * p.k >= 4294967296.0 || (a.vec && tiles_many >= kNumSms));
  const int bt = many_rows ? 128 : p.m <= 16 ? 16 : p.m <= 32 ? 32 : p.m <= 64 ? 64 : 128;
  if (p.k > 0) {
    const void *x = p.x, *w = p.w;
    int64_t ldx = row_stride(p.ldx, p.m, p.k), ldw = row_stride(p.ldw, p.n, p.k);
    const int64_t need = linear_act_work_bytes(p);
    if (need > 0) {
      if (p.work_bytes < need || !p.work || !align(p.work, 16))
        return bad(FB_ERR_ARG, "rows that do not start on 16 bytes need a workspace (fb_linear_act_work_bytes), 16-byte aligned");
      char* work = static_cast<char*>(p.work);
      auto copy = [&](const void*& q, int64_t& ld, int rows) {
        const int64_t chunks = rows * (up8(p.k) / 8);
        align_rows_kernel<<<static_cast<unsigned>(std::min<int64_t>((chunks + 255) / 256, 16 * kNumSms)), 256, 0, st>>>(static_cast<const uint16_t*>(q), ld, rows, p.k,
                                                                       reinterpret_cast<uint16_t*>(work), up8(p.k));
        q = work;
        ld = up8(p.k);
        work += copy_bytes(rows, p.k);
      };
      if (!tma_rows(p.x, p.ldx, p.m, p.k)) copy(x, ldx, p.m);
      if (!tma_rows(p.w, p.ldw, p.n, p.k)) copy(w, ldw, p.n);
      const cudaError_t e = cudaGetLastError();
      if (e != cudaSuccess) {
        err = std::string("fb_linear_act: ") + cudaGetErrorString(e);
        return FB_ERR_CUDA;
      }
    }
    int rc = encode_rows(&a.tma_w, w, p.n, p.k, ldw, kFeat, half, err);
    if (!rc) rc = encode_rows(&a.tma_x, x, p.m, p.k, ldx, bt, half, err);
    if (rc) return rc;
  }
  a.bias = p.bias;
  a.residual = p.residual;
  a.out = p.out;
  a.ld_res = p.ld_residual;
  a.ld_out = p.ld_out;
  a.m = p.m;
  a.n = p.n;
  a.half = half;
  a.res_f32 = p.residual_dtype == FB_F32;
  a.out_f32 = p.out_dtype == FB_F32;
  a.idesc = many_rows ? idesc_bf16_f32(256, 256, false) : idesc_bf16_f32(kFeat, bt, false);
  if (half) a.idesc &= ~((1u << 7) | (1u << 10));  // operand format 0: fp16
  a.status = dev->status;
  cudaError_t e;
  if (many_rows) {
    a.tiles_f = (p.n + 255) / 256;
    a.tiles_t = (p.m + 255) / 256;
    if (tiles_many > (1ll << 30)) return bad(FB_ERR_UNSUPPORTED, "too many output tiles");
    a.group = a.tiles_f <= 16 ? 4 : 16;
    const int pairs = dev->sm_count / 2;
    // Pairs that share a tile, as long as each gets two stages of K and the clusters all run at once.
    a.splits = 1;
    for (int s = 2; s <= many::kMaxSplits; ++s)
      if (tiles_many <= g_clusters[s].load(std::memory_order_relaxed) && a.num_kb >= 4 * s) a.splits = s;
    e = with_act(p.act, [&](auto c) {
      constexpr int ACT = decltype(c)::value;
      if (a.splits > 1)
        return launch(many::many_kernel<ACT, true>, a, static_cast<int>(2 * a.splits * tiles_many), 2 * a.splits, many::kThreads,
                      many::kSmemBytes, st);
      return launch(many::many_kernel<ACT, false>, a, static_cast<int>(2 * std::min<int64_t>(tiles_many, pairs)), 2, many::kThreads,
                    many::kSmemBytes, st);
    });
  } else {
    a.tiles_f = (p.n + kFeat - 1) / kFeat;
    a.tiles_t = (p.m + bt - 1) / bt;
    const int64_t tiles = static_cast<int64_t>(a.tiles_f) * a.tiles_t;
    if (tiles > (1ll << 27)) return bad(FB_ERR_UNSUPPORTED, "too many output tiles");
    // Split K over a cluster, at most two CTAs per SM and four K blocks at least per CTA, so that the busiest SM has the
    // least to do: 24 tiles take six CTAs each (144 SMs busy), 96 tiles three (two per SM instead of 96 SMs with one).
    a.splits = 1;
    for (int s = 2; s <= 8 && tiles * s <= 2 * kNumSms && a.num_kb >= 4 * s; ++s) {
      const int64_t now = (tiles * a.splits + kNumSms - 1) / kNumSms, then = (tiles * s + kNumSms - 1) / kNumSms;
      if (then * a.splits < now * s) a.splits = s;
    }
    const int ctas = static_cast<int>(tiles * a.splits);
    e = with_act(p.act, [&](auto c) { return go_few<decltype(c)::value>(a, bt, ctas, st); });
  }
  if (e != cudaSuccess) {
    err = std::string("fb_linear_act: ") + cudaGetErrorString(e);
    return FB_ERR_CUDA;
  }
  return FB_OK;
}

}  // namespace fb
