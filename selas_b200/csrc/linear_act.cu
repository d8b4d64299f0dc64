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
// Precision: the tensor core adds into its accumulator with less care than an fp32 add (over K = 12288 the error grew to
// 1.3e-5 of the result's norm), so an accumulator takes 1024 of K at most; the epilogue warps then add it to fp32
// registers, which are the sum proper, while the other TMEM buffer takes the next 1024. That costs 2 % of the time at
// most (every 512 cost 10 %) and holds the error of an fp32 output near 1e-6.
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
// z < 0 and z - z h otherwise, h = erfc(|x|) / 2, which keeps the small values of the negative side. With CUDA's erff the
// epilogue of a 256 x 256 tile at K = 3072 took longer than its products. The sigmoids divide by 1 + exp with the
// hardware's exp2 and division (2 ulp); tanh(u) = 2 sigmoid(2u) - 1.
template <int ACT>
__device__ __forceinline__ float activate(float z) {
  if constexpr (ACT == FB_ACT_RELU) return z < 0.f ? 0.f : z;  // keeps a NaN
  if constexpr (ACT == FB_ACT_GELU) {
    const float x = fabsf(z) * 0.70710678118654752f;
    const float t = __fdividef(1.0f, fmaf(0.3275911f, x, 1.0f));
    float h = fmaf(t, 0.5f * 1.061405429f, 0.5f * -1.453152027f);
    h = fmaf(h, t, 0.5f * 1.421413741f);
    h = fmaf(h, t, 0.5f * -0.284496736f);
    h = fmaf(h, t, 0.5f * 0.254829592f);
    const float zh = z * (h * t * __expf(-x * x));
    return z < 0.f ? zh : z - zh;
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
__device__ __forceinline__ float widen(uint32_t v, int half) {
  return half ? __half2float(__ushort_as_half(static_cast<uint16_t>(v))) : __uint_as_float(v << 16);
}
__device__ __forceinline__ uint32_t narrow(float v, int half) {
  return half ? __half_as_ushort(__float2half_rn(v)) : __bfloat16_as_ushort(__float2bfloat16_rn(v));
}
__device__ __forceinline__ float4 widen4(uint2 u, int half) {
  return make_float4(widen(u.x & 0xFFFFu, half), widen(u.x >> 16, half), widen(u.y & 0xFFFFu, half), widen(u.y >> 16, half));
}

__device__ __forceinline__ float4 ld_shared_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// Four consecutive features n0 .. n0 + 3 of a token as aligned vectors (n0 + 4 <= n), and one feature of any alignment.
__device__ __forceinline__ float4 bias4(const Args& a, int n0) {
  if (a.bias == nullptr) return make_float4(0.f, 0.f, 0.f, 0.f);
  return widen4(__ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(a.bias) + n0)), a.half);
}
__device__ __forceinline__ float4 residual4(const Args& a, int token, int n0) {
  if (a.residual == nullptr) return make_float4(0.f, 0.f, 0.f, 0.f);
  const int64_t at = static_cast<int64_t>(token) * a.ld_res + n0;
  if (a.res_f32) return *reinterpret_cast<const float4*>(static_cast<const float*>(a.residual) + at);
  return widen4(*reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(a.residual) + at), a.half);
}
template <int ACT>
__device__ __forceinline__ void finish4(const Args& a, int token, int n0, float4 z, float4 b, float4 r) {
  const float y0 = activate<ACT>(z.x + b.x) + r.x, y1 = activate<ACT>(z.y + b.y) + r.y;
  const float y2 = activate<ACT>(z.z + b.z) + r.z, y3 = activate<ACT>(z.w + b.w) + r.w;
  const int64_t at = static_cast<int64_t>(token) * a.ld_out + n0;
  if (a.out_f32) {
    *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) = make_float4(y0, y1, y2, y3);
  } else {
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + at) =
        make_uint2(narrow(y0, a.half) | narrow(y1, a.half) << 16, narrow(y2, a.half) | narrow(y3, a.half) << 16);
  }
}
__device__ __forceinline__ float bias1(const Args& a, int n) {
  return a.bias == nullptr ? 0.f : widen(__ldg(static_cast<const uint16_t*>(a.bias) + n), a.half);
}
__device__ __forceinline__ float residual1(const Args& a, int token, int n) {
  if (a.residual == nullptr) return 0.f;
  const int64_t at = static_cast<int64_t>(token) * a.ld_res + n;
  return a.res_f32 ? static_cast<const float*>(a.residual)[at] : widen(static_cast<const uint16_t*>(a.residual)[at], a.half);
}
template <int ACT>
__device__ __forceinline__ void finish1(const Args& a, int token, int n, float z, float b, float r) {
  const float y = activate<ACT>(z + b) + r;
  const int64_t at = static_cast<int64_t>(token) * a.ld_out + n;
  if (a.out_f32) {
    static_cast<float*>(a.out)[at] = y;
  } else {
    static_cast<uint16_t*>(a.out)[at] = static_cast<uint16_t>(narrow(y, a.half));
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
  float4 b;  // of features f0 + 4 lane + 0 .. 3, or f0 + lane + 32 * 0 .. 3
  if (whole) {
    b = bias4(a, f0 + 4 * lane);
  } else {
    b.x = f0 + lane < a.n ? bias1(a, f0 + lane) : 0.f;
    b.y = f0 + lane + 32 < a.n ? bias1(a, f0 + lane + 32) : 0.f;
    b.z = f0 + lane + 64 < a.n ? bias1(a, f0 + lane + 64) : 0.f;
    b.w = f0 + lane + 96 < a.n ? bias1(a, f0 + lane + 96) : 0.f;
  }
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

  // U tokens per warp at a time: a lane finishes four features of each.
  constexpr int U = 2;
  const uint32_t base = smem_u32(tile);
  if (whole) {
    const int n0 = f0 + 4 * lane;
#pragma unroll 1
    for (int j = j0 + warp; j < j1; j += U * C::kWarps) {
      float4 r[U], z[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int ju = min(j + u * C::kWarps, BT - 1);  // past the share: read, not written
        z[u] = *reinterpret_cast<const float4*>(tile + ju * kFeat + 4 * lane);
        if (j + u * C::kWarps < j1) r[u] = residual4(a, t0 + j + u * C::kWarps, n0);
      }
      if (a.splits > 1) {
#pragma unroll
        for (int u = 0; u < U; ++u) z[u] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int s = 0; s < a.splits; ++s) {
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int ju = min(j + u * C::kWarps, BT - 1);
            const float4 p = ld_shared_cluster_f4(mapa_shared(base + (ju * kFeat + 4 * lane) * 4, s));
            z[u].x += p.x, z[u].y += p.y, z[u].z += p.z, z[u].w += p.w;
          }
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (j + u * C::kWarps < j1) finish4<ACT>(a, t0 + j + u * C::kWarps, n0, z[u], b, r[u]);
    }
  } else {
    const float bs[4] = {b.x, b.y, b.z, b.w};
#pragma unroll 1
    for (int j = j0 + warp; j < j1; j += U * C::kWarps) {
      float r[U][4], z[U][4];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int ju = j + u * C::kWarps;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int n = f0 + lane + 32 * i;
          r[u][i] = ju < j1 && n < a.n ? residual1(a, t0 + ju, n) : 0.f;
          z[u][i] = 0.f;
        }
      }
#pragma unroll 2
      for (int s = 0; s < a.splits; ++s) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int ju = min(j + u * C::kWarps, BT - 1);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float p;
            if (a.splits > 1) {
              asm volatile("ld.shared::cluster.f32 %0, [%1];"
                           : "=f"(p)
                           : "r"(mapa_shared(base + (ju * kFeat + lane + 32 * i) * 4, s))
                           : "memory");
            } else {
              p = tile[ju * kFeat + lane + 32 * i];
            }
            z[u][i] += p;
          }
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int n = f0 + lane + 32 * i;
          if (j + u * C::kWarps < j1 && n < a.n) finish1<ACT>(a, t0 + j + u * C::kWarps, n, z[u][i], bs[i], r[u][i]);
        }
    }
  }
  __syncwarp();
  if (a.splits > 1) {
    // Nobody reads this CTA's tile any more: what was read has been used, so this barrier orders no memory (with
    // release semantics it would also wait for the outputs to reach L2).
    asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
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
namespace many {
constexpr int kTile = 256;
constexpr int kEpiWarps = 8;
// Three warpgroups: loads and MMAs (two of its warps idle), and the two of the epilogue, which take the registers that
// the first gives back. 128 x 40 + 256 x 232 = 384 x 168, what the block is launched with.
constexpr int kThreads = 128 + 32 * kEpiWarps;
constexpr int kLeanRegs = 40, kEpiRegs = 232;
constexpr int kSub = 2;
constexpr int kStages = 3;
constexpr int kChunkStages = 8;
constexpr int kBoxBytes = 128 * BK * 2;
constexpr int kOpBytes = kSub * kBoxBytes;
constexpr int kStageBytes = 2 * kOpBytes;
constexpr int kPatchBytes = 32 * 32 * 4;
constexpr int kSmemBytes = kStages * kStageBytes + kEpiWarps * kPatchBytes + 256 + 1024;
constexpr uint32_t kTmemCols = 512;

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

template <int ACT>
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
  const int rank = static_cast<int>(cluster_ctarank());
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
  const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;
  const int tiles = a.tiles_f * a.tiles_t;
  const int nstage = (a.num_kb + kSub - 1) / kSub;  // a K tail past the end is zero-filled by TMA

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
        for (int ks = 0; ks < nstage; ++ks) {
          if (!mbar_wait(&empty[stage], phase ^ 1u, abort_flag, a.status, FB_DEV_TIMEOUT_MMA)) {
            ok = false;
            break;
          }
          const uint32_t bar = mapa_shared(smem_u32(&full[stage]), 0);
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
        for (int kc = 0; ok && kc < nstage; kc += kChunkStages) {
          if (!mbar_wait(&acc_empty[acc], acc_phase ^ 1u, abort_flag, a.status, FB_DEV_TIMEOUT_EPI)) {
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * kTile);
          for (int ks = kc; ks < min(kc + kChunkStages, nstage); ++ks) {
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
            umma_commit_pair_both(smem_u32(&empty[stage]));
            if (++stage == kStages) {
              stage = 0;
              phase ^= 1u;
            }
          }
          if (!ok) break;
          umma_commit_pair_both(smem_u32(&acc_full[acc]));
          acc ^= 1;
          if (acc == 0) acc_phase ^= 1u;
        }
      }
      umma_commit_pair(mapa_shared(smem_u32(drain), 0));
      mbar_wait_quiet(drain, 0, kWaitBudgetNs);
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
      const int row0 = mb * kTile + 128 * rank + quarter * 32;
      if (a.residual != nullptr && row0 + lane < a.m) {  // the row's 128 residuals: in L2 by the time the sums are there
        const int n0 = nb * kTile + part * 128, line = a.res_f32 ? 32 : 64;
        for (int n = n0; n < min(n0 + 128, a.n); n += line) {
          const int64_t at = static_cast<int64_t>(row0 + lane) * a.ld_res + n;
          asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const uint8_t*>(a.residual) + (a.res_f32 ? 4 : 2) * at));
        }
      }
      float v[128];
      for (int kc = 0; kc < nstage; kc += kChunkStages) {
        if (!mbar_wait(&acc_full[acc], acc_phase, abort_flag, a.status, FB_DEV_TIMEOUT_MMA)) {
          ok = false;
          break;
        }
        tc_fence_after_sync();
        promote<128, 32>(tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + acc * kTile + part * 128, kc == 0, v);
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive_remote(mapa_shared(smem_u32(&acc_empty[acc]), 0));
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1u;
      }
      if (!ok) break;
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        const int n0 = nb * kTile + part * 128 + 32 * c;
        if (n0 < a.n && row0 < a.m) {
          // the patch: row = lane, the 16-byte unit u of a row at place u ^ (row % 8)
          __syncwarp();
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (c == k) {
#pragma unroll
              for (int u = 0; u < 8; ++u)
                *reinterpret_cast<float4*>(patch + lane * 128 + ((u ^ (lane & 7)) << 4)) =
                    make_float4(v[32 * k + 4 * u], v[32 * k + 4 * u + 1], v[32 * k + 4 * u + 2], v[32 * k + 4 * u + 3]);
            }
          }
          __syncwarp();
          if (a.vec && n0 + 32 <= a.n) {
            const int u = lane & 7, n = n0 + 4 * u;
            const float4 b = bias4(a, n);
            float4 r[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int row = 4 * i + (lane >> 3);
              if (row0 + row < a.m) r[i] = residual4(a, row0 + row, n);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int row = 4 * i + (lane >> 3);
              const float4 z = *reinterpret_cast<const float4*>(patch + row * 128 + ((u ^ (row & 7)) << 4));
              if (row0 + row < a.m) finish4<ACT>(a, row0 + row, n, z, b, r[i]);
            }
          } else {
            const int n = n0 + lane;
            const float b = n < a.n ? bias1(a, n) : 0.f;
            const int rows = n < a.n ? min(32, a.m - row0) : 0;
#pragma unroll 4
            for (int row = 0; row < rows; ++row) {
              const float z = *reinterpret_cast<const float*>(patch + row * 128 + (((lane >> 2) ^ (row & 7)) << 4) + 4 * (lane & 3));
              finish1<ACT>(a, row0 + row, n, z, b, residual1(a, row0 + row, n));
            }
          }
        }
      }
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();  // the peer no longer signals this CTA and nobody reads this CTA's TMEM
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem_base, kTmemCols);
  }
}
}  // namespace many

// Rows of a 16-bit matrix whose start or stride is not a multiple of 16 bytes, copied to rows of `ldo` elements (a
// multiple of 8): what TMA can read. The columns past k are never read (the tensor map ends at k).
__global__ void __launch_bounds__(256) align_rows_kernel(const uint16_t* __restrict__ in, int64_t ld, int64_t rows, int k,
                                                         uint16_t* __restrict__ out, int64_t ldo) {
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x)
    for (int c = threadIdx.x; c < k; c += 256) out[row * ldo + c] = __ldg(in + row * ld + c);
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
      raise(many::many_kernel<ACT>, many::kSmemBytes);
      return cudaSuccess;
    });
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
  DeviceState* dev = current_device(derr);
  if (!dev) {
    err = derr;
    return FB_ERR_INIT;
  }
  Args a;
  memset(&a, 0, sizeof(a));
  const bool half = p.dtype == FB_F16;
  a.num_kb = (p.k + BK - 1) / BK;
  const int64_t tiles_many = ((p.m + 255ll) / 256) * ((p.n + 255ll) / 256);
  const int64_t tiles_few = ((p.m + 127ll) / 128) * ((p.n + 127ll) / 128);
  // many_kernel where 256 x 256 tiles keep the pairs busy.
  static const int force = getenv("LACT") ? atoi(getenv("LACT")) : 0;
  const bool many_rows = force ? force == 2 : p.m > 128 && tiles_many >= 37;
  const int bt = many_rows ? 128 : p.m <= 16 ? 16 : p.m <= 32 ? 32 : p.m <= 64 ? 64 : 128;
  (void)tiles_few;
  if (p.k > 0) {
    const void *x = p.x, *w = p.w;
    int64_t ldx = row_stride(p.ldx, p.m, p.k), ldw = row_stride(p.ldw, p.n, p.k);
    const int64_t need = linear_act_work_bytes(p);
    if (need > 0) {
      if (p.work_bytes < need || !p.work || !align(p.work, 16))
        return bad(FB_ERR_ARG, "rows that do not start on 16 bytes need a workspace (fb_linear_act_work_bytes), 16-byte aligned");
      char* work = static_cast<char*>(p.work);
      auto copy = [&](const void*& q, int64_t& ld, int rows) {
        align_rows_kernel<<<std::min(rows, 16 * kNumSms), 256, 0, st>>>(static_cast<const uint16_t*>(q), ld, rows, p.k,
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
  a.vec = align(p.out, 4 * osz) && p.ld_out % 4 == 0 && align(p.bias, 8) &&
          (!p.residual || (align(p.residual, 4 * rsz) && p.ld_residual % 4 == 0));
  a.idesc = many_rows ? idesc_bf16_f32(256, 256, false) : idesc_bf16_f32(kFeat, bt, false);
  if (half) a.idesc &= ~((1u << 7) | (1u << 10));  // operand format 0: fp16
  a.status = dev->status;
  cudaError_t e;
  if (many_rows) {
    a.tiles_f = (p.n + 255) / 256;
    a.tiles_t = (p.m + 255) / 256;
    if (tiles_many > (1ll << 30)) return bad(FB_ERR_UNSUPPORTED, "too many output tiles");
    a.group = a.tiles_f <= 16 ? 4 : 16;
    const int pairs = static_cast<int>(std::min<int64_t>(tiles_many, dev->sm_count / 2));
    e = with_act(p.act, [&](auto c) {
      return launch(many::many_kernel<decltype(c)::value>, a, 2 * pairs, 2, many::kThreads, many::kSmemBytes, st);
    });
  } else {
    a.tiles_f = (p.n + kFeat - 1) / kFeat;
    a.tiles_t = (p.m + bt - 1) / bt;
    const int64_t tiles = static_cast<int64_t>(a.tiles_f) * a.tiles_t;
    if (tiles > (1ll << 27)) return bad(FB_ERR_UNSUPPORTED, "too many output tiles");
    // Split K over a cluster until every SM has a CTA, as long as each gets four K blocks.
    a.splits = 1;
    while (a.splits < 8 && tiles * (a.splits + 1) <= kNumSms && a.num_kb >= 4 * (a.splits + 1)) ++a.splits;
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
