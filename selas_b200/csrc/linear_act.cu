// linear_act.cu — y = act(x w^T + bias) + residual with one rounding at the end, for any number of rows.
//
//   x [m, k], w [n, k] (nn.Linear), both bf16 or both fp16; bias [n] of their type; residual [m, n] of their type or
//   fp32; y [m, n] of their type or fp32. act: none, ReLU, GELU (erf or tanh), x * sigmoid(1.702 x), SiLU, on the fp32
//   accumulator.
//
// The weight is the tensor cores' M operand here and the tokens are N: a tile is 128 output features by BT = 16 .. 256
// tokens, so a single token costs one 16-column MMA per 16 of K instead of a 128-row tile of padding, and the kernel is
// what a few rows need to be: a stream of the weight through shared memory. Where the tiles are fewer than the SMs, a
// cluster of up to eight CTAs shares one: each takes a run of K, leaves its fp32 partial tile in shared memory, and
// finishes an equal share of the tile's tokens by adding the partials of all of them over distributed shared memory
// in rank order (no workspace, no atomics; the same call always gives the same bits).
//
// One CTA, 192 threads: warp 0 loads (TMA, 128-byte swizzle), warp 1 issues tcgen05.mma, warps 2..5 move the
// accumulator (TMEM lane = feature, column = token) to shared memory as [token][feature], and all six warps write the
// outputs: a warp takes one token's 128 features, four per lane, so bias, residual and output are contiguous accesses.
#include "gemm_common.cuh"

namespace fb {
namespace lact {

using gemm::BK;

constexpr int kFeat = 128;  // output features of a tile
constexpr int kThreads = 192;

struct Args {
  CUtensorMap tma_w, tma_x;
  const void* bias;
  const void* residual;
  void* out;
  int64_t ld_res, ld_out;
  int m, n, num_kb;
  int splits, tiles_f;
  int half;      // operands and 16-bit outputs are fp16 (else bf16)
  int res_f32, out_f32, act;
  int vec;       // four consecutive outputs (and residuals, biases) are aligned vectors
  uint32_t idesc;
  int* status;
};

template <int BT>
struct Cfg {
  // Two CTAs per SM up to 128 tokens, so that up to 296 tiles stream at once; one CTA of 192 KB at 256.
  static constexpr int kStages = BT == 16 ? 6 : BT == 32 ? 5 : BT == 64 ? 4 : BT == 128 ? 3 : 4;
  static constexpr int kWBytes = kFeat * BK * 2;
  static constexpr int kXBytes = BT * BK * 2;
  static constexpr int kStageBytes = kWBytes + kXBytes;
  static constexpr int kSmemBytes = kStages * kStageBytes + 256 + 1024;
  static constexpr int kTmemCols = BT < 32 ? 32 : BT;
  static constexpr int kSlots = BT == 256 ? kNumSms : 2 * kNumSms;  // CTAs resident at once
  static_assert(kStages * kStageBytes >= BT * kFeat * 4, "the fp32 tile takes the operand stages' place");
};

__device__ __forceinline__ float activate(float z, int act) {
  switch (act) {
    case FB_ACT_RELU: return z < 0.f ? 0.f : z;
    case FB_ACT_GELU: return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
    case FB_ACT_GELU_TANH: return gelu_tanh_f32(z);
    case FB_ACT_QUICK_GELU: return z / (1.0f + expf(-1.702f * z));
    case FB_ACT_SILU: return z / (1.0f + expf(-z));
    default: return z;
  }
}

// 16-bit value of the operands' type widened to fp32, and back.
__device__ __forceinline__ float widen(uint16_t v, int half) {
  return half ? __half2float(__ushort_as_half(v)) : bf16_bits_to_f32(v);
}
__device__ __forceinline__ uint16_t narrow(float v, int half) {
  return half ? __half_as_ushort(__float2half_rn(v)) : __bfloat16_as_ushort(__float2bfloat16_rn(v));
}

__device__ __forceinline__ float4 ld_shared_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// Four outputs of one token, features n0 .. n0 + 3 (fewer at the end of a row): bias, activation, residual, rounding.
__device__ __forceinline__ void finish4(const Args& a, int token, int n0, float4 acc) {
  float v[4] = {acc.x, acc.y, acc.z, acc.w};
  const int64_t ro = static_cast<int64_t>(token) * a.ld_res + n0;
  const int64_t oo = static_cast<int64_t>(token) * a.ld_out + n0;
  const uint16_t* bias = static_cast<const uint16_t*>(a.bias);
  if (a.vec && n0 + 4 <= a.n) {
    if (bias) {
      const uint2 u = __ldg(reinterpret_cast<const uint2*>(bias + n0));
      v[0] += widen(u.x & 0xFFFFu, a.half), v[1] += widen(u.x >> 16, a.half);
      v[2] += widen(u.y & 0xFFFFu, a.half), v[3] += widen(u.y >> 16, a.half);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = activate(v[j], a.act);
    if (a.residual) {
      if (a.res_f32) {
        const float4 r = *reinterpret_cast<const float4*>(static_cast<const float*>(a.residual) + ro);
        v[0] += r.x, v[1] += r.y, v[2] += r.z, v[3] += r.w;
      } else {
        const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(a.residual) + ro);
        v[0] += widen(u.x & 0xFFFFu, a.half), v[1] += widen(u.x >> 16, a.half);
        v[2] += widen(u.y & 0xFFFFu, a.half), v[3] += widen(u.y >> 16, a.half);
      }
    }
    if (a.out_f32) {
      *reinterpret_cast<float4*>(static_cast<float*>(a.out) + oo) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
      uint2 u;
      u.x = narrow(v[0], a.half) | static_cast<uint32_t>(narrow(v[1], a.half)) << 16;
      u.y = narrow(v[2], a.half) | static_cast<uint32_t>(narrow(v[3], a.half)) << 16;
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + oo) = u;
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (n0 + j >= a.n) return;
    float z = v[j];
    if (bias) z += widen(__ldg(bias + n0 + j), a.half);
    z = activate(z, a.act);
    if (a.residual)
      z += a.res_f32 ? static_cast<const float*>(a.residual)[ro + j]
                     : widen(static_cast<const uint16_t*>(a.residual)[ro + j], a.half);
    if (a.out_f32) {
      static_cast<float*>(a.out)[oo + j] = z;
    } else {
      static_cast<uint16_t*>(a.out)[oo + j] = narrow(z, a.half);
    }
  }
}

template <int BT>
__global__ void __launch_bounds__(kThreads) linear_act_kernel(const __grid_constant__ Args a) {
  using C = Cfg<BT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sW = smem;
  uint8_t* sX = smem + C::kStages * C::kWBytes;
  float* tile = reinterpret_cast<float*>(smem);  // [BT][128] fp32, once every stage has been consumed
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kStages * C::kStageBytes);
  uint64_t* empty = full + C::kStages;
  uint64_t* done = empty + C::kStages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = warp_id(), lane = lane_id();
  const int rank = a.splits > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int t = blockIdx.x / a.splits;
  const int f0 = (t % a.tiles_f) * kFeat, t0 = (t / a.tiles_f) * BT;
  const int kb0 = static_cast<int>(static_cast<int64_t>(a.num_kb) * rank / a.splits);
  const int kb1 = static_cast<int>(static_cast<int64_t>(a.num_kb) * (rank + 1) / a.splits);

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(done, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&a.tma_w);
    tma_prefetch_desc(&a.tma_x);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0, issued[C::kStages];
      for (int s = 0; s < C::kStages; ++s) issued[s] = 0xFFFFFFFFu;
      bool ok = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&empty[stage], phase ^ 1u, abort_flag, a.status, FB_DEV_TIMEOUT_MMA)) {
          ok = false;
          break;
        }
        mbar_arrive_expect_tx(&full[stage], C::kStageBytes);
        tma_load_2d(&a.tma_w, &full[stage], sW + stage * C::kWBytes, kb * BK, f0);
        tma_load_2d(&a.tma_x, &full[stage], sX + stage * C::kXBytes, kb * BK, t0);
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
      int stage = 0;
      uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&full[stage], phase, abort_flag, a.status, FB_DEV_TIMEOUT_TMA)) break;
        tc_fence_after_sync();
        const uint32_t w0 = smem_u32(sW + stage * C::kWBytes), x0 = smem_u32(sX + stage * C::kXBytes);
#pragma unroll
        for (int k = 0; k < BK / 16; ++k)
          umma_bf16_ss(tmem_base, sdesc_kmajor_sw128(w0 + 32 * k), sdesc_kmajor_sw128(x0 + 32 * k), a.idesc,
                       (kb > kb0 || k > 0) ? 1u : 0u);
        umma_commit(&empty[stage]);
        if (++stage == C::kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      umma_commit(done);  // every MMA issued so far: the accumulator is complete and the stages are free
      mbar_wait_quiet(done, 0, kWaitBudgetNs);
    }
  } else {
    // The accumulator to shared memory. With no K at all (k == 0) it was never written: zeros.
    const int quarter = warp & 3;  // the TMEM lanes a warp may read are fixed by warp % 4
    const bool ok = mbar_wait(done, 0, abort_flag, a.status, FB_DEV_TIMEOUT_MMA);
    tc_fence_after_sync();
    constexpr int CW = BT < 32 ? 16 : 32;
    const int f = quarter * 32 + lane;
#pragma unroll 1
    for (int c = 0; c < BT; c += CW) {
      uint32_t r[CW];
      const uint32_t at = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + c;
      if (ok && kb1 > kb0) {
        if constexpr (CW == 16) {
          tmem_ld_32x32b_x16(at, r);
        } else {
          tmem_ld_32x32b_x32(at, r);
        }
        tmem_ld_wait();
      } else {
#pragma unroll
        for (int j = 0; j < CW; ++j) r[j] = 0u;
      }
#pragma unroll
      for (int j = 0; j < CW; ++j) tile[(c + j) * kFeat + f] = __uint_as_float(r[j]);
    }
  }
  __syncwarp();
  tc_fence_before_sync();
  if (a.splits > 1) {
    cluster_sync_all();
  } else {
    __syncthreads();
  }

  // This CTA's share of the tile's tokens, one token per warp at a time.
  const int live = min(BT, a.m - t0);
  const int j1 = live * (rank + 1) / a.splits;
  const uint32_t base = smem_u32(tile) + 16 * lane;
  for (int j = live * rank / a.splits + warp; j < j1; j += kThreads / 32) {
    float4 v;
    if (a.splits > 1) {
      v = ld_shared_cluster_f4(mapa_shared(base + j * kFeat * 4, 0));
      for (int s = 1; s < a.splits; ++s) {
        const float4 u = ld_shared_cluster_f4(mapa_shared(base + j * kFeat * 4, s));
        v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
      }
    } else {
      v = *reinterpret_cast<const float4*>(tile + j * kFeat + 4 * lane);
    }
    if (f0 + 4 * lane < a.n) finish4(a, t0 + j, f0 + 4 * lane, v);
  }
  __syncwarp();
  if (a.splits > 1) {
    cluster_sync_all();  // nobody reads this CTA's tile any more
  } else {
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, C::kTmemCols);
  }
}

// Rows of a 16-bit matrix whose start or stride is not a multiple of 16 bytes, copied to rows of `ldo` elements (a
// multiple of 8): what TMA can read. The columns past k are never read (the tensor map ends at k).
__global__ void __launch_bounds__(256) align_rows_kernel(const uint16_t* __restrict__ in, int64_t ld, int64_t rows, int k,
                                                         uint16_t* __restrict__ out, int64_t ldo) {
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x)
    for (int c = threadIdx.x; c < k; c += 256) out[row * ldo + c] = __ldg(in + row * ld + c);
}

template <int BT>
static cudaError_t go(const Args& a, int ctas, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas, 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = Cfg<BT>::kSmemBytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = a.splits;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, linear_act_kernel<BT>, a);
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
  e = e ? e : cudaFuncSetAttribute(linear_act_kernel<16>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<16>::kSmemBytes);
  e = e ? e : cudaFuncSetAttribute(linear_act_kernel<32>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<32>::kSmemBytes);
  e = e ? e : cudaFuncSetAttribute(linear_act_kernel<64>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<64>::kSmemBytes);
  e = e ? e : cudaFuncSetAttribute(linear_act_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<128>::kSmemBytes);
  e = e ? e : cudaFuncSetAttribute(linear_act_kernel<256>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<256>::kSmemBytes);
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
  const int bt = p.m <= 16 ? 16 : p.m <= 32 ? 32 : p.m <= 64 ? 64 : p.m <= 128 ? 128 : 256;
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
  a.num_kb = (p.k + BK - 1) / BK;
  a.half = half;
  a.res_f32 = p.residual_dtype == FB_F32;
  a.out_f32 = p.out_dtype == FB_F32;
  a.act = p.act;
  a.vec = align(p.out, 4 * osz) && p.ld_out % 4 == 0 && align(p.bias, 8) &&
          (!p.residual || (align(p.residual, 4 * rsz) && p.ld_residual % 4 == 0));
  a.idesc = idesc_bf16_f32(kFeat, bt, false);
  if (half) a.idesc &= ~((1u << 7) | (1u << 10));  // operand format 0: fp16
  a.status = dev->status;
  a.tiles_f = (p.n + kFeat - 1) / kFeat;
  const int64_t tiles = static_cast<int64_t>(a.tiles_f) * ((p.m + bt - 1) / bt);
  if (tiles > (1ll << 27)) return bad(FB_ERR_UNSUPPORTED, "too many output tiles");
  // Split K over a cluster while that still fits the SMs in one go and leaves every CTA four K steps.
  a.splits = 1;
  while (a.splits < 8 && tiles * (a.splits + 1) <= kNumSms && a.num_kb >= 4 * (a.splits + 1)) ++a.splits;
  const int ctas = static_cast<int>(tiles * a.splits);
  cudaError_t e = bt == 16    ? go<16>(a, ctas, st)
                  : bt == 32  ? go<32>(a, ctas, st)
                  : bt == 64  ? go<64>(a, ctas, st)
                  : bt == 128 ? go<128>(a, ctas, st)
                              : go<256>(a, ctas, st);
  if (e != cudaSuccess) {
    err = std::string("fb_linear_act: ") + cudaGetErrorString(e);
    return FB_ERR_CUDA;
  }
  return FB_OK;
}

}  // namespace fb
