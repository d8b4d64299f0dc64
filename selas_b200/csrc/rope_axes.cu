// rope_axes.cu — rotary positions with several axes, applied straight from the position ids.
//
// Token l has one position per axis a, ids[l, a]; axis a owns d_a / 2 rotation slots with the frequencies
// theta^(-2j / d_a), and the slots of all axes lie one after the other (the order of selas's rope_tables,
// flux.py:106-114). Slot s turns one pair of a head's elements by phi = ids[l, axis(s)] * omega_s: the pair
// (2s, 2s + 1) (interleaved, flux.py:117-121) or (s, s + hd / 2) (halves). The turn is orthogonal, so the
// gradient is the same kernel with -phi.
//
// Angles: phi / 2 pi is formed in 64 bits (one multiply by omega / 2 pi, minus its nearest whole number), which
// keeps positions of millions exact to ~1e-9 turns, and only the fraction in [-1/2, 1/2] goes to sincospif in 32 bits: rounded
// to 2^-26 turns, which moves an fp32 result by 1e-7 of its pair at most and is far below the step of a 16-bit one.
//
// Bound: HBM, every element read once and written once. A group of threads owns a token and up to twelve of its heads, of q
// and of k alike: each thread keeps the sines and cosines of its own slots in registers for all of them, so no table is read
// from memory. Measured (q and k of 24 heads x 128 in bf16): 61440 tokens, 1.51 GB, 229 us = 6.6 TB/s, the speed of a copy;
// 4608 tokens read in place from a fused projection, 113 MB, 22.5 us, of which a copy of that layout takes 22 to 25 too.
#include "fb_internal.h"

namespace fb {
namespace rope {

constexpr int kMaxSlots = 256;  // head_dim <= 512
constexpr int kThreads = 256;

struct Tensor {
  const void* x;
  void* out;
  int64_t xb, xh, xl;  // strides of x: image, head, token (elements)
  int64_t ob, oh, ol;
  int heads;
};

struct Args {
  Tensor t[2];
  int heads;        // of all tensors; head h of tensor 1 is number t[0].heads + h
  int seq;
  uint32_t tokens;  // batch * seq
  uint32_t items;   // tokens * runs of heads
  int per_item;     // consecutive heads of a work item
  int half;         // head_dim / 2
  int tpr;          // threads per head row
  int inverse;
  const void* ids;
  int ids_type;     // fb_ids_type
  int64_t ib, il, ia;
  double turns[kMaxSlots];    // omega / 2 pi of each slot
  uint8_t axis[kMaxSlots];
};

__device__ __forceinline__ double load_id(const Args& a, int64_t at) {
  switch (a.ids_type) {
    case FB_IDS_F32: return static_cast<double>(static_cast<const float*>(a.ids)[at]);
    case FB_IDS_F64: return static_cast<const double*>(a.ids)[at];
    case FB_IDS_I32: return static_cast<double>(static_cast<const int32_t*>(a.ids)[at]);
    default: return static_cast<double>(static_cast<const long long*>(a.ids)[at]);
  }
}

// V consecutive elements of type T. Wide: the 16 bytes of one vector access, worked on as 32-bit words (two 16-bit values
// are widened and rounded as a pair); else element by element.
template <typename T, int V>
struct Chunk;
template <>
struct Chunk<float, 4> {
  float4 v;
  __device__ __forceinline__ void get(float (&f)[4]) const { f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w; }
  __device__ __forceinline__ void set(const float (&f)[4]) { v = make_float4(f[0], f[1], f[2], f[3]); }
};
template <>
struct Chunk<__nv_bfloat16, 8> {
  uint4 v;
  __device__ __forceinline__ void get(float (&f)[8]) const {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
  __device__ __forceinline__ void set(const float (&f)[8]) {
    v = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  }
};
template <>
struct Chunk<__half, 8> {
  uint4 v;
  __device__ __forceinline__ void get(float (&f)[8]) const {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = p.x, f[2 * i + 1] = p.y;
    }
  }
  __device__ __forceinline__ void set(const float (&f)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    v = make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <typename T>
struct Chunk<T, 1> {
  T e;
  __device__ __forceinline__ void get(float (&f)[1]) const { f[0] = static_cast<float>(e); }
  __device__ __forceinline__ void set(const float (&f)[1]) { e = static_cast<T>(f[0]); }
};
template <typename T>
struct Chunk<T, 2> {
  T e[2];
  __device__ __forceinline__ void get(float (&f)[2]) const { f[0] = static_cast<float>(e[0]), f[1] = static_cast<float>(e[1]); }
  __device__ __forceinline__ void set(const float (&f)[2]) { e[0] = static_cast<T>(f[0]), e[1] = static_cast<T>(f[1]); }
};

// Shared memory of a block of 256 threads for the rows on their way: 12 chunks of 16 bytes a thread, four blocks per SM.
constexpr int kRows = 12;

// A work item is one token and a run of heads: a group of `tpr` threads turns its rows, a thread's share of a row being
// one chunk of V elements (interleaved: V / 2 slots), or two chunks half a row apart (halves: V slots). Wide rows are
// all put on their way to shared memory first (each thread its own chunks, so nothing is waited for together) and the
// angles are worked out while they come.
template <typename T, int V, bool HALVES>
__global__ void __launch_bounds__(kThreads, 4) rope_axes_kernel(const __grid_constant__ Args a) {
  constexpr int S = HALVES ? V : V / 2;  // slots of a thread
  constexpr bool WIDE = V * sizeof(T) == 16;
  using C = Chunk<T, V>;
  extern __shared__ __align__(16) uint8_t staged[];
  // The slots' constants are read by different lanes at different places, which the constant cache serves one by one:
  // from shared memory they come at once.
  __shared__ double turns[kMaxSlots];
  __shared__ uint8_t axis[kMaxSlots];
  const int groups = kThreads / a.tpr;
  const int g = threadIdx.x / a.tpr;
  const int r = threadIdx.x - g * a.tpr;
  const uint32_t item = blockIdx.x * static_cast<uint32_t>(groups) + g;
  const bool works = g < groups && item < a.items;
  const uint32_t split = item / a.tokens;
  const uint32_t token = item - split * a.tokens;
  const uint32_t b = token / a.seq, l = token - b * a.seq;
  const int n0 = a.t[0].heads;
  const int h0 = static_cast<int>(split) * a.per_item;
  const int rows = works ? min(a.heads - h0, a.per_item) : 0;
  const T* x0 = static_cast<const T*>(a.t[0].x) + b * a.t[0].xb + l * a.t[0].xl + h0 * a.t[0].xh + r * V;
  const T* x1 = static_cast<const T*>(a.t[1].x) + b * a.t[1].xb + l * a.t[1].xl + (h0 - n0) * a.t[1].xh + r * V;
  C* mine = reinterpret_cast<C*>(staged) + threadIdx.x;
  if constexpr (WIDE) {
    for (int k = 0; k < rows; ++k) {
      const T* at = h0 + k < n0 ? x0 + k * a.t[0].xh : x1 + k * a.t[1].xh;
      const uint32_t dst = smem_u32(mine) + k * (HALVES ? 2 : 1) * kThreads * 16;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(at) : "memory");
      if constexpr (HALVES)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + kThreads * 16), "l"(at + a.half) : "memory");
    }
  }
  for (int i = threadIdx.x; i < a.half; i += kThreads) {
    turns[i] = a.turns[i];
    axis[i] = a.axis[i];
  }
  __syncthreads();
  if (!works) return;
  float c[S], s[S];
#pragma unroll
  for (int j = 0; j < S; ++j) {
    const int slot = r * S + j;
    double t = load_id(a, b * a.ib + l * a.il + axis[slot] * a.ia) * turns[slot];
    t -= rint(t);
    sincospif(2.0f * static_cast<float>(t), &s[j], &c[j]);
    if (a.inverse) s[j] = -s[j];
  }
  if constexpr (WIDE) asm volatile("cp.async.wait_all;" ::: "memory");
  T* o0 = static_cast<T*>(a.t[0].out) + b * a.t[0].ob + l * a.t[0].ol + h0 * a.t[0].oh + r * V;
  T* o1 = static_cast<T*>(a.t[1].out) + b * a.t[1].ob + l * a.t[1].ol + (h0 - n0) * a.t[1].oh + r * V;
#pragma unroll 4
  for (int k = 0; k < rows; ++k) {
    const bool first = h0 + k < n0;
    C p, q;
    if constexpr (WIDE) {
      p = mine[k * (HALVES ? 2 : 1) * kThreads];
      if constexpr (HALVES) q = mine[(2 * k + 1) * kThreads];
    } else {
      const T* at = first ? x0 + k * a.t[0].xh : x1 + k * a.t[1].xh;
      p = *reinterpret_cast<const C*>(at);
      if constexpr (HALVES) q = *reinterpret_cast<const C*>(at + a.half);
    }
    float f[V], e[V];
    p.get(f);
    if constexpr (HALVES) q.get(e);
#pragma unroll
    for (int j = 0; j < S; ++j) {
      float& va = HALVES ? f[j] : f[2 * j];
      float& vb = HALVES ? e[j] : f[2 * j + 1];
      const float ta = va * c[j] - vb * s[j];
      vb = va * s[j] + vb * c[j];
      va = ta;
    }
    T* at = first ? o0 + k * a.t[0].oh : o1 + k * a.t[1].oh;
    p.set(f);
    *reinterpret_cast<C*>(at) = p;
    if constexpr (HALVES) {
      q.set(e);
      *reinterpret_cast<C*>(at + a.half) = q;
    }
  }
}

template <typename T, int V, bool HALVES>
static cudaError_t go(Args& a, cudaStream_t st) {
  a.tpr = HALVES ? a.half / V : 2 * a.half / V;
  const int groups = kThreads / a.tpr;
  // Runs of up to kRows chunks, shorter where that would leave some of the four blocks per SM without work: a single
  // token's heads all go to different groups.
  constexpr int most = HALVES ? kRows / 2 : kRows;
  const int64_t room = 4ll * kNumSms * groups;
  const int64_t fair = (static_cast<int64_t>(a.tokens) * a.heads + room - 1) / room;
  const int64_t runs = (a.heads + most - 1) / most;
  a.per_item = static_cast<int>(std::min<int64_t>(fair, (a.heads + runs - 1) / runs));
  const int64_t items = static_cast<int64_t>(a.tokens) * ((a.heads + a.per_item - 1) / a.per_item);
  if (items > 0x7FFFFFFF) return cudaErrorInvalidConfiguration;  // more than 180 GB hold in any layout but broadcast ones
  a.items = static_cast<uint32_t>(items);
  const unsigned grid = (a.items + groups - 1) / groups;
  const int smem = V * sizeof(T) == 16 ? a.per_item * (HALVES ? 2 : 1) * kThreads * 16 : 0;
  rope_axes_kernel<T, V, HALVES><<<grid, kThreads, smem, st>>>(a);
  return cudaGetLastError();
}

template <typename T>
static cudaError_t go_t(Args& a, bool halves, bool wide, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  if (halves) return wide ? go<T, V, true>(a, st) : go<T, 1, true>(a, st);
  return wide ? go<T, V, false>(a, st) : go<T, 2, false>(a, st);
}

// turns and axis of every slot. A model calls with the same axes again and again: the last ones of this thread are
// kept, since 64 powers cost as much as the launch.
static void fill_slots(int axes, const int32_t* dims, const double* theta, Args& a) {
  struct Last {
    int axes = 0;
    int32_t dims[8];
    double theta[8];
    double turns[kMaxSlots];
    uint8_t axis[kMaxSlots];
  };
  static thread_local Last last;
  bool same = last.axes == axes;
  for (int i = 0; same && i < axes; ++i) same = last.dims[i] == dims[i] && last.theta[i] == theta[i];
  if (!same) {
    int slot = 0;
    for (int i = 0; i < axes; ++i) {
      for (int j = 0; j < dims[i]; j += 2, ++slot) {
        last.turns[slot] = pow(theta[i], -static_cast<double>(j) / dims[i]) * 0.15915494309189533577;  // omega / 2 pi
        last.axis[slot] = static_cast<uint8_t>(i);
      }
      last.dims[i] = dims[i];
      last.theta[i] = theta[i];
    }
    last.axes = axes;
  }
  memcpy(a.turns, last.turns, sizeof(double) * a.half);
  memcpy(a.axis, last.axis, a.half);
}

}  // namespace rope

std::string rope_axes_setup() {
  using namespace rope;
  const int bytes = kRows * kThreads * 16;
  cudaError_t e = cudaSuccess;
  auto raise = [&](auto kernel) {
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  };
  raise(rope_axes_kernel<float, 4, false>);
  raise(rope_axes_kernel<float, 4, true>);
  raise(rope_axes_kernel<__half, 8, false>);
  raise(rope_axes_kernel<__half, 8, true>);
  raise(rope_axes_kernel<__nv_bfloat16, 8, false>);
  raise(rope_axes_kernel<__nv_bfloat16, 8, true>);
  return e == cudaSuccess ? std::string() : std::string("cudaFuncSetAttribute(rope_axes): ") + cudaGetErrorString(e);
}

int launch_rope_axes(const fb_rope_args& p, cudaStream_t st, std::string& err) {
  const int count = p.count, dtype = p.dtype, head_dim = p.head_dim, axes = p.axes, pairs = p.pairs;
  const fb_rope_tensor* ts = p.tensor;
  if (count < 1 || count > 2 || axes < 1 || axes > 8 || p.batch < 0 || p.seq < 0) {
    err = "fb_rope_axes: need 1 or 2 tensors, 1 to 8 axes, batch and seq >= 0";
    return FB_ERR_ARG;
  }
  if (dtype != FB_F32 && dtype != FB_F16 && dtype != FB_BF16) {
    err = "fb_rope_axes: dtype must be FB_F32, FB_F16 or FB_BF16";
    return FB_ERR_ARG;
  }
  if (p.ids_type < FB_IDS_F32 || p.ids_type > FB_IDS_I64 || (pairs != FB_ROPE_INTERLEAVED && pairs != FB_ROPE_HALVES)) {
    err = "fb_rope_axes: unknown ids type or pair order";
    return FB_ERR_ARG;
  }
  int64_t sum = 0;
  for (int i = 0; i < axes; ++i) {
    if (p.axes_dim[i] < 2 || p.axes_dim[i] % 2 != 0 || p.axes_dim[i] > 2 * rope::kMaxSlots || !(p.theta[i] > 0.0)) {
      err = "fb_rope_axes: each axis needs an even number of dims >= 2 and a base > 0";
      return FB_ERR_ARG;
    }
    sum += p.axes_dim[i];
  }
  if (sum != head_dim || head_dim > 2 * rope::kMaxSlots) {
    err = "fb_rope_axes: the axes' dims must add up to head_dim, at most 512";
    return FB_ERR_ARG;
  }
  for (int n = 0; n < count; ++n) {
    if (ts[n].heads < 1 || ts[n].heads > 65536) {
      err = "fb_rope_axes: 1 to 65536 heads";
      return FB_ERR_ARG;
    }
  }
  std::string derr;
  if (!device_for(Operator::kRopeAxes, derr)) {  // raises the kernels' shared-memory limits on this device
    err = derr;
    return FB_ERR_INIT;
  }
  const int64_t tokens = static_cast<int64_t>(p.batch) * p.seq;
  if (tokens == 0) return FB_OK;
  if (tokens > (1ll << 30)) {
    err = "fb_rope_axes: at most 2^30 tokens per call";
    return FB_ERR_UNSUPPORTED;
  }
  if (!p.ids) {
    err = "fb_rope_axes: null ids";
    return FB_ERR_ARG;
  }
  rope::Args a;
  memset(&a, 0, offsetof(rope::Args, turns));
  const int esz = dtype == FB_F32 ? 4 : 2;
  const int v = 16 / esz;
  // 16-byte accesses where every row starts on 16 bytes and a thread's elements stay inside the row (inside its
  // half, for pairs in halves); any other layout goes element by element.
  bool wide = pairs == FB_ROPE_HALVES ? (head_dim / 2) % v == 0 : head_dim % v == 0;
  for (int n = 0; n < count; ++n) {
    const fb_rope_tensor& t = ts[n];
    const uintptr_t at = reinterpret_cast<uintptr_t>(t.x) | reinterpret_cast<uintptr_t>(t.out);
    if (!t.x || !t.out || at % esz != 0) {
      err = "fb_rope_axes: null or misaligned tensor";
      return FB_ERR_ARG;
    }
    wide = wide && at % 16 == 0;
    for (int64_t s : {t.x_stride_b, t.x_stride_h, t.x_stride_l, t.out_stride_b, t.out_stride_h, t.out_stride_l})
      wide = wide && s % v == 0;
    a.t[n] = {t.x, t.out, t.x_stride_b, t.x_stride_h, t.x_stride_l, t.out_stride_b, t.out_stride_h, t.out_stride_l,
              t.heads};
    a.heads += t.heads;
  }
  if (count == 1) a.t[1] = a.t[0];  // never read: its heads come after the last
  a.seq = p.seq;
  a.tokens = static_cast<uint32_t>(tokens);
  a.half = head_dim / 2;
  a.inverse = p.inverse != 0;
  a.ids = p.ids;
  a.ids_type = p.ids_type;
  a.ib = p.ids_stride_b;
  a.il = p.ids_stride_l;
  a.ia = p.ids_stride_a;
  rope::fill_slots(axes, p.axes_dim, p.theta, a);
  const bool halves = pairs == FB_ROPE_HALVES;
  cudaError_t e = dtype == FB_F32   ? rope::go_t<float>(a, halves, wide, st)
                  : dtype == FB_F16 ? rope::go_t<__half>(a, halves, wide, st)
                                    : rope::go_t<__nv_bfloat16>(a, halves, wide, st);
  if (e != cudaSuccess) {
    err = std::string("fb_rope_axes: ") + cudaGetErrorString(e);
    return FB_ERR_CUDA;
  }
  return FB_OK;
}

}  // namespace fb
