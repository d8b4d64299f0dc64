// rope_axes.cu — rotary positions with several axes, applied straight from the position ids.
//
// Token l has one position per axis a, ids[l, a]; axis a owns d_a / 2 rotation slots with the frequencies
// theta^(-2j / d_a), and the slots of all axes lie one after the other (the order of selas's rope_tables,
// flux.py:106-114). Slot s turns one pair of a head's elements by phi = ids[l, axis(s)] * omega_s: the pair
// (2s, 2s + 1) (interleaved, flux.py:117-121) or (s, s + hd / 2) (halves). The turn is orthogonal, so the
// gradient is the same kernel with -phi.
//
// Angles: phi / 2 pi is formed in 64 bits (one multiply by omega / 2 pi, minus its nearest whole number), which
// keeps positions of millions exact to ~1e-9 turns, and only the fraction in [-1/2, 1/2] goes to sincospif in 32 bits.
//
// Bound: HBM, every element read once and written once. A group of threads owns one token: each thread keeps the
// sines and cosines of its own slots in registers and walks over the heads of q and of k, 16 bytes at a time, so no
// table is read and an angle is computed once for all the heads that a thread takes.
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
  uint32_t items;   // tokens * splits
  int per_item;     // consecutive heads of one work item
  int half;         // head_dim / 2
  int tpr;          // threads per token
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

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// V consecutive elements: one 16-byte access where V elements are 16 bytes, else element by element.
template <typename T, int V>
struct alignas(V * sizeof(T) == 16 ? 16 : sizeof(T)) Chunk {
  T e[V];
};

constexpr int kInFlight = 8;  // head rows a thread loads before it turns the first

// A thread's share of one head row: one chunk of V elements (interleaved: V / 2 slots), or two chunks half a row
// apart (halves: V slots).
template <typename T, int V, bool HALVES>
__global__ void __launch_bounds__(kThreads) rope_axes_kernel(const __grid_constant__ Args a) {
  constexpr int S = HALVES ? V : V / 2;  // slots of a thread
  constexpr int U = HALVES ? kInFlight / 2 : kInFlight;
  // The slots' constants are read by different lanes at different places, which the constant cache serves one by one:
  // from shared memory they come at once.
  __shared__ double turns[kMaxSlots];
  __shared__ uint8_t axis[kMaxSlots];
  for (int i = threadIdx.x; i < a.half; i += kThreads) {
    turns[i] = a.turns[i];
    axis[i] = a.axis[i];
  }
  __syncthreads();
  const int groups = kThreads / a.tpr;
  const int g = threadIdx.x / a.tpr;
  const int r = threadIdx.x - g * a.tpr;
  const uint32_t item = blockIdx.x * static_cast<uint32_t>(groups) + g;
  if (g >= groups || item >= a.items) return;
  const uint32_t split = item / a.tokens;
  const uint32_t token = item - split * a.tokens;
  const uint32_t b = token / a.seq, l = token - b * a.seq;

  using C = Chunk<T, V>;
  const T* x[2];
  T* o[2];
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    // head h of tensor 1 counts from t[0].heads
    const int64_t h0 = n ? -static_cast<int64_t>(a.t[0].heads) : 0;
    x[n] = static_cast<const T*>(a.t[n].x) + b * a.t[n].xb + l * a.t[n].xl + h0 * a.t[n].xh + r * V;
    o[n] = static_cast<T*>(a.t[n].out) + b * a.t[n].ob + l * a.t[n].ol + h0 * a.t[n].oh + r * V;
  }
  const int h_end = min(a.heads, static_cast<int>(split + 1) * a.per_item);
  int h = static_cast<int>(split) * a.per_item;

  float c[S], s[S];
  for (; h < h_end; h += U) {
    C p[U], q[HALVES ? U : 1];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (h + u < h_end) {
        const int n = h + u >= a.t[0].heads;
        const T* at = (n ? x[1] : x[0]) + (h + u) * (n ? a.t[1].xh : a.t[0].xh);
        p[u] = *reinterpret_cast<const C*>(at);
        if constexpr (HALVES) q[u] = *reinterpret_cast<const C*>(at + a.half);
      }
    }
    if (h == static_cast<int>(split) * a.per_item) {  // the first rows are on their way: the angles meanwhile
#pragma unroll
      for (int i = 0; i < S; ++i) {
        const int slot = r * S + i;
        double t = load_id(a, b * a.ib + l * a.il + axis[slot] * a.ia) * turns[slot];
        t -= rint(t);
        sincospif(2.0f * static_cast<float>(t), &s[i], &c[i]);
        if (a.inverse) s[i] = -s[i];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (h + u < h_end) {
#pragma unroll
        for (int i = 0; i < S; ++i) {
          T& ea = HALVES ? p[u].e[i] : p[u].e[2 * i];
          T& eb = HALVES ? q[u].e[i] : p[u].e[2 * i + 1];
          const float va = to_f32<T>(ea), vb = to_f32<T>(eb);
          ea = from_f32<T>(va * c[i] - vb * s[i]);
          eb = from_f32<T>(va * s[i] + vb * c[i]);
        }
        const int n = h + u >= a.t[0].heads;
        T* at = (n ? o[1] : o[0]) + (h + u) * (n ? a.t[1].oh : a.t[0].oh);
        *reinterpret_cast<C*>(at) = p[u];
        if constexpr (HALVES) *reinterpret_cast<C*>(at + a.half) = q[u];
      }
    }
  }
}

template <typename T, int V, bool HALVES>
static cudaError_t go(Args& a, cudaStream_t st) {
  a.tpr = HALVES ? a.half / V : 2 * a.half / V;
  const int groups = kThreads / a.tpr;
  // Cut the heads of q and k into enough runs to fill the GPU (about eight blocks per SM), of whole batches of loads
  // where tokens are many; a single token spreads over as many groups as there are heads.
  constexpr int U = HALVES ? kInFlight / 2 : kInFlight;
  const int64_t want = (static_cast<int64_t>(kNumSms) * 8 * groups + a.tokens - 1) / a.tokens;
  a.per_item = static_cast<int>(std::max<int64_t>(1, a.heads / want));
  if (a.per_item > U) a.per_item = (a.per_item + U - 1) / U * U;
  a.items = a.tokens * static_cast<uint32_t>((a.heads + a.per_item - 1) / a.per_item);
  const unsigned grid = (a.items + groups - 1) / groups;
  rope_axes_kernel<T, V, HALVES><<<grid, kThreads, 0, st>>>(a);
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
