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
  int count;
  int seq;
  uint32_t tokens;  // batch * seq
  uint32_t items;   // tokens * splits
  int splits;       // the heads of each tensor are cut into this many runs, one per work item
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

// A thread's share of one head row: one chunk of V elements (interleaved: V / 2 slots), or two chunks half a row
// apart (halves: V slots).
template <typename T, int V, bool HALVES>
__global__ void __launch_bounds__(kThreads) rope_axes_kernel(const __grid_constant__ Args a) {
  constexpr int S = HALVES ? V : V / 2;  // slots of a thread
  constexpr int U = 4;                   // head rows in flight per thread
  const int groups = kThreads / a.tpr;
  const int g = threadIdx.x / a.tpr;
  const int r = threadIdx.x - g * a.tpr;
  const uint32_t item = blockIdx.x * static_cast<uint32_t>(groups) + g;
  if (g >= groups || item >= a.items) return;
  const uint32_t split = item / a.tokens;
  const uint32_t token = item - split * a.tokens;
  const uint32_t b = token / a.seq, l = token - b * a.seq;

  float c[S], s[S];
  const int slot0 = r * S;
#pragma unroll
  for (int i = 0; i < S; ++i) {
    const int slot = slot0 + i;
    double t = load_id(a, b * a.ib + l * a.il + a.axis[slot] * a.ia) * a.turns[slot];
    t -= rint(t);
    sincospif(2.0f * static_cast<float>(t), &s[i], &c[i]);
    if (a.inverse) s[i] = -s[i];
  }

  using C = Chunk<T, V>;
  for (int n = 0; n < a.count; ++n) {
    const Tensor& t = a.t[n];
    const int h1 = static_cast<int>(static_cast<int64_t>(t.heads) * (split + 1) / a.splits);
    int h = static_cast<int>(static_cast<int64_t>(t.heads) * split / a.splits);
    const T* x = static_cast<const T*>(t.x) + b * t.xb + l * t.xl + r * V;
    T* o = static_cast<T*>(t.out) + b * t.ob + l * t.ol + r * V;
    for (; h < h1; h += U) {
      C p[U], q[HALVES ? U : 1];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (h + u < h1) {
          p[u] = *reinterpret_cast<const C*>(x + (h + u) * t.xh);
          if constexpr (HALVES) q[u] = *reinterpret_cast<const C*>(x + (h + u) * t.xh + a.half);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (h + u < h1) {
#pragma unroll
          for (int i = 0; i < S; ++i) {
            T& ea = HALVES ? p[u].e[i] : p[u].e[2 * i];
            T& eb = HALVES ? q[u].e[i] : p[u].e[2 * i + 1];
            const float va = to_f32<T>(ea), vb = to_f32<T>(eb);
            ea = from_f32<T>(va * c[i] - vb * s[i]);
            eb = from_f32<T>(va * s[i] + vb * c[i]);
          }
          *reinterpret_cast<C*>(o + (h + u) * t.oh) = p[u];
          if constexpr (HALVES) *reinterpret_cast<C*>(o + (h + u) * t.oh + a.half) = q[u];
        }
      }
    }
  }
}

template <typename T, int V, bool HALVES>
static cudaError_t go(Args& a, cudaStream_t st) {
  a.tpr = HALVES ? a.half / V : 2 * a.half / V;
  const int groups = kThreads / a.tpr;
  // Cut the heads into enough runs to fill the GPU: about eight blocks per SM, at most one run per head. A single
  // token then spreads over as many groups as it has heads.
  int heads = 0;
  for (int n = 0; n < a.count; ++n) heads = std::max(heads, a.t[n].heads);
  const int64_t want = (static_cast<int64_t>(kNumSms) * 8 * groups + a.tokens - 1) / a.tokens;
  a.splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(want, heads)));
  a.items = a.tokens * static_cast<uint32_t>(a.splits);
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

}  // namespace rope

int launch_rope_axes(const fb_rope_tensor* ts, int count, int dtype, int batch, int seq, int head_dim, const void* ids,
                     int ids_type, int64_t ids_stride_b, int64_t ids_stride_l, int64_t ids_stride_a, int axes,
                     const int32_t* axes_dim, const double* theta, int pairs, int inverse, cudaStream_t st,
                     std::string& err) {
  if (count < 1 || count > 2 || !ts || !axes_dim || !theta || axes < 1 || axes > 8 || batch < 0 || seq < 0) {
    err = "fb_rope_axes: need 1 or 2 tensors, 1 to 8 axes, batch and seq >= 0";
    return FB_ERR_ARG;
  }
  if (dtype != FB_F32 && dtype != FB_F16 && dtype != FB_BF16) {
    err = "fb_rope_axes: dtype must be FB_F32, FB_F16 or FB_BF16";
    return FB_ERR_ARG;
  }
  if (ids_type < FB_IDS_F32 || ids_type > FB_IDS_I64 || (pairs != FB_ROPE_INTERLEAVED && pairs != FB_ROPE_HALVES)) {
    err = "fb_rope_axes: unknown ids type or pair order";
    return FB_ERR_ARG;
  }
  int64_t sum = 0;
  for (int i = 0; i < axes; ++i) {
    if (axes_dim[i] < 2 || axes_dim[i] % 2 != 0 || axes_dim[i] > 2 * rope::kMaxSlots || !(theta[i] > 0.0)) {
      err = "fb_rope_axes: each axis needs an even number of dims >= 2 and a base > 0";
      return FB_ERR_ARG;
    }
    sum += axes_dim[i];
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
  const int64_t tokens = static_cast<int64_t>(batch) * seq;
  if (tokens == 0) return FB_OK;
  if (tokens > (1ll << 30)) {
    err = "fb_rope_axes: at most 2^30 tokens per call";
    return FB_ERR_UNSUPPORTED;
  }
  if (!ids) {
    err = "fb_rope_axes: null ids";
    return FB_ERR_ARG;
  }
  rope::Args a;
  memset(&a, 0, sizeof(a));
  const int esz = dtype == FB_F32 ? 4 : 2;
  const int v = 16 / esz;
  // 16-byte accesses where every row starts on 16 bytes and a thread's elements stay inside the row (inside its
  // half, for pairs in halves); any other layout goes element by element.
  bool wide = pairs == FB_ROPE_HALVES ? (head_dim / 2) % v == 0 : head_dim % v == 0;
  for (int n = 0; n < count; ++n) {
    const fb_rope_tensor& t = ts[n];
    const uintptr_t p = reinterpret_cast<uintptr_t>(t.x) | reinterpret_cast<uintptr_t>(t.out);
    if (!t.x || !t.out || p % esz != 0) {
      err = "fb_rope_axes: null or misaligned tensor";
      return FB_ERR_ARG;
    }
    wide = wide && p % 16 == 0;
    for (int64_t s : {t.x_stride_b, t.x_stride_h, t.x_stride_l, t.out_stride_b, t.out_stride_h, t.out_stride_l})
      wide = wide && s % v == 0;
    a.t[n] = {t.x, t.out, t.x_stride_b, t.x_stride_h, t.x_stride_l, t.out_stride_b, t.out_stride_h, t.out_stride_l,
              t.heads};
  }
  a.count = count;
  a.seq = seq;
  a.tokens = static_cast<uint32_t>(tokens);
  a.half = head_dim / 2;
  a.inverse = inverse != 0;
  a.ids = ids;
  a.ids_type = ids_type;
  a.ib = ids_stride_b;
  a.il = ids_stride_l;
  a.ia = ids_stride_a;
  int slot = 0;
  for (int i = 0; i < axes; ++i) {
    for (int j = 0; j < axes_dim[i]; j += 2, ++slot) {
      a.turns[slot] = pow(theta[i], -static_cast<double>(j) / axes_dim[i]) * 0.15915494309189533577;  // omega / 2 pi
      a.axis[slot] = static_cast<uint8_t>(i);
    }
  }
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
