// layer_norm.cu — layer norm with an affine map, and its backward pass with the gradients of the map, for plain norms
// (one weight for every row) and for adaLN (weight 1 + scale[b], bias shift[b] per image).
//
//   forward   y  = xhat * w + b,  xhat = (x - mean) * rstd,  rstd = 1 / sqrt(var + eps)
//   backward  g  = dy * w;  dx = rstd * (g - mean(g) - xhat * mean(g * xhat)) [+ add]
//             dw = sum over rows of dy * xhat,  db = sum over rows of dy
//
// Bound: HBM. Every kernel reads each input once: a row stays in the registers of a group of threads between the
// passes over it (mean first, then the squares of the centred values, so a large mean costs no precision), and the
// backward pass works mean and rstd out again from x, which it has to read anyway, instead of reading saved ones. The
// next rows are on their way to shared memory meanwhile, each thread's elements to places that only it reads. The
// column sums dw and db stay in registers too (a thread owns the same columns of every row it takes), are joined
// across the block's groups in shared memory, and go out as one fp32 partial row per block; a second kernel adds the
// partials in a fixed order, so results do not depend on the order in which blocks run. The blocks of a call with few rows
// are a cluster instead, and add their sums over distributed shared memory in order of rank.
//
// Measured on the device: forward 18432 x 3072 fp32 to bf16 56 us (6.0 TB/s), 65537 x 768 bf16 36 us (5.7); backward
// 65537 x 1280 bf16 96 us (5.3), 18432 x 3072 fp32 with bf16 dy 103 us (5.5), 4608 x 3072 fp32 with the adaLN scale and add
// 43 us (4.6; 31 rows per SM, ten per group of threads, and about 3 us to join the partials). Further from the copy's speed:
// 16-bit rows above some 2000 wide, whose few groups per SM stop at two barriers per row (6000 x 6144 31 us forward, 75
// backward: 4.8 and 3.0 TB/s); widths that are no multiple of four, loaded value by value without rows on their
// way (20000 x 1001 bf16 29 and 56 us: 2.8 and 2.1); above 10240 the 1024 threads' registers spill (4000 x 12288 bf16 70 and
// 129 us: 2.8 and 2.3), and above 16384 a block reads its row again for every pass (3000 x 20000 fp32 1.7 and 1.0 TB/s).
#include <type_traits>

#include "fb_internal.h"

namespace fb {
namespace norm {

constexpr int kMaxCluster = 8;      // blocks of a portable cluster
constexpr int kMaxDimRegs = 16384;  // the widest row that a group of 1024 threads holds in registers

struct Args {
  const void *x, *dy, *add;
  void* out;  // y, or dx
  const void *w, *b;
  float *part, *dw, *db;  // partials [sum group][block][2][dim]; with one block per group dw and db are written directly
  int64_t xo, xi, yo, yi, ao, ai, oo, oi;  // strides of x, dy, add, out: outer index, inner index (elements)
  int64_t w_stride;                        // of w and b per outer index (0: shared)
  int rows;                                // rows of a sum group (forward: all rows)
  int inner;                               // row = outer * inner + index
  int dim;
  int x_type, y_type, w_type;              // fb_dtype; y_type: y (forward) or dy
  int depth, stage_bytes;                  // rows on their way to shared memory, and the bytes of one
  int add_staged;                          // add is one of what comes that way
  int cluster;                             // the blocks of a sum group are a cluster and join their sums themselves
  float w_plus;                            // w is read as w_plus + w (1 for adaLN's scale)
  float eps;
};

// Two fp32 values in one 64-bit register: Blackwell's packed arithmetic does both in one instruction, and the norms'
// inner loops are bound by instruction issue before they are by the arithmetic.
typedef uint64_t f2;
__device__ __forceinline__ f2 pack2(float lo, float hi) {
  f2 v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
  return v;
}
__device__ __forceinline__ float2 unpack2(f2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
  f2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
  f2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
  f2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
// A pair of another block of the cluster, at its own shared-memory address there.
__device__ __forceinline__ f2 ld_cluster2(uint32_t addr, int rank) {
  f2 v;
  asm volatile("ld.shared::cluster.b64 %0, [%1];" : "=l"(v) : "r"(mapa_shared(addr, rank)) : "memory");
  return v;
}
__device__ __forceinline__ float total(f2 v) {
  const float2 r = unpack2(v);
  return r.x + r.y;
}

// Where a group is in its walk over rows: row = outer * inner + index, advanced by a fixed step without divisions.
// Groups smaller than a warp take consecutive rows and walk on as long as the first group of their warp has a row, since
// they shuffle together; a group past the last row works on zeros and writes nothing.
struct Place {
  int row, o, i;
};
__device__ __forceinline__ Place place_of(const Args& a, int first, int row) {
  const int all = first + row;
  return {row, all / a.inner, all % a.inner};
}
struct Step {
  int rows, o, i;
};
__device__ __forceinline__ void advance(Place& p, const Step& s, int inner) {
  p.row += s.rows;
  p.i += s.i;
  p.o += s.o + (p.i >= inner);
  if (p.i >= inner) p.i -= inner;
}

// CH consecutive elements (4: one vector access, 1: any alignment) widened to fp32. KEPT: nothing writes the tensor while the
// kernel runs, so it may be read through the read-only path (not add, which dx may take the place of).
template <bool KEPT, typename T>
__device__ __forceinline__ T read(const T* p) {
  if constexpr (KEPT) {
    return __ldg(p);
  } else {
    return *p;
  }
}
template <int CH, bool KEPT = true>
__device__ __forceinline__ void load_chunk(const void* p, int type, int64_t at, float* f) {
  if (type == FB_F32) {
    const float* s = static_cast<const float*>(p) + at;
    if constexpr (CH == 4) {
      const float4 v = read<KEPT>(reinterpret_cast<const float4*>(s));
      f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w;
    } else {
      f[0] = read<KEPT>(s);
    }
  } else if (type == FB_BF16) {
    const uint16_t* s = static_cast<const uint16_t*>(p) + at;
    if constexpr (CH == 4) {
      const uint2 u = read<KEPT>(reinterpret_cast<const uint2*>(s));
      f[0] = __uint_as_float(u.x << 16), f[1] = __uint_as_float(u.x & 0xFFFF0000u);
      f[2] = __uint_as_float(u.y << 16), f[3] = __uint_as_float(u.y & 0xFFFF0000u);
    } else {
      f[0] = bf16_bits_to_f32(read<KEPT>(s));
    }
  } else {
    const __half* s = static_cast<const __half*>(p) + at;
    if constexpr (CH == 4) {
      const uint2 u = read<KEPT>(reinterpret_cast<const uint2*>(s));
      const float2 lo = __half22float2(*reinterpret_cast<const __half2*>(&u.x));
      const float2 hi = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
      f[0] = lo.x, f[1] = lo.y, f[2] = hi.x, f[3] = hi.y;
    } else {
      f[0] = __half2float(read<KEPT>(s));
    }
  }
}

template <int CH>
__device__ __forceinline__ void store_chunk(void* p, int type, int64_t at, const float* f) {
  if (type == FB_F32) {
    float* d = static_cast<float*>(p) + at;
    if constexpr (CH == 4) {
      *reinterpret_cast<float4*>(d) = make_float4(f[0], f[1], f[2], f[3]);
    } else {
      d[0] = f[0];
    }
  } else if (type == FB_BF16) {
    uint16_t* d = static_cast<uint16_t*>(p) + at;
    if constexpr (CH == 4) {
      *reinterpret_cast<uint2*>(d) = make_uint2(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]));
    } else {
      *reinterpret_cast<__nv_bfloat16*>(d) = __float2bfloat16_rn(f[0]);
    }
  } else {
    __half* d = static_cast<__half*>(p) + at;
    if constexpr (CH == 4) {
      const __half2 lo = __floats2half2_rn(f[0], f[1]), hi = __floats2half2_rn(f[2], f[3]);
      *reinterpret_cast<uint2*>(d) =
          make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    } else {
      d[0] = __float2half_rn(f[0]);
    }
  }
}

// Widens CH elements that lie in shared memory or registers as raw bytes.
__device__ __forceinline__ void widen4(const uint8_t* p, int type, float* f) {
  if (type == FB_F32) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w;
  } else if (type == FB_BF16) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    f[0] = __uint_as_float(u.x << 16), f[1] = __uint_as_float(u.x & 0xFFFF0000u);
    f[2] = __uint_as_float(u.y << 16), f[3] = __uint_as_float(u.y & 0xFFFF0000u);
  } else {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    const float2 lo = __half22float2(*reinterpret_cast<const __half2*>(&u.x));
    const float2 hi = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
    f[0] = lo.x, f[1] = lo.y, f[2] = hi.x, f[3] = hi.y;
  }
}

// The elements of a row that one thread of its group holds: NCH chunks of CH, chunk c at column CH * (t + GT * c);
// zeros past the end (FULL: the row ends with the last thread's last chunk). The type branch is outside the loop, so the loads of a row go out together.
template <int GT, int NCH, int CH, bool FULL, bool KEPT>
__device__ __forceinline__ void load_row(const void* p, int type, int64_t base, int t, int dim, float (&f)[NCH * CH]) {
  auto each = [&](int ty) {
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int col = CH * (t + GT * c);
      if ((FULL && GT >= 32) || col < dim) {  // small groups: dim is 0 for one without a row
        load_chunk<CH, KEPT>(p, ty, base + col, f + CH * c);
      } else {
#pragma unroll
        for (int j = 0; j < CH; ++j) f[CH * c + j] = 0.f;
      }
    }
  };
  if (type == FB_F32) {
    each(FB_F32);
  } else if (type == FB_BF16) {
    each(FB_BF16);
  } else {
    each(FB_F16);
  }
}

template <int GT, int NCH, int CH, bool FULL>
__device__ __forceinline__ void store_row(void* p, int type, int64_t base, int t, int dim, const float (&f)[NCH * CH]) {
  auto each = [&](int ty) {
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int col = CH * (t + GT * c);
      if (FULL || col < dim) store_chunk<CH>(p, ty, base + col, f + CH * c);
    }
  };
  if (type == FB_F32) {
    each(FB_F32);
  } else if (type == FB_BF16) {
    each(FB_BF16);
  } else {
    each(FB_F16);
  }
}

// Asynchronous copy of a thread's own chunks of a row to its own places in shared memory, chunk c at
// dst + c * T * bytes(chunk): no other thread reads them, so waiting for the copies needs no barrier.
template <int GT, int NCH, int T, bool FULL>
__device__ __forceinline__ void fetch_row(uint32_t dst, const void* p, int type, int64_t base, int t, int dim) {
  if (type == FB_F32) {
    const float* s = static_cast<const float*>(p) + base;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int col = 4 * (t + GT * c);
      if (FULL || col < dim) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + c * T * 16), "l"(s + col) : "memory");
    }
  } else {
    const uint16_t* s = static_cast<const uint16_t*>(p) + base;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int col = 4 * (t + GT * c);
      if (FULL || col < dim) asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst + c * T * 8), "l"(s + col) : "memory");
    }
  }
}

// The fetched row, widened.
template <int GT, int NCH, int T, bool FULL>
__device__ __forceinline__ void take_row(const uint8_t* src, int type, int t, int dim, float (&f)[NCH * 4]) {
  auto each = [&](int ty, int bytes) {
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      if ((FULL && GT >= 32) || 4 * (t + GT * c) < dim) {
        widen4(src + c * T * bytes, ty, f + 4 * c);
      } else {
        f[4 * c] = f[4 * c + 1] = f[4 * c + 2] = f[4 * c + 3] = 0.f;
      }
    }
  };
  if (type == FB_F32) {
    each(FB_F32, 16);
  } else if (type == FB_BF16) {
    each(FB_BF16, 8);
  } else {
    each(FB_F16, 8);
  }
}

__device__ __forceinline__ void commit_fetch() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Waits until at most `newer` of this thread's newest fetches are on their way (0..3).
__device__ __forceinline__ void wait_fetch(int newer) {
  if (newer == 0) {
    asm volatile("cp.async.wait_group 0;" ::: "memory");
  } else if (newer == 1) {
    asm volatile("cp.async.wait_group 1;" ::: "memory");
  } else if (newer == 2) {
    asm volatile("cp.async.wait_group 2;" ::: "memory");
  } else {
    asm volatile("cp.async.wait_group 3;" ::: "memory");
  }
}

// Sums of two values over a group of GT threads (all of them get both). Up to a warp: shuffles, the whole warp together.
// More: one entry per warp in shared memory and a barrier of the group's own; `buf` alternates between calls, so one
// barrier per sum is enough.
template <int GT>
__device__ __forceinline__ float2 group_sum2(float a, float b, int group, float2* slots, int& buf) {
  // the lower half of the group's lanes adds up a, the upper half b
  constexpr int L = GT < 32 ? GT : 32;
  const bool upper = threadIdx.x & (L / 2);
  float v = (upper ? b : a) + __shfl_xor_sync(0xffffffffu, upper ? a : b, L / 2);
#pragma unroll
  for (int o = L / 4; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if constexpr (GT <= 32) return make_float2(__shfl_sync(0xffffffffu, v, 0, L), __shfl_sync(0xffffffffu, v, L / 2, L));
  constexpr int W = GT / 32;
  float2* s = slots + (buf * (blockDim.x / GT) + group) * W;
  buf ^= 1;
  const int warp = (threadIdx.x % GT) >> 5;
  if ((threadIdx.x & 15) == 0) (upper ? s[warp].y : s[warp].x) = v;
  asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(GT) : "memory");
  float2 r = s[0];
#pragma unroll
  for (int w = 1; w < W; ++w) r.x += s[w].x, r.y += s[w].y;
  return r;
}

// Threads of a block (whole groups of GT), and blocks per SM that a kernel is compiled for (registers) and its grid and
// shared memory are sized for. Forward: blocks of 256 threads, as many as their registers allow. Backward: one block per SM, so that the
// groups' column sums are joined in shared memory and one partial row per SM goes to memory.
constexpr int fwd_threads(int gt) { return gt < 256 ? 256 : gt; }
constexpr int fwd_blocks(int gt, int e) { return gt >= 512 ? (gt == 512 ? 2 : 1) : e <= 4 ? 4 : e <= 12 ? 3 : 2; }
constexpr int bwd_threads(int gt, int e) {
  const int most = e <= 4 ? 1024 : e <= 8 ? 768 : e <= 16 ? 512 : e <= 24 ? 384 : 256;
  return most < gt ? gt : most / gt * gt;  // whole groups: their barriers count on it
}

// One row of up to GT * NCH * CH elements per group of GT threads at a time; a group walks over rows
// blockIdx.x * NG + group, + gridDim.x * NG, ... of sum group blockIdx.y, the next `depth` rows on their way to shared
// memory while it works on one (CH == 4; the rows of odd sizes and alignments, CH == 1, are loaded where they are used).
// How many rows ahead of its warp's first group a group is.
template <int GT>
__device__ __forceinline__ int ahead_of_warp() {
  return GT < 32 ? static_cast<int>(threadIdx.x % 32) / GT : 0;
}

template <int GT, int NCH, int CH, bool FULL, int THREADS>
struct Walk {
  static constexpr int T = THREADS, NG = T / GT, E = NCH * CH, P = E / 2;
  static_assert(T % GT == 0 && T <= 1024 && (GT <= 32 || NG <= 15), "whole groups, a barrier of its own for each");
  // Pair k of a thread's elements lies in the chunks of columns 2k .. 2k + 1; both are inside the row or both past its
  // end for chunks of four, each by itself for single elements.
  static __device__ __forceinline__ int column(int t, int e) { return CH * (t + GT * (e / CH)) + e % CH; }
  static __device__ __forceinline__ f2 inside(int t, int k, int dim, float v) {
    if constexpr (FULL) {
      return pack2(v, v);
    } else if constexpr (CH == 4) {
      const float m = column(t, 2 * k) < dim ? v : 0.f;
      return pack2(m, m);
    } else {
      return pack2(column(t, 2 * k) < dim ? v : 0.f, column(t, 2 * k + 1) < dim ? v : 0.f);
    }
  }
  static __device__ __forceinline__ void pairs(const float (&f)[E], f2 (&v)[P]) {
#pragma unroll
    for (int k = 0; k < P; ++k) v[k] = pack2(f[2 * k], f[2 * k + 1]);
  }
  template <bool KEPT = true>
  static __device__ __forceinline__ void load(const void* p, int type, int64_t base, int t, int dim, f2 (&v)[P]) {
    float f[E];
    load_row<GT, NCH, CH, FULL, KEPT>(p, type, base, t, dim, f);
    pairs(f, v);
  }
  static __device__ __forceinline__ void take(const uint8_t* src, int type, int t, int dim, f2 (&v)[P]) {
    if constexpr (CH == 4) {
      float f[E];
      take_row<GT, NCH, T, FULL>(src, type, t, dim, f);
      pairs(f, v);
    }
  }
  static __device__ __forceinline__ void store(void* p, int type, int64_t base, int t, int dim, const f2 (&v)[P]) {
    float f[E];
#pragma unroll
    for (int k = 0; k < P; ++k) {
      const float2 r = unpack2(v[k]);
      f[2 * k] = r.x, f[2 * k + 1] = r.y;
    }
    store_row<GT, NCH, CH, FULL>(p, type, base, t, dim, f);
  }
  // w of outer index o, as it multiplies: w_plus + w, or ones
  static __device__ __forceinline__ void weight(const Args& a, int o, int t, f2 (&w)[P]) {
    if (a.w != nullptr) {
      load(a.w, a.w_type, o * a.w_stride, t, a.dim, w);
      const f2 plus = pack2(a.w_plus, a.w_plus);
#pragma unroll
      for (int k = 0; k < P; ++k) w[k] = add2(w[k], plus);
    } else {
#pragma unroll
      for (int k = 0; k < P; ++k) w[k] = pack2(1.f, 1.f);
    }
  }
};

template <int GT, int NCH, int CH, bool FULL>
__global__ void __launch_bounds__(fwd_threads(GT), fwd_blocks(GT, NCH* CH)) fwd_kernel(const __grid_constant__ Args a) {
  using W = Walk<GT, NCH, CH, FULL, fwd_threads(GT)>;
  constexpr int P = W::P, T = W::T, NG = W::NG;
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ float2 slots[GT > 32 ? 2 * NG * (GT / 32) : 1];
  const int group = threadIdx.x / GT, t = threadIdx.x % GT;
  const int rows_step = gridDim.x * NG;
  const Step step = {rows_step, rows_step / a.inner, rows_step % a.inner};
  const uint8_t* mine = ring + threadIdx.x * (a.x_type == FB_F32 ? 16 : 8);
  Place at = place_of(a, 0, blockIdx.x * NG + group), ahead = at;
  auto fetch = [&](int stage) {
    if (ahead.row < a.rows) {
      fetch_row<GT, NCH, T, FULL>(smem_u32(mine) + stage * a.stage_bytes, a.x, a.x_type, ahead.o * a.xo + ahead.i * a.xi, t, a.dim);
    }
    commit_fetch();
    advance(ahead, step, a.inner);
  };
  if constexpr (CH == 4) {
    for (int k = 0; k < a.depth; ++k) fetch(k);
  }
  const float inv = 1.0f / static_cast<float>(a.dim);
  f2 w[P], b[P];
  int have = -1;  // the outer index whose w and b are in registers
  int buf = 0, stage = 0;
  for (; at.row - ahead_of_warp<GT>() < a.rows; advance(at, step, a.inner)) {
    const bool live = GT >= 32 || at.row < a.rows;
    if (live && (have < 0 || (a.w_stride != 0 && have != at.o))) {
      have = at.o;
      W::weight(a, at.o, t, w);
      if (a.b != nullptr) {
        W::load(a.b, a.w_type, at.o * a.w_stride, t, a.dim, b);
      } else {
#pragma unroll
        for (int k = 0; k < P; ++k) b[k] = pack2(0.f, 0.f);
      }
    }
    f2 x[P];
    if constexpr (CH == 4) {
      wait_fetch(a.depth - 1);
      W::take(mine + stage * a.stage_bytes, a.x_type, t, live ? a.dim : 0, x);
    } else {
      W::load(a.x, a.x_type, at.o * a.xo + at.i * a.xi, t, live ? a.dim : 0, x);
    }
    f2 s[2], q[2];  // two running sums: the additions of one would wait for one another
    s[0] = s[1] = q[0] = q[1] = pack2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < P; ++k) s[k & 1] = add2(s[k & 1], x[k]);
    const float mean = group_sum2<GT>(total(add2(s[0], s[1])), 0.f, group, slots, buf).x * inv;
    if constexpr (CH == 4) {
      fetch(stage);  // the stage's values are in registers
      if (++stage == a.depth) stage = 0;
    }
#pragma unroll
    for (int k = 0; k < P; ++k) {
      x[k] = add2(x[k], W::inside(t, k, a.dim, -mean));
      q[k & 1] = fma2(x[k], x[k], q[k & 1]);
    }
    const float rstd = rsqrtf(group_sum2<GT>(total(add2(q[0], q[1])), 0.f, group, slots, buf).x * inv + a.eps);
    const f2 r = pack2(rstd, rstd);
#pragma unroll
    for (int k = 0; k < P; ++k) x[k] = fma2(mul2(x[k], r), w[k], b[k]);
    if (live) W::store(a.out, a.y_type, at.o * a.oo + at.i * a.oi, t, a.dim, x);
  }
}

template <int GT, int NCH, int CH, bool FULL>
__global__ void __launch_bounds__(bwd_threads(GT, NCH* CH), 1) bwd_kernel(const __grid_constant__ Args a) {
  using W = Walk<GT, NCH, CH, FULL, bwd_threads(GT, NCH * CH)>;
  constexpr int E = W::E, P = W::P, T = W::T, NG = W::NG;
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ float2 slots[GT > 32 ? 2 * NG * (GT / 32) : 1];
  const int group = threadIdx.x / GT, t = threadIdx.x % GT;
  const int rows_step = gridDim.x * NG;
  const Step step = {rows_step, rows_step / a.inner, rows_step % a.inner};
  // a stage holds the block's chunks of x, then of dy, then of add
  const int xb = a.x_type == FB_F32 ? 16 : 8, yb = a.y_type == FB_F32 ? 16 : 8;
  const uint8_t* mx = ring + threadIdx.x * xb;
  const uint8_t* my = ring + NCH * T * xb + threadIdx.x * yb;
  const uint8_t* ma = ring + NCH * T * (xb + yb) + threadIdx.x * xb;
  Place at = place_of(a, blockIdx.y * a.rows, blockIdx.x * NG + group), ahead = at;
  auto fetch = [&](int stage) {
    if (ahead.row < a.rows) {
      const int off = stage * a.stage_bytes;
      fetch_row<GT, NCH, T, FULL>(smem_u32(mx) + off, a.x, a.x_type, ahead.o * a.xo + ahead.i * a.xi, t, a.dim);
      fetch_row<GT, NCH, T, FULL>(smem_u32(my) + off, a.dy, a.y_type, ahead.o * a.yo + ahead.i * a.yi, t, a.dim);
      if (a.add_staged)
        fetch_row<GT, NCH, T, FULL>(smem_u32(ma) + off, a.add, a.x_type, ahead.o * a.ao + ahead.i * a.ai, t, a.dim);
    }
    commit_fetch();
    advance(ahead, step, a.inner);
  };
  if constexpr (CH == 4) {
    for (int k = 0; k < a.depth; ++k) fetch(k);
  }
  const float inv = 1.0f / static_cast<float>(a.dim);
  int buf = 0, stage = 0;
  f2 dw[P], db[P];
#pragma unroll
  for (int k = 0; k < P; ++k) dw[k] = db[k] = pack2(0.f, 0.f);
  // w waits in shared memory, once for all groups: the sums need its registers. All rows of a block have the same w (a
  // w per outer index comes with a sum group per outer index).
  ulonglong2* ws = reinterpret_cast<ulonglong2*>(ring + (CH == 4 ? a.depth * a.stage_bytes : 0)) + t;
  if (group == 0) {
    f2 w[P];
    W::weight(a, at.o, t, w);
#pragma unroll
    for (int k = 0; k < P; k += 2) ws[(k / 2) * GT] = make_ulonglong2(w[k], w[k + 1]);
  }
  __syncthreads();
  for (; at.row - ahead_of_warp<GT>() < a.rows; advance(at, step, a.inner)) {
    const bool live = GT >= 32 || at.row < a.rows;
    const int dim = live ? a.dim : 0;
    f2 x[P], g[P];
    if constexpr (CH == 4) {
      wait_fetch(a.depth - 1);
      W::take(mx + stage * a.stage_bytes, a.x_type, t, dim, x);
      W::take(my + stage * a.stage_bytes, a.y_type, t, dim, g);
    } else {
      W::load(a.x, a.x_type, at.o * a.xo + at.i * a.xi, t, dim, x);
      W::load(a.dy, a.y_type, at.o * a.yo + at.i * a.yi, t, dim, g);
    }
    // two running sums of each kind: the additions of one would wait for one another
    f2 sx[2], sg[2];
    sx[0] = sx[1] = sg[0] = sg[1] = pack2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < P; k += 2) {
      const ulonglong2 w = ws[(k / 2) * GT];
      sx[0] = add2(sx[0], x[k]);
      sx[1] = add2(sx[1], x[k + 1]);
      sg[0] = fma2(g[k], w.x, sg[0]);
      sg[1] = fma2(g[k + 1], w.y, sg[1]);
    }
    const float2 m = group_sum2<GT>(total(add2(sx[0], sx[1])), total(add2(sg[0], sg[1])), group, slots, buf);
    const float mean = m.x * inv;
    f2 qx[2], qg[2];
    qx[0] = qx[1] = qg[0] = qg[1] = pack2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < P; k += 2) {
      const ulonglong2 w = ws[(k / 2) * GT];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        x[k + j] = add2(x[k + j], W::inside(t, k + j, a.dim, -mean));
        qx[j] = fma2(x[k + j], x[k + j], qx[j]);
        qg[j] = fma2(mul2(g[k + j], j ? w.y : w.x), x[k + j], qg[j]);
      }
    }
    const float2 v = group_sum2<GT>(total(add2(qx[0], qx[1])), total(add2(qg[0], qg[1])), group, slots, buf);
    const float rstd = live ? rsqrtf(v.x * inv + a.eps) : 0.f;  // 0: nothing for the sums, not even 0 * inf
    // dx = rstd (g w - mean(g w) - xhat mean(g w xhat)), xhat = x rstd
    const float c0 = -rstd * m.y * inv, c1 = -rstd * (v.y * inv * rstd);
    const f2 r = pack2(rstd, rstd), k0 = pack2(c0, c0), k1 = pack2(c1, c1);
#pragma unroll
    for (int k = 0; k < P; k += 2) {
      const ulonglong2 w = ws[(k / 2) * GT];
#pragma unroll
      for (int j = k; j < k + 2; ++j) {
        const f2 h = mul2(x[j], r);
        x[j] = fma2(mul2(g[j], j == k ? w.x : w.y), r, fma2(h, k1, k0));
        dw[j] = fma2(g[j], h, dw[j]);
        db[j] = add2(db[j], g[j]);
      }
    }
    if (a.add != nullptr) {
      f2 ad[P];
      if (CH == 4 && a.add_staged) {
        W::take(ma + stage * a.stage_bytes, a.x_type, t, dim, ad);
      } else {
        W::template load<false>(a.add, a.x_type, at.o * a.ao + at.i * a.ai, t, dim, ad);
      }
#pragma unroll
      for (int k = 0; k < P; ++k) x[k] = add2(x[k], ad[k]);
    }
    if (live) W::store(a.out, a.x_type, at.o * a.oo + at.i * a.oi, t, a.dim, x);
    if constexpr (CH == 4) {
      fetch(stage);  // every value of the stage has been used
      if (++stage == a.depth) stage = 0;
    }
  }
  if (a.dw == nullptr) return;
  if constexpr (CH == 4) wait_fetch(0);  // the ring is free
  // Join the groups' sums. A pair of columns is added up by several threads, each over a run of the groups, and their
  // sums in the order of the runs by the first group's thread that owns the pair.
  if constexpr (NG > 1) {
    constexpr int PAIRS = P * GT, RUNS = T / PAIRS > 1 ? T / PAIRS : 1;
    f2* join = reinterpret_cast<f2*>(ring);
    for (int s = 0; s < 2; ++s) {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < P; ++k) join[k * T + threadIdx.x] = s ? db[k] : dw[k];
      __syncthreads();
      if constexpr (RUNS > 1) {
        const int q = threadIdx.x % PAIRS, run = threadIdx.x / PAIRS;
        f2 v = pack2(0.f, 0.f);
        if (run < RUNS) {
          const f2* p = join + q / GT * T + q % GT;
          for (int n = NG * run / RUNS; n < NG * (run + 1) / RUNS; ++n) v = add2(v, p[n * GT]);
        }
        __syncthreads();
        if (run < RUNS) join[run * PAIRS + q] = v;
        __syncthreads();
      }
      if (group == 0) {
#pragma unroll
        for (int k = 0; k < P; ++k) {
          f2 v = join[RUNS > 1 ? k * GT + t : k * T + t];
          for (int n = 1; n < (RUNS > 1 ? RUNS : NG); ++n) v = add2(v, join[RUNS > 1 ? n * PAIRS + k * GT + t : k * T + n * GT + t]);
          (s ? db[k] : dw[k]) = v;
        }
      }
    }
  }
  if (a.cluster) {
    // The blocks' sums, added in order of rank by the blocks alike, each its share of the columns.
    constexpr int PAIRS = P * GT;
    f2* sums = reinterpret_cast<f2*>(ring);  // [dw, db][pair]
    __syncthreads();                         // nobody reads the ring any more
    if (group == 0) {
#pragma unroll
      for (int k = 0; k < P; ++k) sums[k * GT + t] = dw[k], sums[PAIRS + k * GT + t] = db[k];
    }
    __syncwarp();
    cluster_sync_all();
    for (int q = blockIdx.x * T + threadIdx.x; q < 2 * PAIRS; q += gridDim.x * T) {
      const uint32_t at = smem_u32(sums + q);
      f2 part[kMaxCluster];
#pragma unroll
      for (int r = 0; r < kMaxCluster; ++r) part[r] = ld_cluster2(at, min(r, static_cast<int>(gridDim.x) - 1));
      f2 v = part[0];
#pragma unroll
      for (int r = 1; r < kMaxCluster; ++r)
        if (r < gridDim.x) v = add2(v, part[r]);
      const int p = q < PAIRS ? q : q - PAIRS, c0 = W::column(p % GT, p / GT * 2), c1 = W::column(p % GT, p / GT * 2 + 1);
      float* d = (q < PAIRS ? a.dw : a.db) + static_cast<int64_t>(blockIdx.y) * a.dim;
      const float2 s = unpack2(v);
      if (FULL || c0 < a.dim) d[c0] = s.x;
      if (FULL || c1 < a.dim) d[c1] = s.y;
    }
    __syncwarp();
    cluster_sync_all();  // nobody reads this block's sums any more
    return;
  }
  if (NG > 1 && group != 0) return;
  float *pw, *pb;
  if (gridDim.x == 1) {
    pw = a.dw + static_cast<int64_t>(blockIdx.y) * a.dim;
    pb = a.db + static_cast<int64_t>(blockIdx.y) * a.dim;
  } else {
    pw = a.part + (static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x) * 2 * a.dim;
    pb = pw + a.dim;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int col = W::column(t, e);
    const float2 vw = unpack2(dw[e / 2]), vb = unpack2(db[e / 2]);
    if (FULL || col < a.dim) pw[col] = e % 2 ? vw.y : vw.x, pb[col] = e % 2 ? vb.y : vb.x;
  }
}

// dw, db [sum group][dim] = the partials' sums. 32 columns x 32 runs of the partials per block, joined in order: with a
// partial per SM a thread has four or five loads, all on their way at once.
__global__ void __launch_bounds__(1024) join_kernel(const float* part, int blocks, int dim, float* __restrict__ dw,
                                                    float* __restrict__ db) {
  __shared__ float s[32][33];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31, run = threadIdx.x >> 5;
  const int64_t n2 = 2ll * dim;
  const int64_t col = static_cast<int64_t>(blockIdx.x) * 32 + lane;  // over dw, then db
  const float* p = part + static_cast<int64_t>(blockIdx.y) * blocks * n2 + col;
  float v = 0.f;
  if (col < n2) {
    const int lo = blocks * run / 32, hi = blocks * (run + 1) / 32;
#pragma unroll 5
    for (int k = lo; k < hi; ++k) v += p[k * n2];
  }
  s[run][lane] = v;
  __syncthreads();
  if (run == 0 && col < n2) {
#pragma unroll
    for (int r = 1; r < 32; ++r) v += s[r][lane];
    float* d = col < dim ? dw : db - dim;
    d[static_cast<int64_t>(blockIdx.y) * dim + col] = v;
  }
}

// ---- rows wider than kMaxDimRegs: one block per row, the row read again for each pass (from L2)

template <typename F>
__device__ __forceinline__ float2 wide_sum2(int dim, float2* slots, F f) {
  float a = 0.f, b = 0.f;
  for (int col = threadIdx.x; col < dim; col += 1024) f(col, a, b);
  int buf = 0;
  const float2 r = group_sum2<1024>(a, b, 0, slots, buf);
  __syncthreads();  // the slots are free again
  return r;
}

__global__ void __launch_bounds__(1024) fwd_wide_kernel(const __grid_constant__ Args a) {
  __shared__ float2 slots[2 * 32];
  const int64_t row = blockIdx.x, o = row / a.inner, i = row - o * a.inner;
  const int64_t xb = o * a.xo + i * a.xi, ob = o * a.oo + i * a.oi, wb = o * a.w_stride;
  const float inv = 1.0f / static_cast<float>(a.dim);
  auto at = [](const void* p, int type, int64_t k) {
    float f;
    load_chunk<1>(p, type, k, &f);
    return f;
  };
  const float mean = wide_sum2(a.dim, slots, [&](int c, float& s, float&) { s += at(a.x, a.x_type, xb + c); }).x * inv;
  const float var = wide_sum2(a.dim, slots, [&](int c, float& s, float&) {
    const float d = at(a.x, a.x_type, xb + c) - mean;
    s += d * d;
  }).x * inv;
  const float rstd = 1.0f / sqrtf(var + a.eps);
  for (int c = threadIdx.x; c < a.dim; c += 1024) {
    float y = (at(a.x, a.x_type, xb + c) - mean) * rstd;
    if (a.w) y *= a.w_plus + at(a.w, a.w_type, wb + c);
    if (a.b) y += at(a.b, a.w_type, wb + c);
    store_chunk<1>(a.out, a.y_type, ob + c, &y);
  }
}

// dx of a row, and its mean and rstd into part[row][2] for the column sums.
__global__ void __launch_bounds__(1024) bwd_wide_kernel(const __grid_constant__ Args a) {
  __shared__ float2 slots[2 * 32];
  const int64_t row = blockIdx.x, o = row / a.inner, i = row - o * a.inner;
  const int64_t xb = o * a.xo + i * a.xi, yb = o * a.yo + i * a.yi, ab = o * a.ao + i * a.ai, ob = o * a.oo + i * a.oi;
  const int64_t wb = o * a.w_stride;
  const float inv = 1.0f / static_cast<float>(a.dim);
  auto at = [](const void* p, int type, int64_t k) {
    float f;
    load_chunk<1>(p, type, k, &f);
    return f;
  };
  auto weight = [&](int c) { return a.w ? a.w_plus + at(a.w, a.w_type, wb + c) : 1.0f; };
  const float2 m = wide_sum2(a.dim, slots, [&](int c, float& s, float& g) {
    s += at(a.x, a.x_type, xb + c);
    g += at(a.dy, a.y_type, yb + c) * weight(c);
  });
  const float mean = m.x * inv, gmean = m.y * inv;
  const float2 v = wide_sum2(a.dim, slots, [&](int c, float& s, float& g) {
    const float d = at(a.x, a.x_type, xb + c) - mean;
    s += d * d;
    g += at(a.dy, a.y_type, yb + c) * weight(c) * d;
  });
  const float rstd = 1.0f / sqrtf(v.x * inv + a.eps), gx = v.y * inv * rstd;
  if (threadIdx.x == 0 && a.dw) a.part[2 * row] = mean, a.part[2 * row + 1] = rstd;
  for (int c = threadIdx.x; c < a.dim; c += 1024) {
    const float h = (at(a.x, a.x_type, xb + c) - mean) * rstd;
    float dx = rstd * (at(a.dy, a.y_type, yb + c) * weight(c) - gmean - h * gx);
    if (a.add) {
      float ad;
      load_chunk<1, false>(a.add, a.x_type, ab + c, &ad);
      dx += ad;
    }
    store_chunk<1>(a.out, a.x_type, ob + c, &dx);
  }
}

// dw, db of 32 columns of one sum group: 8 warps take every 8th row.
__global__ void __launch_bounds__(256) sums_wide_kernel(const __grid_constant__ Args a) {
  __shared__ float sw[8][32], sb[8][32];
  const int lane = threadIdx.x & 31, run = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float w = 0.f, b = 0.f;
  if (c < a.dim) {
    for (int64_t r = run; r < a.rows; r += 8) {
      const int64_t row = static_cast<int64_t>(blockIdx.y) * a.rows + r, o = row / a.inner, i = row - o * a.inner;
      float x, g;
      load_chunk<1>(a.x, a.x_type, o * a.xo + i * a.xi + c, &x);
      load_chunk<1>(a.dy, a.y_type, o * a.yo + i * a.yi + c, &g);
      w += g * ((x - a.part[2 * row]) * a.part[2 * row + 1]);
      b += g;
    }
  }
  sw[run][lane] = w, sb[run][lane] = b;
  __syncthreads();
  if (run == 0 && c < a.dim) {
#pragma unroll
    for (int r = 1; r < 8; ++r) w += sw[r][lane], b += sb[r][lane];
    a.dw[static_cast<int64_t>(blockIdx.y) * a.dim + c] = w;
    a.db[static_cast<int64_t>(blockIdx.y) * a.dim + c] = b;
  }
}

// ---------------------------------------------------------------------------------------------- host

static int size_of(int t) { return t == FB_F32 ? 4 : 2; }

// The group of threads for a row of `dim` elements. Few threads with many elements each cost the fewest barriers,
// shuffles and addresses per element, and the independent arithmetic of many elements hides latency better than more
// warps do (65537 x 768 in bf16, forward and backward: 47 and 84 us with 12 to 16 elements a thread, 39 and 66 with 24;
// 6000 x 6144 backward: 110 with 12, 78 with 24). The bound is what the registers hold: x, w and b forward at two blocks
// of 256 threads per SM, x, dy and the two running column sums backward, where blocks get smaller as threads hold more.
static int group_threads(int dim, bool vec, int most) {
  int gt = 8;
  while (gt * (gt < 32 ? 8 : vec ? most : 16) < dim && gt < 1024) gt *= 2;
  return gt;
}
// The most elements a thread holds: forward 32 of 16-bit rows, whose widening costs instructions, and 20 of fp32 rows,
// which need the warps more (18432 x 3072 57 us with 12, 61 with 24); 20 where wider rows would spill.
static int most_fwd(int dim, int x_type) { return x_type != FB_F32 && dim <= 8192 ? 32 : 20; }
static int most_bwd(int dim) { return dim <= 10240 ? 40 : 20; }
static int elements(int dim, int gt, bool vec) { return vec ? 4 * ((dim + 4 * gt - 1) / (4 * gt)) : gt < 32 ? 8 : 16; }

// Rows per group of threads up to which a sum group's rows go to one cluster of up to eight blocks, which joins its sums
// without a second launch. Measured, partial rows and a second launch against a cluster, bf16: 77 x 768 a call 16.9 / 14.7 us
// (device 10.3 / 10.0), 8 x 12288 22.1 / 16.4 on the device; at three rows per group the longer walk costs what the join
// saved (256 x 768 12.3 / 14.3).
constexpr int kClusterSteps = 2;
// Blocks per sum group of the backward pass: the SMs shared out over the groups, fewer where there are fewer rows than
// groups of threads. The share is a whole number, so sum groups (images) of 75 to 147 get a block each and leave SMs idle
// (fp32 3072 wide, 64 rows an image: 80 images 55 us, 147 images 57), and 50 to 74 get two (74 images 82 us).
struct Blocks {
  int64_t n;
  bool cluster;
};
static Blocks bwd_blocks(int64_t rows, int dim, int64_t sum_groups, bool vec, bool sums) {
  const int gt = group_threads(dim, vec, most_bwd(dim)), ng = bwd_threads(gt, elements(dim, gt, vec)) / gt;
  const int64_t need = std::max<int64_t>(1, (rows + ng - 1) / ng);
  const int64_t few = std::min<int64_t>(need, kMaxCluster);
  if (sums && need > 1 && need <= kClusterSteps * kMaxCluster && sum_groups * few <= kNumSms / 2) return {few, true};
  return {std::max<int64_t>(1, std::min<int64_t>(need, kNumSms / std::max<int64_t>(1, sum_groups))), false};
}

constexpr int kRingPerSm = 208 * 1024;  // shared memory of an SM that the rows on their way (and w) may take

template <int GT, int NCH, int CH, bool FULL>
static cudaError_t go_fwd(Args a, cudaStream_t st) {
  constexpr int T = fwd_threads(GT), NG = T / GT, per_sm = fwd_blocks(GT, NCH * CH);
  int smem = 0;
  if (CH == 4) {
    a.stage_bytes = 4 * NCH * T * size_of(a.x_type);
    a.depth = std::max(1, std::min(4, kRingPerSm / per_sm / a.stage_bytes));
    smem = a.depth * a.stage_bytes;
  }
  const int64_t need = (static_cast<int64_t>(a.rows) + NG - 1) / NG;
  fwd_kernel<GT, NCH, CH, FULL><<<static_cast<unsigned>(std::min<int64_t>(need, per_sm * kNumSms)), T, smem, st>>>(a);
  return cudaGetLastError();
}

template <int GT, int NCH, int CH, bool FULL>
static cudaError_t go_bwd(Args a, int64_t sum_groups, cudaStream_t st) {
  constexpr int T = bwd_threads(GT, NCH * CH), w_bytes = NCH * CH * GT * 4;
  int smem = w_bytes;
  if (CH == 4) {
    const int xb = size_of(a.x_type), yb = size_of(a.y_type);
    const int two = 4 * NCH * T * (xb + yb), three = two + 4 * NCH * T * xb;
    a.add_staged = a.add && three + w_bytes <= kRingPerSm;
    a.stage_bytes = a.add_staged ? three : two;
    a.depth = std::max(1, std::min(4, (kRingPerSm - w_bytes) / a.stage_bytes));
    smem += a.depth * a.stage_bytes;
  }
  const Blocks blocks = bwd_blocks(a.rows, a.dim, sum_groups, CH == 4, a.dw != nullptr);
  a.cluster = blocks.cluster;
  // after the walk, the groups' sums, then the block's
  smem = std::max(smem, std::max(NCH * CH * T * 4, a.cluster ? NCH * CH * GT * 8 : 0));
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3(static_cast<unsigned>(blocks.n), static_cast<unsigned>(sum_groups));
  cfg.blockDim = dim3(T);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 0;
  if (a.cluster) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(blocks.n);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.numAttrs = 1;
  }
  cudaError_t e = cudaLaunchKernelEx(&cfg, bwd_kernel<GT, NCH, CH, FULL>, a);
  if (e == cudaSuccess && a.dw != nullptr && blocks.n > 1 && !a.cluster) {
    // launched without a gap when the last block of the walk ends; it waits for their writes before it reads
    cfg.gridDim = dim3(static_cast<unsigned>((2ll * a.dim + 31) / 32), static_cast<unsigned>(sum_groups));
    cfg.blockDim = dim3(1024);
    cfg.dynamicSmemBytes = 0;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, join_kernel, static_cast<const float*>(a.part), static_cast<int>(blocks.n), a.dim, a.dw, a.db);
  }
  return e;
}

// f(GT, NCH, CH) as integral constants for a row of `dim` elements: every instance there is, and the only ones.
template <int N>
using Int = std::integral_constant<int, N>;
template <int GT, int FROM, int TO, typename F>
static cudaError_t with_chunks(int chunks, F f) {
  if constexpr (FROM < TO) {
    if (chunks > FROM) return with_chunks<GT, FROM + 1, TO>(chunks, f);
  }
  return f(Int<GT>(), Int<FROM>(), Int<4>());
}
template <typename F>
static cudaError_t with_fwd(int dim, bool vec, int x_type, F f) {
  const int gt = group_threads(dim, vec, most_fwd(dim, x_type)), chunks = (dim + 4 * gt - 1) / (4 * gt);
  switch (gt) {
    case 8: return vec ? with_chunks<8, 1, 2>(chunks, f) : f(Int<8>(), Int<8>(), Int<1>());
    case 16: return vec ? with_chunks<16, 2, 2>(chunks, f) : f(Int<16>(), Int<8>(), Int<1>());
    case 32: return vec ? with_chunks<32, 2, 8>(chunks, f) : f(Int<32>(), Int<16>(), Int<1>());
    case 64: return vec ? with_chunks<64, 3, 8>(chunks, f) : f(Int<64>(), Int<16>(), Int<1>());
    case 128: return vec ? with_chunks<128, 3, 8>(chunks, f) : f(Int<128>(), Int<16>(), Int<1>());
    case 256: return vec ? with_chunks<256, 3, 8>(chunks, f) : f(Int<256>(), Int<16>(), Int<1>());
    case 512: return vec ? with_chunks<512, 3, 5>(chunks, f) : f(Int<512>(), Int<16>(), Int<1>());
    default: return vec ? with_chunks<1024, 3, 4>(chunks, f) : f(Int<1024>(), Int<16>(), Int<1>());
  }
}
template <typename F>
static cudaError_t with_bwd(int dim, bool vec, F f) {
  const int gt = group_threads(dim, vec, most_bwd(dim)), chunks = (dim + 4 * gt - 1) / (4 * gt);
  switch (gt) {
    case 8: return vec ? with_chunks<8, 1, 2>(chunks, f) : f(Int<8>(), Int<8>(), Int<1>());
    case 16: return vec ? with_chunks<16, 2, 2>(chunks, f) : f(Int<16>(), Int<8>(), Int<1>());
    case 32: return vec ? with_chunks<32, 2, 10>(chunks, f) : f(Int<32>(), Int<16>(), Int<1>());
    case 64: return vec ? with_chunks<64, 6, 10>(chunks, f) : f(Int<64>(), Int<16>(), Int<1>());
    case 128: return vec ? with_chunks<128, 6, 10>(chunks, f) : f(Int<128>(), Int<16>(), Int<1>());
    case 256: return vec ? with_chunks<256, 6, 10>(chunks, f) : f(Int<256>(), Int<16>(), Int<1>());
    case 512: return f(Int<512>(), Int<16>(), Int<1>());
    default: return vec ? with_chunks<1024, 3, 4>(chunks, f) : f(Int<1024>(), Int<16>(), Int<1>());
  }
}

static cudaError_t dispatch(const Args& a, bool bwd, int64_t sum_groups, bool vec, cudaStream_t st) {
  if (a.dim > kMaxDimRegs) {
    if (!bwd) {
      fwd_wide_kernel<<<static_cast<unsigned>(a.rows), 1024, 0, st>>>(a);
      return cudaGetLastError();
    }
    bwd_wide_kernel<<<static_cast<unsigned>(a.rows) * static_cast<unsigned>(sum_groups), 1024, 0, st>>>(a);
    cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess && a.dw != nullptr) {
      sums_wide_kernel<<<dim3((a.dim + 31) / 32, static_cast<unsigned>(sum_groups)), 256, 0, st>>>(a);
      e = cudaGetLastError();
    }
    return e;
  }
  auto run = [&](auto gt, auto nch, auto ch) {
    constexpr int GT = decltype(gt)::value, NCH = decltype(nch)::value, CH = decltype(ch)::value;
    if constexpr (CH == 4) {
      if (a.dim == 4 * GT * NCH) return go_fwd<GT, NCH, CH, true>(a, st);
    }
    return go_fwd<GT, NCH, CH, false>(a, st);
  };
  auto back = [&](auto gt, auto nch, auto ch) {
    constexpr int GT = decltype(gt)::value, NCH = decltype(nch)::value, CH = decltype(ch)::value;
    if constexpr (CH == 4) {
      if (a.dim == 4 * GT * NCH) return go_bwd<GT, NCH, CH, true>(a, sum_groups, st);
    }
    return go_bwd<GT, NCH, CH, false>(a, sum_groups, st);
  };
  return bwd ? with_bwd(a.dim, vec, back) : with_fwd(a.dim, vec, a.x_type, run);
}

// Raises the shared-memory limits of every instance (ring of up to kRingPerSm bytes).
static cudaError_t setup() {
  cudaError_t e = cudaSuccess;
  auto raise = [&](auto kernel) {
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingPerSm);
  };
  auto fwd = [&](auto gt, auto nch, auto ch) {
    constexpr int GT = decltype(gt)::value, NCH = decltype(nch)::value, CH = decltype(ch)::value;
    raise(fwd_kernel<GT, NCH, CH, false>);
    if constexpr (CH == 4) raise(fwd_kernel<GT, NCH, CH, true>);
    return e;
  };
  auto bwd = [&](auto gt, auto nch, auto ch) {
    constexpr int GT = decltype(gt)::value, NCH = decltype(nch)::value, CH = decltype(ch)::value;
    raise(bwd_kernel<GT, NCH, CH, false>);
    if constexpr (CH == 4) raise(bwd_kernel<GT, NCH, CH, true>);
    return e;
  };
  for (int vec = 0; vec < 2; ++vec)
    for (int dim = 32; dim <= kMaxDimRegs; dim += dim < 128 ? 32 : 128) {
      with_fwd(dim, vec, FB_F32, fwd);
      with_fwd(dim, vec, FB_BF16, fwd);
      with_bwd(dim, vec, bwd);
    }
  return e;
}

static bool is_dtype(int t) { return t == FB_F32 || t == FB_F16 || t == FB_BF16; }
// Whether chunks of four elements of this tensor are aligned vectors.
static bool vec4(const void* p, int type, std::initializer_list<int64_t> strides) {
  if (reinterpret_cast<uintptr_t>(p) % (4 * size_of(type)) != 0) return false;
  for (int64_t s : strides)
    if (s % 4 != 0) return false;
  return true;
}
static bool misaligned(const void* p, int type) { return reinterpret_cast<uintptr_t>(p) % size_of(type) != 0; }

}  // namespace norm

std::string layer_norm_setup() {
  const cudaError_t e = norm::setup();
  return e == cudaSuccess ? std::string() : std::string("cudaFuncSetAttribute(layer_norm): ") + cudaGetErrorString(e);
}

int64_t layer_norm_work_floats(int64_t outer, int64_t inner, int32_t dim, int32_t per_outer) {
  const int64_t rows = per_outer ? inner : outer * inner, groups = per_outer ? outer : 1;
  if (rows <= 0 || groups <= 0 || dim <= 0) return 0;
  if (dim > norm::kMaxDimRegs) return 2 * rows * groups;
  // which of the two layouts runs depends on alignments that are not known here: room for either
  int64_t blocks = 1;
  for (int vec = 0; vec < (dim % 4 == 0 ? 2 : 1); ++vec) {
    const norm::Blocks b = norm::bwd_blocks(rows, dim, groups, vec, true);
    if (!b.cluster) blocks = std::max(blocks, b.n);
  }
  return blocks > 1 ? groups * blocks * 2 * dim : 0;
}

int launch_layer_norm(const fb_layer_norm_args& p, bool bwd, cudaStream_t st, std::string& err) {
  const char* who = bwd ? "fb_layer_norm_backward" : "fb_layer_norm";
  auto bad = [&](int code, const char* what) {
    err = std::string(who) + ": " + what;
    return code;
  };
  if (p.outer < 0 || p.inner < 0 || p.dim < 1) return bad(FB_ERR_ARG, "need outer, inner >= 0 and dim >= 1");
  if (p.dim > (1 << 30)) return bad(FB_ERR_UNSUPPORTED, "at most 2^30 elements per row");
  if (!norm::is_dtype(p.x_dtype) || !norm::is_dtype(p.y_dtype) || !norm::is_dtype(p.w_dtype))
    return bad(FB_ERR_ARG, "dtypes must be FB_F32, FB_F16 or FB_BF16");
  if (!(p.eps >= 0.0f)) return bad(FB_ERR_ARG, "eps must be >= 0");
  const bool sums = bwd && (p.dweight || p.dbias);
  if (sums && (!p.dweight || !p.dbias)) return bad(FB_ERR_ARG, "dweight and dbias come together");
  const int64_t rows_all = (p.inner > 0 && p.outer > (1ll << 31) / p.inner) ? (1ll << 40) : p.outer * p.inner;
  if (rows_all > (1ll << 30)) return bad(FB_ERR_UNSUPPORTED, "at most 2^30 rows per call");
  // A block of the backward pass works with one w, so a w per outer index makes a sum group of each.
  const bool per_outer = bwd && ((sums && p.sum_per_outer) || p.w_outer_stride != 0);
  if (sums && per_outer && !p.sum_per_outer) return bad(FB_ERR_UNSUPPORTED, "a weight per outer index has sums per outer index");
  const int64_t groups = per_outer ? p.outer : 1;
  if (groups > 65535) return bad(FB_ERR_UNSUPPORTED, "at most 65535 gradients of their own per call");
  if (rows_all == 0) {
    if (sums && groups > 0) {  // sums over no rows
      const size_t n = static_cast<size_t>(groups) * p.dim * sizeof(float);
      cudaError_t e = cudaMemsetAsync(p.dweight, 0, n, st);
      if (e == cudaSuccess) e = cudaMemsetAsync(p.dbias, 0, n, st);
      if (e != cudaSuccess) {
        err = std::string(who) + ": " + cudaGetErrorString(e);
        return FB_ERR_CUDA;
      }
    }
    return FB_OK;
  }
  if (!p.x || !p.out || (bwd && !p.dy)) return bad(FB_ERR_ARG, "null pointer");
  if (p.out == p.x || (bwd && p.out == p.dy)) return bad(FB_ERR_ARG, "out must not be x or dy");  // rows may be read again
  if (norm::misaligned(p.x, p.x_dtype) || norm::misaligned(p.out, bwd ? p.x_dtype : p.y_dtype) ||
      (bwd && (norm::misaligned(p.dy, p.y_dtype) || (p.add && norm::misaligned(p.add, p.x_dtype)))) ||
      (p.weight && norm::misaligned(p.weight, p.w_dtype)) || (p.bias && norm::misaligned(p.bias, p.w_dtype)) ||
      norm::misaligned(p.dweight, FB_F32) || norm::misaligned(p.dbias, FB_F32) || norm::misaligned(p.work, FB_F32))
    return bad(FB_ERR_ALIGN, "a pointer is not aligned to its elements");
  std::string derr;
  if (!device_for(Operator::kLayerNorm, derr)) {  // raises the kernels' shared-memory limits on this device
    err = derr;
    return FB_ERR_INIT;
  }
  norm::Args a;
  memset(&a, 0, sizeof(a));
  a.x = p.x;
  a.dy = p.dy;
  a.add = bwd ? p.add : nullptr;
  a.out = p.out;
  a.w = p.weight;
  a.b = p.bias;
  a.xo = p.x_outer_stride, a.xi = p.x_inner_stride;
  a.yo = p.dy_outer_stride, a.yi = p.dy_inner_stride;
  a.ao = p.add_outer_stride, a.ai = p.add_inner_stride;
  a.oo = p.out_outer_stride, a.oi = p.out_inner_stride;
  a.w_stride = p.w_outer_stride;
  a.inner = static_cast<int>(p.inner);
  a.rows = static_cast<int>(per_outer ? p.inner : rows_all);
  a.dim = p.dim;
  a.x_type = p.x_dtype;
  a.y_type = p.y_dtype;
  a.w_type = p.w_dtype;
  a.w_plus = p.weight_plus_one ? 1.0f : 0.0f;
  a.eps = p.eps;
  if (sums) {
    const int64_t need = layer_norm_work_floats(p.outer, p.inner, p.dim, p.sum_per_outer);
    if (p.work_floats < need || (need > 0 && !p.work)) return bad(FB_ERR_ARG, "workspace too small");
    a.part = p.work;
    a.dw = p.dweight;
    a.db = p.dbias;
  }
  bool vec = p.dim % 4 == 0 && norm::vec4(p.x, p.x_dtype, {a.xo, a.xi}) &&
             norm::vec4(p.out, bwd ? p.x_dtype : p.y_dtype, {a.oo, a.oi});
  if (bwd) vec = vec && norm::vec4(p.dy, p.y_dtype, {a.yo, a.yi}) && (!p.add || norm::vec4(p.add, p.x_dtype, {a.ao, a.ai}));
  if (p.weight) vec = vec && norm::vec4(p.weight, p.w_dtype, {a.w_stride});
  if (p.bias) vec = vec && norm::vec4(p.bias, p.w_dtype, {a.w_stride});
  const cudaError_t e = norm::dispatch(a, bwd, groups, vec, st);
  if (e != cudaSuccess) {
    err = std::string(who) + ": " + cudaGetErrorString(e);
    return FB_ERR_CUDA;
  }
  return FB_OK;
}

}  // namespace fb
