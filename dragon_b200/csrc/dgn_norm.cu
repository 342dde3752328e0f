// Root-mean-square norm with the residual's addition, its output in the input's
// type or in 8 bits with scales, and its backward pass.
//
//   h = T(x + r)                    rounded once to the storage type, so that the backward pass sees the same h
//   rstd = (mean(h^2) + eps)^(-1/2)
//   y = h * rstd * w
//   codes = rn(y * L / amax), scale = amax / L       per group of columns; L the largest value of the 8-bit type
//
//   g = dy * w,  n = h * rstd
//   dh = rstd * (g - n * mean(g * n)) + dres         (the gradient of x and of r alike)
//   dw = sum over rows of dy * n
//
// Sums are held in 32 bits.  A row is read once: it stays in registers, packed in
// its storage type, between the sum of squares and the output.
//
// Bound by memory: 8192 rows of 4096 bfloat16 columns with a residual take 42.9 us forward
// (6.3 TB/s, 97 % of the measured copy rate) and 44.8 us backward (93 %: 41 without the
// weight gradient, whose partial sums go through the second cache and a second kernel).
// With 8-bit output it is the instructions, 44.7 us for bytes of 36.3: each value is rounded,
// multiplied twice, compared and converted.  Rows that are not aligned move by single or
// paired elements and are bound by their number: 4097 columns take 96 us forward, 277 backward.
#include <cuda_fp8.h>
#include <math.h>

#include "dgn_kernels.cuh"
#include "dgn_ops.h"

namespace {

using namespace dgn;

constexpr int kMaxCols = 32768;
constexpr int kSMs = 148;
constexpr float kSmallestAmax = 0x1p-40f;  // groups whose largest value is below this take this one's scale
constexpr int kThreads = 256;              // of a block whose rows belong to teams of its threads

struct NormParams {
  const char* x;
  const char* residual;  // may be null
  const char* weight;    // may be null
  char* hidden;          // may be null when residual is
  char* out;
  float* scales;
  float* rstd;
  long long rows, x_stride, residual_stride, hidden_stride;  // strides in elements
  int cols, group_shift, groups;  // columns per scale as a power of two; scales per row
  int weight_f32, code;
  float eps, inv_cols, largest, inv_largest;  // the largest code
};

// Threads and columns.  A row belongs to a team of `team` threads; each of them holds NV
// parts of E elements (16 bytes), made of words of W neighbouring elements.  W = E: rows
// aligned to 16 bytes.  W = 2 (16-bit types, an even number of columns) and W = 1: other rows.
// Neighbouring threads have neighbouring words, so that narrow loads still fill whole lines.
template <int BYTES> struct Word;
template <> struct Word<2> { typedef unsigned short type; };
template <> struct Word<4> { typedef unsigned type; };

template <typename T, int W>
__device__ __forceinline__ int column(int i, int e, int thread, int team) {
  constexpr int Q = Elem<T>::E / W;
  return ((i * Q + e / W) * team + thread) * W + e % W;
}

template <typename T, int W>
__device__ __forceinline__ uint4 load_part(const char* row, int i, int thread, int team, int cols) {
  constexpr int E = Elem<T>::E;
  if constexpr (W == E) {
    const int c = column<T, W>(i, 0, thread, team);
    return c < cols ? *reinterpret_cast<const uint4*>(row + (size_t)c * sizeof(T)) : make_uint4(0, 0, 0, 0);
  } else {
    typedef typename Word<W * sizeof(T)>::type U;
    uint4 v = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int e = 0; e < E; e += W) {
      const int c = column<T, W>(i, e, thread, team);
      if (c < cols) reinterpret_cast<U*>(&v)[e / W] = *reinterpret_cast<const U*>(row + (size_t)c * sizeof(T));
    }
    return v;
  }
}
template <typename T, int W>
__device__ __forceinline__ void store_part(char* row, int i, int thread, int team, int cols, uint4 v) {
  constexpr int E = Elem<T>::E;
  if constexpr (W == E) {
    const int c = column<T, W>(i, 0, thread, team);
    if (c < cols) *reinterpret_cast<uint4*>(row + (size_t)c * sizeof(T)) = v;
  } else {
    typedef typename Word<W * sizeof(T)>::type U;
#pragma unroll
    for (int e = 0; e < E; e += W) {
      const int c = column<T, W>(i, e, thread, team);
      if (c < cols) *reinterpret_cast<U*>(row + (size_t)c * sizeof(T)) = reinterpret_cast<const U*>(&v)[e / W];
    }
  }
}

// The weights of a part in float32: ones without a weight, zeros behind the last column.
template <typename T, int W>
__device__ __forceinline__ void load_weight(const char* weight, int f32, int i, int thread, int team, int cols, float* w) {
  constexpr int E = Elem<T>::E;
  if (!weight) {
#pragma unroll
    for (int e = 0; e < E; ++e) w[e] = 1.f;
  } else if (!f32) {
    Elem<T>::unpack(load_part<T, W>(weight, i, thread, team, cols), w);
  } else if (W == E) {
    const int c = column<T, W>(i, 0, thread, team);
#pragma unroll
    for (int e = 0; e < E; e += 4) {
      const float4 f = c < cols ? *reinterpret_cast<const float4*>(weight + (size_t)(c + e) * 4) : make_float4(0, 0, 0, 0);
      w[e] = f.x; w[e + 1] = f.y; w[e + 2] = f.z; w[e + 3] = f.w;
    }
  } else {
#pragma unroll
    for (int e = 0; e < E; e += W) {
      const int c = column<T, W>(i, e, thread, team);
      const bool there = c < cols;
      if (W == 2) {
        const float2 f = there ? *reinterpret_cast<const float2*>(weight + (size_t)c * 4) : make_float2(0, 0);
        w[e] = f.x; w[e + 1] = f.y;
      } else {
        w[e] = there ? *reinterpret_cast<const float*>(weight + (size_t)c * 4) : 0.f;
      }
    }
  }
}

// Two float32 values in one instruction (add, mul and fma of f32x2, each rounded as the single one is).
struct Pair {
  u64 v;
  __device__ Pair() {}
  __device__ Pair(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
  __device__ float2 get() const {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
    return f;
  }
};
__device__ __forceinline__ Pair operator+(Pair a, Pair b) {
  asm("add.rn.f32x2 %0, %0, %1;" : "+l"(a.v) : "l"(b.v));
  return a;
}
__device__ __forceinline__ Pair operator*(Pair a, Pair b) {
  asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(a.v) : "l"(b.v));
  return a;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(c.v) : "l"(a.v), "l"(b.v));
  return c;
}
__device__ __forceinline__ Pair twice(float a) { return Pair(a, a); }

// The E values of a part as pairs, and back.
template <typename T> __device__ __forceinline__ void unpack2(uint4 v, Pair* a) {
  float f[Elem<T>::E];
  Elem<T>::unpack(v, f);
#pragma unroll
  for (int e = 0; e < Elem<T>::E; e += 2) a[e / 2] = Pair(f[e], f[e + 1]);
}
template <typename T> __device__ __forceinline__ uint4 pack2(const Pair* a) {
  float f[Elem<T>::E];
#pragma unroll
  for (int e = 0; e < Elem<T>::E; e += 2) {
    const float2 p = a[e / 2].get();
    f[e] = p.x; f[e + 1] = p.y;
  }
  return Elem<T>::pack(f);
}
template <typename T, int W>
__device__ __forceinline__ void load_weight2(const char* weight, int f32, int i, int thread, int team, int cols, Pair* w) {
  float f[Elem<T>::E];
  load_weight<T, W>(weight, f32, i, thread, team, cols, f);
#pragma unroll
  for (int e = 0; e < Elem<T>::E; e += 2) w[e / 2] = Pair(f[e], f[e + 1]);
}

struct Sum { static __device__ float of(float a, float b) { return a + b; } };
// The larger magnitude; a NaN stays one.
struct Largest { static __device__ float of(float a, float b) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(fabsf(a)), "f"(fabsf(b)));
  return m;
} };

// One value of each of RU rows for all threads of their team: TEAM lanes of a warp, or
// (TEAM 0) the block, whose warps meet in `slot`.  A slot is written again only behind
// another barrier of the caller's: two of them take turns.
template <typename Op, int TEAM, int RU>
__device__ __forceinline__ void team_reduce(float (&v)[RU], float* slot) {
#pragma unroll
  for (int d = (TEAM ? TEAM : 32) / 2; d; d >>= 1)
#pragma unroll
    for (int u = 0; u < RU; ++u) v[u] = Op::of(v[u], __shfl_xor_sync(0xffffffffu, v[u], d));
  if (TEAM) return;
  const int warps = blockDim.x >> 5;
  if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = v[0];
  if (threadIdx.x >= warps && threadIdx.x < 32) slot[threadIdx.x] = 0.f;
  __syncthreads();
  float all = 0.f;
  for (int w = 0; w < warps; w += 4) {
    const float4 f = *reinterpret_cast<const float4*>(slot + w);
    all = Op::of(all, Op::of(Op::of(f.x, f.y), Op::of(f.z, f.w)));
  }
  v[0] = all;
}

__device__ __forceinline__ unsigned encode1(float a, int code) {
  if (code == DGN_CODE_I8) return (unsigned)min(max(__float2int_rn(a), -127), 127) & 255;  // NaN -> 0
  return __nv_cvt_float_to_fp8(a, __NV_SATFINITE, code == DGN_CODE_E4M3 ? __NV_E4M3 : __NV_E5M2);
}
// E codes, the first in the lowest byte.
template <int E>
__device__ __forceinline__ uint2 encode(const Pair* a, int code) {
  unsigned w[4] = {0, 0, 0, 0};
  if (code == DGN_CODE_I8) {
#pragma unroll
    for (int e = 0; e < E / 2; ++e) {
      const float2 f = a[e].get();
      w[e] = encode1(f.x, DGN_CODE_I8) | encode1(f.y, DGN_CODE_I8) << 8;
    }
  } else if (code == DGN_CODE_E4M3) {
#pragma unroll
    for (int e = 0; e < E / 2; ++e) w[e] = __nv_cvt_float2_to_fp8x2(a[e].get(), __NV_SATFINITE, __NV_E4M3);
  } else {
#pragma unroll
    for (int e = 0; e < E / 2; ++e) w[e] = __nv_cvt_float2_to_fp8x2(a[e].get(), __NV_SATFINITE, __NV_E5M2);
  }
  return make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
}

// (mean + eps)^(-1/2); 0 where the mean is infinite.
__device__ __forceinline__ float inverse_root(float v) { return __frsqrt_rn(v); }

// Codes of values h * w * rstd from u = h * w alone: with m the largest |u| of the group, code = rn(u * (L / m)) and
// scale = m * rstd / L, so that rstd's rounding does not move a code.  L / m is kept as a quotient and its remainder's (the
// double-length division of Dekker, 1971): of values of few bits u L / m often lies halfway between two codes, and one
// float32 for L / m would leave that place by its rounding (27 codes of a million of bfloat16 rows and weights went to the
// wrong neighbour; with both the product is rounded once).
__device__ __forceinline__ float2 code_factor(float m, float rstd, float largest, float inv_largest) {
  const float top = m * rstd;
  if (!(top < __uint_as_float(0x7f800000u))) return make_float2(__uint_as_float(0x7fffffffu), 0.f);  // NaN, infinity: NaN
  if (top < kSmallestAmax) return make_float2(largest * rstd * (1.f / kSmallestAmax), 0.f);
  const float f = __fdividef(0.25f * largest, 0.25f * m);  // a quarter: the call gives 0 for divisors above 2^126
  return make_float2(f, fmaf(-f, m, largest) * (f * inv_largest));
}
__device__ __forceinline__ float times(float u, float2 f) { return fmaf(u, f.x, u * f.y); }
__device__ __forceinline__ float code_scale(float m, float rstd, float inv_largest) {
  const float top = m * rstd;
  return top < __uint_as_float(0x7f800000u) ? fmaxf(top, kSmallestAmax) * inv_largest : __uint_as_float(0x7fffffffu);
}

// One row for a block (TEAM 0), or RU rows for a team of TEAM lanes; rows that are read
// together lie next to each other.
template <typename T, int TEAM, int NV, int W, bool CODES>
__global__ void __launch_bounds__(TEAM || (NV == 2 && W == Elem<T>::E) ? kThreads : NV == 2 ? 512 : 1024)
    rms_norm_kernel(const __grid_constant__ NormParams p) {
  constexpr int E = Elem<T>::E;
  constexpr bool VEC = W == E;
  constexpr int RU = !TEAM || !VEC ? 1 : NV == 1 ? 4 : NV == 2 ? 2 : 1;
  constexpr long long S = sizeof(T);
  __shared__ __align__(16) float slot[2][32];
  __shared__ float chunk[VEC || !CODES ? 1 : 1024];  // largest magnitude of 32 columns each
  __shared__ float2 factor[VEC || !CODES ? 1 : 1024];
  const int team = TEAM ? TEAM : blockDim.x, me = threadIdx.x, cols = p.cols;
  const long long first = (long long)blockIdx.x * blockDim.y * RU + threadIdx.y;
  uint4 h[RU][NV], r[RU][NV];
#pragma unroll
  for (int u = 0; u < RU; ++u) {
    const long long row = first + u * blockDim.y;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      h[u][i] = r[u][i] = make_uint4(0, 0, 0, 0);
      if (row < p.rows) {
        h[u][i] = load_part<T, W>(p.x + row * p.x_stride * S, i, me, team, cols);
        if (p.residual) r[u][i] = load_part<T, W>(p.residual + row * p.residual_stride * S, i, me, team, cols);
      }
    }
  }
  float sum[RU], rstd[RU];
#pragma unroll
  for (int u = 0; u < RU; ++u) {
    const long long row = first + u * blockDim.y;
    Pair squares(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      Pair a[E / 2];
      unpack2<T>(h[u][i], a);
      if (p.residual) {
        Pair b[E / 2];
        unpack2<T>(r[u][i], b);
#pragma unroll
        for (int e = 0; e < E / 2; ++e) a[e] = a[e] + b[e];
        h[u][i] = pack2<T>(a);
        if (sizeof(T) < 4) unpack2<T>(h[u][i], a);
        if (row < p.rows) store_part<T, W>(p.hidden + row * p.hidden_stride * S, i, me, team, cols, h[u][i]);
      }
#pragma unroll
      for (int e = 0; e < E / 2; ++e) squares = fma2(a[e], a[e], squares);
    }
    sum[u] = squares.get().x + squares.get().y;
  }
  team_reduce<Sum, TEAM>(sum, slot[0]);
#pragma unroll
  for (int u = 0; u < RU; ++u) {
    const long long row = first + u * blockDim.y;
    rstd[u] = inverse_root(fmaf(sum[u], p.inv_cols, p.eps));
    if (me == 0 && row < p.rows) p.rstd[row] = rstd[u];
  }

  if (!CODES) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      Pair w[E / 2];
      load_weight2<T, W>(p.weight, p.weight_f32, i, me, team, cols, w);
#pragma unroll
      for (int u = 0; u < RU; ++u) {
        const long long row = first + u * blockDim.y;
        Pair a[E / 2];
        unpack2<T>(h[u][i], a);
#pragma unroll
        for (int e = 0; e < E / 2; ++e) a[e] = a[e] * twice(rstd[u]) * w[e];
        if (row < p.rows) store_part<T, W>(p.out + row * cols * S, i, me, team, cols, pack2<T>(a));
      }
    }
    return;
  }

  // 8-bit codes.  Aligned rows: a group of at most 128 columns lies in neighbouring lanes of one warp.  Other rows: 32
  // columns lie in the lanes of a warp, and larger groups are put together in shared memory.
  const float largest = p.largest;
  const bool whole = p.groups == 1;
  float top[RU];
  if (whole || !VEC) {
#pragma unroll
    for (int u = 0; u < RU; ++u) top[u] = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float w[E];
      load_weight<T, W>(p.weight, p.weight_f32, i, me, team, cols, w);
#pragma unroll
      for (int u = 0; u < RU; ++u) {
        float a[E];
        Elem<T>::unpack(h[u][i], a);
        if (VEC || whole) {
#pragma unroll
          for (int e = 0; e < E; ++e) top[u] = Largest::of(top[u], a[e] * w[e]);
        } else {
#pragma unroll
          for (int e = 0; e < E; e += W) {  // 32 / W lanes hold a chunk's words
            float m = fabsf(a[e] * w[e]);
            if (W == 1) {
              m = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(m)));  // by its bits a NaN is largest
            } else {
              m = Largest::of(m, a[e + 1] * w[e + 1]);
#pragma unroll
              for (int d = 8; d; d >>= 1) m = Largest::of(m, __shfl_xor_sync(0xffffffffu, m, d));
            }
            const int c = column<T, W>(i, e, me, team);
            if ((c & 31) == 0 && c < cols) chunk[threadIdx.y * 32 + (c >> 5)] = m;
          }
        }
      }
    }
    const auto meet = [] { TEAM ? __syncwarp() : __syncthreads(); };
    if (whole) {
      team_reduce<Largest, TEAM>(top, slot[1]);
    } else {
      meet();
      const int chunks = (cols + 31) >> 5, of_group = 1 << (p.group_shift - 5);
      for (int g = me; g < p.groups; g += team) {
        float m = 0.f;
        for (int k = g * of_group; k < min((g + 1) * of_group, chunks); ++k) m = Largest::of(m, chunk[threadIdx.y * 32 + k]);
        factor[threadIdx.y * 32 + g] = code_factor(m, rstd[0], largest, p.inv_largest);
        if (first < p.rows) p.scales[first * p.groups + g] = code_scale(m, rstd[0], p.inv_largest);
      }
      meet();
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    Pair w[E / 2];
    load_weight2<T, W>(p.weight, p.weight_f32, i, me, team, cols, w);
#pragma unroll
    for (int u = 0; u < RU; ++u) {
      const long long row = first + u * blockDim.y;
      unsigned char* out = reinterpret_cast<unsigned char*>(p.out) + row * cols;
      Pair a[E / 2];
      unpack2<T>(h[u][i], a);
#pragma unroll
      for (int e = 0; e < E / 2; ++e) a[e] = a[e] * w[e];
      if (VEC) {
        const int c = column<T, W>(i, 0, me, team);
        float m = 0.f;
        if (whole) {
          m = top[u];
        } else {
#pragma unroll
          for (int e = 0; e < E / 2; ++e) m = Largest::of(m, Largest::of(a[e].get().x, a[e].get().y));
          for (int d = (1 << p.group_shift) / E / 2; d; d >>= 1) m = Largest::of(m, __shfl_xor_sync(0xffffffffu, m, d));
        }
        if (c >= cols || row >= p.rows) continue;
        if (whole ? c == 0 : (c & ((1 << p.group_shift) - 1)) == 0)
          p.scales[row * p.groups + (whole ? 0 : c >> p.group_shift)] = code_scale(m, rstd[u], p.inv_largest);
        const float2 f = code_factor(m, rstd[u], largest, p.inv_largest);
#pragma unroll
        for (int e = 0; e < E / 2; ++e) a[e] = fma2(a[e], twice(f.x), a[e] * twice(f.y));
        const uint2 codes = encode<E>(a, p.code);
        if (E == 8) *reinterpret_cast<uint2*>(out + c) = codes;
        else *reinterpret_cast<unsigned*>(out + c) = codes.x;
      } else {
        const float2 all = code_factor(top[u], rstd[u], largest, p.inv_largest);
        if (whole && me == 0 && i == 0 && row < p.rows) p.scales[row] = code_scale(top[u], rstd[u], p.inv_largest);
#pragma unroll
        for (int e = 0; e < E; e += W) {
          const int c = column<T, W>(i, e, me, team);
          if (c >= cols || row >= p.rows) continue;
          const float2 f = whole ? all : factor[threadIdx.y * 32 + (c >> p.group_shift)];
          const float2 v = a[e / 2].get();
          if (W == 2)
            *reinterpret_cast<unsigned short*>(out + c) =
                (unsigned short)(encode1(times(v.x, f), p.code) | encode1(times(v.y, f), p.code) << 8);
          else
            out[c] = (unsigned char)encode1(times(e & 1 ? v.y : v.x, f), p.code);
        }
      }
    }
  }
}

struct NormGradParams {
  const char* grad_out;
  const char* grad_hidden;  // may be null
  const char* hidden;
  const char* weight;       // may be null
  const float* rstd;
  char* grad_x;
  float* partial;           // [gridDim.x][cols]; null without a weight
  long long rows, grad_out_stride, grad_hidden_stride, hidden_stride;
  int cols, weight_f32;
};

// How much of h the gradient loses: with d = sum(dy w h), rstd n mean(dy w n) = h * rstd^3 d / cols, one factor at a time.
__device__ __forceinline__ float along(float d, float rstd, int cols) { return d * rstd / (float)cols * rstd * rstd; }

// Writes a block's sums of the weight gradient to its row of the partial sums; teams that
// share the block are added in shared memory, in their order.
template <typename T, int TEAM, int NV, int W>
__device__ __forceinline__ void store_partial(const NormGradParams& p, const Pair* sums, float* shared) {
  constexpr int E = Elem<T>::E;
  constexpr bool VEC = W == E;
  const int team = TEAM ? TEAM : blockDim.x, me = threadIdx.x, cols = p.cols;
  float* mine = p.partial + (long long)blockIdx.x * cols;
  float* to = TEAM ? shared + threadIdx.y * cols : mine;
  float acc[NV * E];
#pragma unroll
  for (int i = 0; i < NV * E; ++i) acc[i] = i & 1 ? sums[i / 2].get().y : sums[i / 2].get().x;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = column<T, W>(i, 0, me, team);
    if (VEC && c < cols) {
#pragma unroll
      for (int e = 0; e < E; e += 4)
        *reinterpret_cast<float4*>(to + c + e) = make_float4(acc[i * E + e], acc[i * E + e + 1], acc[i * E + e + 2], acc[i * E + e + 3]);
    } else if (!VEC) {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (column<T, W>(i, e, me, team) < cols) to[column<T, W>(i, e, me, team)] = acc[i * E + e];
    }
  }
  if (!TEAM) return;
  __syncthreads();
  for (int c = threadIdx.y * TEAM + me; c < cols; c += kThreads) {
    float s = 0.f;
    for (int y = 0; y < (int)blockDim.y; ++y) s += shared[y * cols + c];
    mine[c] = s;
  }
}

// The plain form: rows straight into registers.  Taken by rows that are not aligned, by
// short ones (a team of 8 or 16 lanes, four rows at a time) and by those too long for the ring below.
template <typename T, int TEAM, int NV, int W, int MOST = TEAM ? kThreads : 512>
__global__ void __launch_bounds__(MOST, TEAM ? 2 : 1) rms_norm_grad_kernel(const __grid_constant__ NormGradParams p) {
  constexpr int E = Elem<T>::E, RU = TEAM && W == E ? 4 : 1;
  constexpr long long S = sizeof(T);
  extern __shared__ __align__(16) float shared[];  // teams * cols floats
  __shared__ __align__(16) float slot[2][32];
  allow_next();
  const int team = TEAM ? TEAM : blockDim.x, me = threadIdx.x, cols = p.cols;
  Pair acc[NV * E / 2];
#pragma unroll
  for (int i = 0; i < NV * E / 2; ++i) acc[i] = twice(0.f);
  int turn = 0;
  for (long long base = (long long)blockIdx.x * blockDim.y * RU; base < p.rows;
       base += (long long)gridDim.x * blockDim.y * RU, turn ^= 1) {
    uint4 g[RU][NV], h[RU][NV], r[RU][NV];
    float dot[RU], rstd[RU];
#pragma unroll
    for (int u = 0; u < RU; ++u) {
      const long long row = base + u * blockDim.y + threadIdx.y;
      rstd[u] = row < p.rows ? p.rstd[row] : 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        g[u][i] = h[u][i] = r[u][i] = make_uint4(0, 0, 0, 0);
        if (row < p.rows) {
          g[u][i] = load_part<T, W>(p.grad_out + row * p.grad_out_stride * S, i, me, team, cols);
          h[u][i] = load_part<T, W>(p.hidden + row * p.hidden_stride * S, i, me, team, cols);
          if (p.grad_hidden) r[u][i] = load_part<T, W>(p.grad_hidden + row * p.grad_hidden_stride * S, i, me, team, cols);
        }
      }
      dot[u] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      Pair w[E / 2];
      load_weight2<T, W>(p.weight, p.weight_f32, i, me, team, cols, w);
#pragma unroll
      for (int u = 0; u < RU; ++u) {
        Pair a[E / 2], b[E / 2], d(0.f, 0.f);
        unpack2<T>(g[u][i], a);
        unpack2<T>(h[u][i], b);
#pragma unroll
        for (int e = 0; e < E / 2; ++e) {
          d = fma2(a[e] * w[e], b[e], d);
          acc[i * E / 2 + e] = fma2(a[e], b[e] * twice(rstd[u]), acc[i * E / 2 + e]);
        }
        dot[u] += d.get().x + d.get().y;
      }
    }
    team_reduce<Sum, TEAM>(dot, slot[turn]);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      Pair w[E / 2];
      load_weight2<T, W>(p.weight, p.weight_f32, i, me, team, cols, w);
#pragma unroll
      for (int u = 0; u < RU; ++u) {
        const long long row = base + u * blockDim.y + threadIdx.y;
        const Pair back = twice(-along(dot[u], rstd[u], cols)), scale = twice(rstd[u]);
        Pair a[E / 2], b[E / 2], c[E / 2];
        unpack2<T>(g[u][i], a);
        unpack2<T>(h[u][i], b);
        unpack2<T>(r[u][i], c);
#pragma unroll
        for (int e = 0; e < E / 2; ++e) a[e] = fma2(a[e] * w[e], scale, fma2(back, b[e], c[e]));
        if (row < p.rows) store_part<T, W>(p.grad_x + row * cols * S, i, me, team, cols, pack2<T>(a));
      }
    }
  }
  if (p.partial) store_partial<T, TEAM, NV, W>(p, acc, shared);
}

// Stages of a ring: four, or two where a thread has four parts.
__host__ __device__ constexpr int ring_stages(int vectors) { return vectors == 4 ? 2 : 4; }

__device__ __forceinline__ void copy_async(uint4* to, const char* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((unsigned)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}

// Aligned rows (8192 x 4096 bfloat16: 41 us of 41.5 at the copy rate, 62 for the plain form with as
// many blocks).  Each thread copies its own vectors of the rows to come into its own places of a ring in shared memory
// (cp.async), so the loads of STAGES - 1 rows are in flight while one is worked on and nobody waits for another
// thread's copy; the sums of the weight gradient (and up to 16 weights a thread) stay in
// registers for all of the block's rows.
template <typename T, int TEAM, int NV, bool RESIDUAL, int MOST = NV == 4 ? 512 : kThreads>
__global__ void __launch_bounds__(MOST) rms_norm_grad_ring_kernel(const __grid_constant__ NormGradParams p) {
  constexpr int E = Elem<T>::E, STAGES = ring_stages(NV), TENSORS = RESIDUAL ? 3 : 2;
  constexpr long long S = sizeof(T);
  extern __shared__ __align__(16) uint4 ring[];  // [STAGES][TENSORS][NV][threads]
  __shared__ __align__(16) float slot[2][32];
  allow_next();
  const int team = TEAM ? TEAM : blockDim.x, me = threadIdx.x, cols = p.cols;
  const int threads = blockDim.x * blockDim.y, place = threadIdx.y * blockDim.x + me;
  const long long step = (long long)gridDim.x * blockDim.y;
  auto fetch = [&](int stage, long long row) {
    uint4* to = ring + (size_t)stage * TENSORS * NV * threads + place;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = column<T, Elem<T>::E>(i, 0, me, team);
      if (row < p.rows && c < cols) {
        copy_async(to + (0 * NV + i) * threads, p.grad_out + (row * p.grad_out_stride + c) * S);
        copy_async(to + (1 * NV + i) * threads, p.hidden + (row * p.hidden_stride + c) * S);
        if (RESIDUAL) copy_async(to + (2 * NV + i) * threads, p.grad_hidden + (row * p.grad_hidden_stride + c) * S);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  long long row = (long long)blockIdx.x * blockDim.y + threadIdx.y;
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) fetch(s, row + s * step);
  constexpr bool KEEP = NV <= 2;  // the weights in registers; those of four parts are read again for each row
  Pair w[(KEEP ? NV * E : E) / 2], acc[NV * E / 2];
  if (KEEP) {
#pragma unroll
    for (int i = 0; i < NV; ++i) load_weight2<T, Elem<T>::E>(p.weight, p.weight_f32, i, me, team, cols, w + i * E / 2);
  }
#pragma unroll
  for (int i = 0; i < NV * E / 2; ++i) acc[i] = twice(0.f);
  int stage = 0, turn = 0;
  float next_rstd = row < p.rows ? p.rstd[row] : 0.f;
  for (; row < p.rows; row += step, turn ^= 1) {
    const float rstd = next_rstd;
    if (row + step < p.rows) next_rstd = p.rstd[row + step];
    // The stage that the previous row has left.
    fetch(stage == 0 ? STAGES - 1 : stage - 1, row + (STAGES - 1) * step);
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
    const uint4* from = ring + (size_t)stage * TENSORS * NV * threads + place;
    uint4 g[NV], h[NV];
    float dot[1] = {0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      g[i] = h[i] = make_uint4(0, 0, 0, 0);
      if (column<T, Elem<T>::E>(i, 0, me, team) < cols) {
        g[i] = from[(0 * NV + i) * threads];
        h[i] = from[(1 * NV + i) * threads];
      }
      Pair a[E / 2], b[E / 2], *wi = w + (KEEP ? i * E / 2 : 0), d(0.f, 0.f);
      if (!KEEP) load_weight2<T, Elem<T>::E>(p.weight, p.weight_f32, i, me, team, cols, wi);
      unpack2<T>(g[i], a);
      unpack2<T>(h[i], b);
#pragma unroll
      for (int e = 0; e < E / 2; ++e) {
        d = fma2(a[e] * wi[e], b[e], d);
        acc[i * E / 2 + e] = fma2(a[e], b[e] * twice(rstd), acc[i * E / 2 + e]);
      }
      dot[0] += d.get().x + d.get().y;
    }
    team_reduce<Sum, TEAM>(dot, slot[turn]);
    const Pair back = twice(-along(dot[0], rstd, cols)), scale = twice(rstd);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = column<T, Elem<T>::E>(i, 0, me, team);
      if (c >= cols) continue;
      Pair a[E / 2], b[E / 2], f[E / 2], *wi = w + (KEEP ? i * E / 2 : 0);
      if (!KEEP) load_weight2<T, Elem<T>::E>(p.weight, p.weight_f32, i, me, team, cols, wi);
      unpack2<T>(g[i], a);
      unpack2<T>(h[i], b);
      if (RESIDUAL) unpack2<T>(from[(2 * NV + i) * threads], f);
#pragma unroll
      for (int e = 0; e < E / 2; ++e) a[e] = fma2(a[e] * wi[e], scale, RESIDUAL ? fma2(back, b[e], f[e]) : back * b[e]);
      *reinterpret_cast<uint4*>(p.grad_x + (row * cols + c) * S) = pack2<T>(a);
    }
    stage = stage == STAGES - 1 ? 0 : stage + 1;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  if (!p.partial) return;
  if (TEAM) __syncthreads();  // the ring becomes the teams' meeting place
  store_partial<T, TEAM, NV, Elem<T>::E>(p, acc, reinterpret_cast<float*>(ring));
}

// Sum of the partial rows: a block of 32 x 32 threads takes 32 columns, a warp every 32nd partial row.
template <typename W>
__global__ void __launch_bounds__(1024) norm_weight_grad_kernel(const float* partial, W* grad, int parts, int cols) {
  __shared__ float s[32][33];
  await_previous();
  const int c = blockIdx.x * 32 + threadIdx.x;
  float v = 0.f;
  if (c < cols) {
#pragma unroll 8
    for (int i = threadIdx.y; i < parts; i += 32) v += partial[(long long)i * cols + c];
  }
  s[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  v = s[threadIdx.x][threadIdx.y];
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  const int o = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && o < cols) grad[o] = W(v);
}

// Launch shape of a row kernel: a team of `team` threads with `vectors` parts each, `teams` of them in a block.
struct RowShape {
  int team, vectors, teams;
  int lanes() const { return teams > 1 ? team : 0; }  // the kernels' TEAM
};

// Two parts a thread up to 512: with four, 4096 columns of bfloat16 in 8 bits took 45.0 us instead of 42.6 (codes of one
// rounded factor; 44.7 with the quotient and its remainder's).
// Rows of up to 128 parts go to a warp or a half or quarter of one and need no barrier; longer ones to a block, with
// more parts for a thread where the threads would pass 512.
RowShape row_shape(int cols, int elems, bool vec) {
  const int parts = (int)ceil_div(cols, elems);
  if (parts <= 128) {
    const int team = !vec ? 32 : parts <= 8 ? 8 : parts <= 16 ? 16 : 32;
    return {team, parts <= 32 ? 1 : parts <= 64 ? 2 : 4, kThreads / team};
  }
  const int vectors = parts <= (vec ? 512 : 1024) ? 2 : parts <= 4096 ? 4 : 8;
  return {(int)ceil_div(ceil_div(parts, vectors), 32) * 32, vectors, 1};
}

// The backward pass keeps the weights and their gradient in registers: two parts a thread wherever 512 threads will do.
// With four, whose weights are read again for each row, 32768 rows of 1024 bfloat16 columns took 55.7 us instead of 46.7;
// two for each of 1024 threads spill (2048 rows of 16384 columns: 85 us, 78 with four for 512).
RowShape grad_shape(int cols, int elems, bool vec) {
  const int parts = (int)ceil_div(cols, elems);
  if (!vec || parts <= 64 || parts > 1024) return row_shape(cols, elems, vec);
  return {(int)ceil_div(parts, 64) * 32, 2, 1};
}

template <typename T, int W, bool CODES>
const void* norm_kernel_of(const RowShape& s) {
  if constexpr (W == Elem<T>::E) {
    if (s.lanes() == 8) return (const void*)rms_norm_kernel<T, 8, 1, W, CODES>;
    if (s.lanes() == 16) return (const void*)rms_norm_kernel<T, 16, 1, W, CODES>;
  }
  if (s.lanes() == 32) {
    if (s.vectors == 1) return (const void*)rms_norm_kernel<T, 32, 1, W, CODES>;
    if (s.vectors == 2) return (const void*)rms_norm_kernel<T, 32, 2, W, CODES>;
    return (const void*)rms_norm_kernel<T, 32, 4, W, CODES>;
  }
  if (s.vectors == 2) return (const void*)rms_norm_kernel<T, 0, 2, W, CODES>;
  if constexpr (Elem<T>::E == 4)  // more than 4096 parts: float32 only
    if (s.vectors == 8) return (const void*)rms_norm_kernel<T, 0, 8, W, CODES>;
  return (const void*)rms_norm_kernel<T, 0, 4, W, CODES>;
}
template <typename T, int W>
const void* norm_kernel_of(const RowShape& s, bool codes) {
  return codes ? norm_kernel_of<T, W, true>(s) : norm_kernel_of<T, W, false>(s);
}
template <typename T>
const void* norm_kernel(const RowShape& s, int word, bool codes) {
  if (word == Elem<T>::E) return norm_kernel_of<T, Elem<T>::E>(s, codes);
  if constexpr (sizeof(T) == 2)
    if (word == 2) return norm_kernel_of<T, 2>(s, codes);
  return norm_kernel_of<T, 1>(s, codes);
}

// Whether the ring takes a row: aligned, more than 16 parts, and two stages of 512 threads' parts are enough.
bool ring_takes(const RowShape& s, bool vec) { return vec && s.team > 16 && s.team <= 512; }

template <typename T, int W>
const void* norm_grad_kernel_of(const RowShape& s) {
  if constexpr (W == Elem<T>::E) {
    if (s.lanes() == 8) return (const void*)rms_norm_grad_kernel<T, 8, 1, W>;
    if (s.lanes() == 16) return (const void*)rms_norm_grad_kernel<T, 16, 1, W>;
  } else {
    if (s.lanes() == 32) {
      if (s.vectors == 1) return (const void*)rms_norm_grad_kernel<T, 32, 1, W>;
      if (s.vectors == 2) return (const void*)rms_norm_grad_kernel<T, 32, 2, W>;
      return (const void*)rms_norm_grad_kernel<T, 32, 4, W>;
    }
    if (s.vectors == 2) return (const void*)rms_norm_grad_kernel<T, 0, 2, W>;
    if (s.team <= 512) return (const void*)rms_norm_grad_kernel<T, 0, 4, W>;
  }
  if constexpr (Elem<T>::E == 4)
    if (s.vectors == 8) return (const void*)rms_norm_grad_kernel<T, 0, 8, W, 1024>;
  return (const void*)rms_norm_grad_kernel<T, 0, 4, W, 1024>;
}
template <typename T, bool RESIDUAL>
const void* norm_grad_ring_of(const RowShape& s) {
  if (s.lanes() == 32)
    return s.vectors == 1 ? (const void*)rms_norm_grad_ring_kernel<T, 32, 1, RESIDUAL>
                          : (const void*)rms_norm_grad_ring_kernel<T, 32, 2, RESIDUAL>;
  if (s.vectors == 4) return (const void*)rms_norm_grad_ring_kernel<T, 0, 4, RESIDUAL>;
  return s.team <= kThreads ? (const void*)rms_norm_grad_ring_kernel<T, 0, 2, RESIDUAL>
                            : (const void*)rms_norm_grad_ring_kernel<T, 0, 2, RESIDUAL, 512>;
}
template <typename T>
const void* norm_grad_kernel(const RowShape& s, int word, bool residual) {
  constexpr int E = Elem<T>::E;
  if (ring_takes(s, word == E)) return residual ? norm_grad_ring_of<T, true>(s) : norm_grad_ring_of<T, false>(s);
  if (word == E) return norm_grad_kernel_of<T, E>(s);
  if constexpr (sizeof(T) == 2)
    if (word == 2) return norm_grad_kernel_of<T, 2>(s);
  return norm_grad_kernel_of<T, 1>(s);
}

// Shared memory of a backward block.
size_t grad_shared(const RowShape& s, bool vec, bool residual, int64_t cols) {
  if (ring_takes(s, vec)) return (size_t)ring_stages(s.vectors) * (residual ? 3 : 2) * s.vectors * s.team * s.teams * 16;
  return s.teams > 1 ? (size_t)s.teams * cols * sizeof(float) : 0;
}

// Blocks of the backward pass: as many as fit an SM by their shared memory and at 128 registers a thread, eight at most,
// and no more than there are rows for.
int grad_blocks(const RowShape& s, size_t shared, int64_t rows) {
  const int64_t by_shared = shared ? (int64_t)(220 << 10) / (int64_t)shared : 8, by_threads = 512 / (s.team * s.teams);
  const int64_t fit = by_shared < by_threads ? by_shared : by_threads;
  const int64_t most = kSMs * (fit < 1 ? 1 : fit > 8 ? 8 : fit), sets = ceil_div(rows, s.teams);
  return (int)(sets < most ? sets : most);
}

int check_matrix(int64_t rows, int64_t cols, int dtype) {
  if (!float_dtype(dtype)) return report_error(DGN_ERR_UNSUPPORTED, "the norm takes float16, bfloat16 or float32");
  if (rows < 0 || rows > INT32_MAX) return report_error(DGN_ERR_ARG, "the norm takes 0..2^31-1 rows");
  if (cols < 1 || cols > kMaxCols) return report_error(DGN_ERR_ARG, "the norm takes rows of 1..32768 columns");
  return DGN_OK;
}

}  // namespace

extern "C" int dgn_rms_norm(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride,
                            const void* weight, int weight_dtype, void* hidden, int64_t hidden_stride, void* out,
                            int code, int64_t group, float* scales, float* rstd, int64_t rows, int64_t cols, float eps,
                            int dtype, int device, void* stream) {
  int rc = check_matrix(rows, cols, dtype);
  if (rc != DGN_OK) return rc;
  // Not below the normal numbers: rstd of a row of zeros times the inverse of the smallest scale stays finite.
  if (!(eps >= 0x1p-126f) || isinf(eps)) return report_error(DGN_ERR_ARG, "eps must be a positive number, 2^-126 at least");
  if (code < DGN_CODE_NONE || code > DGN_CODE_E5M2) return report_error(DGN_ERR_ARG, "unknown 8-bit code");
  if (group != 0 && group != 32 && group != 64 && group != 128)
    return report_error(DGN_ERR_ARG, "a scale covers 32, 64 or 128 columns, or the row (0)");
  if (weight && weight_dtype != dtype && weight_dtype != DGN_F32)
    return report_error(DGN_ERR_ARG, "the weight is float32 or of the input's type");
  if (rows == 0) return DGN_OK;
  if (!x || !out || !rstd || (residual && !hidden) || (code && !scales))
    return report_error(DGN_ERR_ARG, "dgn_rms_norm: null pointer");
  if (x_stride < cols || (residual && (residual_stride < cols || hidden_stride < cols)))
    return report_error(DGN_ERR_ARG, "a row stride is shorter than the row");
  if (residual && hidden == residual && hidden_stride != residual_stride)
    return report_error(DGN_ERR_ARG, "in place, hidden has the residual's stride");
  const int es = (int)dgn_dtype_size(dtype), elems = 16 / es;
  const size_t ws = weight_dtype == DGN_F32 ? 4 : es;
  if (!aligned(x, es) || !aligned(residual, es) || !aligned(hidden, es) || !aligned(out, code ? 1 : es) ||
      (weight && !aligned(weight, ws)) || !aligned(scales, 4) || !aligned(rstd, 4))
    return report_error(DGN_ERR_ARG, "a pointer is not aligned to its element size");
  // Whether words of `w` elements divide the rows and what they lie in.
  const auto fits = [&](int w) {
    const size_t bytes = (size_t)w * es;
    return cols % w == 0 && x_stride % w == 0 && aligned(x, bytes) && aligned(out, code ? w : bytes) &&
           (!weight || aligned(weight, w * ws > 16 ? 16 : w * ws)) &&
           (!residual || (residual_stride % w == 0 && hidden_stride % w == 0 && aligned(residual, bytes) && aligned(hidden, bytes)));
  };
  const int word = fits(elems) ? elems : es == 2 && fits(2) ? 2 : 1;
  const bool vec = word == elems;
  const RowShape s = row_shape((int)cols, elems, vec);
  NormParams p;
  p.x = static_cast<const char*>(x);
  p.residual = static_cast<const char*>(residual);
  p.weight = static_cast<const char*>(weight);
  p.hidden = static_cast<char*>(hidden);
  p.out = static_cast<char*>(out);
  p.scales = scales;
  p.rstd = rstd;
  p.rows = rows;
  p.x_stride = x_stride;
  p.residual_stride = residual_stride;
  p.hidden_stride = hidden_stride;
  p.cols = (int)cols;
  p.group_shift = group == 32 ? 5 : group == 64 ? 6 : 7;
  p.groups = group ? (int)ceil_div(cols, group) : 1;
  p.weight_f32 = weight_dtype == DGN_F32;
  p.code = code;
  p.eps = eps;
  p.inv_cols = 1.f / (float)cols;
  p.largest = code == DGN_CODE_I8 ? 127.f : code == DGN_CODE_E4M3 ? 448.f : 57344.f;
  p.inv_largest = 1.f / p.largest;
  const void* fn = dtype == DGN_F32   ? norm_kernel<float>(s, word, code != 0)
                   : dtype == DGN_F16 ? norm_kernel<__half>(s, word, code != 0)
                                      : norm_kernel<__nv_bfloat16>(s, word, code != 0);
  OnDevice on(device);
  if (on.error() != cudaSuccess) return report_error(DGN_ERR_CUDA, cudaGetErrorString(on.error()));
  // Rows of a block, as in the kernel: short aligned rows are taken four (one part) or two (two parts) at a time.
  const int set = s.teams == 1 || !vec ? s.teams : s.teams * (s.vectors == 1 ? 4 : s.vectors == 2 ? 2 : 1);
  void* args[] = {&p};
  return launch(fn, dim3((unsigned)ceil_div(rows, set)), dim3(s.team, s.teams), 0, stream, args);
}

extern "C" int64_t dgn_rms_norm_grad_workspace(int64_t rows, int64_t cols, int dtype) {
  if (!float_dtype(dtype) || rows < 1 || cols < 1 || cols > kMaxCols) return 0;
  // Enough for either alignment of the rows, with a residual's gradient or without: one sum for each block.
  int64_t most = 0;
  for (int vec = 0; vec < 2; ++vec)
    for (int residual = 0; residual < 2; ++residual) {
      const RowShape s = grad_shape((int)cols, 16 / (int)dgn_dtype_size(dtype), vec);
      const int64_t blocks = grad_blocks(s, grad_shared(s, vec, residual, cols), rows);
      most = blocks > most ? blocks : most;
    }
  return most * cols * (int64_t)sizeof(float);
}

extern "C" int dgn_rms_norm_grad(const void* grad_out, int64_t grad_out_stride, const void* grad_hidden,
                                 int64_t grad_hidden_stride, const void* hidden, int64_t hidden_stride,
                                 const void* weight, int weight_dtype, const float* rstd, void* grad_x,
                                 void* grad_weight, void* workspace, int64_t workspace_bytes, int64_t rows,
                                 int64_t cols, int dtype, int device, void* stream) {
  int rc = check_matrix(rows, cols, dtype);
  if (rc != DGN_OK) return rc;
  if (weight && weight_dtype != dtype && weight_dtype != DGN_F32)
    return report_error(DGN_ERR_ARG, "the weight is float32 or of the input's type");
  if (grad_weight && !weight) return report_error(DGN_ERR_ARG, "a weight gradient needs the weight");
  const int es = (int)dgn_dtype_size(dtype), elems = 16 / es;
  const size_t ws = weight_dtype == DGN_F32 ? 4 : es;
  if (grad_weight && !aligned(grad_weight, ws))
    return report_error(DGN_ERR_ARG, "a pointer is not aligned to its element size");
  if (rows == 0) {
    if (!grad_weight) return DGN_OK;
    OnDevice on(device);
    if (on.error() != cudaSuccess) return report_error(DGN_ERR_CUDA, cudaGetErrorString(on.error()));
    cudaError_t e = cudaMemsetAsync(grad_weight, 0, (size_t)cols * ws, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? DGN_OK : report_error(DGN_ERR_CUDA, cudaGetErrorString(e));
  }
  if (!grad_out || !hidden || !rstd || !grad_x || (grad_weight && !workspace))
    return report_error(DGN_ERR_ARG, "dgn_rms_norm_grad: null pointer");
  if (grad_out_stride < cols || hidden_stride < cols || (grad_hidden && grad_hidden_stride < cols))
    return report_error(DGN_ERR_ARG, "a row stride is shorter than the row");
  if (!aligned(grad_out, es) || !aligned(hidden, es) || !aligned(grad_hidden, es) || !aligned(grad_x, es) ||
      (weight && !aligned(weight, ws)) || !aligned(rstd, 4) || !aligned(workspace, 4))
    return report_error(DGN_ERR_ARG, "a pointer is not aligned to its element size");
  const auto fits = [&](int w) {
    const size_t bytes = (size_t)w * es;
    return cols % w == 0 && grad_out_stride % w == 0 && hidden_stride % w == 0 && aligned(grad_out, bytes) &&
           aligned(hidden, bytes) && aligned(grad_x, bytes) && (!weight || aligned(weight, w * ws > 16 ? 16 : w * ws)) &&
           (w == 1 || aligned(workspace, 16)) &&
           (!grad_hidden || (grad_hidden_stride % w == 0 && aligned(grad_hidden, bytes)));
  };
  const int word = fits(elems) ? elems : es == 2 && fits(2) ? 2 : 1;
  const bool vec = word == elems;
  const RowShape s = grad_shape((int)cols, elems, vec);
  const size_t smem = grad_shared(s, vec, grad_hidden != nullptr, cols);
  const int parts = grad_blocks(s, smem, rows);
  if (grad_weight && workspace_bytes < (int64_t)parts * cols * (int64_t)sizeof(float))
    return report_error(DGN_ERR_ARG, "dgn_rms_norm_grad: workspace too small");
  NormGradParams p;
  p.grad_out = static_cast<const char*>(grad_out);
  p.grad_hidden = static_cast<const char*>(grad_hidden);
  p.hidden = static_cast<const char*>(hidden);
  p.weight = static_cast<const char*>(weight);
  p.rstd = rstd;
  p.grad_x = static_cast<char*>(grad_x);
  p.partial = grad_weight ? static_cast<float*>(workspace) : nullptr;
  p.rows = rows;
  p.grad_out_stride = grad_out_stride;
  p.grad_hidden_stride = grad_hidden_stride;
  p.hidden_stride = hidden_stride;
  p.cols = (int)cols;
  p.weight_f32 = weight_dtype == DGN_F32;
  OnDevice on(device);
  if (on.error() != cudaSuccess) return report_error(DGN_ERR_CUDA, cudaGetErrorString(on.error()));
  const bool residual = grad_hidden != nullptr;
  const void* fn = dtype == DGN_F32   ? norm_grad_kernel<float>(s, word, residual)
                   : dtype == DGN_F16 ? norm_grad_kernel<__half>(s, word, residual)
                                      : norm_grad_kernel<__nv_bfloat16>(s, word, residual);
  void* args[] = {&p};
  rc = launch(fn, dim3(parts), dim3(s.team, s.teams), smem, stream, args);
  if (rc != DGN_OK || !grad_weight) return rc;
  int nparts = parts, ncols = (int)cols;
  const float* partial = p.partial;
  void* args2[] = {&partial, &grad_weight, &nparts, &ncols};
  const void* fn2 = weight_dtype == DGN_F32 ? (const void*)norm_weight_grad_kernel<float>
                    : dtype == DGN_F16      ? (const void*)norm_weight_grad_kernel<__half>
                                            : (const void*)norm_weight_grad_kernel<__nv_bfloat16>;
  return launch_behind(fn2, dim3((unsigned)ceil_div(cols, 32)), dim3(32, 32), 0, stream, args2);
}
