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
#include <cuda_fp8.h>
#include <math.h>

#include "dgn_kernels.cuh"
#include "dgn_ops.h"

namespace {

using namespace dgn;

constexpr int kMaxCols = 32768;
constexpr int kMaxPartials = 592;         // rows of the weight gradient's partial sums: four blocks on each of 148 SMs
constexpr float kSmallestAmax = 0x1p-40f;  // groups whose largest value is below this take this one's scale

struct NormParams {
  const char* x;
  const char* residual;  // may be null
  const char* weight;    // may be null
  char* hidden;          // may be null when residual is
  char* out;
  float* scales;
  float* rstd;
  long long rows, x_stride, residual_stride, hidden_stride;  // strides in elements
  int cols, group, groups;  // group: columns per scale; groups: scales per row
  int weight_f32, code;
  float eps;
};

// E consecutive elements from column c of a row, zeros behind the last column.
template <typename T, bool VEC>
__device__ __forceinline__ uint4 load_part(const char* row, int c, int cols) {
  if (VEC) return *reinterpret_cast<const uint4*>(row + (size_t)c * sizeof(T));
  const T* p = reinterpret_cast<const T*>(row) + c;
  uint4 v = make_uint4(0, 0, 0, 0);
  T* e = reinterpret_cast<T*>(&v);
#pragma unroll
  for (int i = 0; i < Elem<T>::E; ++i)
    if (c + i < cols) e[i] = p[i];
  return v;
}
template <typename T, bool VEC>
__device__ __forceinline__ void store_part(char* row, int c, int cols, uint4 v) {
  if (VEC) {
    *reinterpret_cast<uint4*>(row + (size_t)c * sizeof(T)) = v;
    return;
  }
  T* p = reinterpret_cast<T*>(row) + c;
  const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
  for (int i = 0; i < Elem<T>::E; ++i)
    if (c + i < cols) p[i] = e[i];
}

// The weights of E columns in float32 (ones without a weight).
template <typename T, bool VEC>
__device__ __forceinline__ void load_weight(const char* weight, int f32, int c, int cols, float* w) {
  constexpr int E = Elem<T>::E;
  if (!weight) {
#pragma unroll
    for (int i = 0; i < E; ++i) w[i] = 1.f;
  } else if (!f32) {
    Elem<T>::unpack(load_part<T, VEC>(weight, c, cols), w);
  } else if (VEC) {
#pragma unroll
    for (int i = 0; i < E; i += 4) {
      const float4 f = *reinterpret_cast<const float4*>(weight + (size_t)(c + i) * 4);
      w[i] = f.x; w[i + 1] = f.y; w[i + 2] = f.z; w[i + 3] = f.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) w[i] = c + i < cols ? reinterpret_cast<const float*>(weight)[c + i] : 0.f;
  }
}

struct Sum { static __device__ float of(float a, float b) { return a + b; } };
// Largest magnitude by the bits of |v|: NaN beats infinity beats every number.
struct Largest { static __device__ float of(float a, float b) {
  return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b))); } };

// One value for all threads of a row: a warp's lanes, then its row's warps through
// shared memory.  `slot` has 32 entries for each row of the block.
template <typename Op>
__device__ __forceinline__ float row_reduce(float v, float* slot) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v = Op::of(v, __shfl_xor_sync(0xffffffffu, v, d));
  const int warps = blockDim.x >> 5;
  if (warps == 1) return v;
  if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = v;
  __syncthreads();
  v = (threadIdx.x & 31) < warps ? slot[threadIdx.x & 31] : 0.f;
#pragma unroll
  for (int d = 16; d; d >>= 1) v = Op::of(v, __shfl_xor_sync(0xffffffffu, v, d));
  __syncthreads();
  return v;
}

__device__ __forceinline__ unsigned encode2(float a, float b, int code) {
  if (code == DGN_CODE_I8) {
    const int i = min(max(__float2int_rn(a), -127), 127), j = min(max(__float2int_rn(b), -127), 127);  // NaN -> 0
    return (unsigned)(i & 255) | (unsigned)(j & 255) << 8;
  }
  return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, code == DGN_CODE_E4M3 ? __NV_E4M3 : __NV_E5M2);
}
__device__ __forceinline__ float largest_code(int code) {
  return code == DGN_CODE_I8 ? 127.f : code == DGN_CODE_E4M3 ? 448.f : 57344.f;
}

// Threads (x, y): x works on row blockIdx.x * blockDim.y + y, which takes blockDim.x * NV * E >= cols columns.
template <typename T, int NV, bool VEC, bool CODES>
__global__ void __launch_bounds__(NV <= 2 ? 512 : 1024) rms_norm_kernel(const __grid_constant__ NormParams p) {
  constexpr int E = Elem<T>::E;
  __shared__ float slot[32];
  const long long row = (long long)blockIdx.x * blockDim.y + threadIdx.y;
  if (row >= p.rows) return;  // rows share a block only when each has one warp: nobody waits for this one
  const char* x = p.x + row * p.x_stride * (long long)sizeof(T);
  const char* r = p.residual ? p.residual + row * p.residual_stride * (long long)sizeof(T) : nullptr;
  char* hidden = r ? p.hidden + row * p.hidden_stride * (long long)sizeof(T) : nullptr;
  uint4 h[NV];
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * blockDim.x + threadIdx.x) * E;
    h[i] = make_uint4(0, 0, 0, 0);
    if (c < p.cols) {
      h[i] = load_part<T, VEC>(x, c, p.cols);
      if (r) {
        float a[E], b[E];
        Elem<T>::unpack(h[i], a);
        Elem<T>::unpack(load_part<T, VEC>(r, c, p.cols), b);
#pragma unroll
        for (int e = 0; e < E; ++e) a[e] += b[e];
        h[i] = Elem<T>::pack(a);
        store_part<T, VEC>(hidden, c, p.cols, h[i]);
      }
    }
    float a[E];
    Elem<T>::unpack(h[i], a);
#pragma unroll
    for (int e = 0; e < E; ++e) sum = fmaf(a[e], a[e], sum);
  }
  sum = row_reduce<Sum>(sum, slot);
  const float rstd = 1.f / sqrtf(sum / (float)p.cols + p.eps);
  if (threadIdx.x == 0) p.rstd[row] = rstd;

  if (!CODES) {
    char* out = p.out + row * p.cols * (long long)sizeof(T);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * blockDim.x + threadIdx.x) * E;
      if (c >= p.cols) break;
      float a[E], w[E];
      Elem<T>::unpack(h[i], a);
      load_weight<T, VEC>(p.weight, p.weight_f32, c, p.cols, w);
#pragma unroll
      for (int e = 0; e < E; ++e) a[e] = a[e] * rstd * w[e];
      store_part<T, VEC>(out, c, p.cols, Elem<T>::pack(a));
    }
    return;
  }

  // 8-bit codes.  A group of at most 128 columns lies in the lanes of one warp (E = 4: 32 lanes); a scale per row
  // takes one more reduction over the row.
  const float largest = largest_code(p.code);
  unsigned char* out = reinterpret_cast<unsigned char*>(p.out) + row * p.cols;
  float whole = 0.f;
  if (p.groups == 1) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * blockDim.x + threadIdx.x) * E;
      if (c >= p.cols) break;
      float a[E], w[E];
      Elem<T>::unpack(h[i], a);
      load_weight<T, VEC>(p.weight, p.weight_f32, c, p.cols, w);
#pragma unroll
      for (int e = 0; e < E; ++e) whole = Largest::of(whole, fabsf(a[e] * rstd * w[e]));
    }
    whole = row_reduce<Largest>(whole, slot);
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * blockDim.x + threadIdx.x) * E;
    float a[E], w[E], amax = 0.f;
    Elem<T>::unpack(h[i], a);
    if (c < p.cols) {
      load_weight<T, VEC>(p.weight, p.weight_f32, c, p.cols, w);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        a[e] = a[e] * rstd * w[e];
        if (VEC || c + e < p.cols) amax = Largest::of(amax, fabsf(a[e]));
      }
    }
    if (p.groups == 1) {
      amax = whole;
    } else {
      for (int d = p.group / E / 2; d; d >>= 1) amax = Largest::of(amax, __shfl_xor_sync(0xffffffffu, amax, d));
    }
    if (c >= p.cols) continue;
    // A group with a NaN or an infinity has no scale: it reads as NaN.
    const bool finite = __float_as_uint(amax) < 0x7f800000u;
    const float top = fmaxf(amax, kSmallestAmax);
    const float inv = finite ? largest / top : __uint_as_float(0x7fffffffu);
    if (c % p.group == 0) p.scales[row * p.groups + c / p.group] = finite ? top / largest : __uint_as_float(0x7fffffffu);
    unsigned code[E / 2];
#pragma unroll
    for (int e = 0; e < E; e += 2) code[e / 2] = encode2(a[e] * inv, a[e + 1] * inv, p.code);
    if (VEC) {
      const unsigned lo = code[0] | code[1] << 16;
      if (E == 8) *reinterpret_cast<uint2*>(out + c) = make_uint2(lo, code[E / 2 - 2] | code[E / 2 - 1] << 16);
      else *reinterpret_cast<unsigned*>(out + c) = lo;
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (c + e < p.cols) out[c + e] = (unsigned char)(code[e / 2] >> (8 * (e & 1)));
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

// Threads as above; a block takes every gridDim.x-th row (or set of blockDim.y rows) and keeps the weight gradient of
// its rows in registers, so that the partial sums are as many as the blocks and their order is fixed.
template <typename T, int NV, bool VEC>
__global__ void __launch_bounds__(NV <= 2 ? 512 : 1024) rms_norm_grad_kernel(const __grid_constant__ NormGradParams p) {
  constexpr int E = Elem<T>::E;
  extern __shared__ float shared[];  // several rows a block: blockDim.y * cols floats
  __shared__ float slot[32];
  float acc[NV * E];
#pragma unroll
  for (int i = 0; i < NV * E; ++i) acc[i] = 0.f;
  for (long long row = (long long)blockIdx.x * blockDim.y + threadIdx.y; row < p.rows;
       row += (long long)gridDim.x * blockDim.y) {
    const char* gp = p.grad_out + row * p.grad_out_stride * (long long)sizeof(T);
    const char* hp = p.hidden + row * p.hidden_stride * (long long)sizeof(T);
    const char* rp = p.grad_hidden ? p.grad_hidden + row * p.grad_hidden_stride * (long long)sizeof(T) : nullptr;
    const float rstd = p.rstd[row];
    uint4 g[NV], h[NV];
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * blockDim.x + threadIdx.x) * E;
      g[i] = h[i] = make_uint4(0, 0, 0, 0);
      if (c < p.cols) {
        g[i] = load_part<T, VEC>(gp, c, p.cols);
        h[i] = load_part<T, VEC>(hp, c, p.cols);
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * blockDim.x + threadIdx.x) * E;
      if (c >= p.cols) break;
      float a[E], b[E], w[E];
      Elem<T>::unpack(g[i], a);
      Elem<T>::unpack(h[i], b);
      load_weight<T, VEC>(p.weight, p.weight_f32, c, p.cols, w);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float n = b[e] * rstd;
        dot = fmaf(a[e] * w[e], n, dot);
        acc[i * E + e] = fmaf(a[e], n, acc[i * E + e]);
      }
    }
    dot = row_reduce<Sum>(dot, slot) / (float)p.cols;
    char* out = p.grad_x + row * p.cols * (long long)sizeof(T);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * blockDim.x + threadIdx.x) * E;
      if (c >= p.cols) break;
      float a[E], b[E], w[E];
      Elem<T>::unpack(g[i], a);
      Elem<T>::unpack(h[i], b);
      load_weight<T, VEC>(p.weight, p.weight_f32, c, p.cols, w);
#pragma unroll
      for (int e = 0; e < E; ++e) a[e] = rstd * (a[e] * w[e] - b[e] * rstd * dot);
      if (rp) {
        Elem<T>::unpack(load_part<T, VEC>(rp, c, p.cols), b);
#pragma unroll
        for (int e = 0; e < E; ++e) a[e] += b[e];
      }
      store_part<T, VEC>(out, c, p.cols, Elem<T>::pack(a));
    }
  }
  if (!p.partial) return;
  float* mine = p.partial + (long long)blockIdx.x * p.cols;
  if (blockDim.y == 1) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * blockDim.x + threadIdx.x) * E;
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (c + e < p.cols) mine[c + e] = acc[i * E + e];
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * blockDim.x + threadIdx.x) * E;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (c + e < p.cols) shared[threadIdx.y * p.cols + c + e] = acc[i * E + e];
  }
  __syncthreads();
  for (int c = threadIdx.y * blockDim.x + threadIdx.x; c < p.cols; c += blockDim.x * blockDim.y) {
    float s = 0.f;
    for (int y = 0; y < (int)blockDim.y; ++y) s += shared[y * p.cols + c];
    mine[c] = s;
  }
}

// Sum of the partial rows: a block of 32 x 32 threads takes 32 columns, a warp every 32nd partial row.
template <typename W>
__global__ void __launch_bounds__(1024) norm_weight_grad_kernel(const float* partial, W* grad, int parts, int cols) {
  __shared__ float s[32][33];
  const int c = blockIdx.x * 32 + threadIdx.x;
  float v = 0.f;
  if (c < cols)
    for (int i = threadIdx.y; i < parts; i += 32) v += partial[(long long)i * cols + c];
  s[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  v = s[threadIdx.x][threadIdx.y];
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  const int o = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && o < cols) grad[o] = W(v);
}

// Launch shape of a row kernel: `threads` for a row, `vectors` for a thread, `rows` for a block.
struct RowShape {
  int threads, vectors, rows;
};
RowShape row_shape(int64_t rows, int cols, int elems) {
  const int nvec = (int)ceil_div(cols, elems);
  RowShape s;
  s.rows = 1;
  if (nvec <= 128) {  // a warp for a row needs no barrier
    s.threads = 32;
    s.vectors = nvec <= 32 ? 1 : nvec <= 64 ? 2 : 4;
    s.rows = 4;
    return s;
  }
  s.vectors = nvec <= 1024 ? 2 : nvec <= 4096 ? 4 : 8;
  s.threads = (int)ceil_div(ceil_div(nvec, s.vectors), 32) * 32;
  return s;
}

template <typename T, bool VEC, bool CODES>
const void* norm_kernel_nv(int nv) {
  switch (nv) {
    case 1: return (const void*)rms_norm_kernel<T, 1, VEC, CODES>;
    case 2: return (const void*)rms_norm_kernel<T, 2, VEC, CODES>;
    case 4: return (const void*)rms_norm_kernel<T, 4, VEC, CODES>;
    default: break;
  }
  if constexpr (Elem<T>::E == 4) {  // more than 4096 vectors a row: float32 only
    return (const void*)rms_norm_kernel<T, 8, VEC, CODES>;
  } else {
    return nullptr;
  }
}
template <typename T>
const void* norm_kernel(int nv, bool vec, bool codes) {
  if (vec) return codes ? norm_kernel_nv<T, true, true>(nv) : norm_kernel_nv<T, true, false>(nv);
  return codes ? norm_kernel_nv<T, false, true>(nv) : norm_kernel_nv<T, false, false>(nv);
}
template <typename T, bool VEC>
const void* norm_grad_kernel_nv(int nv) {
  switch (nv) {
    case 1: return (const void*)rms_norm_grad_kernel<T, 1, VEC>;
    case 2: return (const void*)rms_norm_grad_kernel<T, 2, VEC>;
    case 4: return (const void*)rms_norm_grad_kernel<T, 4, VEC>;
    default: break;
  }
  if constexpr (Elem<T>::E == 4) {
    return (const void*)rms_norm_grad_kernel<T, 8, VEC>;
  } else {
    return nullptr;
  }
}
template <typename T>
const void* norm_grad_kernel(int nv, bool vec) {
  return vec ? norm_grad_kernel_nv<T, true>(nv) : norm_grad_kernel_nv<T, false>(nv);
}

int partial_rows(int64_t rows, const RowShape& s) {
  const int64_t sets = ceil_div(rows, s.rows);
  return (int)(sets < kMaxPartials ? sets : kMaxPartials);
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
  if (!(eps > 0.f) || isinf(eps)) return report_error(DGN_ERR_ARG, "eps must be a positive number");
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
  const int es = (int)dgn_dtype_size(dtype), elems = 16 / es;
  const size_t ws = weight_dtype == DGN_F32 ? 4 : es;
  if (!aligned(x, es) || !aligned(residual, es) || !aligned(hidden, es) || !aligned(out, code ? 1 : es) ||
      (weight && !aligned(weight, ws)) || !aligned(scales, 4) || !aligned(rstd, 4))
    return report_error(DGN_ERR_ARG, "a pointer is not aligned to its element size");
  const bool vec = cols % elems == 0 && aligned(x, 16) && x_stride % elems == 0 && aligned(out, 16) &&
                   (!weight || aligned(weight, 16)) &&
                   (!residual || (aligned(residual, 16) && aligned(hidden, 16) && residual_stride % elems == 0 &&
                                  hidden_stride % elems == 0));
  const RowShape s = row_shape(rows, (int)cols, elems);
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
  p.group = group && group < cols ? (int)group : (int)cols;
  p.groups = (int)ceil_div(cols, p.group);
  p.weight_f32 = weight_dtype == DGN_F32;
  p.code = code;
  p.eps = eps;
  const void* fn = dtype == DGN_F32   ? norm_kernel<float>(s.vectors, vec, code != 0)
                   : dtype == DGN_F16 ? norm_kernel<__half>(s.vectors, vec, code != 0)
                                      : norm_kernel<__nv_bfloat16>(s.vectors, vec, code != 0);
  OnDevice on(device);
  if (on.error() != cudaSuccess) return report_error(DGN_ERR_CUDA, cudaGetErrorString(on.error()));
  void* args[] = {&p};
  return launch(fn, dim3((unsigned)ceil_div(rows, s.rows)), dim3(s.threads, s.rows), 0, stream, args);
}

extern "C" int64_t dgn_rms_norm_grad_workspace(int64_t rows, int64_t cols, int dtype) {
  if (!float_dtype(dtype) || rows < 1 || cols < 1 || cols > kMaxCols) return 0;
  const RowShape s = row_shape(rows, (int)cols, 16 / (int)dgn_dtype_size(dtype));
  return (int64_t)partial_rows(rows, s) * cols * (int64_t)sizeof(float);
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
  OnDevice on(device);
  if (on.error() != cudaSuccess) return report_error(DGN_ERR_CUDA, cudaGetErrorString(on.error()));
  if (rows == 0) {
    if (!grad_weight) return DGN_OK;
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
  const RowShape s = row_shape(rows, (int)cols, elems);
  const int parts = partial_rows(rows, s);
  if (grad_weight && workspace_bytes < (int64_t)parts * cols * (int64_t)sizeof(float))
    return report_error(DGN_ERR_ARG, "dgn_rms_norm_grad: workspace too small");
  const bool vec = cols % elems == 0 && aligned(grad_out, 16) && grad_out_stride % elems == 0 && aligned(hidden, 16) &&
                   hidden_stride % elems == 0 && aligned(grad_x, 16) && (!weight || aligned(weight, 16)) &&
                   (!grad_hidden || (aligned(grad_hidden, 16) && grad_hidden_stride % elems == 0));
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
  const void* fn = dtype == DGN_F32   ? norm_grad_kernel<float>(s.vectors, vec)
                   : dtype == DGN_F16 ? norm_grad_kernel<__half>(s.vectors, vec)
                                      : norm_grad_kernel<__nv_bfloat16>(s.vectors, vec);
  void* args[] = {&p};
  const size_t smem = s.rows > 1 ? (size_t)s.rows * cols * sizeof(float) : 0;
  rc = launch(fn, dim3(parts), dim3(s.threads, s.rows), smem, stream, args);
  if (rc != DGN_OK || !grad_weight) return rc;
  int nparts = parts, ncols = (int)cols;
  const float* partial = p.partial;
  void* args2[] = {&partial, &grad_weight, &nparts, &ncols};
  const void* fn2 = weight_dtype == DGN_F32 ? (const void*)norm_weight_grad_kernel<float>
                    : dtype == DGN_F16      ? (const void*)norm_weight_grad_kernel<__half>
                                            : (const void*)norm_weight_grad_kernel<__nv_bfloat16>;
  return launch(fn2, dim3((unsigned)ceil_div(cols, 32)), dim3(32, 32), 0, stream, args2);
}
