// Passes over activations: packing to eight bits and back, the gradient through an activation with the bias gradient, rows
// copied to a stride that TMA takes.  All are bound by memory: a thread moves 16 bytes a time, four such loads in flight, where
// rows start on 16 bytes; else a warp moves 32 neighbouring values.
#include <algorithm>

#include "wino_e4m3.cuh"
#include "wino_linear.h"

namespace wino {
namespace e4m3 {

using sm100::Pair16;

constexpr int THREADS = 256, UNROLL = 4;

// Row and place within it of item `i` of rows of `per` items.
__device__ __forceinline__ void split_index(unsigned long long i, unsigned per, long long &row, unsigned &at) {
  if (i <= 0xFFFFFFFFull) {
    const unsigned r = (unsigned)i / per;
    row = r;
    at = (unsigned)i - r * per;
  } else {
    row = (long long)(i / per);
    at = (unsigned)(i - (unsigned long long)row * per);
  }
}

// Items of eight values, four lanes to a block.
template <typename T>
__global__ void __launch_bounds__(THREADS) pack_kernel(const T *__restrict__ x, long long x_stride, uint8_t *__restrict__ q, uint8_t *__restrict__ scale,
                                                       unsigned long long n_items, unsigned per_row, int cols) {
  const unsigned long long i0 = (unsigned long long)blockIdx.x * (THREADS * UNROLL) + threadIdx.x;
  uint4 v[UNROLL];
  long long row[UNROLL];
  unsigned at[UNROLL];
  bool in[UNROLL];
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    const unsigned long long i = i0 + u * THREADS;
    split_index(i, per_row, row[u], at[u]);
    in[u] = i < n_items && (int)(at[u] * 8) < cols;
    v[u] = in[u] ? *reinterpret_cast<const uint4 *>(x + row[u] * x_stride + at[u] * 8) : make_uint4(0u, 0u, 0u, 0u);
  }
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    const uint32_t w[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
    float f[8], top = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 p = Pair16<T>::unpack(w[j]);
      f[2 * j] = p.x;
      f[2 * j + 1] = p.y;
      top = fmaxf(top, fmaxf(finite_magnitude(p.x), finite_magnitude(p.y)));
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const uint32_t byte = scale_byte(top);
    const float inv = inverse_scale(byte);
    const uint2 r = make_uint2(pack2(f[0], f[1], inv) | (pack2(f[2], f[3], inv) << 16), pack2(f[4], f[5], inv) | (pack2(f[6], f[7], inv) << 16));
    if (in[u]) {
      *reinterpret_cast<uint2 *>(q + row[u] * cols + at[u] * 8) = r;
      if ((threadIdx.x & 3) == 0) scale[row[u] * (per_row >> 2) + (at[u] >> 2)] = (uint8_t)byte;
    }
  }
}

// A warp to a block, for rows of any length and place.
template <typename T>
__global__ void __launch_bounds__(THREADS) pack_ragged_kernel(const T *__restrict__ x, long long x_stride, uint8_t *__restrict__ q,
                                                              uint8_t *__restrict__ scale, unsigned long long n_blocks, unsigned per_row, int cols) {
  const int lane = threadIdx.x & 31;
  const unsigned long long b0 = (unsigned long long)blockIdx.x * (THREADS / 32 * UNROLL) + (threadIdx.x >> 5);
  float v[UNROLL];
  long long row[UNROLL];
  unsigned at[UNROLL];
  bool in[UNROLL];
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    const unsigned long long b = b0 + u * (THREADS / 32);
    split_index(b, per_row, row[u], at[u]);
    in[u] = b < n_blocks && (int)(at[u] * BLOCK) + lane < cols;
    v[u] = in[u] ? Elem<T>::load(x + row[u] * x_stride + at[u] * BLOCK + lane) : 0.f;
  }
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    float top = finite_magnitude(v[u]);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    const uint32_t byte = scale_byte(top);
    if (in[u]) {
      q[row[u] * cols + at[u] * BLOCK + lane] = (uint8_t)pack2(v[u], 0.f, inverse_scale(byte));
      if (lane == 0) scale[row[u] * per_row + at[u]] = (uint8_t)byte;
    }
  }
}

template <typename T> __device__ __forceinline__ uint32_t values2(uint32_t q, float s) {
  const float2 f = unpack2(q);
  return Pair16<T>::round(within<T>(f.x * s), within<T>(f.y * s));
}

template <typename T>
__global__ void __launch_bounds__(THREADS) unpack_kernel(const uint8_t *__restrict__ q, const uint8_t *__restrict__ scale, T *__restrict__ x,
                                                         long long x_stride, unsigned long long n_items, unsigned per_row, int cols) {
  const unsigned long long i0 = (unsigned long long)blockIdx.x * (THREADS * UNROLL) + threadIdx.x;
  uint2 v[UNROLL];
  uint32_t byte[UNROLL];
  long long row[UNROLL];
  unsigned at[UNROLL];
  bool in[UNROLL];
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    const unsigned long long i = i0 + u * THREADS;
    split_index(i, per_row, row[u], at[u]);
    in[u] = i < n_items && (int)(at[u] * 8) < cols;
    v[u] = make_uint2(0u, 0u);
    byte[u] = 0u;
    if (in[u]) {
      v[u] = *reinterpret_cast<const uint2 *>(q + row[u] * cols + at[u] * 8);
      byte[u] = scale[row[u] * (per_row >> 2) + (at[u] >> 2)];
    }
  }
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    const float s = scale_of(byte[u]);
    if (in[u])
      *reinterpret_cast<uint4 *>(x + row[u] * x_stride + at[u] * 8) =
          make_uint4(values2<T>(v[u].x & 0xFFFFu, s), values2<T>(v[u].x >> 16, s), values2<T>(v[u].y & 0xFFFFu, s), values2<T>(v[u].y >> 16, s));
  }
}

template <typename T>
__global__ void __launch_bounds__(THREADS) unpack_ragged_kernel(const uint8_t *__restrict__ q, const uint8_t *__restrict__ scale, T *__restrict__ x,
                                                                long long x_stride, unsigned long long n_blocks, unsigned per_row, int cols) {
  const int lane = threadIdx.x & 31;
  const unsigned long long b0 = (unsigned long long)blockIdx.x * (THREADS / 32 * UNROLL) + (threadIdx.x >> 5);
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    const unsigned long long b = b0 + u * (THREADS / 32);
    long long row;
    unsigned at;
    split_index(b, per_row, row, at);
    if (b < n_blocks && (int)(at * BLOCK) + lane < cols) {
      const float f = unpack2(q[row * cols + at * BLOCK + lane]).x * scale_of(scale[row * per_row + at]);
      Elem<T>::store(x + row * x_stride + at * BLOCK + lane, within<T>(f));
    }
  }
}

// Rows copied with zeros behind them; T is any 16-bit type.
__global__ void __launch_bounds__(THREADS) pad_rows_kernel(const uint16_t *__restrict__ x, long long x_stride, uint16_t *__restrict__ y, long long out_stride,
                                                           unsigned long long n_items, unsigned per_row, int cols) {
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    const unsigned long long i = (unsigned long long)blockIdx.x * (THREADS * UNROLL) + threadIdx.x + u * THREADS;
    if (i >= n_items) return;
    long long row;
    unsigned at;
    split_index(i, per_row, row, at);
    const uint16_t *src = x + row * x_stride + at * 2;
    const uint32_t a = (int)(at * 2) < cols ? src[0] : 0u, b = (int)(at * 2 + 1) < cols ? src[1] : 0u;
    *reinterpret_cast<uint32_t *>(y + row * out_stride + at * 2) = a | (b << 16);
  }
}

// ---- gradient through the activation ---------------------------------------------------------------------------------
// A block takes a strip of 32 x V columns and a run of rows, eight rows at a time; every thread adds up its own V columns in
// fp32, the eight sums of a column are added in order, and a second kernel adds the runs in order: no atomics, the same bits
// every time.
constexpr int ROWS = 8;

template <typename T, int V> struct Run {
  static __device__ __forceinline__ void load(const T *p, float (&f)[V]) {
    if constexpr (V == 8) {
      const uint4 v = *reinterpret_cast<const uint4 *>(p);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 t = Pair16<T>::unpack(w[j]);
        f[2 * j] = t.x;
        f[2 * j + 1] = t.y;
      }
    } else f[0] = Elem<T>::load(p);
  }
  static __device__ __forceinline__ void store(T *p, const float (&f)[V]) {
    if constexpr (V == 8)
      *reinterpret_cast<uint4 *>(p) = make_uint4(Pair16<T>::round(f[0], f[1]), Pair16<T>::round(f[2], f[3]), Pair16<T>::round(f[4], f[5]), Pair16<T>::round(f[6], f[7]));
    else Elem<T>::store(p, f[0]);
  }
};

template <typename T, int V>
__global__ void __launch_bounds__(THREADS) act_grad_kernel(const __grid_constant__ ActGrad a, int chunks) {
  const int lane = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int c = (blockIdx.x * 32 + lane) * V;
  const long long r0 = a.rows * blockIdx.y / chunks, r1 = a.rows * (blockIdx.y + 1) / chunks;
  const unsigned n_blk = (unsigned)((a.cols + BLOCK - 1) / BLOCK);
  float sum[V];
#pragma unroll
  for (int j = 0; j < V; ++j) sum[j] = 0.f;
  if (c < a.cols) {
#pragma unroll 2
    for (long long r = r0 + ty; r < r1; r += ROWS) {
      float g[V], z[V];
      Run<T, V>::load((const T *)a.gy + r * a.gy_stride + c, g);
      if (a.z8) {
        const float s = scale_of(a.z8_scale[r * n_blk + c / BLOCK]);
        const uint8_t *src = a.z8 + r * a.cols + c;
        if constexpr (V == 8) {
          const uint2 v = *reinterpret_cast<const uint2 *>(src);
          const uint32_t w[4] = {v.x & 0xFFFFu, v.x >> 16, v.y & 0xFFFFu, v.y >> 16};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 t = unpack2(w[j]);
            z[2 * j] = within<T>(t.x * s);
            z[2 * j + 1] = within<T>(t.y * s);
          }
        } else z[0] = within<T>(unpack2(*src).x * s);
      } else if (a.z) Run<T, V>::load((const T *)a.z + r * a.z_stride + c, z);
      if (a.act != WINOCONV_ACT_NONE) {
#pragma unroll
        for (int j = 0; j < V; ++j) g[j] *= act::slope(z[j], a.act);
      }
#pragma unroll
      for (int j = 0; j < V; ++j) sum[j] += g[j];
      if (a.dz) Run<T, V>::store((T *)a.dz + r * a.dz_stride + c, g);
    }
  }
  if (!a.dbias) return;
  __shared__ float part[ROWS][32 * V + 1];
#pragma unroll
  for (int j = 0; j < V; ++j) part[ty][j * 32 + lane] = sum[j];
  __syncthreads();
  for (int t = threadIdx.x; t < 32 * V; t += THREADS) {
    const int l = t / V, j = t - l * V, col = (blockIdx.x * 32 + l) * V + j;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) s += part[i][j * 32 + l];
    if (col < a.cols) a.ws[(long long)blockIdx.y * a.cols + col] = s;
  }
}

template <typename O>
__global__ void __launch_bounds__(THREADS) column_sum_kernel(const float *__restrict__ ws, O *__restrict__ out, int cols, int chunks) {
  __shared__ float part[ROWS][32];
  const int lane = threadIdx.x & 31, ty = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (c < cols)
    for (int i = ty; i < chunks; i += ROWS) s += ws[(long long)i * cols + c];
  part[ty][lane] = s;
  __syncthreads();
  if (ty == 0 && c < cols) {
#pragma unroll
    for (int i = 1; i < ROWS; ++i) s += part[i][lane];
    Elem<O>::store(out + c, s);
  }
}

bool on16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
unsigned blocks_of(unsigned long long n, unsigned per) { return (unsigned)((n + per - 1) / per); }

template <typename T>
cudaError_t pack(const void *x, long long x_stride, long long rows, int cols, uint8_t *q, uint8_t *scale, cudaStream_t s) {
  const unsigned n_blk = (unsigned)((cols + BLOCK - 1) / BLOCK);
  if (cols % 8 == 0 && on16(x) && x_stride % 8 == 0 && (reinterpret_cast<uintptr_t>(q) & 7u) == 0) {
    const unsigned long long n = (unsigned long long)rows * n_blk * 4;
    pack_kernel<T><<<blocks_of(n, THREADS * UNROLL), THREADS, 0, s>>>((const T *)x, x_stride, q, scale, n, n_blk * 4, cols);
  } else {
    const unsigned long long n = (unsigned long long)rows * n_blk;
    pack_ragged_kernel<T><<<blocks_of(n, THREADS / 32 * UNROLL), THREADS, 0, s>>>((const T *)x, x_stride, q, scale, n, n_blk, cols);
  }
  return cudaGetLastError();
}
template <typename T>
cudaError_t unpack(const uint8_t *q, const uint8_t *scale, long long rows, int cols, void *x, long long x_stride, cudaStream_t s) {
  const unsigned n_blk = (unsigned)((cols + BLOCK - 1) / BLOCK);
  if (cols % 8 == 0 && on16(x) && x_stride % 8 == 0 && (reinterpret_cast<uintptr_t>(q) & 7u) == 0) {
    const unsigned long long n = (unsigned long long)rows * n_blk * 4;
    unpack_kernel<T><<<blocks_of(n, THREADS * UNROLL), THREADS, 0, s>>>(q, scale, (T *)x, x_stride, n, n_blk * 4, cols);
  } else {
    const unsigned long long n = (unsigned long long)rows * n_blk;
    unpack_ragged_kernel<T><<<blocks_of(n, THREADS / 32 * UNROLL), THREADS, 0, s>>>(q, scale, (T *)x, x_stride, n, n_blk, cols);
  }
  return cudaGetLastError();
}

template <typename T> cudaError_t act_grad(const ActGrad &a, cudaStream_t s) {
  const bool wide = a.cols % 8 == 0 && on16(a.gy) && a.gy_stride % 8 == 0 && (!a.z || (on16(a.z) && a.z_stride % 8 == 0)) &&
                    (!a.z8 || (reinterpret_cast<uintptr_t>(a.z8) & 7u) == 0) && (!a.dz || (on16(a.dz) && a.dz_stride % 8 == 0));
  const int chunks = act_grad_chunks(a.rows, a.cols), v = wide ? 8 : 1;
  const dim3 grid((unsigned)((a.cols + 32 * v - 1) / (32 * v)), (unsigned)chunks);
  if (wide) act_grad_kernel<T, 8><<<grid, THREADS, 0, s>>>(a, chunks);
  else act_grad_kernel<T, 1><<<grid, THREADS, 0, s>>>(a, chunks);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || !a.dbias) return e;
  const unsigned n = (unsigned)((a.cols + 31) / 32);
  if (a.dbias_dtype == WINOCONV_F32) column_sum_kernel<float><<<n, THREADS, 0, s>>>(a.ws, (float *)a.dbias, a.cols, chunks);
  else if (a.dbias_dtype == WINOCONV_F16) column_sum_kernel<__half><<<n, THREADS, 0, s>>>(a.ws, (__half *)a.dbias, a.cols, chunks);
  else column_sum_kernel<__nv_bfloat16><<<n, THREADS, 0, s>>>(a.ws, (__nv_bfloat16 *)a.dbias, a.cols, chunks);
  return cudaGetLastError();
}

}  // namespace e4m3

using namespace e4m3;

cudaError_t launch_e4m3_pack(int dtype, const void *x, long long x_stride, long long rows, int cols, uint8_t *q, uint8_t *scale, cudaStream_t s) {
  return dtype == WINOCONV_F16 ? pack<__half>(x, x_stride, rows, cols, q, scale, s) : pack<__nv_bfloat16>(x, x_stride, rows, cols, q, scale, s);
}
cudaError_t launch_e4m3_unpack(int dtype, const uint8_t *q, const uint8_t *scale, long long rows, int cols, void *x, long long x_stride, cudaStream_t s) {
  return dtype == WINOCONV_F16 ? unpack<__half>(q, scale, rows, cols, x, x_stride, s) : unpack<__nv_bfloat16>(q, scale, rows, cols, x, x_stride, s);
}
cudaError_t launch_pad_rows(const void *x, long long x_stride, void *y, long long out_stride, long long rows, int cols, cudaStream_t s) {
  const unsigned per = (unsigned)(out_stride / 2);
  const unsigned long long n = (unsigned long long)rows * per;
  pad_rows_kernel<<<blocks_of(n, THREADS * UNROLL), THREADS, 0, s>>>((const uint16_t *)x, x_stride, (uint16_t *)y, out_stride, n, per, cols);
  return cudaGetLastError();
}
// Runs of rows: enough blocks for four on every SM, at least 32 rows to a run (so that the partial sums stay a few per cent of
// what is read), at most 65535.
int act_grad_chunks(long long rows, int cols) {
  const long long strips = (cols + 255) / 256, want = std::max<long long>(1, (4LL * 148 + strips - 1) / strips);
  return (int)std::max<long long>(1, std::min({want, (rows + 31) / 32, 65535LL}));
}
cudaError_t launch_act_grad(const ActGrad &a, cudaStream_t s) {
  return a.dtype == WINOCONV_F16 ? act_grad<__half>(a, s) : act_grad<__nv_bfloat16>(a, s);
}

}  // namespace wino
