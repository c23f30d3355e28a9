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

// Where item `i` of eight values lies: in rows x_stride apart, among the eight-bit rows, and its block.  FLAT: rows without gaps
// and of whole blocks, no division by a row's length.
template <bool FLAT>
__device__ __forceinline__ bool place(unsigned long long i, unsigned long long n_items, unsigned per_row, int cols, long long x_stride, long long &wide,
                                      long long &dense, long long &block) {
  if constexpr (FLAT) {
    wide = dense = (long long)(i * 8);
    block = (long long)(i >> 2);
    return i < n_items;
  } else {
    long long row;
    unsigned at;
    split_index(i, per_row, row, at);
    wide = row * x_stride + at * 8;
    dense = row * cols + at * 8;
    block = row * (per_row >> 2) + (at >> 2);
    return i < n_items && (int)(at * 8) < cols;
  }
}
// The kernels start while the one before them ends (programmatic dependent launch): nothing is read or written before this.
// (Their pointers are not declared restrict: the compiler may move a load that it takes for one of unchanging memory.)
__device__ __forceinline__ void grid_start() {
  sm100::grid_launch_dependents();
  sm100::grid_dependency_wait();
}

// Items of eight values, four lanes to a block.
template <typename T, bool FLAT>
__global__ void __launch_bounds__(THREADS) pack_kernel(const T *x, long long x_stride, uint8_t *q, uint8_t *scale,
                                                       unsigned long long n_items, unsigned per_row, int cols) {
  const unsigned long long i0 = (unsigned long long)blockIdx.x * (THREADS * UNROLL) + threadIdx.x;
  uint4 v[UNROLL];
  long long to[UNROLL], block[UNROLL];
  bool in[UNROLL];
  grid_start();
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    const unsigned long long i = i0 + u * THREADS;
    long long from;
    in[u] = place<FLAT>(i, n_items, per_row, cols, x_stride, from, to[u], block[u]);
    v[u] = in[u] ? *reinterpret_cast<const uint4 *>(x + from) : make_uint4(0u, 0u, 0u, 0u);
  }
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    const uint32_t w[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
    uint32_t m = 0u;      // (a packed maximum leaves NaN out)
#pragma unroll
    for (int j = 0; j < 4; ++j) m = Pair16<T>::max2(m, w[j] & 0x7FFF7FFFu);
    m = Pair16<T>::max2(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = Pair16<T>::max2(m, __shfl_xor_sync(0xffffffffu, m, 2));
    const float2 m2 = Pair16<T>::unpack(m);
    float f[8], top = fmaxf(m2.x, m2.y);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 p = Pair16<T>::unpack(w[j]);
      f[2 * j] = p.x;
      f[2 * j + 1] = p.y;
    }
    if (__any_sync(0xffffffffu, top == __uint_as_float(0x7F800000u))) {      // rare: an infinity takes no part in the scale and is kept as NaN
      top = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        top = fmaxf(top, finite_magnitude(f[j]));
        f[j] = fabsf(f[j]) < __uint_as_float(0x7F800000u) ? f[j] : __uint_as_float(0x7FC00000u);
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    }
    const uint32_t byte = scale_byte(top);
    const float inv = inverse_scale(byte);
    const uint2 r = make_uint2(pack2_finite(f[0], f[1], inv) | (pack2_finite(f[2], f[3], inv) << 16), pack2_finite(f[4], f[5], inv) | (pack2_finite(f[6], f[7], inv) << 16));
    if (in[u]) {
      *reinterpret_cast<uint2 *>(q + to[u]) = r;
      if ((threadIdx.x & 3) == 0) scale[block[u]] = (uint8_t)byte;
    }
  }
}

// A warp to a block, for rows of any length and place.
template <typename T>
__global__ void __launch_bounds__(THREADS) pack_ragged_kernel(const T *x, long long x_stride, uint8_t *q,
                                                              uint8_t *scale, unsigned long long n_blocks, unsigned per_row, int cols) {
  const int lane = threadIdx.x & 31;
  const unsigned long long b0 = (unsigned long long)blockIdx.x * (THREADS / 32 * UNROLL) + (threadIdx.x >> 5);
  float v[UNROLL];
  long long row[UNROLL];
  unsigned at[UNROLL];
  bool in[UNROLL];
  grid_start();
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

// Four values in 16 bits; only a block with the largest scales can reach beyond the type.
template <typename T> __device__ __forceinline__ uint2 values4(uint32_t q, uint32_t byte, float s) {
  float2 a = unpack2(q & 0xFFFFu), b = unpack2(q >> 16);
  a.x *= s; a.y *= s; b.x *= s; b.y *= s;
  if (byte > safe_byte<T>()) { a.x = within<T>(a.x); a.y = within<T>(a.y); b.x = within<T>(b.x); b.y = within<T>(b.y); }
  return make_uint2(Pair16<T>::round(a.x, a.y), Pair16<T>::round(b.x, b.y));
}

template <typename T, bool FLAT>
__global__ void __launch_bounds__(THREADS) unpack_kernel(const uint8_t *q, const uint8_t *scale, T *x,
                                                         long long x_stride, unsigned long long n_items, unsigned per_row, int cols) {
  const unsigned long long i0 = (unsigned long long)blockIdx.x * (THREADS * UNROLL) + threadIdx.x;
  uint2 v[UNROLL];
  uint32_t byte[UNROLL];
  long long to[UNROLL];
  bool in[UNROLL];
  grid_start();
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    const unsigned long long i = i0 + u * THREADS;
    long long from, block;
    in[u] = place<FLAT>(i, n_items, per_row, cols, x_stride, to[u], from, block);
    v[u] = make_uint2(0u, 0u);
    byte[u] = 0u;
    if (in[u]) {
      v[u] = *reinterpret_cast<const uint2 *>(q + from);
      byte[u] = scale[block];
    }
  }
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    const float s = scale_of(byte[u]);
    if (in[u]) {
      const uint2 a = values4<T>(v[u].x, byte[u], s), b = values4<T>(v[u].y, byte[u], s);
      *reinterpret_cast<uint4 *>(x + to[u]) = make_uint4(a.x, a.y, b.x, b.y);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(THREADS) unpack_ragged_kernel(const uint8_t *q, const uint8_t *scale, T *x,
                                                                long long x_stride, unsigned long long n_blocks, unsigned per_row, int cols) {
  const int lane = threadIdx.x & 31;
  const unsigned long long b0 = (unsigned long long)blockIdx.x * (THREADS / 32 * UNROLL) + (threadIdx.x >> 5);
  grid_start();
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

// ---- a ReLU's signs ---------------------------------------------------------------------------------------------------
// Eight values and their byte a thread, four times.
template <typename T>
__global__ void __launch_bounds__(THREADS) sign_pack_kernel(const T *y, unsigned long long n, uint8_t *bits) {
  grid_start();
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    const unsigned long long i = (unsigned long long)blockIdx.x * (THREADS * UNROLL) + threadIdx.x + u * THREADS;
    if (i * 8 >= n) return;
    uint32_t w[4] = {0u, 0u, 0u, 0u};
    if (i * 8 + 8 <= n) {
      const uint4 v = reinterpret_cast<const uint4 *>(y)[i];
      w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    } else {
      for (int j = 0; j < (int)(n - i * 8); ++j) w[j >> 1] |= (uint32_t)reinterpret_cast<const uint16_t *>(y)[i * 8 + j] << (16 * (j & 1));
    }
    uint32_t b = 0u;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = Pair16<T>::unpack(w[j]);
      b |= (f.x > 0.f ? 1u : 0u) << (2 * j) | (f.y > 0.f ? 2u : 0u) << (2 * j);
    }
    bits[i] = (uint8_t)b;
  }
}
template <typename T>
__global__ void __launch_bounds__(THREADS) sign_apply_kernel(const T *gy, const uint8_t *bits, unsigned long long n, T *gx) {
  grid_start();
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    const unsigned long long i = (unsigned long long)blockIdx.x * (THREADS * UNROLL) + threadIdx.x + u * THREADS;
    if (i * 8 >= n) return;
    const uint32_t b = bits[i];
    if (i * 8 + 8 <= n) {
      const uint4 v = reinterpret_cast<const uint4 *>(gy)[i];
      uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {      // a product, not a choice: what is not finite stays visible
        const float2 f = Pair16<T>::unpack(w[j]);
        w[j] = Pair16<T>::round(f.x * (float)((b >> (2 * j)) & 1u), f.y * (float)((b >> (2 * j + 1)) & 1u));
      }
      reinterpret_cast<uint4 *>(gx)[i] = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      for (int j = 0; j < (int)(n - i * 8); ++j) Elem<T>::store(gx + i * 8 + j, Elem<T>::load(gy + i * 8 + j) * (float)((b >> j) & 1u));
    }
  }
}

// Rows copied with zeros behind them, eight values a thread; the second matrix by blocks of its own.
__global__ void __launch_bounds__(THREADS) pad_rows_kernel(const __grid_constant__ PadRows p) {
  const auto &m = p.m[blockIdx.y];
  const unsigned per_row = (unsigned)(m.y_stride / 8);
  const unsigned long long n_items = (unsigned long long)m.rows * per_row;
  grid_start();
  for (unsigned long long i = (unsigned long long)blockIdx.x * THREADS + threadIdx.x; i < n_items; i += (unsigned long long)gridDim.x * THREADS) {
    long long row;
    unsigned at;
    split_index(i, per_row, row, at);
    const int c = (int)at * 8;
    const long long from = row * m.x_stride + c;
    uint32_t w[4];
    if (m.in_dtype == WINOCONV_F32) {
      const float *src = (const float *)m.x + from;
      float f[8];
      if (c + 8 <= m.cols && (reinterpret_cast<uintptr_t>(src) & 15u) == 0) {
        const float4 a = reinterpret_cast<const float4 *>(src)[0], b = reinterpret_cast<const float4 *>(src)[1];
        f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = c + j < m.cols ? src[j] : 0.f;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        w[j] = m.dtype == WINOCONV_F16 ? Pair16<__half>::round(f[2 * j], f[2 * j + 1]) : Pair16<__nv_bfloat16>::round(f[2 * j], f[2 * j + 1]);
    } else {
      const uint16_t *src = (const uint16_t *)m.x + from;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t a = c + 2 * j < m.cols ? src[2 * j] : 0u, b = c + 2 * j + 1 < m.cols ? src[2 * j + 1] : 0u;
        w[j] = a | (b << 16);
      }
    }
    *reinterpret_cast<uint4 *>((uint16_t *)m.y + row * m.y_stride + c) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// ---- gradient through the activation ---------------------------------------------------------------------------------
// A block takes a strip of 32 x V columns and a run of rows, eight rows at a time; every thread adds up its own V columns in
// fp32, the eight sums of a column are added in order, and a second kernel adds the runs in order: no atomics, the same bits
// every time.  dz is rounded to the layer's type because the tensor cores read it for both products (their results carry the square
// root of two times a single rounding's error for it); the bias gradient is summed from the values before that rounding.
constexpr int ROWS = 8;

using act::F2;
template <typename T> __device__ __forceinline__ F2 pair_of(uint32_t v) {
  const float2 t = Pair16<T>::unpack(v);
  return F2(t.x, t.y);
}
// Values by pairs; of one value the second half of the pair is of no meaning.
template <typename T, int V> struct Run;
template <typename T> struct Run<T, 8> {
  using Raw = uint4;
  using Raw8 = uint2;
  static __device__ __forceinline__ F2 pair(const uint4 &v, int j) { return pair_of<T>(j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w); }
  static __device__ __forceinline__ F2 pair8(const uint2 &v, int j) {
    const float2 t = unpack2(((j & 2) ? v.y : v.x) >> (16 * (j & 1)));
    return F2(t.x, t.y);
  }
  static __device__ __forceinline__ void store(T *p, const uint32_t (&w)[4]) { *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]); }
};
template <typename T> struct Run<T, 1> {
  using Raw = uint16_t;
  using Raw8 = uint8_t;
  static __device__ __forceinline__ F2 pair(uint16_t v, int) { return pair_of<T>(v); }
  static __device__ __forceinline__ F2 pair8(uint8_t v, int) {
    const float2 t = unpack2(v);
    return F2(t.x, t.y);
  }
  static __device__ __forceinline__ void store(T *p, const uint32_t (&w)[1]) { *reinterpret_cast<uint16_t *>(p) = (uint16_t)w[0]; }
};

// Two rows of 16 bytes a thread in flight and four blocks to an SM: 35.8 us for 4096 x 8192 of bf16 through gelu_tanh, 201 MB at 5.6
// TB/s, and as long for 168 MB where z is in eight bits (four rows and three blocks 38.7 and 43.7, one row and six blocks 46.0 and 49.5).
// ACT, Z8: what z is, known when the kernel is compiled (-1: looked up for each value, for rows that take no vectors).
template <typename T, int V, int ACT, bool Z8>
__global__ void __launch_bounds__(THREADS, 4) act_grad_kernel(const __grid_constant__ ActGrad a, int chunks) {
  constexpr int DEEP = 2;      // rows whose loads are in flight together
  const int lane = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int c = (blockIdx.x * 32 + lane) * V;
  const long long r0 = a.rows * blockIdx.y / chunks, r1 = a.rows * (blockIdx.y + 1) / chunks;
  const unsigned n_blk = (unsigned)((a.cols + BLOCK - 1) / BLOCK);
  const int kind = ACT < 0 ? a.act : ACT;
  const bool z8 = ACT < 0 ? a.z8 != nullptr : Z8;
  constexpr int P = (V + 1) / 2;
  using R = Run<T, V>;
  F2 sum[P];
#pragma unroll
  for (int j = 0; j < P; ++j) sum[j] = F2(0.f);
  grid_start();
  if (c < a.cols) {
    for (long long r = r0 + ty; r < r1; r += ROWS * DEEP) {
      typename R::Raw g_raw[DEEP], z_raw[DEEP];
      typename R::Raw8 q_raw[DEEP];
      uint32_t byte[DEEP];
#pragma unroll
      for (int u = 0; u < DEEP; ++u) {
        const long long at = r + u * ROWS;
        if (at >= r1) break;
        g_raw[u] = *reinterpret_cast<const typename R::Raw *>((const T *)a.gy + at * a.gy_stride + c);
        if (kind != WINOCONV_ACT_NONE) {
          if (z8) {
            q_raw[u] = *reinterpret_cast<const typename R::Raw8 *>(a.z8 + at * a.cols + c);
            byte[u] = a.z8_scale[at * n_blk + c / BLOCK];
          } else z_raw[u] = *reinterpret_cast<const typename R::Raw *>((const T *)a.z + at * a.z_stride + c);
        }
      }
#pragma unroll
      for (int u = 0; u < DEEP; ++u) {
        const long long at = r + u * ROWS;
        if (at >= r1) break;
        uint32_t w[P];
        // (every slope is 0 or 1 long before 2^100: a block beyond that is read as one up to there, which does not overflow)
        const F2 scale(z8 && kind != WINOCONV_ACT_NONE ? scale_of(byte[u] == 255u ? 255u : min(byte[u], 227u)) : 1.f);
#pragma unroll
        for (int j = 0; j < P; ++j) {
          F2 g = R::pair(g_raw[u], j);
          if (kind != WINOCONV_ACT_NONE) {
            g = g * act::slope(z8 ? R::pair8(q_raw[u], j) * scale : R::pair(z_raw[u], j), kind);
          }
          sum[j] = sum[j] + g;
          w[j] = Pair16<T>::round(g.lo(), g.hi());
        }
        if (a.dz) R::store((T *)a.dz + at * a.dz_stride + c, w);
      }
    }
  }
  if (!a.dbias) return;
  __shared__ float part[ROWS][32 * V + 1];
#pragma unroll
  for (int j = 0; j < V; ++j) part[ty][j * 32 + lane] = (j & 1) ? sum[j / 2].hi() : sum[j / 2].lo();
  __syncthreads();
  for (int t = threadIdx.x; t < 32 * V; t += THREADS) {
    const int l = t / V, j = t - l * V, col = (blockIdx.x * 32 + l) * V + j;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) s += part[i][j * 32 + l];
    if (col >= a.cols) continue;
    if (chunks > 1) a.ws[(long long)blockIdx.y * a.cols + col] = s;
    else if (a.dbias_dtype == WINOCONV_F32) ((float *)a.dbias)[col] = s;      // one run: nothing left to add
    else if (a.dbias_dtype == WINOCONV_F16) Elem<__half>::store((__half *)a.dbias + col, s);
    else Elem<__nv_bfloat16>::store((__nv_bfloat16 *)a.dbias + col, s);
  }
}

template <typename O>
__global__ void __launch_bounds__(THREADS) column_sum_kernel(const float *ws, O *out, int cols, int chunks) {
  __shared__ float part[ROWS][32];
  const int lane = threadIdx.x & 31, ty = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float s = 0.f;
  grid_start();
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
bool on8(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 7u) == 0; }
unsigned blocks_of(unsigned long long n, unsigned per) { return (unsigned)((n + per - 1) / per); }

template <typename... P, typename... A> cudaError_t launch(void (*kern)(P...), dim3 grid, cudaStream_t s, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid; cfg.blockDim = dim3(THREADS); cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr; cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, P(args)...);
}

template <typename T>
cudaError_t pack(const void *x, long long x_stride, long long rows, int cols, uint8_t *q, uint8_t *scale, cudaStream_t s) {
  const unsigned n_blk = (unsigned)((cols + BLOCK - 1) / BLOCK);
  const unsigned long long n = (unsigned long long)rows * n_blk;
  if (cols % 8 == 0 && on16(x) && x_stride % 8 == 0 && on8(q)) {
    const bool flat = cols % BLOCK == 0 && (x_stride == cols || rows == 1);
    return launch(flat ? pack_kernel<T, true> : pack_kernel<T, false>, blocks_of(n * 4, THREADS * UNROLL), s, (const T *)x, x_stride, q, scale, n * 4, n_blk * 4, cols);
  }
  return launch(pack_ragged_kernel<T>, blocks_of(n, THREADS / 32 * UNROLL), s, (const T *)x, x_stride, q, scale, n, n_blk, cols);
}
template <typename T>
cudaError_t unpack(const uint8_t *q, const uint8_t *scale, long long rows, int cols, void *x, long long x_stride, cudaStream_t s) {
  const unsigned n_blk = (unsigned)((cols + BLOCK - 1) / BLOCK);
  const unsigned long long n = (unsigned long long)rows * n_blk;
  if (cols % 8 == 0 && on16(x) && x_stride % 8 == 0 && on8(q)) {
    const bool flat = cols % BLOCK == 0 && (x_stride == cols || rows == 1);
    return launch(flat ? unpack_kernel<T, true> : unpack_kernel<T, false>, blocks_of(n * 4, THREADS * UNROLL), s, q, scale, (T *)x, x_stride, n * 4, n_blk * 4, cols);
  }
  return launch(unpack_ragged_kernel<T>, blocks_of(n, THREADS / 32 * UNROLL), s, q, scale, (T *)x, x_stride, n, n_blk, cols);
}

template <typename T, int ACT> auto act_grad_kernel_of(bool z8) { return z8 ? act_grad_kernel<T, 8, ACT, true> : act_grad_kernel<T, 8, ACT, false>; }
template <typename T> cudaError_t act_grad(const ActGrad &a, cudaStream_t s) {
  const bool wide = a.cols % 8 == 0 && on16(a.gy) && a.gy_stride % 8 == 0 && (!a.z || (on16(a.z) && a.z_stride % 8 == 0)) && (!a.z8 || on8(a.z8)) &&
                    (!a.dz || (on16(a.dz) && a.dz_stride % 8 == 0));
  const int chunks = act_grad_chunks(a.rows, a.cols), v = wide ? 8 : 1;
  auto kern = act_grad_kernel<T, 1, -1, false>;
  if (wide) {
    switch (a.act) {
      case WINOCONV_ACT_RELU: kern = act_grad_kernel_of<T, WINOCONV_ACT_RELU>(a.z8); break;
      case WINOCONV_ACT_GELU: kern = act_grad_kernel_of<T, WINOCONV_ACT_GELU>(a.z8); break;
      case WINOCONV_ACT_GELU_TANH: kern = act_grad_kernel_of<T, WINOCONV_ACT_GELU_TANH>(a.z8); break;
      case WINOCONV_ACT_SILU: kern = act_grad_kernel_of<T, WINOCONV_ACT_SILU>(a.z8); break;
      default: kern = act_grad_kernel<T, 8, WINOCONV_ACT_NONE, false>;
    }
  }
  const cudaError_t e = launch(kern, dim3((unsigned)((a.cols + 32 * v - 1) / (32 * v)), (unsigned)chunks), s, a, chunks);
  if (e != cudaSuccess || !a.dbias || chunks == 1) return e;
  const unsigned n = (unsigned)((a.cols + 31) / 32);
  if (a.dbias_dtype == WINOCONV_F32) return launch(column_sum_kernel<float>, n, s, a.ws, (float *)a.dbias, a.cols, chunks);
  if (a.dbias_dtype == WINOCONV_F16) return launch(column_sum_kernel<__half>, n, s, a.ws, (__half *)a.dbias, a.cols, chunks);
  return launch(column_sum_kernel<__nv_bfloat16>, n, s, a.ws, (__nv_bfloat16 *)a.dbias, a.cols, chunks);
}

}  // namespace e4m3

using namespace e4m3;

cudaError_t launch_e4m3_pack(int dtype, const void *x, long long x_stride, long long rows, int cols, uint8_t *q, uint8_t *scale, cudaStream_t s) {
  return dtype == WINOCONV_F16 ? pack<__half>(x, x_stride, rows, cols, q, scale, s) : pack<__nv_bfloat16>(x, x_stride, rows, cols, q, scale, s);
}
cudaError_t launch_e4m3_unpack(int dtype, const uint8_t *q, const uint8_t *scale, long long rows, int cols, void *x, long long x_stride, cudaStream_t s) {
  return dtype == WINOCONV_F16 ? unpack<__half>(q, scale, rows, cols, x, x_stride, s) : unpack<__nv_bfloat16>(q, scale, rows, cols, x, x_stride, s);
}
cudaError_t launch_pad_rows(const PadRows &p, cudaStream_t s) {
  unsigned long long n = 1;
  for (int i = 0; i < p.count; ++i) n = std::max(n, (unsigned long long)p.m[i].rows * (unsigned long long)(p.m[i].y_stride / 8));
  return launch(pad_rows_kernel, dim3((unsigned)std::min<unsigned long long>((n + THREADS - 1) / THREADS, 16 * 148), (unsigned)p.count), s, p);
}
cudaError_t launch_sign_pack(int dtype, const void *y, long long n, uint8_t *bits, cudaStream_t s) {
  const unsigned blocks = blocks_of((unsigned long long)(n + 7) / 8, THREADS * UNROLL);
  return dtype == WINOCONV_F16 ? launch(sign_pack_kernel<__half>, blocks, s, (const __half *)y, (unsigned long long)n, bits)
                               : launch(sign_pack_kernel<__nv_bfloat16>, blocks, s, (const __nv_bfloat16 *)y, (unsigned long long)n, bits);
}
cudaError_t launch_sign_apply(int dtype, const void *gy, const uint8_t *bits, long long n, void *gx, cudaStream_t s) {
  const unsigned blocks = blocks_of((unsigned long long)(n + 7) / 8, THREADS * UNROLL);
  return dtype == WINOCONV_F16 ? launch(sign_apply_kernel<__half>, blocks, s, (const __half *)gy, bits, (unsigned long long)n, (__half *)gx)
                               : launch(sign_apply_kernel<__nv_bfloat16>, blocks, s, (const __nv_bfloat16 *)gy, bits, (unsigned long long)n, (__nv_bfloat16 *)gx);
}
// Runs of rows: equal shares of 32 rows or a multiple of that on average (a block has 16 in flight), short enough for three waves of
// four blocks on every SM, so that the last wave costs little, and at most 65535 of them.  A run's partial sums cost 8 bytes a column,
// written and read, of 32 or more (from 33 rows on: two runs of 16 and 17) that are read of gy alone.
int act_grad_chunks(long long rows, int cols) {
  const long long strips = (cols + 255) / 256, groups = (rows + 31) / 32;
  const long long per = std::max<long long>({1, groups * strips / (4 * 3 * 148), (groups + 65534) / 65535});
  return (int)((groups + per - 1) / per);
}
cudaError_t launch_act_grad(const ActGrad &a, cudaStream_t s) {
  return a.dtype == WINOCONV_F16 ? act_grad<__half>(a, s) : act_grad<__nv_bfloat16>(a, s);
}

}  // namespace wino
