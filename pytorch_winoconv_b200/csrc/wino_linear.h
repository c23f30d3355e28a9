// Fully connected layers and 8-bit activation checkpoints: what wino_capi.cu asks of wino_linear.cu and wino_e4m3.cu.
#pragma once

#include <cuda_runtime.h>

#include "wino_common.cuh"

namespace wino {

// out[row][col] = sum over red of R[row, red] C[col, red].  An operand lies with its reduction contiguous (mn = 0: [rows][red])
// or with its rows contiguous (mn = 1: [red][rows]); `stride` is the element distance of its slow dimension, a multiple of 8.
struct MatOperand {
  const void *ptr;
  long long stride;
  int mn;
};
struct LinearProblem {
  int dtype;                 // of R and C, and of y unless out_f32
  int rows, cols, red;
  MatOperand r, c;
  int layer;                 // 1: z = product + bias, y = act(z) + residual; 0: y = product
  int act, bias_f32, out_f32;
  const void *bias;          // [cols] or null
  const void *residual;      // or null
  void *y, *z;               // z: pre-activation in dtype, or null
  uint8_t *z8, *z8_scale;    // pre-activation in 8 bits [rows][cols] and its scales [rows][ceil(cols / 32)], or null
  long long residual_stride, y_stride, z_stride;
};
// pair: columns (256, 128 or 64) of a tile of 256 rows by two CTAs, tiles walked by a persistent grid.  Else a tile of `tile_rows` x
// 128 by a cluster of `split` CTAs that share its reduction.  by_rows: a layer's few rows without the tensor cores.
struct LinearPlan {
  int by_rows, pair;
  int tile_rows, split, stages;
};
LinearPlan linear_plan(const LinearProblem &p);
bool linear_by_rows(long long rows, int layer, bool z8);      // such a problem's operands may lie anywhere
cudaError_t launch_linear(const LinearProblem &p, const LinearPlan &plan, cudaStream_t s, const char **detail);
cudaError_t read_and_clear_linear_error(cudaStream_t s, unsigned int *code);

// One or two matrices copied to rows y_stride apart (a multiple of 8), zeros behind them; f32 rounded to dtype.
struct PadRows {
  struct {
    const void *x;
    void *y;
    long long x_stride, y_stride, rows;
    int cols, in_dtype, dtype;
  } m[2];
  int count;
};
cudaError_t launch_pad_rows(const PadRows &p, cudaStream_t s);

// dz = gy * act'(z) and the sums of its columns.  z in dtype, or in 8 bits with its scales; dz may be null (act none), dbias too.
struct ActGrad {
  int dtype, act;
  long long rows;
  int cols;
  const void *gy, *z;
  const uint8_t *z8, *z8_scale;
  void *dz, *dbias;
  int dbias_dtype;
  long long gy_stride, z_stride, dz_stride;
  float *ws;                 // act_grad_chunks() x cols floats where dbias is asked for
};
int act_grad_chunks(long long rows, int cols);
cudaError_t launch_act_grad(const ActGrad &a, cudaStream_t s);

// x [rows][cols] -> q [rows][cols] e4m3, scale [rows][ceil(cols / 32)] powers of two as biased exponents; and back.
cudaError_t launch_e4m3_pack(int dtype, const void *x, long long x_stride, long long rows, int cols, uint8_t *q, uint8_t *scale, cudaStream_t s);
cudaError_t launch_e4m3_unpack(int dtype, const uint8_t *q, const uint8_t *scale, long long rows, int cols, void *x, long long x_stride, cudaStream_t s);

// Signs of a ReLU's result, eight to a byte, and a gradient times them.
cudaError_t launch_sign_pack(int dtype, const void *y, long long n, uint8_t *bits, cudaStream_t s);
cudaError_t launch_sign_apply(int dtype, const void *gy, const uint8_t *bits, long long n, void *gx, cudaStream_t s);

}  // namespace wino
