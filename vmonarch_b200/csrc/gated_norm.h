// Parameter block of the gated residual norm (gated_norm.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace vmb {

struct GatedNormParams {
  const void *x, *y;                 // [rows][cols], row strides x_row, y_row; y may be NULL
  void *x_new, *h;                   // [rows][cols] dense; x_new unused without y
  const void *gate, *scale, *shift;  // [seqs][cols] or NULL
  const void *weight, *post_weight;  // [cols] or NULL
  float* stats;                      // [3][rows]: ry, mean, rx (written forward where not NULL, read backward)
  const int32_t* seq_start;          // [seqs], first row of each sequence; NULL with one sequence
  const void *dx_new, *dh;           // backward: gradients in, row strides; either may be NULL (zero)
  void *dx, *dy;                     // [rows][cols] dense
  void *dgate, *dscale, *dshift, *dweight, *dpost_weight;  // any may be NULL
  float *part, *seq_part;            // column sums: [blocks + seqs][3][cols], [seqs][cols][2]; NULL: not wanted
  int64_t rows;                      // below 2^31, as the strides
  int x_row, y_row, dx_new_row, dh_row;
  int cols, seqs, layer;
  float eps;
  int tpr, stages;                   // set at launch
};

int gated_norm_blocks(const GatedNormParams& p);  // blocks of a backward call
cudaError_t gated_norm(const GatedNormParams& p, bool bf16, bool f32_params, bool bwd, cudaStream_t st);

}  // namespace vmb
