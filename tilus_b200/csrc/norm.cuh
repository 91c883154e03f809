// Parameter blocks of the row-wise kernels: the per-token int8 cast, the block norm and its gradient (norm_kernel.cu).
#pragma once
#include "common.cuh"

namespace b200q {

constexpr int NORM_ROWS_FROM = 888;   // rows from which a block norm has its rows copied ahead (three to a CTA)
constexpr int NORM_ROWS_STAGES = 4;   // rows in shared memory then
constexpr int NORM_BACK_THREADS = 512;  // of an SM in the gradient's kernel, which takes up to 128 registers a thread
constexpr int NORM_BACK_STAGES = 4;     // rows in shared memory

struct CastIntParams {
  const unsigned short* x;  // [T, D], row stride ldx, fp16 or bf16
  signed char* out;         // [T, D], row stride ldo
  float* out_sf;            // [T]
  int T, D, ldx, ldo;
};

// What norm_kernel.cu computes, for each row t of [T, D]:
//   n  = block * rsqrt(mean(block^2) + eps) * post      (block itself where post is null)
//   r' = scale * residual + gate * n                    (gate: one row for each tokens_per_gate rows; null: 1)
//   x  = r' * rsqrt(mean(r'^2) + eps) * weight
struct NormParams {
  const unsigned short *block, *weight, *post, *gate;  // of the activation type; weight, post [D], gate [T / tokens_per_gate, D]
  const void* residual;                                // of the activation type or fp32; null: zero
  unsigned short* x;                                   // one of x and
  signed char* x_int;                                  // x_int with x_sf
  float* x_sf;
  void* new_residual;                                  // of the residual's type
  int T, D, tokens_per_gate;
  long long ldb, ldr, ldg, ldx, ldn;                   // row strides of block, residual, gate, x / x_int, new_residual
  float scale, eps;
  int sms;                                             // of the GPU
};
struct NormBackwardParams {
  const unsigned short *block, *weight, *post, *gate, *grad_x;
  const void *residual, *grad_new;  // null: zero
  unsigned short* grad_block;
  void* grad_residual;              // null: not wanted
  float *grad_weight, *grad_post, *grad_gate;  // [D], [D], [gates, D] fp32
  float* partial;                   // [2][CTAs][D]: shares of grad_weight, and of grad_post or S
  int* status;                      // workspace status header
  int T, D, gates, tokens_per_gate;
  int ctas_per_gate, grid;          // CTAs that share a gate's rows; several gates to a CTA where it is 1
  int sums_runs, sums_per, gate_per;  // runs of a gate's shares in the second kernel; 65536 / runs + 1; 65536 / ctas_per_gate + 1
  int threads, vectors, stages, smem;  // threads of a row, its vectors of a thread, rows in shared memory and their bytes
  long long ldb, ldr, ldg, lddx, lddn, lddb, lddr;
  float scale, eps;
};

void norm_backward_shape(int D, bool residual_f32, int gates, int tokens_per_gate, int sms, int max_smem, NormBackwardParams* p);
cudaError_t cast_int_launch(const CastIntParams& p, int act, cudaStream_t stream);
cudaError_t norm_launch(const NormParams& p, int act, bool residual_f32, cudaStream_t stream);
cudaError_t norm_backward_launch(const NormBackwardParams& p, int act, bool residual_f32, cudaStream_t stream);

}  // namespace b200q
