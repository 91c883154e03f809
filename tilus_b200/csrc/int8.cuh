// Parameter blocks of the 8-bit integer products (int8_kernel.cu) and of the host code (int8_api.cu), and what that shares with api.cu.
#pragma once
#include <cuda.h>

#include "common.cuh"

namespace b200q {

struct Int8Params {
  const signed char *a, *b;    // [M, K], [rows, K], row strides lda and ldb (the row kernel; the others have tensor maps of them)
  long long lda, ldb;
  const float* a_sf;           // [M] scales of the rows of A
  const float* b_sf;           // [columns of the product] scales of the rows of B
  const unsigned short* bias;  // [N] of the output type, or null
  unsigned short* c;           // [M, N], leading dimension ldc
  int* status;                 // workspace status header
  int M, N, K, ldc;            // N: columns of the output (gated: half the rows of B)
  int kblocks;                 // ceil(K / 128): stages of the pipelines
  int act;                     // type of C and the bias: 0 fp16, 1 bf16
  int use_clamp;               // gated: clamp the gate from above and the other factor on both sides
  float clamp;
  int tiles, m_tiles, n_tiles, m_group;  // pair kernel: output tiles and their raster groups
  int rows, width, wide;       // stream kernel: rows of A rounded up to 16; output columns of the first `wide` CTAs (or clusters)
  int cluster, stages, smem;   // CTAs that share K, ring slots, dynamic shared memory
  int early;                   // stream and row kernels: B was complete when the kernel before this one started
};

// api.cu
struct DeviceInfo {
  int sm_count = 0;
  int max_smem = 0;
};
DeviceInfo device_info();
int cuda_failed(int code);  // remembers a CUDA error for b200q_last_cuda_error and returns ST_CUDA
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_tiled_fn();

// int8_kernel.cu
int int8_pair_smem_bytes(int cols);
int int8_stream_smem_bytes(int M, bool gated, int width, int cluster, int stages);
cudaError_t int8_pair_launch(const Int8Params& p, bool gated, int cols, const CUtensorMap& ta, const CUtensorMap& tb,
                             const CUtensorMap& tc, int grid, cudaStream_t stream);
const int* int8_stream_clusters(const DeviceInfo& di);
cudaError_t int8_row_launch(const Int8Params& p, bool gated, int grid, cudaStream_t stream);
cudaError_t int8_stream_launch(const Int8Params& p, bool gated, const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tb_less,
                               cudaStream_t stream);

}  // namespace b200q
