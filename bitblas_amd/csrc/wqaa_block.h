// wqaa_block.h - the block-scaled 8-bit path: shared declarations of its product, quantiser and norm (not part of the ABI)
#pragma once
#include "wqaa_common.h"

namespace wqaa {

constexpr int kBlock = 128;                  // k per scale (and weight rows per scale)

struct BlockGemmArgs {
  const unsigned char* A;                    // (M, K) 8-bit floats, rows K bytes apart
  const unsigned char* W;                    // (N, K)
  const float* sa;                           // scale of (row m, block b) at sa[b * sa_ld + m]
  const float* sw;                           // scale of (tile t, block b) at sw[t * KB + b]
  const void* bias;                          // (N,) of the output type, or null
  void* C;                                   // (M, N)
  float* ws;                                 // partial tiles of the K slices: (tile behind the whole ones, slice, BM, BN)
  long sa_ld;
  int M, N, K, KB;                           // KB = ceil(K / 128)
  int out_dtype;                             // wqaa_dtype
  int tiles_m, tiles_n;
  // the first `whole` tiles have a workgroup each; the others `split`, slice z of them k-blocks [z * split_len, min(KB, (z + 1) * split_len))
  int whole, split, split_len;
  int group_m;                               // M-tiles that share an N-tile back to back
};

int block_gemm_plan(const wqaa_block_desc& d, int m, wqaa_plan* plan);
size_t block_gemm_workspace_bytes(const wqaa_block_desc& d, int m);
int block_gemm_launch(const wqaa_block_desc& d, const void* A, const void* W, const float* sa, int64_t sa_ld, const float* sw, const void* bias,
                      void* C, int m, void* workspace, uint64_t workspace_bytes, hipStream_t stream);
// what a launch could not hold, refused before anything touches the device: rows and grids beyond 31 bits, a grid of 2^32 threads
int block_gemm_check(const wqaa_block_desc& d, int m);
int block_quantize_check(const wqaa_block_quant& q);
int residual_norm_check(const wqaa_residual_norm_args& n);
int block_quantize_launch(const wqaa_block_quant& q, hipStream_t stream);
int residual_norm_launch(const wqaa_residual_norm_args& n, hipStream_t stream);
void block_init();

}  // namespace wqaa
