// The paged 8-bit cache: what its kernels share on the host.
#pragma once
#include <ATen/core/Tensor.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace q8 {

struct ChunkArgs {
  const void* q;                 // [T, nq, D] bf16, row stride q_row
  int64_t q_row;
  const uint8_t *kc, *vc;        // [pages, nkv, bs, D]
  const float *ks, *vs;          // [pages, nkv]
  const int* tables;             // [B, width]
  const int *lens, *news;        // [B]
  void* out;                     // [T, nq, D]
  int B, T, width, nq, nkv, bs, pages;
  int min_new;                   // sequences with fewer new tokens are left out
  float scale;                   // softmax scale times log2 e
};

// whether the cache and the tables are as the kernels take them
bool cache_fits(const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& ks, const at::Tensor& vs, const at::Tensor& tables,
                const at::Tensor& lens, const c10::optional<at::Tensor>& news, c10::Device dev);

bool chunk_supported(int rep);
void launch_chunk(const ChunkArgs& a, int D, int dev, cudaStream_t st);

}  // namespace q8
