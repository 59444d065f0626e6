// Low-rank adapters beside a shared projection (lora.cu), for the forward pass.
#pragma once
#include "common.cuh"

namespace ms {

// One fused projection's adapters and the call's tensors (ms_lora_add's arguments).
struct LoraCall {
  const void* x;
  int64_t x_stride;
  const float* base;
  int64_t base_stride;
  void* out;
  int64_t out_stride;
  const void* a;
  const void* b;
  int K, N, n_slices;
  int slice_end[3];  // column ends of the first slices (contiguous slices)
  bool interleaved;  // two slices alternating every 8 columns (gate | up)
  bool swiglu;
  int dtype, out_dtype;
};

size_t lora_workspace_size(int n_tokens, int n_slices, int max_rank);
int lora_add(const LoraCall& c, const ms_lora_adapters& ad, const ms_lora_plan& plan,
             void* workspace, size_t workspace_bytes, cudaStream_t s);
int validate_lora(const ms_lora_adapters* ad, const ms_lora_plan* plan);

}  // namespace ms
