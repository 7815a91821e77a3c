// layer.h -- what layer.cpp shares with verify.cpp: the decode step of the Llama
// layer with its cache append and attention left to the caller.
#pragma once

#include "../../include/reef_b200.h"
#include "ops.h"

namespace reef {

// The two pieces of a decode step that differ between one new token per sequence
// and several drafted ones.
struct DecodeHooks {
  // the QKV projection's split-K partials -> q8 / q_scale and the cache rows
  virtual int append(const int32_t* part, int splits, const float* x_scale, int8_t* q8,
                     float* q_scale, int* lens, cudaStream_t st) = 0;
  // attention of q8 over the cache -> out [rows][heads_q * 128]; partial:
  // decode_attn_partial_floats() of scratch
  virtual int attend(const int8_t* q8, const float* q_scale, const int* lens, float* partial,
                     float* out, cudaStream_t st) = 0;

 protected:
  ~DecodeHooks() = default;
};

// Workspace bytes of decode_run on layer->batch rows (0: invalid).
size_t decode_run_bytes(const reef_b200_llama_layer* layer, size_t max_len);
// The decode step on layer->batch rows x -> y (arguments checked by the caller).
int decode_run(const reef_b200_llama_layer* layer, const float* x, float* y, size_t max_len,
               void* workspace, size_t workspace_bytes, DecodeHooks& hooks, cudaStream_t st);

}  // namespace reef
