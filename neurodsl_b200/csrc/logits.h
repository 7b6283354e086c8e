// logits.h — launcher of the penalties, biases and grammar mask on logits.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>

namespace nd {

struct LogitsPenalty {
  const void* logits;          // [rows][ld], bf16 or fp32
  bool in_f32;
  long long ld;
  int rows, V;
  const int* history;          // [rows][history_ld]; negative: no token
  long long history_ld;
  int n_history;               // 0 without a history
  const int* history_lens;     // [rows] or null (n_history)
  const float* repetition;     // [rows] or null
  const float* presence;
  const float* frequency;
  const int* bias_ids;         // [rows][n_bias] or null; negative: no entry
  const float* bias;           // [rows][n_bias]
  int n_bias;
  const unsigned int* mask;    // [rows][mask_ld] words or null; bit v % 32 of word v / 32
  long long mask_ld;
  void* out;                   // [rows][out_ld]
  bool out_f32;
  long long out_ld;
  int* idx;                    // [rows] or null
};
cudaError_t launch_logits_penalty(cudaStream_t stream, const LogitsPenalty& a, int* err_word);

}  // namespace nd
