// Parameters of drawing tokens from the algebraic likelihood (head_sample.hip).
#pragma once

#include <stdint.h>

namespace alg {

struct HeadSampleParams {
  const void* z;  // (N, V) logits, f32 or bf16, rows `stride` elements apart
  long stride;
  int z_bf16;
  int N, V;
  const void* u;    // (N) uniform numbers, f32 or f64
  int u_f64;
  // Settings, one a row or (pointer nullptr) one for all.
  const float *temperature, *top_p, *min_p;
  const int* top_k;
  float temperature_all, top_p_all, min_p_all;
  int top_k_all;
  double n, inv_c, clamp;  // x = min(z inv_c, clamp)
  float z_clamp;           // the least float whose x reaches the clamp
  int bits;                // a weight of 1 counts 2^bits: V of them stay under 2^62
  int64_t* token;
  float* logprob;
};

}  // namespace alg
