// Parameters of the head's logits (head_logits.hip).
#pragma once

namespace alg {

struct HeadLogitsParams {
  const void* h;  // (N, d)
  const void* e;  // (V, d), of h's type
  float* z;       // (N, V)
  int bf16_in;
  int N, d, V;
};

}  // namespace alg
