// Parameters of the token embedding and its gradient (embedding.hip).
#pragma once

#include <stdint.h>

namespace alg {

struct EmbeddingParams {
  const void* tokens;  // (N), int32 or int64
  int tokens64;
  const void* table;   // (V, d), f32 or bf16
  int table_bf16;
  void* y;             // forward: (N, d); backward: its cotangent
  int y_bf16;
  float scale;
  int N, d, V;
  // Backward.
  void* grad;          // (V, d), of the table's type
  int* keys[2];        // (N) tokens, and where they stood, sorted from one into the other
  int* pos[2];
  int* hist;           // (256, blocks), then 256 sums
  int blocks, passes;
  float* part;         // (2 chunks, d): sums of the runs that reach over a chunk's borders
  int chunk, chunks;   // sorted tokens in chunks of this many
};

}  // namespace alg
