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
  // Few rows: what the tiles of each row found before (nullptr: nothing).
  unsigned long long* best;  // (N, tiles): the largest key, and the complement of its first token; all ones: a NaN
  unsigned long long* bins;  // (N, SAMPLE_BINS) the first histogram
  unsigned long long* sums;  // (N, tiles, SAMPLE_WAVES) kept weights, of rows without top-k and top-p
};

constexpr int SAMPLE_THREADS = 1024, SAMPLE_WAVES = SAMPLE_THREADS / 64;
constexpr int SAMPLE_TILE = 4 * SAMPLE_THREADS;  // tokens of a tile
constexpr int SAMPLE_TILES = 256;                // tiles of the largest vocabulary
constexpr int SAMPLE_BINS = 2048;
inline int sample_tiles(int V) { return (V + SAMPLE_TILE - 1) / SAMPLE_TILE; }

}  // namespace alg
