// The token embedding y_t = s E[token_t] and its gradient dE_v = s sum of dy_t over the tokens equal v
// (src/algebraic/model.py: the table that the head reads as well).
//
// A token outside [0, V) has no row: below 0 (padding) it gets zeros, from V on NaN, and no gradient.
//
// The gradient's sums run in the order of the tokens, whatever runs when, so that a step gives the same bits
// each time; atomic adds would not, and would read and write the f32 table again for every token. So the
// tokens are sorted (stably, 8 bits a pass, in whole numbers), which makes equal ones neighbours, and one
// launch reads each dy row once, adds up runs of equal tokens in f32, and writes every row of dE once, zeros
// included. A run may be of any length (a few tokens make up much of a text), so the work is cut into chunks
// of sorted tokens, not into runs: a chunk writes the runs that lie within it, and leaves the sums of those
// that reach over its borders for a second launch, which adds them in order.
//
// Bytes bound it. 16384 tokens of a text, d 2048, V 32000, f32 table: lookup 28 us (156 MB, 5.7 TB/s), the gradient 69
// (333 MB, 4.8 TB/s, 265 of them written; zeros in stores of 16 neighbouring bytes a lane: 6 less than of 32; stores
// that pass the caches by took 116 for 82 then), its sort 16, the join 5.
#include <type_traits>

#include "common.h"
#include "embedding.h"
#include "launchers.h"

namespace alg {

namespace {

constexpr int EMB_THREADS = 256;
constexpr int SORT_BLOCK = 1024;  // tokens a workgroup of a pass takes, one a lane
constexpr int SORT_WAVES = SORT_BLOCK / 64;
constexpr int SORT_COUNT = 4;     // blocks up to which each counts all tokens
constexpr int SORT_SUM = 128;      // blocks up to which each adds up the counts of all
constexpr int ZERO_ROWS = 16;     // rows of the table that a workgroup looks after for zeros
constexpr int EMB_COLS = 512;     // columns a wave takes: 8 a lane

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(p);
    *reinterpret_cast<float4*>(x + 4) = *reinterpret_cast<const float4*>(p + 4);
  } else {
    const bf16x8 v = *reinterpret_cast<const bf16x8*>(p);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = (float)v[e];
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = *reinterpret_cast<const float4*>(x);
    *reinterpret_cast<float4*>(p + 4) = *reinterpret_cast<const float4*>(x + 4);
  } else {
    bf16x8 v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = f2bf(x[e]);
    *reinterpret_cast<bf16x8*>(p) = v;
  }
}

__device__ __forceinline__ long token_at(const EmbeddingParams& p, int i) {
  return p.tokens64 ? (long)static_cast<const int64_t*>(p.tokens)[i] : (long)static_cast<const int*>(p.tokens)[i];
}
// The key that a token is sorted by: V where it has no row.
__device__ __forceinline__ int token_key(const EmbeddingParams& p, int i) {
  const long t = token_at(p, i);
  return t >= 0 && t < p.V ? (int)t : p.V;
}
__device__ __forceinline__ int sort_key(const EmbeddingParams& p, int pass, int i) {
  return pass ? p.keys[(pass - 1) & 1][i] : token_key(p, i);
}

}  // namespace

// Eight elements a lane, rows one after the other.
template <typename E, typename Y>
__global__ __launch_bounds__(EMB_THREADS) void embedding_fwd_kernel(EmbeddingParams p) {
  const int each = p.d / 8;
  const size_t id = (size_t)blockIdx.x * EMB_THREADS + threadIdx.x;
  const size_t row = id / each;
  if (row >= (size_t)p.N) return;
  const int col = 8 * (int)(id - row * each);
  const long t = token_at(p, (int)row);
  float x[8];
  if (t >= 0 && t < p.V) {
    load8(static_cast<const E*>(p.table) + (size_t)t * p.d + col, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] *= p.scale;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = t < 0 ? 0.0f : __builtin_nanf("");
  }
  store8(static_cast<Y*>(p.y) + row * p.d + col, x);
}

// How often each value of 8 bits of the key occurs in each block of tokens.
__global__ __launch_bounds__(SORT_BLOCK) void embedding_hist_kernel(EmbeddingParams p, int pass) {
  __shared__ int count[256];
  const int i = blockIdx.x * SORT_BLOCK + threadIdx.x;
  if (threadIdx.x < 256) count[threadIdx.x] = 0;
  __syncthreads();
  if (i < p.N) atomicAdd(&count[(sort_key(p, pass, i) >> (8 * pass)) & 255], 1);
  __syncthreads();
  if (threadIdx.x < 256) p.hist[threadIdx.x * p.blocks + blockIdx.x] = count[threadIdx.x];
}

// Of many blocks, each value's counts made those of the blocks before, and their sum: a workgroup a value. (All passes
// of 65536 tokens 26 us so, 22 without; 131072 26 and 27; 1048576 47 to 51 and 270.)
__global__ __launch_bounds__(SORT_BLOCK) void embedding_sum_kernel(EmbeddingParams p) {
  __shared__ int sums[SORT_WAVES];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int* counts = p.hist + (size_t)blockIdx.x * p.blocks;
  int before = 0;
  for (int b0 = 0; b0 < p.blocks; b0 += SORT_BLOCK) {
    const int b = b0 + threadIdx.x, c = b < p.blocks ? counts[b] : 0;
    int upto = c;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      const int below = __shfl_up(upto, m, 64);
      if (lane >= m) upto += below;
    }
    if (lane == 63) sums[wave] = upto;
    __syncthreads();
    int all = 0;
    for (int w = 0; w < SORT_WAVES; ++w) {
      if (w < wave) upto += sums[w];
      all += sums[w];
    }
    if (b < p.blocks) counts[b] = before + upto - c;
    before += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) p.hist[(size_t)256 * p.blocks + blockIdx.x] = before;
}

// Each token to its place in the order of these 8 bits, equal ones as they stand: a workgroup 1024 tokens, a wave
// 64, whose lanes of equal bits find each other by ballots. With few tokens every workgroup counts them all
// itself, which saves a launch that counts them (both passes: 4096 tokens 15 to 16 us so, 17 with it; 8161 19 to 22,
// 18; 16384 25 to 32, the more so the more tokens are equal, 18). Tokens of one block are one workgroup's,
// which makes all passes (1024 tokens 10 us).
template <bool COUNT>
__device__ __forceinline__ void scatter(const EmbeddingParams& p, int pass) {
  __shared__ int base[SORT_WAVES][256], sums[256], before[256];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, begin = blockIdx.x * SORT_BLOCK;
  const int i = begin + tid;
  const bool live = i < p.N;
  const int key = live ? sort_key(p, pass, i) : 0, bits = (key >> (8 * pass)) & 255;
  const int where = live && pass ? p.pos[(pass - 1) & 1][i] : i;
  // How many tokens of value `tid` there are, and how many in the blocks before this one.
  int total = 0, earlier = 0;
  if constexpr (COUNT) {
    if (tid < 256) sums[tid] = before[tid] = 0;
    __syncthreads();
    for (int k0 = tid; k0 < p.N; k0 += 8 * SORT_BLOCK) {
      int k[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int at = k0 + e * SORT_BLOCK;
        k[e] = at < p.N ? (sort_key(p, pass, at) >> (8 * pass)) & 255 : -1;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (k[e] >= 0) atomicAdd(k0 + e * SORT_BLOCK < begin ? &before[k[e]] : &sums[k[e]], 1);
    }
    __syncthreads();
    if (tid < 256) {
      earlier = before[tid];
      total = earlier + sums[tid];
    }
    __syncthreads();
  } else if (p.blocks > SORT_SUM) {
    if (tid < 256) {
      earlier = p.hist[(size_t)tid * p.blocks + blockIdx.x];
      total = p.hist[(size_t)256 * p.blocks + tid];
    }
  } else if (tid < 256) {
#pragma unroll 8
    for (int b = 0; b < p.blocks; ++b) {
      const int c = p.hist[tid * p.blocks + b];
      if (b < (int)blockIdx.x) earlier += c;
      total += c;
    }
  }
  // The tokens of lower values: a sum over 256 lanes, four waves.
  int upto = total;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const int below = __shfl_up(upto, m, 64);
    if (lane >= m) upto += below;
  }
  if (tid < 256 && lane == 63) sums[wave] = upto;
  // The wave's lanes of the same bits.
  unsigned long long same = __ballot(live);
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const unsigned long long set = __ballot((bits >> k) & 1);
    same &= (bits >> k) & 1 ? set : ~set;
  }
  for (int w = tid; w < SORT_WAVES * 256; w += SORT_BLOCK) (&base[0][0])[w] = 0;
  __syncthreads();
  const int rank = __popcll(same & ((1ull << lane) - 1));
  if (live && rank == 0) base[wave][bits] = __popcll(same);
  if (tid < 256)
    for (int w = 0; w < wave; ++w) upto += sums[w];
  __syncthreads();
  if (tid < 256) {
    int at = upto - total + earlier;
#pragma unroll
    for (int w = 0; w < SORT_WAVES; ++w) {
      const int c = base[w][tid];
      base[w][tid] = at;
      at += c;
    }
  }
  __syncthreads();
  if (live) {
    const int to = base[wave][bits] + rank;
    p.keys[pass & 1][to] = key;
    p.pos[pass & 1][to] = where;
  }
}
template <bool COUNT>
__global__ __launch_bounds__(SORT_BLOCK) void embedding_scatter_kernel(EmbeddingParams p, int pass) {
  scatter<COUNT>(p, pass);
}
__global__ __launch_bounds__(SORT_BLOCK) void embedding_sort_kernel(EmbeddingParams p) {
  for (int pass = 0; pass < p.passes; ++pass) {
    if (pass) __syncthreads();  // what the pass before wrote
    scatter<true>(p, pass);
  }
}

// The first of n sorted keys, `apart` from each other, that is not below v: 64 of them looked at each time.
__device__ __forceinline__ int lower_bound(const int* keys, int n, int v, int apart = 1) {
  const int lane = threadIdx.x & 63;
  int lo = 0;
  while (n > 0) {
    const int step = (n + 63) / 64, at = lane * step;
    const int c = __popcll(__ballot(at < n && keys[(size_t)(lo + at) * apart] < v));
    if (c == 0) break;
    lo += (c - 1) * step + 1;
    n = min(step, n - (c - 1) * step) - 1;
  }
  return lo;
}

// Runs of equal tokens: a wave one chunk of sorted tokens and EMB_COLS columns, BATCH rows' loads under way at a
// time; the workgroups behind those the rows without a token.
template <typename E, typename Y>
__global__ __launch_bounds__(EMB_THREADS) void embedding_bwd_kernel(EmbeddingParams p) {
  constexpr int BATCH = sizeof(Y) == 2 ? 16 : 8;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int* keys = p.keys[(p.passes - 1) & 1];
  const int* pos = p.pos[(p.passes - 1) & 1];
  const int strips = (p.d + EMB_COLS - 1) / EMB_COLS, units = p.chunks * strips;
  const int work = (units + EMB_THREADS / 64 - 1) / (EMB_THREADS / 64);
  E* grad = static_cast<E*>(p.grad);
  if ((int)blockIdx.x >= work) {
    __shared__ int ends[2];
    __shared__ int held[ZERO_ROWS];
    const int v0 = (blockIdx.x - work) * ZERO_ROWS;
    if (threadIdx.x < ZERO_ROWS) held[threadIdx.x] = 0;
    if (wave < 2) {
      const int at = lower_bound(keys, p.N, v0 + wave * ZERO_ROWS);
      if (lane == 0) ends[wave] = at;
    }
    __syncthreads();
    for (int i = ends[0] + threadIdx.x; i < ends[1]; i += EMB_THREADS)
      if (keys[i] < p.V) held[keys[i] - v0] = 1;
    __syncthreads();
    const int pieces = p.d * (int)sizeof(E) / 16;
    for (int r = 0; r < min(ZERO_ROWS, p.V - v0); ++r)
      if (!held[r])
        for (int c = threadIdx.x; c < pieces; c += EMB_THREADS)
          reinterpret_cast<float4*>(grad + (size_t)(v0 + r) * p.d)[c] = float4{};
    return;
  }
  const int unit = blockIdx.x * (EMB_THREADS / 64) + wave;
  if (unit >= units) return;
  const int j = unit / strips, col = (unit - j * strips) * EMB_COLS + 8 * lane;
  const bool live = col < p.d;
  const int begin = j * p.chunk, end = min(p.N, begin + p.chunk);
  const Y* dy = static_cast<const Y*>(p.y) + (live ? col : 0);
  float sum[8] = {};
  int run = __builtin_amdgcn_readfirstlane(keys[begin]);
  bool head = begin > 0 && keys[begin - 1] == run;  // the run began before the chunk
  const bool tail = end < p.N && keys[end] == keys[end - 1];
  const auto leave = [&](bool tail) {
    if (run < p.V && live) {
      if (head || tail) {
        store8(p.part + ((size_t)2 * j + (head ? 0 : 1)) * p.d + col, sum);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] *= p.scale;
        store8(grad + (size_t)run * p.d + col, sum);
      }
    }
    head = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[e] = 0.0f;
  };
  for (int i0 = begin; i0 < end; i0 += 64) {
    const int n = min(64, end - i0);
    const int at = i0 + min(lane, n - 1), my_key = keys[at], my_pos = pos[at];
    for (int b = 0; b < n; b += BATCH) {
      Y x[BATCH][8];
#pragma unroll
      for (int e = 0; e < BATCH; ++e) {  // rows past the end again the last one
        const int row = __builtin_amdgcn_readlane(my_pos, min(b + e, n - 1));
        __builtin_memcpy(x[e], __builtin_assume_aligned(dy + (size_t)row * p.d, 16), sizeof x[e]);
      }
#pragma unroll
      for (int e = 0; e < BATCH; ++e) {
        if (b + e >= n) break;
        const int key = __builtin_amdgcn_readlane(my_key, b + e);
        if (key != run) {
          leave(false);
          run = key;
        }
#pragma unroll
        for (int c = 0; c < 8; ++c) sum[c] += (float)x[e][c];
      }
    }
  }
  leave(tail);
}

// Runs over several chunks: the workgroup of the chunk where one begins adds up its parts, each wave a quarter of
// them in order, then the quarters in order. (16384 tokens of 64 columns, a
// third of them one, 14 us, of one wave for all 47; a text's, 2048 columns, 8 and 10.)
template <typename E>
__global__ __launch_bounds__(EMB_THREADS) void embedding_join_kernel(EmbeddingParams p) {
  constexpr int WAVES = EMB_THREADS / 64;
  __shared__ float quarter[WAVES - 1][EMB_COLS];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int* keys = p.keys[(p.passes - 1) & 1];
  const int strips = (p.d + EMB_COLS - 1) / EMB_COLS, j = blockIdx.x / strips;
  const int col = (blockIdx.x - j * strips) * EMB_COLS + 8 * lane;
  const int end = (j + 1) * p.chunk;
  if (end >= p.N) return;
  const int run = keys[end - 1], next = keys[end], last = j > 0 ? keys[j * p.chunk - 1] : -1;
  if (run >= p.V || next != run || last == run) return;
  // The chunks that begin with the run: j + 1 to j + n.
  const int n = lower_bound(keys + end, p.chunks - j - 1, run + 1, p.chunk);
  const int each = (n + WAVES - 1) / WAVES, stop = min(n, (wave + 1) * each);
  const bool live = col < p.d;
  const float* part = p.part + (live ? col : 0);
  float sum[8] = {};
  if (wave == 0) load8(part + ((size_t)2 * j + 1) * p.d, sum);
  const auto add = [&](int b, auto batch) {
    constexpr int B = decltype(batch)::value;
    float x[B][8];
#pragma unroll
    for (int e = 0; e < B; ++e) load8(part + (size_t)2 * (j + 1 + min(b + e, stop - 1)) * p.d, x[e]);
#pragma unroll
    for (int e = 0; e < B; ++e) {
      if (b + e >= stop) break;
#pragma unroll
      for (int c = 0; c < 8; ++c) sum[c] += x[e][c];
    }
  };
  int b = wave * each;
  for (; b + 8 < stop; b += 16) add(b, std::integral_constant<int, 16>{});
  for (; b < stop; b += 2) add(b, std::integral_constant<int, 2>{});
  if (wave) store8(&quarter[wave - 1][8 * lane], sum);
  __syncthreads();
  if (wave || !live) return;
#pragma unroll
  for (int w = 0; w < WAVES - 1; ++w) {
    float x[8];
    load8(&quarter[w][8 * lane], x);
#pragma unroll
    for (int c = 0; c < 8; ++c) sum[c] += x[c];
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) sum[e] *= p.scale;
  store8(static_cast<E*>(p.grad) + (size_t)run * p.d + col, sum);
}

namespace {

template <typename F>
void by_types(const EmbeddingParams& p, F f) {
  if (p.table_bf16) p.y_bf16 ? f(bf16{}, bf16{}) : f(bf16{}, float{});
  else p.y_bf16 ? f(float{}, bf16{}) : f(float{}, float{});
}

}  // namespace

int embedding_sort_blocks(int N) { return (N + SORT_BLOCK - 1) / SORT_BLOCK; }

hipError_t launch_embedding_fwd(const EmbeddingParams& p, hipStream_t st) {
  KTimer t("embedding_fwd", st);
  const size_t lanes = (size_t)p.N * (p.d / 8);
  const dim3 grid((unsigned)((lanes + EMB_THREADS - 1) / EMB_THREADS));
  by_types(p, [&](auto e, auto y) {
    hipLaunchKernelGGL((embedding_fwd_kernel<decltype(e), decltype(y)>), grid, dim3(EMB_THREADS), 0, st, p);
  });
  return hipGetLastError();
}

hipError_t launch_embedding_bwd(const EmbeddingParams& p, hipStream_t st) {
  if (p.N) {
    KTimer t("embedding_sort", st);
    if (p.blocks == 1) hipLaunchKernelGGL(embedding_sort_kernel, dim3(1), dim3(SORT_BLOCK), 0, st, p);
    for (int pass = 0; pass < p.passes && p.blocks > 1; ++pass) {
      if (p.blocks <= SORT_COUNT) {
        hipLaunchKernelGGL(embedding_scatter_kernel<true>, dim3(p.blocks), dim3(SORT_BLOCK), 0, st, p, pass);
      } else {
        hipLaunchKernelGGL(embedding_hist_kernel, dim3(p.blocks), dim3(SORT_BLOCK), 0, st, p, pass);
        if (p.blocks > SORT_SUM) hipLaunchKernelGGL(embedding_sum_kernel, dim3(256), dim3(SORT_BLOCK), 0, st, p);
        hipLaunchKernelGGL(embedding_scatter_kernel<false>, dim3(p.blocks), dim3(SORT_BLOCK), 0, st, p, pass);
      }
    }
  }
  const long strips = (p.d + EMB_COLS - 1) / EMB_COLS, work = (p.chunks * strips + 3) / 4;
  {
    KTimer t("embedding_bwd", st);
    by_types(p, [&](auto e, auto y) {
      hipLaunchKernelGGL((embedding_bwd_kernel<decltype(e), decltype(y)>), dim3((unsigned)(work + (p.V + ZERO_ROWS - 1) / ZERO_ROWS)),
                         dim3(EMB_THREADS), 0, st, p);
    });
  }
  if (p.chunks > 1) {
    KTimer t("embedding_join", st);
    if (p.table_bf16) hipLaunchKernelGGL(embedding_join_kernel<bf16>, dim3((unsigned)(p.chunks * strips)), dim3(EMB_THREADS), 0, st, p);
    else hipLaunchKernelGGL(embedding_join_kernel<float>, dim3((unsigned)(p.chunks * strips)), dim3(EMB_THREADS), 0, st, p);
  }
  return hipGetLastError();
}

}  // namespace alg
