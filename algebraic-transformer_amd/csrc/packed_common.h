// Attention over packed sequences and over a paged cache: parameters, the weights' arithmetic and
// the mapping of workgroups to sequences, shared by packed_fwd.hip, packed_bwd.hip and
// paged_decode.hip.
//
// Weights without a pass ahead of them. With x = q.k alpha, alpha = 1/(sqrt(D) c), the weight of a
// key is rho(x)^n, rho(x) = x + sqrt(1 + x^2). The kernels form s = (q 2^-e).k (a power of two:
// exact) and t = s + sqrt(s^2 + b), b = 1/a^2, a = alpha 2^e; then t = rho(x) / a, and the factor
// a^-n, common to a row's weights and its sink, cancels in the normalisation. No rounding of a
// scaled query and no multiplication per score is left. e makes a in [R, 2 R), R the rho of X =
// 1.875 (n <= 16) or 0.75 (n = 32), so that t^n is at most 1 for x up to X.
// The plain form sums t^n and t^n v in f32 as they are, which is exact enough for a row whose sum
// lies in [low count, 2^30], low = (R a)^-n the weight at x = -X and count its keys. Above, a weight
// may have overflowed, or its product with v. Below, the mean key lies under -X, where s + sqrt(s^2
// + b) cancels: a key at x contributes at most (2/|x|)^n 4 n x^2 eps low of error, 32 eps low at the
// least n, so that a sum above low count has lost no more than 2^-19 of itself, and a weight no
// more than 2^-19 of its row's mean one. The sum is all that
// is looked at, once a row, and nothing per score; if a row fails, its workgroup (or wave) does its
// rows again in the careful form: a running maximum per row, and rho of a negative x as 1/rho(-x).
// The row statistic is rs = (row's shift) Z^(-1/n), so that a normalised weight is (t rs)^n in
// either form; its sign tells the backward pass which form the row took (negative: careful).
//
// Rows. The H query heads share Hkv key heads in groups of G = H / Hkv. The G queries of one token
// at one key head are neighbours in a row index r = t G + g of the sequence, so that a tile of 128
// rows holds 128 / G tokens, K and V are read once for the group, dK and dV add up over the group
// inside one workgroup, and a single token's G queries share a tile.
//
// Sequences. cu[s] is the first token of sequence s. Sequence s owns the work slots from
// cu[s] G / ROWS + s on: at least as many as it has tiles, so that a workgroup finds its sequence
// by a search over cu, without a list made ahead; a slot past a sequence's tiles ends at once
// (at most one a sequence). The tokens from cu[S] on belong to no sequence: their outputs and
// gradients are zero.
#pragma once

#include "attn_common.h"

namespace alg {

constexpr int PK_ROWS = 128;  // rows (token, head of the group) per workgroup of the prompt kernels
constexpr int PK_BK = 64;     // keys per LDS tile
constexpr int DECODE_RANGE = 256;  // keys that a range holds at least, but for a sequence's last
constexpr int MAX_RANGES = 256;    // ranges that packed_combine_kernel joins

// How scores become weights for one call (host: attn_scale).
struct AttnScale {
  int log2n;
  float qmul;   // 2^-e, applied to the queries (exact in bf16 but for subnormals)
  float a;      // alpha 2^e: x = a s
  float b;      // 1 / a^2
  float low;    // least mean weight of the plain form; infinite: every row takes the careful form
};

struct PackedParams {
  const bf16* q;   // (N, H, D)
  const bf16* k;   // packed: (N, Hkv, D); paged: pages of (Hkv, page, D)
  const bf16* v;
  bf16* o;         // (N, H, D), contiguous
  float* stat;     // (Hkv, N G) row statistics, or nullptr
  const void* sink;  // logits, `sink_count` (1 or H) of them, f32 or bf16, or nullptr
  int sink_count, sink_bf16;
  float c;
  const int* cu;   // (S + 1)
  const int* kv_lens;  // paged: (S) keys held, the new tokens among them
  const int* table;    // paged: (S, width) page numbers
  int width, page, pages;
  long q_ts, q_hs;             // elements between tokens, between heads
  long k_ts, k_hs, k_ps;       // tokens, heads, pages
  long v_ts, v_hs, v_ps;
  int N, S, H, Hkv, G;
  AttnScale sc;
  // Keys in `nsplit` ranges, each with its own partial row: f32 sums of t^n v, then per row Z and
  // the shift's reciprocal (negative: the careful form).
  int nsplit;
  float* part_o;   // (nsplit, Hkv N G, D)
  float* part_zt;  // (nsplit, Hkv N G, 2)
};

// New tokens' queries, keys and values on their way into a paged cache (paged_append.hip).
struct PagedAppendParams {
  const bf16 *q, *k, *v;  // raw projections (N, H or Hkv, D)
  long q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;
  bf16 *kp, *vp;          // pages of (Hkv, page, D)
  long kp_ps, kp_hs, kp_ts, vp_ps, vp_hs, vp_ts;
  bf16* qo;               // (N, H, D) contiguous
  const int *cu, *kv_lens, *table;
  int width, page, pages;
  const void *q_gain, *k_gain;   // (D), f32 or bf16, or nullptr
  int gain_bf16;
  const float *cos, *sin;        // (>= width page, D / 2) or nullptr
  float eps;
  int N, S, H, Hkv, D;
};

// Whether a row of `count` keys whose weights sum to `sum` needs the careful form (a NaN does).
__device__ __forceinline__ bool needs_care(float sum, int count, float low) {
  return count > 0 && !(sum >= low * (float)count && sum <= 0x1p30f);
}

struct PackedBwdParams {
  const bf16 *q, *k, *v, *o, *dO;
  const float* stat;  // (Hkv, N G)
  float* ndi;         // (Hkv, N G), - sum_d dO o, written by the dQ kernel
  int* care;          // (slots, Hkv): whether the slot's rows took the careful form, likewise
  const void* sink;
  int sink_count, sink_bf16;
  float c;
  const int* cu;
  long q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, do_ts, do_hs;
  bf16 *dq, *dk, *dv;  // contiguous
  void* dsink;         // (H) gradients per head, f32 or bf16, or nullptr
  int dsink_bf16;
  int N, S, H, Hkv, G;
  AttnScale sc;
  // dQ's keys and dK/dV's rows in ranges, of which each leaves its f32 sums (1: none; the gradients
  // themselves are written); packed_join_kernel adds them up.
  int dq_parts, dkdv_parts;
  float* dq_sum;              // (dq_parts, N, H, D)
  float *dk_sum, *dv_sum;     // (dkdv_parts, N, Hkv, D)
};

// Values formed here whatever is selected of them afterwards: without it the arithmetic of a masked
// element moves behind a branch of its own, a branch an element.
__device__ __forceinline__ void keep_here(float& a) { asm volatile("" : "+v"(a)); }
__device__ __forceinline__ void keep_here(float& a, float& b) { asm volatile("" : "+v"(a), "+v"(b)); }

template <typename P>
__device__ __forceinline__ float sink_score(const P& p, int head) {
  const int i = p.sink_count == 1 ? 0 : head;
  const float logit = p.sink_bf16 ? (float)static_cast<const bf16*>(p.sink)[i] : static_cast<const float*>(p.sink)[i];
  return logit / (p.c * p.sc.a);
}

// t and r = 1/sqrt(s^2 + b) of the plain form.
__device__ __forceinline__ float weight_t(float s, float b, float& r) {
  const float rad = __builtin_fmaf(s, s, b);
  r = rsq(rad);
  return __builtin_fmaf(rad, r, s);
}
// The careful form, as exact for either sign: t = b / (|s| + sqrt(s^2 + b)) below zero. Past
// |s| = 2^60 the square root is |s| itself (b is at most 1), and rad would overflow.
__device__ __forceinline__ float weight_t_careful(float s, float b, float& r) {
  const float as = __builtin_fabsf(s);
  const bool far = as > 0x1p60f;
  const float rad = __builtin_fmaf(s, s, b);
  r = far ? __builtin_amdgcn_rcpf(as) : rsq(rad);
  const float u = as + (far ? as : rad * r);
  return s < 0.0f ? b * __builtin_amdgcn_rcpf(u) : u;
}

// A sink's weight beside the shift T >= ts, its own. A sink of -inf (ts = 0) has none, also where no
// key gives T another value than 0.
__device__ __forceinline__ float sink_weight(float ts, float T, int log2n) {
  return ts == 0.0f ? 0.0f : pow2n<0>(ts / T, log2n);
}

// Slots of a launch, and the sequence of slot `slot` (S: the tokens behind the last sequence).
__host__ __device__ inline int packed_slots(int N, int G, int S, int rows) { return (int)((long)N * G / rows) + S + 1; }

struct PackedSeq {
  int s;      // S: behind the last sequence
  int start;  // first token
  int len;    // tokens
  int tile;   // tile of `rows` rows within the sequence
};
// First token of entry s, whatever the caller wrote there: in [0, N].
__device__ __forceinline__ int packed_start(const int* cu, int s, int N) {
  return s == 0 ? 0 : min(max(cu[s], 0), N);
}
// Up to 64 sequences, one a lane of the wave: the tiles are counted by a sum over the lanes, and a
// launch's first items are tiles, without the gaps of the slots (empty workgroups between others
// leave the CUs unevenly filled: 8 requests of 8000 keys, 8 heads in 4 ranges, 58 us instead of 47).
// The tokens behind the last sequence come last.
struct PackedLanes {
  int s, start, len, tiles;  // of the lane's sequence
};
__device__ __forceinline__ PackedLanes packed_lanes(const int* cu, int N, int S, int G, int rows) {
  const int lane = threadIdx.x & 63;
  PackedLanes a{lane, 0, 0, 0};
  if (lane < S) {
    a.start = packed_start(cu, lane, N);
    a.len = max(packed_start(cu, lane + 1, N) - a.start, 0);
  }
  a.tiles = (a.len * G + rows - 1) / rows;
  return a;
}
__device__ __forceinline__ int lane_value(int v, int lane) { return __builtin_amdgcn_readfirstlane(__shfl(v, lane, 64)); }
__device__ __forceinline__ PackedSeq packed_tail(const int* cu, int N, int S, int tile) {
  PackedSeq f;
  f.s = S;
  f.start = __builtin_amdgcn_readfirstlane(packed_start(cu, S, N));
  f.len = N - f.start;
  f.tile = tile;
  return f;
}
// The lanes' sequences by rising number of keys: over a cache, where a launch is a round or two of
// workgroups and a sequence's work goes with the keys it holds, not with its tokens. (701 tokens each
// over 12000, 8000 and 4000 keys, 16 heads over 4, two ranges: 230 us, 178 with the longest first; 459
// each over 6000 and eleven of 2064 keys, 8 heads over 1: 106, 82. Packed sequences alone, of many more
// workgroups, gained nothing: nine documents of 16384 tokens 203, 205.)
__device__ __forceinline__ void packed_sort(PackedLanes& a, int S, const int* kv_lens) {
  const int lane = threadIdx.x & 63;
  const int key = lane < S ? kv_lens[lane] : 0;
  int rank = 0;
  for (int i = 0; i < S; ++i) {
    const int k = __builtin_amdgcn_readlane(key, i);
    rank += k < key || (k == key && i < lane);
  }
  if (lane >= S) rank = lane;
  const int from = __builtin_amdgcn_ds_permute(4 * rank, lane);  // lane `rank` receives this lane
  a.s = from;
  a.start = __shfl(a.start, from, 64);
  a.len = __shfl(a.len, from, 64);
  a.tiles = __shfl(a.tiles, from, 64);
}
// Item `item` of a launch of `slots` of them: sequence after sequence (kv_lens: sorted), or backwards.
template <bool BACKWARDS>
__device__ __forceinline__ PackedSeq packed_find(const int* cu, int N, int S, int G, int rows, int item, int slots,
                                                 const int* kv_lens = nullptr) {
  const int lane = threadIdx.x & 63;
  if (S <= 64) {
    PackedLanes a = packed_lanes(cu, N, S, G, rows);
    if (kv_lens && S > 1) packed_sort(a, S, kv_lens);
    int upto = a.tiles;  // tiles of the sequences up to the lane's
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      const int below = __shfl_up(upto, m, 64);
      if (lane >= m) upto += below;
    }
    const int total = lane_value(upto, 63);
    if (item >= total) return packed_tail(cu, N, S, item - total);
    if (BACKWARDS) item = total - 1 - item;
    PackedSeq f;
    const int at = __builtin_amdgcn_readfirstlane(__popcll(__ballot(upto <= item)));
    f.s = lane_value(a.s, at);
    f.start = lane_value(a.start, at);
    f.len = lane_value(a.len, at);
    f.tile = item - lane_value(upto - a.tiles, at);
    return f;
  }
  const int slot = BACKWARDS ? slots - 1 - item : item;
  int lo = 0, n = S + 1;
  while (n > 1) {  // 64 candidates at a time: two steps up to 4095 sequences
    const int step = (n + 63) / 64;
    const int at = lane * step;
    bool ok = false;
    if (at < n) {
      const int s = lo + at;
      ok = packed_start(cu, s, N) * G / rows + s <= slot;
    }
    const int c = max((int)__popcll(__ballot(ok)), 1) - 1;
    lo += c * step;
    n = min(step, n - c * step);
  }
  PackedSeq f;
  f.s = __builtin_amdgcn_readfirstlane(min(lo, S));
  f.start = __builtin_amdgcn_readfirstlane(packed_start(cu, f.s, N));
  const int end = f.s == S ? N : __builtin_amdgcn_readfirstlane(packed_start(cu, f.s + 1, N));
  f.len = max(end - f.start, 0);
  f.tile = slot - (f.start * G / rows + f.s);
  return f;
}
// A tile's slot.
__device__ __forceinline__ int packed_slot(const PackedSeq& f, int G, int rows) { return f.start * G / rows + f.s + f.tile; }

// The same for a kernel whose work grows with the tile's number: by falling tile number over all
// sequences, so that the longest work starts first wherever its sequence lies. With f(l) the number
// of tiles numbered l or more, item i has the largest l with f(l) > i, found by halving. From 65
// sequences on, packed_find's order backwards. (dK/dV of nine documents, 16384 tokens, 16 heads over
// 4, D = 128: 454 us then, 486 in packed_find's order; of 13 documents, 8161 tokens, 16 heads, D = 64,
// which are more workgroups of more equal work: 63 and 60.)
__device__ __forceinline__ PackedSeq packed_find_heavy(const int* cu, int N, int S, int G, int rows, int item, int slots) {
  if (S > 64) return packed_find<true>(cu, N, S, G, rows, item, slots);
  const int lane = threadIdx.x & 63;
  const PackedLanes a = packed_lanes(cu, N, S, G, rows);
  const auto f = [&](int l) {
    int c = max(a.tiles - l, 0);
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) c += __shfl_xor(c, m, 64);
    return __builtin_amdgcn_readfirstlane(c);
  };
  const int total = f(0);
  if (item >= total) return packed_tail(cu, N, S, item - total);
  int lo = 0, hi = slots;  // f(lo) > item, f(hi) <= item: every tile's number is below `slots`
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (f(mid) > item) lo = mid;
    else hi = mid;
  }
  const int k = item - f(lo + 1);  // k-th of the sequences that have a tile `lo`
  const unsigned long long has = __ballot(a.tiles > lo);
  const int before = __popcll(has & ((1ull << lane) - 1));
  const unsigned long long at = __ballot(a.tiles > lo && before == k);
  PackedSeq r;
  r.s = __builtin_amdgcn_readfirstlane(at ? __builtin_ctzll(at) : 0);
  r.start = lane_value(a.start, r.s);
  r.len = lane_value(a.len, r.s);
  r.tile = at ? lo : -1;
  return r;
}

// Where row `r` of a sequence lies: its token, head, and elements in the outputs and statistics.
struct PackedRow {
  int tok, head;
  size_t out, stat;
};
template <int D, typename P>
__device__ __forceinline__ PackedRow packed_row(const P& p, const PackedSeq& f, int kvh, int r) {
  PackedRow a;
  a.tok = r / p.G;
  a.head = kvh * p.G + r - a.tok * p.G;
  a.out = ((size_t)(f.start + a.tok) * p.H + a.head) * D;
  a.stat = (size_t)kvh * p.N * p.G + (size_t)f.start * p.G + r;
  return a;
}
// A lane's row formed again where it is used (registers are short in the main loops).
__device__ __forceinline__ int again(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

// One 16-row group of a K / V tile: where its rows start, and how many of them exist.
struct KvGroup {
  const bf16* k;
  const bf16* v;
  int rows;
};

}  // namespace alg
