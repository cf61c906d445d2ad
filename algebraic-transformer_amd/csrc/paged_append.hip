// New tokens into a paged cache, bf16: QK RMS norm with gain and the Cayley rotation at each
// token's position (src/algebraic/model.py:170-174 with algebraic.py:76-83, 172-179, for a token
// that continues a cached sequence), the queries to a packed output, keys and values to their
// pages.
//
// A row of D elements is split over D / 16 lanes; lane li holds the 16-byte chunk li of both
// halves, so that the pairs (x_j, x_{j + D/2}) that a rotation mixes sit in one lane and only the
// sum of squares crosses lanes. One workgroup takes the H + 2 Hkv rows of a token: its sequence,
// position and page are found once per wave and are wave-uniform. y = rot((x tau) gain) is
// computed in f32 and rounded once (the training prologue rounds after the norm, in the tables and
// after every product, as the reference does in bf16; a cache holds what it holds for long, and
// here each of those roundings can be left out). Bytes bound it: each row is read and written
// once. 8000 prompt tokens, 16 heads of 64, 96 MB: 20.7 us, 4.7 TB/s; 64 single tokens, 32 heads over 8 of
// 128: 5.4 us, the latency of the search, the page's entry and a row.
#include "launchers.h"
#include "packed_common.h"

namespace alg {

namespace {

template <int CH>
__device__ __forceinline__ void load8(const bf16* p, float (&x)[CH]) {
  bf16 v[8];
  *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(p);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = (float)v[e];
}
__device__ __forceinline__ void store8(bf16* p, const float (&x)[8]) {
  bf16 v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = f2bf(x[e]);
  *reinterpret_cast<uint4*>(p) = *reinterpret_cast<uint4*>(v);
}
__device__ __forceinline__ void loadf8(const float* p, float (&x)[8]) {
  *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(p);
  *reinterpret_cast<float4*>(x + 4) = *reinterpret_cast<const float4*>(p + 4);
}

}  // namespace

template <int D>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedAppendParams p) {
  constexpr int LPR = D / 16, HALF = D / 2;  // lanes a row
  constexpr int RPB = 256 / LPR;             // rows in flight a workgroup
  const int tok = blockIdx.x;
  const int li = threadIdx.x % LPR, c0 = 8 * li;
  // The token's sequence: with one row a slot, slots are tokens plus sequences passed. The last
  // entry that starts at or before the token is found as in packed_find.
  int lo = 0, n = p.S + 1;
  const int lane = threadIdx.x & 63;
  while (n > 1) {
    const int step = (n + 63) / 64, at = lane * step;
    const bool ok = at < n && packed_start(p.cu, lo + at, p.N) <= tok;
    const int c = max((int)__popcll(__ballot(ok)), 1) - 1;
    lo += c * step;
    n = min(step, n - c * step);
  }
  const int s = __builtin_amdgcn_readfirstlane(min(lo, p.S));
  const bool held = s < p.S;  // else behind the last sequence: no place, and a query of zeros
  int pos = -1;
  if (held) pos = max(p.kv_lens[s], 0) - packed_start(p.cu, s + 1, p.N) + tok;
  const bool placed = held && pos >= 0 && pos < p.width * p.page;
  int id = -1, slot = 0;
  if (placed) {
    const int pi = pos / p.page;
    slot = pos - pi * p.page;
    id = p.table[(size_t)s * p.width + pi];
  }
  const bool write = (unsigned)id < (unsigned)p.pages;

  float cs[8], sn[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    cs[e] = 1.0f;
    sn[e] = 0.0f;
  }
  if (p.cos && placed) {
    loadf8(p.cos + (size_t)pos * HALF + c0, cs);
    loadf8(p.sin + (size_t)pos * HALF + c0, sn);
  }
  const int rows = p.H + 2 * p.Hkv;
  for (int r = threadIdx.x / LPR; r < rows; r += RPB) {
    const bool isq = r < p.H, isv = r >= p.H + p.Hkv;
    const int head = isq ? r : (isv ? r - p.H - p.Hkv : r - p.H);
    const bf16* src = isq ? p.q + (size_t)tok * p.q_ts + (size_t)head * p.q_hs
                          : (isv ? p.v + (size_t)tok * p.v_ts + (size_t)head * p.v_hs
                                 : p.k + (size_t)tok * p.k_ts + (size_t)head * p.k_hs);
    bf16* dst = isq ? p.qo + ((size_t)tok * p.H + head) * D
                    : (isv ? p.vp + (size_t)max(id, 0) * p.vp_ps + (size_t)head * p.vp_hs + (size_t)slot * p.vp_ts
                           : p.kp + (size_t)max(id, 0) * p.kp_ps + (size_t)head * p.kp_hs + (size_t)slot * p.kp_ts);
    float a[8], b[8];
    load8(src + c0, a);
    load8(src + HALF + c0, b);
    float ss = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss += a[e] * a[e] + b[e] * b[e];
#pragma unroll
    for (int m = 1; m < LPR; m <<= 1) ss += __shfl_xor(ss, m, 64);
    if (!isv) {
      const float tau = 1.0f / sqrtf(ss * (1.0f / D) + p.eps);
      const void* gain = isq ? p.q_gain : p.k_gain;
      float ga[8], gb[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) ga[e] = gb[e] = 1.0f;
      if (gain && p.gain_bf16) {
        load8(static_cast<const bf16*>(gain) + c0, ga);
        load8(static_cast<const bf16*>(gain) + HALF + c0, gb);
      } else if (gain) {
        loadf8(static_cast<const float*>(gain) + c0, ga);
        loadf8(static_cast<const float*>(gain) + HALF + c0, gb);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float ya = a[e] * tau * ga[e], yb = b[e] * tau * gb[e];
        a[e] = placed ? ya * cs[e] - yb * sn[e] : 0.0f;
        b[e] = placed ? ya * sn[e] + yb * cs[e] : 0.0f;
      }
    }
    if (isq || write) {
      store8(dst + c0, a);
      store8(dst + HALF + c0, b);
    }
  }
}

hipError_t launch_paged_append(const PagedAppendParams& p, hipStream_t st) {
  KTimer t("paged_append", st);
  if (p.D == 64) hipLaunchKernelGGL(paged_append_kernel<64>, dim3(p.N), dim3(256), 0, st, p);
  else hipLaunchKernelGGL(paged_append_kernel<128>, dim3(p.N), dim3(256), 0, st, p);
  return hipGetLastError();
}

}  // namespace alg
