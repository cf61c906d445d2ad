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
#include <type_traits>

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

// e4m3 of eight values, a power of two scaled away.
__device__ __forceinline__ uint2 bytes8(const float (&x)[8], float unit) {
  int lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * unit, x[1] * unit, 0, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[2] * unit, x[3] * unit, lo, true);
  int hi = __builtin_amdgcn_cvt_pk_fp8_f32(x[4] * unit, x[5] * unit, 0, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(x[6] * unit, x[7] * unit, hi, true);
  return make_uint2(lo, hi);
}

// Where token `tok` stands: its sequence (S: behind the last), position, page and place in it.
struct TokenPlace {
  int s, pos, id, slot;
  bool placed;  // at a position that the table reaches
};
template <typename P>
__device__ __forceinline__ TokenPlace token_place(const P& p, int tok) {
  TokenPlace a;
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
  a.s = __builtin_amdgcn_readfirstlane(min(lo, p.S));
  const bool held = a.s < p.S;  // else behind the last sequence: no place
  a.pos = -1;
  if (held) a.pos = max(p.kv_lens[a.s], 0) - packed_start(p.cu, a.s + 1, p.N) + tok;
  a.placed = held && a.pos >= 0 && a.pos < p.width * p.page;
  a.id = -1;
  a.slot = 0;
  if (a.placed) {
    const int pi = a.pos / p.page;
    a.slot = a.pos - pi * p.page;
    a.id = p.table[(size_t)a.s * p.width + pi];
  }
  return a;
}

}  // namespace

// Into 8 bits the norm and rotation run in f64: a key that f32's few roundings carry over the border
// between two of its steps is 2^-3 away. Results go through f32 on their way to 8 bits or (queries) bf16, 2^-24
// beside half a step of 2^-4 or 2^-8. 7688 prompt tokens, 16 heads of 64, 80 MB: 30 us, 2.7 TB/s; in f32 it
// took 6 less, without the scales' bytes 2; neighbouring tokens on one XCD: no difference. 64 single
// tokens, 32 heads over 8 of 128: 6 us.
template <int D, bool FP8>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedAppendParams p) {
  typedef std::conditional_t<FP8, double, float> W;
  constexpr int LPR = D / 16, HALF = D / 2;  // lanes a row
  constexpr int RPB = 256 / LPR;             // rows in flight a workgroup
  const int tok = blockIdx.x;
  const int li = threadIdx.x % LPR, c0 = 8 * li;
  const TokenPlace at = token_place(p, tok);
  const int pos = at.pos, id = at.id, slot = at.slot;
  const bool placed = at.placed, write = (unsigned)id < (unsigned)p.pages;

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
    float a[8], b[8];
    load8(src + c0, a);
    load8(src + HALF + c0, b);
    W ss = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss += (W)a[e] * (W)a[e] + (W)b[e] * (W)b[e];
#pragma unroll
    for (int m = 1; m < LPR; m <<= 1) ss += __shfl_xor(ss, m, 64);
    if (!isv) {
      const W tau = (W)1 / sqrt(ss * ((W)1 / D) + (W)p.eps);
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
        const W ya = a[e] * tau * ga[e], yb = b[e] * tau * gb[e];
        a[e] = placed ? (float)(ya * cs[e] - yb * sn[e]) : 0.0f;
        b[e] = placed ? (float)(ya * sn[e] + yb * cs[e]) : 0.0f;
      }
    }
    if (isq) {
      bf16* dst = p.qo + ((size_t)tok * p.H + head) * D;
      store8(dst + c0, a);
      store8(dst + HALF + c0, b);
      continue;
    }
    const size_t dst = isv ? (size_t)max(id, 0) * p.vp_ps + (size_t)head * p.vp_hs + (size_t)slot * p.vp_ts
                           : (size_t)max(id, 0) * p.kp_ps + (size_t)head * p.kp_hs + (size_t)slot * p.kp_ts;
    if constexpr (!FP8) {
      if (write) {
        bf16* to = static_cast<bf16*>(isv ? p.vp : p.kp) + dst;
        store8(to + c0, a);
        store8(to + HALF + c0, b);
      }
    } else {
      unsigned top = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        top = max(top, max(__builtin_bit_cast(unsigned, a[e]) & 0x7FFFFFFFu, __builtin_bit_cast(unsigned, b[e]) & 0x7FFFFFFFu));
#pragma unroll
      for (int m = 1; m < LPR; m <<= 1) top = max(top, (unsigned)__shfl_xor((int)top, m, 64));
      const int byte = scale_byte(top);
      const float unit = scale_value(254 - min(byte, 254));
      uint2 lo = bytes8(a, unit), hi = bytes8(b, unit);
      if (byte == 255) {
        // A row with a value that is not finite: NaN keys, whose scores are NaN where they are seen;
        // values of zero, which leave alone the rows that do not see them (the scale is NaN).
        const unsigned fill = isv ? 0u : 0x7F7F7F7Fu;
        lo = hi = make_uint2(fill, fill);
      }
      if (write) {
        uint8_t* to = static_cast<uint8_t*>(isv ? p.vp : p.kp) + dst;
        *reinterpret_cast<uint2*>(to + c0) = lo;
        *reinterpret_cast<uint2*>(to + HALF + c0) = hi;
        if (li == 0)
          (isv ? p.vs + (size_t)id * p.vs_ps + (size_t)head * p.vs_hs
               : p.ks + (size_t)id * p.ks_ps + (size_t)head * p.ks_hs)[slot] = (uint8_t)byte;
      }
    }
  }
}

// The tokens' keys and values out of an 8-bit cache again, as the bf16 numbers they are. A workgroup a
// token as above, a lane 16 bytes of a row. 7688 tokens, 16 heads of 64, 49 MB: 11.7 us, 4.2 TB/s.
template <int D>
__global__ __launch_bounds__(256) void paged_read_kernel(PagedReadParams p) {
  constexpr int LPR = D / 16, RPB = 256 / LPR;
  const int tok = blockIdx.x;
  const int li = threadIdx.x % LPR, c0 = 16 * li;
  const TokenPlace at = token_place(p, tok);
  const bool found = (unsigned)at.id < (unsigned)p.pages;
  // Behind the last sequence and before position 0 there is nothing: zeros. A page that is none, and a
  // position that the table does not reach: NaN.
  const bool lost = !found && at.s < p.S && at.pos >= 0;
  for (int r = threadIdx.x / LPR; r < 2 * p.Hkv; r += RPB) {
    const bool isv = r >= p.Hkv;
    const int head = isv ? r - p.Hkv : r;
    bf16x8 x[2] = {};
    if (found) {
      const uint8_t* from = isv ? p.vp + (size_t)at.id * p.vp_ps + (size_t)head * p.vp_hs + (size_t)at.slot * p.vp_ts
                                : p.kp + (size_t)at.id * p.kp_ps + (size_t)head * p.kp_hs + (size_t)at.slot * p.kp_ts;
      const int byte = isv ? p.vs[(size_t)at.id * p.vs_ps + (size_t)head * p.vs_hs + at.slot]
                           : p.ks[(size_t)at.id * p.ks_ps + (size_t)head * p.ks_hs + at.slot];
      const int4 raw = *reinterpret_cast<const int4*>(from + c0);
      x[0] = values8(raw.x, raw.y, scale_value(byte));
      x[1] = values8(raw.z, raw.w, scale_value(byte));
      if (byte == 255) x[0] = x[1] = (bf16)__builtin_nanf("");
    } else if (lost) {
      x[0] = x[1] = (bf16)__builtin_nanf("");
    }
    bf16* to = (isv ? p.vo : p.ko) + ((size_t)tok * p.Hkv + head) * D + c0;
    *reinterpret_cast<bf16x8*>(to) = x[0];
    *reinterpret_cast<bf16x8*>(to + 8) = x[1];
  }
}

template <bool FP8>
static void launch_append(const PagedAppendParams& p, hipStream_t st) {
  if (p.D == 64) hipLaunchKernelGGL((paged_append_kernel<64, FP8>), dim3(p.N), dim3(256), 0, st, p);
  else hipLaunchKernelGGL((paged_append_kernel<128, FP8>), dim3(p.N), dim3(256), 0, st, p);
}

hipError_t launch_paged_append(const PagedAppendParams& p, hipStream_t st) {
  KTimer t(p.ks ? "paged_append_fp8" : "paged_append", st);
  if (p.ks) launch_append<true>(p, st);
  else launch_append<false>(p, st);
  return hipGetLastError();
}

hipError_t launch_paged_read(const PagedReadParams& p, hipStream_t st) {
  KTimer t("paged_read_fp8", st);
  if (p.D == 64) hipLaunchKernelGGL(paged_read_kernel<64>, dim3(p.N), dim3(256), 0, st, p);
  else hipLaunchKernelGGL(paged_read_kernel<128>, dim3(p.N), dim3(256), 0, st, p);
  return hipGetLastError();
}

}  // namespace alg
