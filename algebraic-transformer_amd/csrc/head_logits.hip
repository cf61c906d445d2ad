// Logits of the tied head, z = h E^T (src/algebraic/model.py:225-230 without the likelihood), summed and written in
// f32. For the tokens of a serving step reading E bounds it, for many the products of gemm_core.h.
//
// Few tokens (and f32): a wave takes 16 rows of E and up to 64 tokens. E goes from memory to registers in
// its own order, 128 bytes of each row at a time (16x16 MFMA, A = E; lane group g holds 16-byte pieces g and
// g + 4 of the 128, and h is laid out alike), h through LDS, which the workgroup's waves share. Lane l then
// holds four neighbouring logits of token l % 16. 5 tokens, d 2048, V 32000, the table from memory: 29 us, 4.5
// TB/s (22 of two tables in turn, which the last cache holds).
#include <type_traits>

#include "gemm_core.h"
#include "head_logits.h"
#include "launchers.h"

namespace alg {

namespace {

constexpr int LG_WAVES = 8, LG_THREADS = 64 * LG_WAVES;
constexpr int DEPTH = 4;  // steps of 128 bytes a row
constexpr int LG_LDS = 64 * 1024;  // bytes of h in LDS, beside the rows' padding

template <typename T, int NT>
struct LogitsShape {
  static constexpr int TOK = 16 * NT;
  static constexpr int STEP = 128 / (int)sizeof(T);           // elements of a row and step
  static constexpr int KC = LG_LDS / TOK / (int)sizeof(T);    // elements of a row of h that LDS holds
  static constexpr int PITCH = KC * (int)sizeof(T) + 16;      // bytes; 16 rows at one place lie in 16 parts of the banks
};

// One 16-byte piece of 16 rows of E with the same of each token (f32: four products of K = 4 each).
template <typename T, int NT>
__device__ __forceinline__ void logits_mfma(const u32x4& a, const u32x4 (&b)[NT], floatx4 (&c)[NT]) {
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) c[nt] = mfma16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b[nt]), c[nt]);
  } else {
    const floatx4 x = __builtin_bit_cast(floatx4, a);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        c[nt] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], __builtin_bit_cast(floatx4, b[nt])[j], c[nt], 0, 0, 0);
  }
}

}  // namespace

// `kw` of the workgroup's waves (a power of two) share 16 rows of E, each every kw-th step of them, and add up their
// sums at the end, in order: for few rows, which would otherwise leave CUs idle.
template <typename T, int NT>
__global__ __launch_bounds__(LG_THREADS) void head_logits_kernel(HeadLogitsParams p, int kw) {
  typedef LogitsShape<T, NT> S;
  __shared__ __attribute__((aligned(16))) char hs[S::TOK * S::PITCH];
  static_assert(sizeof(hs) >= LG_WAVES * NT * 64 * sizeof(floatx4), "the waves' sums fit h's place");
  const int lane = threadIdx.x & 63, g = lane >> 4, l16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), part = wave & (kw - 1);
  const int n0 = blockIdx.y * S::TOK;
  const int v0 = (blockIdx.x * LG_WAVES + wave) / kw * 16;
  const char* row = static_cast<const char*>(p.e) + (size_t)min(v0 + l16, p.V - 1) * p.d * sizeof(T) + 16 * g;
  const int row_bytes = p.d * (int)sizeof(T);  // of 16-byte pieces
  floatx4 acc[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) acc[nt] = floatx4{};
  // h's piece, PIECE bytes a row, goes through registers: the next one is under way while one is used. Zeros past its
  // end and past the last token.
  constexpr int PIECE = S::KC * (int)sizeof(T), HOLD = S::TOK * PIECE / 16 / LG_THREADS;
  u32x4 hold[HOLD];
  const auto fetch = [&](int k0) {
#pragma unroll
    for (int j = 0; j < HOLD; ++j) {
      const int i = threadIdx.x + j * LG_THREADS, t = i / (PIECE / 16), c = k0 + 16 * (i % (PIECE / 16));
      hold[j] = u32x4{};
      if (n0 + t < p.N && c < row_bytes)
        hold[j] = *reinterpret_cast<const u32x4*>(static_cast<const char*>(p.h) + (size_t)(n0 + t) * row_bytes + c);
    }
  };
  fetch(0);
  for (int k0 = 0; k0 < row_bytes; k0 += PIECE) {
    const int len = min(PIECE, row_bytes - k0), whole = len / 128, steps = (len + 127) / 128;
    const int full = (whole - part + kw - 1) / kw;  // this wave's whole steps: part, part + kw, ...
    const char* from = row + k0 + 128 * part;
    // DEPTH steps of E are always under way, from before h's piece is there.
    u32x4 a[DEPTH][2];
    const auto load = [&](int s, u32x4 (&x)[2]) {
      x[0] = *reinterpret_cast<const u32x4*>(from + 128 * kw * s);
      x[1] = *reinterpret_cast<const u32x4*>(from + 128 * kw * s + 64);
    };
#pragma unroll
    for (int i = 0; i < DEPTH; ++i)
      if (i < full) load(i, a[i]);
    if (k0) __syncthreads();
#pragma unroll
    for (int j = 0; j < HOLD; ++j) {
      const int i = threadIdx.x + j * LG_THREADS;
      *reinterpret_cast<u32x4*>(hs + i / (PIECE / 16) * S::PITCH + 16 * (i % (PIECE / 16))) = hold[j];
    }
    __syncthreads();
    if (k0 + PIECE < row_bytes) fetch(k0 + PIECE);
    const char* B = hs + l16 * S::PITCH + 16 * g + 128 * part;
    const auto multiply = [&](int s, const u32x4 (&x)[2]) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        u32x4 b[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) b[nt] = *reinterpret_cast<const u32x4*>(B + 16 * nt * S::PITCH + 128 * kw * s + 64 * i);
        logits_mfma<T, NT>(x[i], b, acc);
      }
    };
    int s = 0;
    for (; s + 2 * DEPTH <= full; s += DEPTH) {
#pragma unroll
      for (int i = 0; i < DEPTH; ++i) {
        multiply(s + i, a[i]);
        load(s + DEPTH + i, a[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < DEPTH; ++i)
      if (s + i < full) multiply(s + i, a[i]);
    for (s += DEPTH; s < full; ++s) {
      u32x4 x[2];
      load(s, x);
      multiply(s, x);
    }
    if (whole < steps && (whole & (kw - 1)) == part) {  // the end of a row
      u32x4 x[2] = {};
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (128 * whole + 64 * i + 16 * g < len) x[i] = *reinterpret_cast<const u32x4*>(row + k0 + 128 * whole + 64 * i);
      multiply(full, x);
    }
  }
  if (kw > 1) {
    floatx4* sums = reinterpret_cast<floatx4*>(hs);
    __syncthreads();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) sums[(wave * NT + nt) * 64 + lane] = acc[nt];
    __syncthreads();
    if (part) return;
    for (int w = 1; w < kw; ++w)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) acc[nt] += sums[((wave + w) * NT + nt) * 64 + lane];
  }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int n = n0 + 16 * nt + l16, v = v0 + 4 * g;
    if (n >= p.N) continue;
    float* z = p.z + (size_t)n * p.V + v;
    if (v + 4 <= p.V) {
      __builtin_memcpy(z, &acc[nt], 16);  // rows start anywhere
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (v + i < p.V) z[i] = acc[nt][i];
    }
  }
}

// Many tokens, bf16: the products of gemm_core.h, rows of C tokens, columns the vocabulary, so that a store
// instruction writes two rows' 128 bytes. Each XCD's share of the tiles is compact. 509 tokens, d 768, V 50257: 55 us,
// 394 tiles in two rounds of which the second is half full, matrix cores 44 % busy.
template <class C>
__global__ __launch_bounds__(C::THREADS, 2) void head_logits_gemm_kernel(HeadLogitsParams p) {
  int tv, tn;
  xcd_tile(blockIdx.x, (p.V + C::TN - 1) / C::TN, (p.N + C::TM - 1) / C::TM, tv, tn);
  const int m0 = tn * C::TM, n0 = tv * C::TN;  // tokens, vocabulary
  const GemmOperand A{static_cast<const bf16*>(p.h), p.d, p.N, p.d, (long)p.N * p.d};
  const GemmOperand B{static_cast<const bf16*>(p.e), p.d, p.V, p.d, (long)p.V * p.d};
  floatx16 acc[C::MB][C::NB];
  gemm_tile<KMAJOR, KMAJOR, C>(A, B, m0, n0, 0, p.d, acc);
  const int lane = threadIdx.x & 63, h = lane >> 5, l32 = lane & 31;
  int wm, wn;
  wave_coords<C>(wm, wn);
  const int mw = m0 + wm * C::WTM, nw = n0 + wn * C::WTN + l32;
  float* z = p.z + (size_t)mw * p.V + nw;
#pragma unroll
  for (int mb = 0; mb < C::MB; ++mb)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int row = mb * 32 + 8 * (i >> 2) + 4 * h + (i & 3);
#pragma unroll
      for (int nb = 0; nb < C::NB; ++nb)
        if (mw + row < p.N && nw + nb * 32 < p.V) z[(size_t)row * p.V + nb * 32] = acc[mb][nb][i];
    }
}

template <typename T, int NT>
static void launch_logits(const HeadLogitsParams& p, hipStream_t st) {
  const int blocks = (p.V + 15) / 16, tiles = (p.N + 16 * NT - 1) / (16 * NT);
  int kw = 1;
  while (kw < LG_WAVES && 2L * blocks * tiles * kw <= 256 * LG_WAVES) kw *= 2;
  hipLaunchKernelGGL((head_logits_kernel<T, NT>), dim3((blocks * kw + LG_WAVES - 1) / LG_WAVES, tiles), dim3(LG_THREADS), 0, st, p, kw);
}
template <class C>
static void launch_logits_gemm(const HeadLogitsParams& p, hipStream_t st) {
  const dim3 grid(((p.V + C::TN - 1) / C::TN) * ((p.N + C::TM - 1) / C::TM));
  hipLaunchKernelGGL(head_logits_gemm_kernel<C>, grid, dim3(C::THREADS), 0, st, p);
}

// bf16: a wave's rows of E up to 16 tokens, and where the rows are so few that waves share them; else the tiles of the
// least gemm_tile_time (launchers.h). us for rows of E / tiles of 64 / 128 / 256, the table not in a cache: d 2048, V
// 32000: 5 tokens 28 28 34 56, 64 tokens 42 30 35 57, 128 tokens 55 43 37 58, 509 tokens 197 132 125 68; d
// 768, V 50257: 5 tokens 17 19 28 26, 64 tokens 23 22 28 28, 509 tokens 135 96 90 63. Rows of E shared, and the
// tiles' best: d 2048, V 2000: 32 tokens 8 16, 128 tokens 9 16; V 4000: 64 tokens 11 16, 128 tokens 13 17; V 8000: 32
// tokens 9 16, 64 tokens 13 11, 128 tokens 20 11; V 16000: 32 tokens 15 17, 64 tokens 20 13. f32: rows of
// E always (64 tokens, d 2048, V 32000: 86 us; 300 tokens 395, of which the matrix cores' rate makes 254).
hipError_t launch_head_logits(const HeadLogitsParams& p, hipStream_t st) {
  KTimer t("head_logits", st);
  const long blocks = (p.V + 15) / 16 * ((p.N + 63) / 64);
  const auto rows = [&](auto type) {
    typedef decltype(type) T;
    if (p.N <= 16) launch_logits<T, 1>(p, st);
    else if (p.N <= 32) launch_logits<T, 2>(p, st);
    else launch_logits<T, 4>(p, st);
  };
  if (!p.bf16_in) {
    rows(float{});
  } else if (p.N <= 16 || blocks <= (p.N <= 32 ? 1024 : 512)) {
    rows(bf16{});
  } else {
    const auto time = [&](int tile) {
      return gemm_tile_time(tile, ((p.V + tile - 1) / tile) * ((p.N + tile - 1) / tile), p.d, p.N, p.V);
    };
    const double t64 = time(64), t128 = time(128), t256 = time(256);
    if (t64 <= t128 && t64 <= t256) launch_logits_gemm<GemmCfg<64, 64, 2, 2>>(p, st);
    else if (t128 <= t256) launch_logits_gemm<GemmCfg<128, 128, 2, 2>>(p, st);
    else launch_logits_gemm<HeadGemm>(p, st);
  }
  return hipGetLastError();
}

}  // namespace alg
