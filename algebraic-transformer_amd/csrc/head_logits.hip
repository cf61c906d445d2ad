// Logits of the tied head, z = h E^T (src/algebraic/model.py:225-230 without the likelihood), summed and written in
// f32, for the tokens of a serving step: E is read once and bounds it.
//
// A wave takes 16 rows of E and up to 64 tokens: E goes from memory to registers in its own order, 128 bytes
// of each row at a time (16x16 MFMA, A = E; lane group g holds 16-byte pieces g and g + 4 of the 128, and h
// is laid out alike), h through LDS, which the workgroup's waves share. Lane l then holds four neighbouring
// logits of token l % 16.
#include <type_traits>

#include "common.h"
#include "head_logits.h"
#include "launchers.h"

namespace alg {

namespace {

constexpr int LG_WAVES = 8, LG_THREADS = 64 * LG_WAVES;
constexpr int LG_LDS = 64 * 1024;  // bytes of h in LDS, beside the rows' padding

template <typename T, int NT>
struct LogitsShape {
  static constexpr int TOK = 16 * NT;
  static constexpr int STEP = 128 / (int)sizeof(T);           // elements of a row and step
  static constexpr int KC = LG_LDS / TOK / (int)sizeof(T);    // elements of a row of h that LDS holds
  static constexpr int PITCH = KC * (int)sizeof(T) + 16;      // bytes; 16 rows at one place lie in 16 parts of the banks
};

template <typename T>
__device__ __forceinline__ floatx4 logits_mfma(const u32x4& a, const u32x4& b, floatx4 c) {
  if constexpr (sizeof(T) == 2) {
    return mfma16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c);
  } else {
    const floatx4 x = __builtin_bit_cast(floatx4, a), y = __builtin_bit_cast(floatx4, b);
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], y[j], c, 0, 0, 0);
    return c;
  }
}

}  // namespace

template <typename T, int NT>
__global__ __launch_bounds__(LG_THREADS) void head_logits_kernel(HeadLogitsParams p) {
  typedef LogitsShape<T, NT> S;
  __shared__ __attribute__((aligned(16))) char hs[S::TOK * S::PITCH];
  const int lane = threadIdx.x & 63, g = lane >> 4, l16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = blockIdx.y * S::TOK;
  const int v0 = (blockIdx.x * LG_WAVES + wave) * 16;
  const char* row = static_cast<const char*>(p.e) + (size_t)min(v0 + l16, p.V - 1) * p.d * sizeof(T) + 16 * g;
  const int row_bytes = p.d * (int)sizeof(T);  // of 16-byte pieces
  floatx4 acc[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) acc[nt] = floatx4{};
  for (int k0 = 0; k0 < row_bytes; k0 += S::KC * (int)sizeof(T)) {
    const int len = min(S::KC * (int)sizeof(T), row_bytes - k0);
    const int steps = (len + 127) / 128;
    if (k0) __syncthreads();
    // h's piece, zeros past its end and past the last token.
    for (int i = threadIdx.x; i < S::TOK * 8 * steps; i += LG_THREADS) {
      const int t = i / (8 * steps), c = 16 * (i - t * 8 * steps);
      u32x4 x = {};
      if (n0 + t < p.N && c < len)
        x = *reinterpret_cast<const u32x4*>(static_cast<const char*>(p.h) + (size_t)(n0 + t) * row_bytes + k0 + c);
      *reinterpret_cast<u32x4*>(hs + t * S::PITCH + c) = x;
    }
    __syncthreads();
    const char* B = hs + l16 * S::PITCH + 16 * g;
    for (int s = 0; s < steps; ++s) {
      u32x4 a[2] = {};
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (128 * s + 64 * i + 16 * g < len) a[i] = *reinterpret_cast<const u32x4*>(row + k0 + 128 * s + 64 * i);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          acc[nt] = logits_mfma<T>(a[i], *reinterpret_cast<const u32x4*>(B + 16 * nt * S::PITCH + 128 * s + 64 * i), acc[nt]);
    }
  }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int n = n0 + 16 * nt + l16, v = v0 + 4 * g;
    if (n >= p.N) continue;
    float* z = p.z + (size_t)n * p.V + v;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (v + i < p.V) z[i] = acc[nt][i];
  }
}

template <typename T>
static void launch_logits(const HeadLogitsParams& p, hipStream_t st) {
  const int rows = LG_WAVES * 16;
  const auto grid = [&](int tokens) { return dim3((p.V + rows - 1) / rows, (p.N + tokens - 1) / tokens); };
  if (p.N <= 16) hipLaunchKernelGGL((head_logits_kernel<T, 1>), grid(16), dim3(LG_THREADS), 0, st, p);
  else if (p.N <= 32) hipLaunchKernelGGL((head_logits_kernel<T, 2>), grid(32), dim3(LG_THREADS), 0, st, p);
  else hipLaunchKernelGGL((head_logits_kernel<T, 4>), grid(64), dim3(LG_THREADS), 0, st, p);
}

hipError_t launch_head_logits(const HeadLogitsParams& p, hipStream_t st) {
  KTimer t("head_logits", st);
  if (p.bf16_in) launch_logits<bf16>(p, st);
  else launch_logits<float>(p, st);
  return hipGetLastError();
}

}  // namespace alg
