// Tokens drawn from the algebraic likelihood of a row of logits (src/algebraic/algebraic.py:223-265: p is
// proportional to rho(x)^n, x = min(z / c, X)), with temperature (rho^(n / T)), top-k, top-p and min-p, from a
// given uniform number.
//
// Which token a number selects depends on sums over the vocabulary to their last bits wherever the number lies
// next to a border, and V = 32000 borders lie everywhere. So the weights are f64, relative to the
// row's largest, and are summed as whole numbers of 2^-bits (2^62 / V): such sums are equal in any order,
// among any number of lanes and atomics, and a row's token depends on its inputs alone.
//
// Order: logits falling, equal ones by their index. The kept tokens are a prefix of it, so that a pair (key, last
// index of that key) says which: `Prefix`. Top-k and top-p ask for the shortest prefix that sums to something (a
// count, a mass). select() finds it without sorting: a histogram over 2048 ranges of the logits, the
// range where the sum is reached, and if that holds few tokens their exact ranks, else a histogram of its
// keys' bits (at most three more); tokens of one single logit are counted.
//
// One workgroup a row, 16 waves. A lane takes four neighbouring tokens of a tile of 4096, so that a wave's
// tokens are neighbours and the draw needs the sums of waves, then of one wave's lanes.
#include <hip/hip_runtime.h>

#include "common.h"
#include "head_sample.h"
#include "launchers.h"

namespace alg {

namespace {

typedef unsigned long long u64;
constexpr int SAMPLE_THREADS = 1024, SAMPLE_WAVES = SAMPLE_THREADS / 64;
constexpr int SAMPLE_TILE = 4 * SAMPLE_THREADS;  // tokens of a tile
constexpr int SAMPLE_TILES = 256;                // tiles of the largest vocabulary
constexpr int SAMPLE_BINS = 2048;
constexpr int SAMPLE_LIST = 1024;                // tokens that are ranked one against the other
constexpr unsigned KEY_CLAMPED = 0xFF800000u;    // +infinity's: a logit at the clamp or above

// Logits as whole numbers of the same order; 0: no token (a logit of -infinity, or none).
__device__ __forceinline__ unsigned logit_key(float z, float z_clamp) {
  if (z >= z_clamp) return KEY_CLAMPED;
  const unsigned b = __builtin_bit_cast(unsigned, z + 0.0f);  // one zero
  if (b >= 0xFF800000u) return 0;  // -infinity (and NaN of that sign, which the caller has seen)
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_logit(unsigned k) {
  return __builtin_bit_cast(float, k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

__device__ __forceinline__ u64 wave_sum(u64 v) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m, 64);
  return v;
}

struct Prefix {
  unsigned key;
  int last;
};
__device__ __forceinline__ bool in_prefix(const Prefix& p, unsigned key, int i) {
  return key > p.key || (key == p.key && i <= p.last);
}

struct SampleShared {
  u64 bins[SAMPLE_BINS];
  u64 list[SAMPLE_LIST];  // key, and the index's complement: falling order
  u64 value[SAMPLE_LIST];
  u64 tile[SAMPLE_TILES][SAMPLE_WAVES];
  u64 wave[SAMPLE_WAVES];
  unsigned lo, hi, count;
  int bin;
  u64 above;
  Prefix found;
};

template <typename T>
struct Sampler {
  const HeadSampleParams& p;
  SampleShared& s;
  const T* row;
  int tid, lane, wave, tiles;
  unsigned top;          // the largest logit's key
  double power, log_top;  // n / T, log2 rho of the largest

  __device__ Sampler(const HeadSampleParams& p_, SampleShared& s_)
      : p(p_), s(s_), row(static_cast<const T*>(p_.z) + (size_t)blockIdx.x * p_.stride), tid(threadIdx.x),
        lane(threadIdx.x & 63), wave(threadIdx.x >> 6), tiles((p_.V + SAMPLE_TILE - 1) / SAMPLE_TILE) {}

  __device__ __forceinline__ int first(int t) const { return t * SAMPLE_TILE + 4 * tid; }
  __device__ __forceinline__ void logits(int t, float (&z)[4]) const {
    const int i = first(t);
    if (p.vec && i + 4 <= p.V) {
      if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(z) = *reinterpret_cast<const float4*>(row + i);
      } else {
        const bf16x4 v = *reinterpret_cast<const bf16x4*>(row + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) z[e] = (float)v[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) z[e] = i + e < p.V ? (float)row[i + e] : -INFINITY;
    }
  }
  __device__ __forceinline__ void keys(int t, unsigned (&k)[4]) const {
    float z[4];
    logits(t, z);
#pragma unroll
    for (int e = 0; e < 4; ++e) k[e] = logit_key(z[e], p.z_clamp);
  }
  // f(key, token) for every token that the prefix holds.
  template <typename F>
  __device__ __forceinline__ void each(const Prefix& in, F f) const {
    for (int t = 0; t < tiles; ++t) {
      unsigned k[4];
      keys(t, k);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (k[e] != 0 && in_prefix(in, k[e], first(t) + e)) f(k[e], first(t) + e);
    }
  }

  __device__ __forceinline__ double log2_rho(unsigned key) const {
    const double x = key == KEY_CLAMPED ? p.clamp : (double)key_logit(key) * p.inv_c, a = fabs(x);
    return copysign(log2(a + sqrt(1.0 + a * a)), x);
  }
  __device__ __forceinline__ double weight(unsigned key) const { return exp2(power * (log2_rho(key) - log_top)); }
  __device__ __forceinline__ u64 mass(unsigned key) const { return (u64)rint(ldexp(weight(key), p.bits)); }

  // The workgroup's sum.
  __device__ u64 total(u64 v) {
    v = wave_sum(v);
    __syncthreads();
    if (lane == 0) s.wave[wave] = v;
    __syncthreads();
    u64 sum = 0;
    for (int w = 0; w < SAMPLE_WAVES; ++w) sum += s.wave[w];
    return sum;
  }
  // The sum over the lanes up to this one's.
  __device__ u64 scan(u64 v) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      const u64 below = __shfl_up(v, m, 64);
      if (lane >= m) v += below;
    }
    __syncthreads();
    if (lane == 63) s.wave[wave] = v;
    __syncthreads();
    for (int w = 0; w < wave; ++w) v += s.wave[w];
    return v;
  }

  // The token at which the running sum of value(key, i), over tokens by their index, first passes `target`
  // (less than the whole sum).
  template <typename F>
  __device__ int draw(u64 target, F value) {
    for (int t = 0; t < tiles; ++t) {
      unsigned k[4];
      keys(t, k);
      u64 v = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) v += value(k[e], first(t) + e);
      v = wave_sum(v);
      if (lane == 0) s.tile[t][wave] = v;
    }
    __syncthreads();
    int t = 0, w = 0;
    u64 below = 0;
    for (; t < tiles; ++t) {
      u64 sum = 0;
      for (int i = 0; i < SAMPLE_WAVES; ++i) sum += s.tile[t][i];
      if (below + sum > target || t == tiles - 1) break;
      below += sum;
    }
    for (; w < SAMPLE_WAVES - 1; ++w) {
      if (below + s.tile[t][w] > target) break;
      below += s.tile[t][w];
    }
    if (wave == w) {
      unsigned k[4];
      keys(t, k);
      u64 v[4], sum = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) sum += v[e] = value(k[e], first(t) + e);
      u64 upto = sum;
#pragma unroll
      for (int m = 1; m < 64; m <<= 1) {
        const u64 x = __shfl_up(upto, m, 64);
        if (lane >= m) upto += x;
      }
      below += upto - sum;  // up to this lane's tokens
      if (below <= target && below + sum > target) {
        int e = 0;
        while (below + v[e] <= target) below += v[e++];
        s.found.last = first(t) + e;
      }
    }
    __syncthreads();
    const int got = s.found.last;
    __syncthreads();
    return got;
  }

  // The shortest prefix, within `in`, whose values sum to `need` (at least 1, at most their sum).
  template <typename F>
  __device__ Prefix select(const Prefix& in, u64 need, F value) {
    unsigned lo = 0, hi = top;
    u64 above = 0;
    // First by ranges of the logits themselves (a monotone function of the key, whatever it rounds), of 1/64 of
    // the scale or as wide as 2048 of them have to be.
    const float z_top = top == KEY_CLAMPED ? p.z_clamp : key_logit(top);
    const float z_step = (float)(64.0 * p.inv_c);
    for (int round = 0;; ++round) {
      const int shift = max(0, 21 - (int)__builtin_clz((hi - lo) | 1u));  // (hi - lo) >> shift < 2048
      const auto bin = [&](unsigned k) {
        if (round == 0) return (int)fminf((z_top - (k == KEY_CLAMPED ? p.z_clamp : key_logit(k))) * z_step, SAMPLE_BINS - 1.0f);
        return (int)((hi - k) >> shift);
      };
      __syncthreads();
      for (int i = tid; i < SAMPLE_BINS; i += SAMPLE_THREADS) s.bins[i] = 0;
      if (tid == 0) {
        s.lo = 0xFFFFFFFFu;
        s.hi = s.count = 0;
      }
      __syncthreads();
      each(in, [&](unsigned k, int i) {
        if (k >= lo && k <= hi) atomicAdd(&s.bins[bin(k)], value(k, i));
      });
      __syncthreads();
      const u64 a = s.bins[2 * tid], b = s.bins[2 * tid + 1];
      const u64 upto = above + scan(a + b);
      const u64 before = upto - a - b;
      if (before < need && before + a >= need) {
        s.bin = 2 * tid;
        s.above = before;
      } else if (before + a < need && upto >= need) {
        s.bin = 2 * tid + 1;
        s.above = before + a;
      }
      __syncthreads();
      const int at = s.bin;
      above = s.above;
      // The tokens of that range: into the list, as many as it holds, with their extremes.
      each(in, [&](unsigned k, int i) {
        if (k < lo || k > hi || bin(k) != at) return;
        const unsigned n = atomicAdd(&s.count, 1u);
        atomicMin(&s.lo, k);
        atomicMax(&s.hi, k);
        if (n < SAMPLE_LIST) {
          s.list[n] = (u64)k << 32 | (unsigned)~i;
          s.value[n] = value(k, i);
        }
      });
      __syncthreads();
      const int count = (int)s.count;
      lo = s.lo;
      hi = s.hi;
      if (count <= SAMPLE_LIST) {
        if (tid < count) {
          const u64 mine = s.list[tid];
          u64 sum = above;
          for (int i = 0; i < count; ++i)
            if (s.list[i] > mine) sum += s.value[i];
          if (sum < need && sum + s.value[tid] >= need) s.found = Prefix{(unsigned)(mine >> 32), (int)~(unsigned)mine};
        }
        __syncthreads();
        const Prefix got = s.found;
        __syncthreads();
        return got;
      }
      if (lo == hi) {  // one logit: as many of its tokens as it takes
        const u64 each_one = value(lo, 0), wanted = (need - above + each_one - 1) / each_one;
        const int last = draw(wanted - 1, [&](unsigned k, int i) { return (u64)(k == lo && in_prefix(in, k, i)); });
        return Prefix{lo, last};
      }
    }
  }

  __device__ void run() {
    const int r = blockIdx.x;
    const float temperature = p.temperature ? p.temperature[r] : p.temperature_all;
    const float top_p = p.top_p ? p.top_p[r] : p.top_p_all;
    const float least = p.min_p ? p.min_p[r] : p.min_p_all;
    const double min_p = least > 0.0f ? fminf(least, 1.0f) : 0.0f;  // the likeliest token stays
    const int top_k = p.top_k ? p.top_k[r] : p.top_k_all;
    // The largest logit, its first token, and whether one is NaN.
    u64 best = 0;
    bool nan = false;
    for (int t = 0; t < tiles; ++t) {
      float z[4];
      logits(t, z);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        nan |= z[e] != z[e];
        const u64 c = (u64)logit_key(z[e], p.z_clamp) << 32 | (unsigned)~(first(t) + e);
        if (c > best) best = c;
      }
    }
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      const u64 o = __shfl_xor(best, m, 64);
      if (o > best) best = o;
    }
    if (lane == 0) s.wave[wave] = best;
    nan = __syncthreads_or(nan) != 0;
    for (int w = 0; w < SAMPLE_WAVES; ++w)
      if (s.wave[w] > best) best = s.wave[w];
    __syncthreads();
    top = (unsigned)(best >> 32);
    if (nan || top == 0 || !(temperature >= 0.0f)) {
      if (tid == 0) {
        p.token[r] = -1;
        p.logprob[r] = __builtin_nanf("");
      }
      return;
    }
    if (temperature == 0.0f) {
      if (tid == 0) {
        p.token[r] = (int)~(unsigned)best;
        p.logprob[r] = 0.0f;
      }
      return;
    }
    power = p.n / (double)temperature;
    log_top = log2_rho(top);
    Prefix in{0, p.V};
    if (top_k > 0 && top_k < p.V) {
      u64 tokens = 0;
      each(in, [&](unsigned, int) { ++tokens; });
      if ((u64)top_k < total(tokens)) in = select(in, top_k, [](unsigned, int) { return (u64)1; });
    }
    if (top_p < 1.0f) {
      u64 m = 0;
      each(in, [&](unsigned k, int) { m += mass(k); });
      const double want = ceil((double)top_p * (double)total(m));
      in = select(in, want >= 1.0 ? (u64)want : 1, [&](unsigned k, int) { return mass(k); });
    }
    const auto kept = [&](unsigned k, int i) {
      if (k == 0 || !in_prefix(in, k, i)) return (u64)0;
      const double w = weight(k);
      return w >= min_p ? (u64)rint(ldexp(w, p.bits)) : (u64)0;
    };
    u64 m = 0;
    each(in, [&](unsigned k, int i) { m += kept(k, i); });
    const u64 whole = total(m);
    double u = p.u_f64 ? static_cast<const double*>(p.u)[r] : (double)static_cast<const float*>(p.u)[r];
    u = u >= 0.0 ? u : 0.0;  // NaN too
    const double at = floor(u * (double)whole);
    const u64 target = at < (double)whole ? min((u64)at, whole - 1) : whole - 1;
    const int token = draw(target, kept);
    if (tid == 0) {
      p.token[r] = token;
      const unsigned k = logit_key((float)row[token], p.z_clamp);
      p.logprob[r] = (float)log((double)kept(k, token) / (double)whole);
    }
  }
};

}  // namespace

template <typename T>
__global__ __launch_bounds__(SAMPLE_THREADS) void head_sample_kernel(HeadSampleParams p) {
  __shared__ SampleShared s;
  Sampler<T>(p, s).run();
}

hipError_t launch_head_sample(const HeadSampleParams& p, hipStream_t st) {
  KTimer t("head_sample", st);
  if (p.z_bf16) hipLaunchKernelGGL(head_sample_kernel<bf16>, dim3(p.N), dim3(SAMPLE_THREADS), 0, st, p);
  else hipLaunchKernelGGL(head_sample_kernel<float>, dim3(p.N), dim3(SAMPLE_THREADS), 0, st, p);
  return hipGetLastError();
}

}  // namespace alg
