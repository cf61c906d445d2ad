// Tokens drawn from the algebraic likelihood of a row of logits (src/algebraic/algebraic.py:223-265: p is
// proportional to rho(x)^n, x = min(z / c, X)), with temperature (rho^(n / T)), top-k, top-p and min-p, from a
// given uniform number.
//
// Which token a number selects depends on sums over the vocabulary to their last bits wherever the number lies
// next to a border, and V = 32000 borders lie everywhere. So the weights are f64, relative to the
// row's largest (to 2^-40 or better), and are summed as whole numbers of 2^-bits (2^62 / V): such sums are
// equal in any order, among any number of lanes and atomics, and a row's token depends on the row alone.
//
// Order: logits falling, equal ones by their index. The kept tokens are a prefix of it. Where a
// histogram over 2048 ranges of the logits (by count for top-k, by weight for top-p) says that no more than
// 1024 tokens can be in it, those are sorted in LDS and everything else happens among them. Otherwise
// the prefix is a pair (key, last index of that key), found without sorting: the exact ranks within the range
// where the sum is reached, or if that is crowded too, histograms of its keys' bits (at most three more);
// tokens of one single logit are counted.
//
// One workgroup a row, 16 waves. A lane takes four neighbouring tokens of a tile of 4096, so that a wave's
// tokens are neighbours and a draw among all tokens needs the sums of waves, then of one wave's lanes.
#include <hip/hip_runtime.h>

#include "common.h"
#include "head_sample.h"
#include "launchers.h"

namespace alg {

namespace {

typedef unsigned long long u64;
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

struct Prefix {
  unsigned key;
  int last;
};
__device__ __forceinline__ bool in_prefix(const Prefix& p, unsigned key, int i) {
  return key > p.key || (key == p.key && i <= p.last);
}

struct SampleShared {
  u64 bins[SAMPLE_BINS];
  int counts[SAMPLE_BINS];
  u64 list[SAMPLE_LIST];  // key, and the index's complement: falling order
  u64 value[SAMPLE_LIST];
  u64 tile[SAMPLE_TILES][SAMPLE_WAVES];
  double2 logs[128];  // 1 / m and -log2 of that, m the middles of [1, 2)'s 128 parts
  double exps[64];    // 2^(i / 64)
  u64 wave[SAMPLE_WAVES];
  unsigned lo, hi, count;
  int bin, upto;
  u64 above;
  Prefix found;
};

// READY: the row's best, and the histogram or sums that it needs first, are there.
template <typename T, bool READY>
struct Sampler {
  const HeadSampleParams& p;
  SampleShared& s;
  const int r;  // the row
  const T* row;
  int tid, lane, wave, tiles;
  unsigned top;             // the largest logit's key
  double power, log_top;    // n / temperature, log2 rho of the largest

  // The row's settings.
  float temperature, top_p;
  double floor_v;  // the least weight kept, times 2^bits
  int top_k;
  bool cut_k, cut_p;

  __device__ Sampler(const HeadSampleParams& p_, SampleShared& s_, int r_)
      : p(p_), s(s_), r(r_), row(static_cast<const T*>(p_.z) + (size_t)r_ * p_.stride), tid(threadIdx.x),
        lane(threadIdx.x & 63), wave(threadIdx.x >> 6), tiles((p_.V + SAMPLE_TILE - 1) / SAMPLE_TILE) {
    temperature = p.temperature ? p.temperature[r] : p.temperature_all;
    top_p = p.top_p ? p.top_p[r] : p.top_p_all;
    top_k = p.top_k ? p.top_k[r] : p.top_k_all;
    const float least = p.min_p ? p.min_p[r] : p.min_p_all;
    floor_v = __builtin_amdgcn_ldexp(least > 0.0f ? (double)fminf(least, 1.0f) : 0.0, p.bits);  // the likeliest token stays
    cut_k = top_k > 0 && top_k < p.V;
    cut_p = top_p < 1.0f;
  }

  __device__ __forceinline__ int first(int t) const { return t * SAMPLE_TILE + 4 * tid; }
  // A lane's four tokens of a tile; none past the row's end. Rows start anywhere.
  __device__ __forceinline__ void logits(int t, T (&z)[4]) const {
    const int i = first(t);
    if (i + 4 <= p.V) {
      __builtin_memcpy(z, row + i, sizeof z);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) z[e] = i + e < p.V ? row[i + e] : (T)-INFINITY;
    }
  }
  // f(logit, token) for every token, the next tiles' loads under way.
  template <typename F>
  __device__ __forceinline__ void sweep(F f) const {
    T z[2][4];
    logits(0, z[0]);
    if (tiles > 1) logits(1, z[1]);
    for (int t = 0; t < tiles; ++t) {
      T now[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        now[e] = z[0][e];
        z[0][e] = z[1][e];
      }
      if (t + 2 < tiles) logits(t + 2, z[1]);
#pragma unroll
      for (int e = 0; e < 4; ++e) f((float)now[e], first(t) + e);
    }
  }
  // f(key, token) for every token that the prefix holds.
  template <typename F>
  __device__ __forceinline__ void each(const Prefix& in, F f) const {
    sweep([&](float z, int i) {
      const unsigned k = logit_key(z, p.z_clamp);
      if (k != 0 && in_prefix(in, k, i)) f(k, i);
    });
  }

  // log2 rho(x), to 2^-43: |x| + sqrt(1 + x^2) = 2^e m, log2 m from the middle of m's 128th part and five
  // terms of the series. The root is s rsqrt(s), the hardware's with one step of Newton's method.
  __device__ __forceinline__ double log2_rho(unsigned key) const {
    const double x = key == KEY_CLAMPED ? p.clamp : (double)key_logit(key) * p.inv_c, a = __builtin_fabs(x);
    const double q = __builtin_fma(a, a, 1.0), y = __builtin_amdgcn_rsq(q), h = q * y;
    const double r = a + __builtin_fma(0.5 * h, __builtin_fma(-h, y, 1.0), h);
    const u64 b = __builtin_bit_cast(u64, r);
    const int high = (int)(b >> 32);
    const double m = __builtin_bit_cast(double, (b & 0x000FFFFFFFFFFFFFull) | 0x3FF0000000000000ull);
    const double2 part = s.logs[(high >> 13) & 127];
    const double t = __builtin_fma(m, part.x, -1.0);
    constexpr double C = 1.4426950408889634;  // 1 / ln 2
    double poly = __builtin_fma(t, C / 5, -C / 4);
    poly = __builtin_fma(t, poly, C / 3);
    poly = __builtin_fma(t, poly, -C / 2);
    poly = __builtin_fma(t, poly, C);
    const double l = __builtin_fma(t, poly, part.y + (double)((high >> 20) - 1023));
    return x < 0.0 ? -l : l;
  }
  // The weight times 2^bits: 2^d of the nearest 64th below a table's and five terms of the series.
  __device__ __forceinline__ double scaled(unsigned key) const {
    const double d = fmax(power * (log2_rho(key) - log_top), -1000.0), j = __builtin_rint(d * 64.0);
    const double f = __builtin_fma(j, -0.015625, d);
    const int ji = (int)j;
    constexpr double L = 0.6931471805599453;
    double poly = __builtin_fma(f, L * L * L * L * L / 120, L * L * L * L / 24);
    poly = __builtin_fma(f, poly, L * L * L / 6);
    poly = __builtin_fma(f, poly, L * L / 2);
    poly = __builtin_fma(f, poly, L);
    poly = __builtin_fma(f, poly, 1.0);
    return __builtin_amdgcn_ldexp(s.exps[ji & 63] * poly, (ji >> 6) + p.bits);
  }
  static __device__ __forceinline__ u64 whole_part(double v) {
    const unsigned high = (unsigned)(v * 0x1p-32);
    return (u64)high << 32 | (unsigned)__builtin_fma((double)high, -0x1p32, v);
  }
  __device__ __forceinline__ u64 mass(unsigned key) const { return whole_part(scaled(key)); }
  __device__ void tables() {
    if (tid < 128) {
      const double inv = 1.0 / (1.0 + (tid + 0.5) / 128.0);
      s.logs[tid] = make_double2(inv, -log2(inv));
    } else if (tid < 192) {
      s.exps[tid - 128] = exp2((tid - 128) / 64.0);
    }
  }

  // The sum over the lanes up to this one's, and over all.
  __device__ u64 scan(u64 v, u64& total) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      const u64 below = __shfl_up(v, m, 64);
      if (lane >= m) v += below;
    }
    __syncthreads();
    if (lane == 63) s.wave[wave] = v;
    __syncthreads();
    total = 0;
#pragma unroll
    for (int w = 0; w < SAMPLE_WAVES; ++w) {
      if (w == wave) v += total;
      total += s.wave[w];
    }
    return v;
  }

  // The lanes' numbers in falling order, a lane each; `size` a power of two, the lanes from there on hold 0.
  template <typename K>
  __device__ K sorted(K v, int size) {
    K* buf = reinterpret_cast<K*>(s.bins);
    for (int block = 2; block <= size; block <<= 1)
      for (int step = block >> 1; step > 0; step >>= 1) {
        K o;
        if (step < 64) {
          o = __shfl_xor(v, step, 64);
        } else {
          __syncthreads();
          buf[tid] = v;
          __syncthreads();
          o = buf[tid ^ step];
        }
        v = ((tid & step) == 0) == ((tid & block) == 0) ? max(v, o) : min(v, o);
      }
    return v;
  }

  // The sum of value(key, i) over all tokens, which pick() then draws from.
  template <typename F>
  __device__ u64 sums(F value) {
    T z[4];
    logits(0, z);
    for (int t = 0; t < tiles; ++t) {
      T now[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) now[e] = z[e];
      if (t + 1 < tiles) logits(t + 1, z);
      u64 v = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) v += value(logit_key((float)now[e], p.z_clamp), first(t) + e);
#pragma unroll
      for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m, 64);
      if (lane == 0) s.tile[t][wave] = v;
    }
    __syncthreads();
    u64 v = 0, total;
    for (int i = tid; i < tiles * SAMPLE_WAVES; i += SAMPLE_THREADS) v += (&s.tile[0][0])[i];
    scan(v, total);
    return total;
  }
  // The token at which the running sum, over tokens by their index, first passes `target` (less than the sum).
  template <typename F>
  __device__ int pick(u64 target, F value) {
    int t = 0, w = 0;
    u64 below = 0;
    for (; t < tiles - 1; ++t) {
      u64 sum = 0;
#pragma unroll
      for (int i = 0; i < SAMPLE_WAVES; ++i) sum += s.tile[t][i];
      if (below + sum > target) break;
      below += sum;
    }
    for (; w < SAMPLE_WAVES - 1; ++w) {
      if (below + s.tile[t][w] > target) break;
      below += s.tile[t][w];
    }
    if (wave == w) {
      T z[4];
      logits(t, z);
      u64 v[4], sum = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) sum += v[e] = value(logit_key((float)z[e], p.z_clamp), first(t) + e);
      u64 upto = sum;
#pragma unroll
      for (int m = 1; m < 64; m <<= 1) {
        const u64 x = __shfl_up(upto, m, 64);
        if (lane >= m) upto += x;
      }
      below += upto - sum;  // up to this lane's tokens
      if (below <= target && below + sum > target) {
        int last = first(t);
#pragma unroll
        for (int e = 0; e < 3; ++e) {
          below += v[e];
          last += below <= target;
        }
        s.found.last = last;
      }
    }
    __syncthreads();
    const int got = s.found.last;
    __syncthreads();
    return got;
  }

  // The first histogram's ranges, of the logits themselves, of 1/64 of the scale: a monotone function of the key,
  // whatever it rounds.
  __device__ __forceinline__ int first_bin(unsigned k) const {
    const float z_top = top == KEY_CLAMPED ? p.z_clamp : key_logit(top), z = k == KEY_CLAMPED ? p.z_clamp : key_logit(k);
    return (int)fminf((z_top - z) * (float)(64.0 * p.inv_c), SAMPLE_BINS - 1.0f);
  }

  // The shortest prefix, within `in`, of whose tokens' values the sum reaches want(their sum) (at least 1, at most
  // the sum; 0: all of `in`). Either a list of no more than SAMPLE_LIST tokens, sorted, with that prefix among its
  // first (`listed` says how many it has), or `in` itself made shorter (`listed` = 0).
  template <typename F, typename W>
  __device__ void select(Prefix& in, int& listed, u64& need, bool ready, F value, W want) {
    unsigned lo = 0, hi = top;
    u64 above = 0;
    for (int round = 0;; ++round) {
      const int shift = max(0, 21 - (int)__builtin_clz((hi - lo) | 1u));  // (hi - lo) >> shift < 2048
      const auto bin = [&](unsigned k) { return round == 0 ? first_bin(k) : (int)((hi - k) >> shift); };
      const bool have = READY && ready && round == 0;
      __syncthreads();
      for (int i = tid; i < SAMPLE_BINS; i += SAMPLE_THREADS) {
        s.bins[i] = have ? p.bins[(size_t)r * SAMPLE_BINS + i] : 0;
        s.counts[i] = have ? p.counts[(size_t)r * SAMPLE_BINS + i] : 0;
      }
      if (tid == 0) {
        s.lo = 0xFFFFFFFFu;
        s.hi = s.count = 0;
      }
      __syncthreads();
      if (!have) {
        each(in, [&](unsigned k, int i) {
          if (k < lo || k > hi) return;
          const int b = bin(k);
          atomicAdd(&s.bins[b], value(k, i));
          atomicAdd(&s.counts[b], 1);
        });
        __syncthreads();
      }
      const u64 a = s.bins[2 * tid], b = s.bins[2 * tid + 1];
      const int ca = s.counts[2 * tid], cb = s.counts[2 * tid + 1];
      u64 total, tokens;
      const u64 upto = above + scan(a + b, total);
      const int held = (int)scan((u64)(ca + cb), tokens);
      if (round == 0) need = want(total);
      if (need == 0) return;
      const u64 before = upto - a - b;
      if (before < need && before + a >= need) {
        s.bin = 2 * tid;
        s.above = before;
        s.upto = held - cb;
      } else if (before + a < need && upto >= need) {
        s.bin = 2 * tid + 1;
        s.above = before + a;
        s.upto = held;
      }
      __syncthreads();
      const int at = s.bin, count = s.counts[at];
      const bool all = round == 0 && s.upto <= SAMPLE_LIST;  // that range's tokens and all above fit the list
      above = s.above;
      each(in, [&](unsigned k, int i) {
        if (k < lo || k > hi) return;
        const int b = bin(k);
        if (b > at || (b < at && !all)) return;
        if (!all) {
          atomicMin(&s.lo, k);
          atomicMax(&s.hi, k);
        }
        const unsigned n = atomicAdd(&s.count, 1u);
        if (n < SAMPLE_LIST) s.list[n] = (u64)k << 32 | (unsigned)~i;
      });
      __syncthreads();
      lo = s.lo;
      hi = s.hi;
      if (all || count <= SAMPLE_LIST) {
        const int n = all ? s.upto : count;
        int size = 64;
        while (size < n) size <<= 1;
        const u64 mine = sorted(tid < n ? s.list[tid] : 0, size);
        __syncthreads();
        s.list[tid] = mine;
        if (all) {
          listed = n;
          __syncthreads();
          return;
        }
        u64 ignored;
        const u64 v = tid < n ? value((unsigned)(mine >> 32), (int)~(unsigned)mine) : 0;
        const u64 sum = above + scan(v, ignored);
        if (sum - v < need && sum >= need) s.found = Prefix{(unsigned)(mine >> 32), (int)~(unsigned)mine};
        __syncthreads();
        in = s.found;
        __syncthreads();
        return;
      }
      if (lo == hi) {  // one logit: as many of its tokens as it takes
        const u64 each_one = value(lo, 0), wanted = (need - above + each_one - 1) / each_one;
        const Prefix from = in;
        const auto it = [&](unsigned k, int i) { return (u64)(k == lo && in_prefix(from, k, i)); };
        sums(it);
        in = Prefix{lo, pick(wanted - 1, it)};
        return;
      }
    }
  }

  __device__ void answer(int token, double logprob) {
    if (tid == 0) {
      p.token[r] = token;
      p.logprob[r] = (float)logprob;
    }
  }

  // The workgroup's largest of the lanes' numbers.
  __device__ u64 largest(u64 c) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) c = max(c, (u64)__shfl_xor(c, m, 64));
    __syncthreads();
    if (lane == 0) s.wave[wave] = c;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < SAMPLE_WAVES; ++w) c = max(c, s.wave[w]);
    return c;
  }
  // The largest logit's key and the complement of its first token, of tiles [begin, end); all ones with a NaN.
  __device__ u64 best(int begin, int end) {
    u64 c = 0;
    for (int t = begin; t < end; ++t) {
      T z[4];
      logits(t, z);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float f = (float)z[e];
        c = max(c, f != f ? ~0ull : (u64)logit_key(f, p.z_clamp) << 32 | (unsigned)~(first(t) + e));
      }
    }
    return largest(c);
  }
  // Takes the row's best; false: it has its answer, or none.
  __device__ bool begin(u64 c) {
    top = (unsigned)(c >> 32);
    if (c == ~0ull || top == 0 || !(temperature >= 0.0f)) {
      answer(-1, __builtin_nan(""));
      return false;
    }
    if (temperature == 0.0f) {
      answer((int)~(unsigned)c, 0.0);
      return false;
    }
    power = p.n / (double)temperature;
    log_top = log2_rho(top);
    return true;
  }
  __device__ __forceinline__ u64 kept(const Prefix& in, unsigned k, int i) const {
    if (k == 0 || !in_prefix(in, k, i)) return 0;
    const double v = scaled(k);
    return v >= floor_v ? whole_part(v) : 0;
  }

  // One tile's share of what the row needs first: the histogram of its cut, or its waves' sums. `s` is clear.
  __device__ void share(int t) {
    T z[4];
    logits(t, z);
    unsigned k[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) k[e] = logit_key((float)z[e], p.z_clamp);
    if (!cut_k && !cut_p) {
      u64 v = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) v += kept(Prefix{0, p.V}, k[e], first(t) + e);
#pragma unroll
      for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m, 64);
      if (lane == 0) p.sums[((size_t)r * tiles + t) * SAMPLE_WAVES + wave] = v;
      return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (k[e] != 0) {
        const int b = first_bin(k[e]);
        atomicAdd(&s.bins[b], cut_k ? (u64)1 : mass(k[e]));
        atomicAdd(&s.counts[b], 1);
      }
    __syncthreads();
    for (int i = tid; i < SAMPLE_BINS; i += SAMPLE_THREADS)
      if (s.counts[i]) {
        atomicAdd(p.bins + (size_t)r * SAMPLE_BINS + i, s.bins[i]);
        atomicAdd(p.counts + (size_t)r * SAMPLE_BINS + i, s.counts[i]);
      }
  }

  __device__ void run() {
    const double u = p.u_f64 ? static_cast<const double*>(p.u)[r] : (double)static_cast<const float*>(p.u)[r];
    tables();
    const u64 c = READY ? largest(tid < tiles ? p.best[(size_t)r * tiles + tid] : 0) : best(0, tiles);
    if (!begin(c)) return;
    Prefix in{0, p.V};
    int listed = 0;
    u64 need = 0;
    if (cut_k)
      select(in, listed, need, true, [](unsigned, int) { return (u64)1; },
             [&](u64 tokens) { return (u64)top_k < tokens ? (u64)top_k : (u64)0; });
    const auto wanted = [&](u64 total) { return max((u64)ceil((double)top_p * (double)total), (u64)1); };
    const int first_k = listed ? top_k : 0;  // of the list
    if (cut_p && !listed) select(in, listed, need, !cut_k, [&](unsigned k, int) { return mass(k); }, wanted);

    // u as a share of `total`, and the tokens that it passes; below 0 or NaN as 0, 1 or more as the largest below.
    const auto target = [&](u64 total) {
      const double at = floor((u >= 0.0 ? u : 0.0) * (double)total);
      return at < (double)total ? min((u64)at, total - 1) : total - 1;
    };
    if (listed) {
      // The list's tokens, a lane each, by falling logit; then the kept ones by their index.
      const u64 mine = s.list[tid];
      const bool is = tid < (first_k ? first_k : listed);
      const double v = is ? scaled((unsigned)(mine >> 32)) : 0.0;
      const u64 m = is ? whole_part(v) : 0;
      u64 total, kept_total;
      const u64 upto = scan(m, total);
      if (first_k) need = cut_p ? wanted(total) : total;
      const bool keep = is && v >= floor_v && (tid == 0 || upto - m < need);
      s.value[tid] = m;
      int size = 64;
      while (size < listed) size <<= 1;
      const unsigned index = ~(unsigned)mine;
      const unsigned by_index = sorted(keep ? ~(index << 10 | (unsigned)tid) : 0u, size);
      __syncthreads();
      const unsigned slot = ~by_index & 1023;
      const u64 w = by_index ? s.value[slot] : 0;
      const u64 sum = scan(w, kept_total), t = target(kept_total);
      if (by_index && sum - w <= t && sum > t) {
        p.token[r] = (int)(~by_index >> 10);
        p.logprob[r] = (float)log((double)w / (double)kept_total);
      }
      return;
    }
    const auto value = [&](unsigned k, int i) { return kept(in, k, i); };
    u64 total;
    if (READY && !cut_k && !cut_p) {
      u64 v = 0;
      for (int i = tid; i < tiles * SAMPLE_WAVES; i += SAMPLE_THREADS)
        v += (&s.tile[0][0])[i] = p.sums[(size_t)r * tiles * SAMPLE_WAVES + i];
      scan(v, total);
    } else {
      total = sums(value);
    }
    const int token = pick(target(total), value);
    answer(token, tid == 0 ? log((double)value(logit_key((float)row[token], p.z_clamp), token) / (double)total) : 0.0);
  }
};

}  // namespace

template <typename T, bool READY>
__global__ __launch_bounds__(SAMPLE_THREADS) void head_sample_kernel(HeadSampleParams p) {
  __shared__ SampleShared s;
  Sampler<T, READY>(p, s, blockIdx.x).run();
}

// Few rows leave most CUs without one, so the passes over a whole row are spread over its tiles, a workgroup each:
// first the largest logit (which clears the row's histogram too), then what share() says. The sums are
// whole numbers: the results are those of one workgroup.
template <typename T>
__global__ __launch_bounds__(SAMPLE_THREADS) void head_sample_best_kernel(HeadSampleParams p) {
  __shared__ SampleShared s;
  Sampler<T, false> row(p, s, blockIdx.y);
  const u64 c = row.best(blockIdx.x, blockIdx.x + 1);
  if (threadIdx.x == 0) p.best[(size_t)blockIdx.y * gridDim.x + blockIdx.x] = c;
  for (int i = blockIdx.x * SAMPLE_THREADS + threadIdx.x; i < SAMPLE_BINS; i += gridDim.x * SAMPLE_THREADS) {
    p.bins[(size_t)blockIdx.y * SAMPLE_BINS + i] = 0;
    p.counts[(size_t)blockIdx.y * SAMPLE_BINS + i] = 0;
  }
}
template <typename T>
__global__ __launch_bounds__(SAMPLE_THREADS) void head_sample_share_kernel(HeadSampleParams p) {
  __shared__ SampleShared s;
  Sampler<T, true> row(p, s, blockIdx.y);
  row.tables();
  for (int i = threadIdx.x; i < SAMPLE_BINS; i += SAMPLE_THREADS) s.bins[i] = s.counts[i] = 0;
  const int tiles = gridDim.x;
  const u64 c = row.largest((int)threadIdx.x < tiles ? p.best[(size_t)blockIdx.y * tiles + threadIdx.x] : 0);
  if (c != ~0ull && c >> 32 && row.temperature > 0.0f) {
    row.begin(c);
    row.share(blockIdx.x);
  }
}

template <typename T>
static void launch_sample(const HeadSampleParams& p, hipStream_t st) {
  const dim3 threads(SAMPLE_THREADS);
  if (!p.best) {
    hipLaunchKernelGGL((head_sample_kernel<T, false>), dim3(p.N), threads, 0, st, p);
    return;
  }
  const dim3 grid(sample_tiles(p.V), p.N);
  hipLaunchKernelGGL(head_sample_best_kernel<T>, grid, threads, 0, st, p);
  hipLaunchKernelGGL(head_sample_share_kernel<T>, grid, threads, 0, st, p);
  hipLaunchKernelGGL((head_sample_kernel<T, true>), dim3(p.N), threads, 0, st, p);
}

hipError_t launch_head_sample(const HeadSampleParams& p, hipStream_t st) {
  KTimer t("head_sample", st);
  if (p.z_bf16) launch_sample<bf16>(p, st);
  else launch_sample<float>(p, st);
  return hipGetLastError();
}

}  // namespace alg
