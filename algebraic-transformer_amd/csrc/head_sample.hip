// Tokens drawn from the algebraic likelihood of a row of logits (src/algebraic/algebraic.py:223-265: p is
// proportional to rho(x)^n, x = min(z / c, X)), with temperature (rho^(n / T)), top-k, top-p and min-p, from a
// given uniform number.
//
// Which token a number selects depends on sums over the vocabulary to their last bits wherever the number lies
// next to a border, and V = 32000 borders lie everywhere. So the weights are f64, relative to the
// row's largest, and are summed as whole numbers of 2^-bits (2^62 / V): such sums are
// equal in any order, among any number of lanes and atomics, and a row's token depends on the row alone.
// log2 rho is good to 2^-44.7 (log2_rho), so a weight to (n / T) 2^-44 of itself, beside 2^-50 for the power of two:
// 2^-41 at n / T = 8, 2^-34 at 1024, and nothing is left of it where n / T passes 2^44. Which logit is the largest, and
// the order by logits, are exact at any temperature.
//
// Order: logits falling, equal ones by their index. The kept tokens are a prefix of it. Where a
// histogram over 2048 ranges of the logits (by count for top-k, by weight for top-p) says that no more than
// 1024 tokens can be in it, those are sorted in LDS and everything else happens among them. Otherwise
// the prefix is a pair (key, last index of that key), found without sorting: the exact ranks within the range
// where the sum is reached, or if that is crowded too, histograms of its keys' bits (at most three more);
// tokens of one single logit are counted.
//
// 64 rows of 32000 with settings of each kind: 31 us (best 5, share 10, row 16), 3 rows of 50257, top-p: 24 (3.5, 6.5,
// 14). Instructions bound the first two (VALU 64 and 72 % busy: a token at a time, f64 weights), latency the last: one
// workgroup a row, which goes over its row once more for the list and then from barrier to barrier (VALU 43 %).
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
constexpr int SAMPLE_LIST = 1024;                // tokens that are sorted
constexpr int SAMPLE_RANKED = 192;               // so many by counting, for each, those before it
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

// The lanes' numbers combined up to each lane (`op` with 0 leaves a number as it is), without a trip through LDS: the
// lanes before it in a row of 16, then the rows before.
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 lanes_before(u64 v) {
  const unsigned lo = __builtin_amdgcn_update_dpp(0, (int)(unsigned)v, CTRL, ROWS, 0xF, true);
  const unsigned hi = __builtin_amdgcn_update_dpp(0, (int)(unsigned)(v >> 32), CTRL, ROWS, 0xF, true);
  return (u64)hi << 32 | lo;
}
template <typename Op>
__device__ __forceinline__ u64 row_scan(u64 v, Op op) {
  v = op(v, lanes_before<0x111, 0xF>(v));
  v = op(v, lanes_before<0x112, 0xF>(v));
  v = op(v, lanes_before<0x114, 0xF>(v));
  return op(v, lanes_before<0x118, 0xF>(v));
}
template <typename Op>
__device__ __forceinline__ u64 wave_scan(u64 v, Op op) {
  v = row_scan(v, op);
  v = op(v, lanes_before<0x142, 0xA>(v));
  return op(v, lanes_before<0x143, 0xC>(v));
}
__device__ __forceinline__ u64 lane_of(u64 v, int lane) {
  return (u64)(unsigned)__builtin_amdgcn_readlane((int)(unsigned)(v >> 32), lane) << 32 |
         (unsigned)__builtin_amdgcn_readlane((int)(unsigned)v, lane);
}
struct Add {
  __device__ __forceinline__ u64 operator()(u64 a, u64 b) const { return a + b; }
};
struct Max {
  __device__ __forceinline__ u64 operator()(u64 a, u64 b) const { return max(a, b); }
};

struct Prefix {
  unsigned key;
  int last;
};
__device__ __forceinline__ bool in_prefix(const Prefix& p, unsigned key, int i) {
  return key > p.key || (key == p.key && i <= p.last);
}

// Tables of log2 and 2^x: 1 / m and log2 m for the middles m of [1, 2)'s 128 parts, and 2^(i / 64). Formed by the
// compiler, from log((1 + y) / (1 - y)) = 2 (y + y^3 / 3 + ...) and the exponential's series.
struct SampleTables {
  double logs[128][2];
  double exps[64];
};
constexpr double LN2 = 0.69314718055994530942;
constexpr SampleTables sample_tables() {
  SampleTables t{};
  for (int i = 0; i < 128; ++i) {
    const double m = 1.0 + (i + 0.5) / 128.0, y = (m - 1.0) / (m + 1.0);
    double sum = 0.0, power = y;
    for (int k = 1; k < 60; k += 2, power *= y * y) sum += power / k;
    t.logs[i][0] = 1.0 / m;
    t.logs[i][1] = 2.0 * sum / LN2;
  }
  for (int i = 0; i < 64; ++i) {
    double sum = 1.0, term = 1.0;
    for (int k = 1; k < 30; ++k) {
      term *= i / 64.0 * LN2 / k;
      sum += term;
    }
    t.exps[i] = sum;
  }
  return t;
}
__device__ constexpr SampleTables SAMPLE_TABLES = sample_tables();

struct SampleShared {
  SampleTables tables;
  u64 bins[SAMPLE_BINS];
  u64 list[SAMPLE_LIST];  // key, and the index's complement: falling order
  u64 value[SAMPLE_LIST];
  u64 tile[SAMPLE_TILES][SAMPLE_WAVES];
  u64 wave[SAMPLE_WAVES];
  unsigned lo, hi, count;
  int bin, token;
  u64 above;
  Prefix found;
};

// log2 of a normal number, to 2^-50: its exponent, and log2 m from the middle of m's 128th part and five terms of
// the series.
typedef __attribute__((address_space(3))) const SampleTables* TablesPtr;
__device__ __noinline__ double log2_of(double v, TablesPtr tables) {
  const u64 b = __builtin_bit_cast(u64, v);
  const int high = (int)(b >> 32), part = (high >> 13) & 127;
  const double m = __builtin_bit_cast(double, (b & 0x000FFFFFFFFFFFFFull) | 0x3FF0000000000000ull);
  const double t = __builtin_fma(m, tables->logs[part][0], -1.0);
  constexpr double C = 1.0 / LN2;
  double poly = __builtin_fma(t, C / 5, -C / 4);
  poly = __builtin_fma(t, poly, C / 3);
  poly = __builtin_fma(t, poly, -C / 2);
  poly = __builtin_fma(t, poly, C);
  return __builtin_fma(t, poly, tables->logs[part][1] + (double)((high >> 20) - 1023));
}

// One row, by one workgroup. What is done to a token stands once in the code and every loop is kept a loop: a
// workgroup goes through it once, and instructions that are fetched for it alone cost more than those that
// are executed (unrolled, 150 KB of them took three times as long).
template <typename T>
struct Sampler {
  const HeadSampleParams& p;
  SampleShared& s;
  const int r;  // the row
  const T* row;
  int tid, lane, wave, tiles;
  unsigned top;           // the largest logit's key
  double power, log_top;  // n / temperature, log2 rho of the largest
  // The row's settings.
  float temperature, top_p;
  double floor_v;  // the least weight kept, times 2^bits
  int top_k;
  bool cut_k, cut_p;

  __device__ __forceinline__ Sampler(const HeadSampleParams& p_, SampleShared& s_, int r_)
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
  __device__ __forceinline__ void tables() {
    constexpr int N = sizeof(SampleTables) / sizeof(double);
    const double* from = reinterpret_cast<const double*>(&SAMPLE_TABLES);
    if (tid < N) reinterpret_cast<double*>(&s.tables)[tid] = from[tid];
  }

  __device__ __forceinline__ int first(int t) const { return t * SAMPLE_TILE + 4 * tid; }
  // A lane's four tokens of a tile; none past the row's end. Rows start anywhere.
  struct Four {
    T z[4];
  };
  __device__ __forceinline__ Four logits(int t) const {
    const int i = first(t);
    Four f;
    if (i + 4 <= p.V) {
      __builtin_memcpy(f.z, row + i, sizeof f.z);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) f.z[e] = i + e < p.V ? row[i + e] : (T)-INFINITY;
    }
    return f;
  }
  // f(logit, token) for every token of tiles [begin, end), and g(t) after each tile, which may end it;
  // four tiles' loads are under way.
  template <typename F, typename G>
  __device__ __forceinline__ void sweep(int begin, int end, F f, G g) const {
    const auto load = [&](int t) { return logits(min(t, end - 1)); };
    Four a = load(begin), b = load(begin + 1), c = load(begin + 2), d = load(begin + 3);
#pragma unroll 1
    for (int t = begin; t < end; ++t) {
      Four now = a;
      a = b;
      b = c;
      c = d;
      if (t + 4 < end) d = logits(t + 4);
#pragma unroll 1
      for (int e = 0; e < 4; ++e) {
        f((float)now.z[0], first(t) + e);
        now.z[0] = now.z[1];
        now.z[1] = now.z[2];
        now.z[2] = now.z[3];
      }
      if (g(t)) break;
    }
  }
  struct Nothing {
    __device__ __forceinline__ bool operator()(int) const { return false; }
  };

  // log2 rho(x) = log2(|x| + sqrt(1 + x^2)), to 2^-44.7: the root is q rsqrt(q), the hardware's (to 2^-23 of itself)
  // with one step of Newton's method, which leaves 3/2 of the square, 2^-45.4; log2 2^-48. (2^22 of both signs: 2^-47.4.)
  __device__ __forceinline__ double log2_rho(unsigned key) const {
    const double x = key == KEY_CLAMPED ? p.clamp : (double)key_logit(key) * p.inv_c, a = __builtin_fabs(x);
    const double q = __builtin_fma(a, a, 1.0), y = __builtin_amdgcn_rsq(q), h = q * y;
    const double l = log2_of(a + __builtin_fma(0.5 * h, __builtin_fma(-h, y, 1.0), h), (TablesPtr)&s.tables);
    return x < 0.0 ? -l : l;
  }
  // The weight times 2^bits: 2^d by the table's nearest 64th and five terms of the series. No key is over the
  // largest, so d is 0 at most. But log2_rho rounds, and logits within 2^-20 c of zero may lie closer than its error
  // (floats further out differ by more): times any n / T such an error could pass every exponent. Held at 0, weights
  // stay within 2^bits, and V of them under 2^62, at any temperature.
  __device__ __forceinline__ double scaled(unsigned key) const {
    const double d = fmin(fmax(power * (log2_rho(key) - log_top), -1000.0), 0.0), j = __builtin_rint(d * 64.0);
    const double f = __builtin_fma(j, -0.015625, d);
    const int ji = (int)j;
    double poly = __builtin_fma(f, LN2 * LN2 * LN2 * LN2 * LN2 / 120, LN2 * LN2 * LN2 * LN2 / 24);
    poly = __builtin_fma(f, poly, LN2 * LN2 * LN2 / 6);
    poly = __builtin_fma(f, poly, LN2 * LN2 / 2);
    poly = __builtin_fma(f, poly, LN2);
    poly = __builtin_fma(f, poly, 1.0);
    return __builtin_amdgcn_ldexp(s.tables.exps[ji & 63] * poly, (ji >> 6) + p.bits);
  }
  static __device__ __forceinline__ u64 whole_part(double v) {
    const unsigned high = (unsigned)(v * 0x1p-32);
    return (u64)high << 32 | (unsigned)__builtin_fma((double)high, -0x1p32, v);
  }
  __device__ __forceinline__ u64 kept(unsigned k) const {
    const double v = scaled(k);
    return v >= floor_v ? whole_part(v) : 0;
  }

  // op over the lanes up to this one, and over all: wave by wave, then a row of 16 lanes over the waves' results.
  template <typename Op>
  __device__ __forceinline__ u64 scan(u64 v, u64& total, Op op) {
    static_assert(SAMPLE_WAVES == 16, "a row of lanes");
    v = wave_scan(v, op);
    __syncthreads();
    if (lane == 63) s.wave[wave] = v;
    __syncthreads();
    const u64 upto = row_scan(s.wave[lane & 15], op);
    total = lane_of(upto, 15);
    return wave > 0 ? op(v, lane_of(upto, max(wave - 1, 0))) : v;
  }
  __device__ __forceinline__ u64 largest(u64 c) {
    scan(c, c, Max());
    return c;
  }
  // The lanes' numbers in falling order, a lane each; `size` a power of two, the lanes from there on hold 0.
  __device__ __forceinline__ u64 sorted(u64 v, int size) {
    u64* buf = s.bins;
#pragma unroll 1
    for (int block = 2; block <= size; block <<= 1)
#pragma unroll 1
      for (int step = block >> 1; step > 0; step >>= 1) {
        u64 o;
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

  // The first histogram's ranges, of the logits themselves, of 1/64 of the scale: a monotone function of the key,
  // whatever it rounds.
  __device__ __forceinline__ int first_bin(unsigned k) const {
    const float z_top = top == KEY_CLAMPED ? p.z_clamp : key_logit(top), z = k == KEY_CLAMPED ? p.z_clamp : key_logit(k);
    return (int)fminf((z_top - z) * (float)(64.0 * p.inv_c), SAMPLE_BINS - 1.0f);
  }

  __device__ __forceinline__ void answer(int token, double logprob) {
    p.token[r] = token;
    p.logprob[r] = (float)logprob;
  }
  __device__ __forceinline__ double log_share(u64 part, u64 whole) const {
    return part == whole ? 0.0 : LN2 * log2_of((double)part / (double)whole, (TablesPtr)&s.tables);
  }
  // The largest logit's key and the complement of its first token, of tiles [begin, end); all ones with a NaN.
  __device__ __forceinline__ u64 best(int begin, int end) {
    u64 c = 0;
    sweep(begin, end, [&](float z, int i) {
      c = max(c, z != z ? ~0ull : (u64)logit_key(z, p.z_clamp) << 32 | (unsigned)~i);
    }, Nothing());
    return largest(c);
  }
  // Takes the row's best; false: it has its answer, or none.
  __device__ __forceinline__ bool begin(u64 c) {
    top = (unsigned)(c >> 32);
    const bool none = c == ~0ull || top == 0 || !(temperature >= 0.0f);
    if (none || temperature == 0.0f) {
      if (tid == 0) answer(none ? -1 : (int)~(unsigned)c, none ? __builtin_nan("") : 0.0);
      return false;
    }
    power = p.n / (double)temperature;
    log_top = log2_rho(top);
    return true;
  }

  // One tile's share of what the row needs first: the histogram of its cut (s.bins clear), or its waves'
  // sums.
  __device__ __forceinline__ void share(int tile) {
    const bool cut = cut_k || cut_p;
    u64 v = 0;
    sweep(tile, tile + 1, [&](float z, int) {
      const unsigned k = logit_key(z, p.z_clamp);
      if (k == 0) return;
      const u64 w = cut_k ? 1 : cut ? whole_part(scaled(k)) : kept(k);
      if (cut) atomicAdd(&s.bins[first_bin(k)], w);
      v += w;
    }, Nothing());
    if (!cut) {
      v = wave_scan(v, Add());
      if (lane == 63) p.sums[((size_t)r * tiles + tile) * SAMPLE_WAVES + wave] = v;
      return;
    }
    __syncthreads();
#pragma unroll
    for (int i = tid; i < SAMPLE_BINS; i += SAMPLE_THREADS)
      if (s.bins[i]) atomicAdd(p.bins + (size_t)r * SAMPLE_BINS + i, s.bins[i]);
  }

  // `ready`: the row's best, and the histogram or sums that it needs first, are there.
  __device__ __forceinline__ void run(bool ready) {
    const double u = p.u_f64 ? static_cast<const double*>(p.u)[r] : (double)static_cast<const float*>(p.u)[r];
    tables();
    u64 c = ready ? (tid < tiles ? p.best[(size_t)r * tiles + tid] : 0) : 0;
    c = ready ? largest(c) : best(0, tiles);
    if (!begin(c)) return;

    // The cuts: by_mass false top-k, true top-p. Each asks for the shortest prefix, within `in`, of whose tokens' values
    // (1, or the weight) the sum reaches `need`; [lo, hi] holds the key where it does, `above` is the sum over it.
    Prefix in{0, p.V};
    bool by_mass = !cut_k, cut = cut_k || cut_p, fresh = true, ties = false;
    unsigned lo = 0, hi = top;
    u64 above = 0, need = 0, wanted_tie = 0;
    int listed = 0, first_k = 0;
    const auto share_of = [&](u64 total) { return max((u64)ceil(fmax((double)top_p, 0.0) * (double)total), (u64)1); };
#pragma unroll 1
    while (true) {
      if (cut) {
        const int shift = max(0, 21 - (int)__builtin_clz((hi - lo) | 1u));  // (hi - lo) >> shift < 2048
        const auto bin = [&](unsigned k) { return fresh ? first_bin(k) : (int)((hi - k) >> shift); };
        u64 a, b;
        if (ready) {
          const ulonglong2 sums = reinterpret_cast<const ulonglong2*>(p.bins + (size_t)r * SAMPLE_BINS)[tid];
          a = sums.x;
          b = sums.y;
          ready = false;
        } else {
          __syncthreads();
#pragma unroll
          for (int i = tid; i < SAMPLE_BINS; i += SAMPLE_THREADS) s.bins[i] = 0;
          __syncthreads();
          sweep(0, tiles, [&](float z, int i) {
            const unsigned k = logit_key(z, p.z_clamp);
            if (k == 0 || k < lo || k > hi || !in_prefix(in, k, i)) return;
            atomicAdd(&s.bins[bin(k)], by_mass ? whole_part(scaled(k)) : 1);
          }, Nothing());
          __syncthreads();
          a = s.bins[2 * tid];
          b = s.bins[2 * tid + 1];
        }
        u64 total;
        const u64 upto = above + scan(a + b, total, Add()), before = upto - a - b;
        if (fresh) need = by_mass ? share_of(total) : (u64)top_k;
        if (!by_mass && fresh && need >= total) {  // top-k takes all
          by_mass = true;
          cut = cut_p;
          continue;
        }
        if (before < need && upto >= need) {
          const bool second = before + a < need;
          s.bin = 2 * tid + second;
          s.above = before + (second ? a : 0);
        }
        // The tokens of that range, and all above if they fit the list.
        const bool round0 = fresh;
        bool all = fresh;
        int n;
#pragma unroll 1
        while (true) {
          if (tid == 0) {
            s.lo = 0xFFFFFFFFu;
            s.hi = s.count = 0;
          }
          __syncthreads();
          const int at = s.bin;
          // What is surely under that range (the first histogram's: by two ranges, and what floats round) is passed
          // over before anything is formed of it; a list that has run over is left.
          const float z_top = top == KEY_CLAMPED ? p.z_clamp : key_logit(top), step = (float)(64.0 * p.inv_c);
          const float z_cut = z_top - (at + 2) / step, z_low = z_cut - 0x1p-20f * (fabsf(z_top) + fabsf(z_cut));
          const float z_min = round0 && at < SAMPLE_BINS - 1 && z_low > -INFINITY && z_low < INFINITY ? z_low : -INFINITY;
          sweep(0, tiles, [&](float z, int i) {
            if (!(z >= z_min)) return;
            const unsigned k = logit_key(z, p.z_clamp);
            if (k == 0 || k < lo || k > hi || !in_prefix(in, k, i)) return;
            const int b = bin(k);
            if (b > at || (b < at && !all)) return;
            if (!all) {
              atomicMin(&s.lo, k);
              atomicMax(&s.hi, k);
            }
            const unsigned n = atomicAdd(&s.count, 1u);
            if (n < SAMPLE_LIST) s.list[n] = (u64)k << 32 | (unsigned)~i;
          }, [&](int) { return all && *(volatile unsigned*)&s.count > SAMPLE_LIST; });
          __syncthreads();
          n = (int)s.count;
          if (n <= SAMPLE_LIST || !all) break;
          all = false;
          __syncthreads();
        }
        above = s.above;
        if (!all) {
          lo = s.lo;
          hi = s.hi;
        }
        fresh = false;
        if (n <= SAMPLE_LIST) {
          u64 mine = tid < n ? s.list[tid] : 0;
          if (n <= SAMPLE_RANKED) {
            int rank = 0;
            if (tid < n)
#pragma unroll 4
              for (int i = 0; i < n; ++i) rank += s.list[i] > mine;
            __syncthreads();
            s.list[tid < n ? rank : tid] = mine;
            __syncthreads();
            mine = s.list[tid];
          } else {
            int size = 64;
            while (size < n) size <<= 1;
            mine = sorted(mine, size);
            __syncthreads();
            s.list[tid] = mine;
          }
          if (all) {
            listed = n;
            first_k = by_mass ? 0 : top_k;
            break;
          }
          u64 ignored;
          const unsigned k = (unsigned)(mine >> 32);
          const u64 v = tid < n ? (by_mass ? whole_part(scaled(k)) : 1) : 0;
          const u64 sum = above + scan(v, ignored, Add());
          if (sum - v < need && sum >= need) s.found = Prefix{k, (int)~(unsigned)mine};
          __syncthreads();
          in = s.found;
        } else if (lo == hi) {  // one logit: as many of its tokens as it takes
          const u64 each = by_mass ? whole_part(scaled(lo)) : 1;
          wanted_tie = (need - above + each - 1) / each;
          ties = true;
        } else {
          continue;
        }
        if (!ties) {  // the next cut
          cut = !by_mass && cut_p;
          by_mass = true;
          fresh = true;
          lo = 0;
          hi = top;
          above = 0;
          continue;
        }
      }
      // A draw: of the wanted one of equal logits, or of the kept tokens. The sums of waves say which wave's.
      const auto value = [&](float z, int i) -> u64 {
        const unsigned k = logit_key(z, p.z_clamp);
        if (k == 0 || !in_prefix(in, k, i)) return 0;
        return ties ? (u64)(k == lo) : kept(k);
      };
      if (ready) {
        for (int i = tid; i < tiles * SAMPLE_WAVES; i += SAMPLE_THREADS)
          (&s.tile[0][0])[i] = p.sums[(size_t)r * tiles * SAMPLE_WAVES + i];
      } else {
        u64 v = 0;
        sweep(0, tiles, [&](float z, int i) { v += value(z, i); }, [&](int t) {
          v = wave_scan(v, Add());
          if (lane == 63) s.tile[t][wave] = v;
          v = 0;
          return false;
        });
      }
      __syncthreads();
      u64 v = 0, total;
      for (int i = tid; i < tiles * SAMPLE_WAVES; i += SAMPLE_THREADS) v += (&s.tile[0][0])[i];
      scan(v, total, Add());
      const u64 target = ties ? wanted_tie - 1 : drawn(u, total);
      int t = 0, w = 0;
      u64 below = 0;
#pragma unroll 1
      for (; t < tiles - 1; ++t) {
        u64 sum = 0;
#pragma unroll
        for (int i = 0; i < SAMPLE_WAVES; ++i) sum += s.tile[t][i];
        if (below + sum > target) break;
        below += sum;
      }
#pragma unroll 1
      for (; w < SAMPLE_WAVES - 1; ++w) {
        if (below + s.tile[t][w] > target) break;
        below += s.tile[t][w];
      }
      if (wave == w) {
        Four z = logits(t);
        u64 got[4], sum = 0;
#pragma unroll 1
        for (int e = 0; e < 4; ++e) {
          const u64 x = value((float)z.z[0], first(t) + e);
          got[0] = got[1];
          got[1] = got[2];
          got[2] = got[3];
          got[3] = x;
          sum += x;
          z.z[0] = z.z[1];
          z.z[1] = z.z[2];
          z.z[2] = z.z[3];
        }
        below += wave_scan(sum, Add()) - sum;  // up to this lane's tokens
        if (below <= target && below + sum > target) {
          int e = 0;
          u64 mine = got[0];
#pragma unroll
          for (int i = 0; i < 3; ++i) {
            below += got[i];
            if (below <= target) {
              ++e;
              mine = got[i + 1];
            }
          }
          if (ties) s.token = first(t) + e;
          else answer(first(t) + e, log_share(mine, total));
        }
      }
      if (!ties) return;
      __syncthreads();
      in = Prefix{lo, s.token};
      ties = false;
      cut = !by_mass && cut_p;
      by_mass = true;
      fresh = true;
      lo = 0;
      hi = top;
      above = 0;
    }

    // The list's tokens, a lane each, by falling logit; then the kept ones by their index.
    const u64 mine = s.list[tid];
    const bool is = tid < (first_k ? first_k : listed);
    const double v = is ? scaled((unsigned)(mine >> 32)) : 0.0;
    const u64 m = is ? whole_part(v) : 0;
    u64 total;
    const u64 upto = scan(m, total, Add());
    if (first_k) need = cut_p ? share_of(total) : total;
    const bool keep = is && v >= floor_v && (tid == 0 || upto - m < need);
    const unsigned index = ~(unsigned)mine;
    s.value[tid] = keep ? m : 0;
    u64 sum = 0, all = 0;  // what the kept tokens of lower index have, and all
    if (listed <= SAMPLE_RANKED) {
      s.list[tid] = index;
      __syncthreads();
      if (!keep) return;
#pragma unroll 4
      for (int i = 0; i < listed; ++i) {
        const u64 w = s.value[i];
        all += w;
        sum += s.list[i] < index ? w : 0;
      }
      const u64 t = drawn(u, all);
      if (sum <= t && sum + m > t) answer((int)index, log_share(m, all));
      return;
    }
    int size = 64;
    while (size < listed) size <<= 1;
    const unsigned by_index = (unsigned)sorted(keep ? (u64) ~(index << 10 | (unsigned)tid) : 0, size);
    __syncthreads();
    const u64 w = by_index ? s.value[~by_index & 1023] : 0;
    sum = scan(w, all, Add());
    const u64 t = drawn(u, all);
    if (by_index && sum - w <= t && sum > t) answer((int)(~by_index >> 10), log_share(w, all));
  }
  // u as a share of `total`, in whole numbers below it: below 0 or NaN as 0, 1 or more as the largest below.
  static __device__ __forceinline__ u64 drawn(double u, u64 total) {
    const double at = floor((u >= 0.0 ? u : 0.0) * (double)total);
    return at < (double)total ? min((u64)at, total - 1) : total - 1;
  }
};

}  // namespace

template <typename T>
__global__ __launch_bounds__(SAMPLE_THREADS) void head_sample_kernel(HeadSampleParams p) {
  __shared__ SampleShared s;
  Sampler<T>(p, s, blockIdx.x).run(p.best != nullptr);
}

// Few rows leave most CUs without one, so the passes over a whole row are spread over its tiles, a workgroup each:
// first the largest logit (which clears the row's histogram too), then what share() says. The sums are
// whole numbers: the results are those of one workgroup.
template <typename T>
__global__ __launch_bounds__(SAMPLE_THREADS) void head_sample_best_kernel(HeadSampleParams p) {
  __shared__ SampleShared s;
  Sampler<T> row(p, s, blockIdx.y);
  const u64 c = row.best(blockIdx.x, blockIdx.x + 1);
  if (threadIdx.x == 0) p.best[(size_t)blockIdx.y * gridDim.x + blockIdx.x] = c;
  for (int i = blockIdx.x * SAMPLE_THREADS + threadIdx.x; i < SAMPLE_BINS; i += gridDim.x * SAMPLE_THREADS) {
    p.bins[(size_t)blockIdx.y * SAMPLE_BINS + i] = 0;
  }
}
template <typename T>
__global__ __launch_bounds__(SAMPLE_THREADS) void head_sample_share_kernel(HeadSampleParams p) {
  __shared__ SampleShared s;
  Sampler<T> row(p, s, blockIdx.y);
  row.tables();
#pragma unroll
  for (int i = threadIdx.x; i < SAMPLE_BINS; i += SAMPLE_THREADS) s.bins[i] = 0;
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
  if (p.best) {
    const dim3 grid(sample_tiles(p.V), p.N);
    hipLaunchKernelGGL(head_sample_best_kernel<T>, grid, threads, 0, st, p);
    hipLaunchKernelGGL(head_sample_share_kernel<T>, grid, threads, 0, st, p);
  }
  hipLaunchKernelGGL(head_sample_kernel<T>, dim3(p.N), threads, 0, st, p);
}

hipError_t launch_head_sample(const HeadSampleParams& p, hipStream_t st) {
  KTimer t("head_sample", st);
  if (p.z_bf16) launch_sample<bf16>(p, st);
  else launch_sample<float>(p, st);
  return hipGetLastError();
}

}  // namespace alg
