// Backward pass of causal algebraic attention over packed sequences with grouped heads, bf16
// (packed_common.h: rows, slots, the weights' two forms; packed_fwd.hip: the forward pass).
//
// With P = (t rs)^n, dP = dO V^T, di = sum_d dO o and r = 1/sqrt(s^2 + b) the score gradient is
// n alpha P (dP - di) / sqrt(1 + x^2) = n 2^-e P (dP - di) r, e the exponent that the queries are
// scaled by; the factor n 2^-e is applied to the sums. Two launches, without atomics (and
// packed_join, where keys or rows are split over workgroups):
//   packed_dq    one workgroup = the 128 rows of a forward workgroup: di, then dQ^T += K^T dS^T
//                over the 64-key tiles up to the diagonal (S^T = K Q^T and dP^T = V dO^T formed
//                again, dS in registers, K^T read transposed from LDS).
//   packed_dkdv  one workgroup = 64 keys of one key head, 16 a wave: dV += P^T dO and
//                dK += dS^T Q over the 64-row tiles (token, head of the group) from the keys'
//                first token on. The rows of all G heads pass one after the other, so the sum
//                over the group that a shared head's gradient is takes place in registers, in a
//                fixed order. Workgroups (key head, g) at the grid's start sum the sinks'
//                gradients, - sum_rows mass di n / (sqrt(1 + x^2) c).
// A row's form (plain or careful) is its forward's, from the sign of its statistic. The dQ kernel's
// workgroups take the careful form where one of their rows does, and leave that in `care`, one
// entry per slot and key head, by which a dK/dV workgroup knows whether one of its rows does; the
// careful form serves either kind of row. Its loops are not pipelined: they are the rare case, and
// in one loop with the plain form they cost that form registers (188 more spilled in dQ at
// D = 128).
// P and dS are rounded to bf16 for their products. Plain form: di is formed of the rounded o, as the
// (B, H, T, D) kernels do in range: dQ and dK are off by these two and their own rounding, 0.003 of their
// size in all, dV by P's and its own. Careful form: di = sum_j P dP from a sweep over the keys of its
// own, as those kernels do out of range, for there dS may be far smaller than dP and di (values near 3
// whose differences are 0.1: dQ off by 0.42 of its size with the rounded o's di, 0.004 so). Sums are f32.
// What bounds it: VALU and matrix issue beside waits for spilled registers and copies. Nine documents of
// 16384 tokens, 16 heads over 4, D = 128: dQ 302 us, 0.80 PFLOP/s (VALU busy 56 % of cycles, matrix cores
// 42 %), dK/dV 408, 0.79 (52, 48); every row careful 980 and 877. 13 documents, 8161 tokens, 16 heads,
// D = 64: 50 and 55 us (64, 23; 66, 26).
// dK/dV with 8 waves, the columns of dK and dV split over them, was slower: 436 us (then 418), and 100 for
// 55 at D = 64.
#include <type_traits>

#include "launchers.h"
#include "packed_common.h"

namespace alg {

// P and dS = P (dP - di) r; `dp` is dP - di.
template <int L2N, bool CARE>
__device__ __forceinline__ void packed_elem(float s, float dp, float rs, float b, int log2n, bool dead, float& pw,
                                            float& ds) {
  float r;
  const float t = CARE ? weight_t_careful(s, b, r) : weight_t(s, b, r);
  pw = pow2n<L2N>(t * __builtin_fabsf(rs), log2n);
  ds = pw * dp * r;
  keep_here(pw, ds);
  if (dead) pw = ds = 0.0f;
}

template <int D, int L2N>
__global__ __launch_bounds__(256, 2) void packed_dq_kernel(PackedBwdParams p) {
  constexpr int BK = PK_BK, CPR = D / 8, NDB = D / 32, NF = D / 16;
  constexpr int RPI = 64 / CPR, PW = 16 / RPI;  // keys per copy instruction; instruction pairs per wave and tile
  __shared__ __attribute__((aligned(16))) bf16 Ks0[BK * D];
  __shared__ __attribute__((aligned(16))) bf16 Ks1[BK * D];
  __shared__ __attribute__((aligned(16))) bf16 Vs0[BK * D];
  __shared__ __attribute__((aligned(16))) bf16 Vs1[BK * D];

  const int lane = threadIdx.x & 63, h = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // wave-uniform
  // Workgroups: key head, range of keys, item.
  const int kvh = blockIdx.x % p.Hkv, unit = blockIdx.x / p.Hkv, range = unit % p.dq_parts;
  const PackedSeq f = packed_find<true>(p.cu, p.N, p.S, p.G, PK_ROWS, unit / p.dq_parts, gridDim.x / p.Hkv / p.dq_parts);
  const int G = p.G, R = f.len * G, r0 = f.tile * PK_ROWS;
  if (f.tile < 0 || r0 >= R) return;
  const int myr = r0 + wave * 32 + l32;
  const bool live = myr < R;
  const PackedRow at = packed_row<D>(p, f, kvh, min(myr, R - 1));
  if (f.s == p.S) {  // tokens behind the last sequence
    const bf16x8 z = {};
    if (live && range == 0) {
      for (int d = 8 * h; d < D; d += 16) *reinterpret_cast<bf16x8*>(p.dq + at.out + d) = z;
      if (h == 0) p.ndi[at.stat] = 0.0f;
    }
    return;
  }
  const int mytok = live ? at.tok : -1;
  const int posmax = (min(r0 + PK_ROWS, R) - 1) / G;
  const int wave_posmax = min(r0 + wave * 32 + 31, R - 1) / G;
  int kt0 = 0, kt1 = posmax / BK + 1;  // this workgroup's key tiles
  if (p.dq_parts > 1) {
    const int per = ceil_div(kt1, p.dq_parts);
    kt0 = min(range * per, kt1);
    kt1 = min(kt0 + per, kt1);
  }
  const int nfull = (r0 / G + 1) / BK;  // tiles before every row's position

  const bf16* kbase = p.k + (size_t)kvh * p.k_hs + (size_t)f.start * p.k_ts;
  const bf16* vbase = p.v + (size_t)kvh * p.v_hs + (size_t)f.start * p.v_ts;
  // The 16 keys of tile kt that this wave copies; past the sequence, and from tile `end` on, they read
  // as zeros.
  auto group = [&](int kt, int end) {
    KvGroup g;
    const int key = kt * BK + 16 * wave;
    g.rows = kt < end ? min(max(f.len - key, 0), 16) : 0;
    const int k = g.rows > 0 ? key : 0;
    g.k = kbase + (size_t)k * p.k_ts;
    g.v = vbase + (size_t)k * p.v_ts;
    return g;
  };
  // Instruction pair j of a copy: a lane's row and swizzled chunk, the same for every tile; the rest
  // of the address is scalar.
  const int lrow = lane / CPR;
  const int k_row = lrow * (int)p.k_ts * 2, v_row = lrow * (int)p.v_ts * 2;
  const int chunkb = 16 * ((lane % CPR) ^ swz_chunk<CPR>(lrow));
  auto dma = [&](bf16* la, bf16* lb, const KvGroup& g, int j) {
    const int kn = g.rows > 0 ? ((g.rows - 1) * (int)p.k_ts + D) * 2 : 0;
    const int vn = g.rows > 0 ? ((g.rows - 1) * (int)p.v_ts + D) * 2 : 0;
    const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc((void*)g.k, (short)0, kn, BUF_RSRC_WORD3);
    const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc((void*)g.v, (short)0, vn, BUF_RSRC_WORD3);
    auto lla = LDS_PTR(bf16, la);
    auto llb = LDS_PTR(bf16, lb);
    asm volatile("" : "+s"(lla), "+s"(llb));
    const int J = wave * PW + j;
    const int col = chunkb ^ (16 * swz_chunk<CPR>(RPI * j));  // 16 rows a wave: the swizzle's period
    const int ko = RPI * j * (int)p.k_ts * 2, vo = RPI * j * (int)p.v_ts * 2;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, lla + J * 512, 16, k_row + col + ko, 0, 0, 0);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, llb + J * 512, 16, v_row + col + vo, 0, 0, 0);
  };

  {
    const KvGroup g = group(kt0, kt1);
#pragma unroll
    for (int j = 0; j < PW; ++j) dma(Ks0, Vs0, g, j);
  }

  // Q (scaled) and dO fragments of this lane's row, its statistic and di; dead rows carry zeros.
  bf16x8 qf[NF], of[NF];
  float di = 0.0f;
  {
    const bf16* Q = p.q + (size_t)(f.start + at.tok) * p.q_ts + (size_t)at.head * p.q_hs + 8 * h;
    const bf16* dO = p.dO + (size_t)(f.start + at.tok) * p.do_ts + (size_t)at.head * p.do_hs + 8 * h;
    const bf16* O = p.o + at.out + 8 * h;
    bf16x8 ov[NF];
#pragma unroll
    for (int s = 0; s < NF; ++s) {
      qf[s] = ld8(Q + 16 * s);
      of[s] = ld8(dO + 16 * s);
      ov[s] = ld8(O + 16 * s);
    }
    keep_own_row<NF>(qf, live);
    keep_own_row<NF>(of, live);
    keep_own_row<NF>(ov, live);
#pragma unroll
    for (int s = 0; s < NF; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        di += (float)of[s][j] * (float)ov[s][j];
        qf[s][j] = f2bf((float)qf[s][j] * p.sc.qmul);
      }
    di += xor32(di);
  }
  const float rs = live ? p.stat[at.stat] : 0.0f;
  const bool careful = __syncthreads_or(rs < 0.0f) != 0;
  if (!careful && live && h == 0 && range == 0) p.ndi[at.stat] = -di;
  if (threadIdx.x == 0 && range == 0) p.care[(size_t)packed_slot(f, G, PK_ROWS) * p.Hkv + kvh] = careful;
  const int log2n = p.sc.log2n;
  const float b2 = p.sc.b;
  // Plain form: dS = (t^n r) fma(rs^n, dP, - rs^n di), one instruction less than P (dP - di) r.
  // Careful form: the statistic itself, and di of its own (below).
  const float pz = careful ? rs : pow2n<0>(rs, log2n);
  const float nzd = -pz * di;
  floatx16 dqa[NDB];
#pragma unroll
  for (int db = 0; db < NDB; ++db) dqa[db] = floatx16{};

  const int tr = (lane & 15) >> 2;
  int row_off[NF];
#pragma unroll
  for (int st = 0; st < NF; ++st) row_off[st] = swz_at<CPR>(l32, 16 * st + 8 * h);
  int tk_lo[NDB];  // transposed K fragments: rows 4h + (0..3); the other half's lie eight rows on
#pragma unroll
  for (int db = 0; db < NDB; ++db) tk_lo[db] = swz_at<CPR>(4 * h + tr, tr_col(db * 32, lane));
  const auto eight_on = [](int at) { return (again(at) ^ 16) + 8 * D; };  // the swizzle's next chunk pair
  bf16x8 rk2[2], rv2[2];  // row fragments of K / V, one step ahead
  __builtin_amdgcn_s_waitcnt(VMCNT0);
  __syncthreads();
  rk2[0] = ld8(Ks0 + row_off[0]);
  rv2[0] = ld8(Vs0 + row_off[0]);
  constexpr int VE = 14;  // VALU instructions per score (scheduling hint)

  // One key tile:
  //   R1 S^T, dP^T of keys 0..31 | the next tile's copy   R2 of 32..63 | dS of 0..31
  //   R3 dQ^T over 0..31 | dS of 32..63                   R4 dQ^T over 32..63
  auto tile = [&](auto bufc, auto maskc, int kt) {
    constexpr int BUF = decltype(bufc)::value;
    constexpr bool MASKED = decltype(maskc)::value;
    const bf16* Ks = BUF ? Ks1 : Ks0;
    const bf16* Vs = BUF ? Vs1 : Vs0;
    bf16* Kn = BUF ? Ks0 : Ks1;
    bf16* Vn = BUF ? Vs0 : Vs1;
    const int kb0 = kt * BK;
    const KvGroup gn = group(kt + 1, kt1);
    if constexpr (MASKED) {
      if (kb0 > wave_posmax) {  // every key lies after this wave's rows
#pragma unroll
        for (int j = 0; j < PW; ++j) dma(Kn, Vn, gn, j);
        __builtin_amdgcn_s_waitcnt(VMCNT0);
        __syncthreads();
        rk2[0] = ld8(Kn + row_off[0]);
        rv2[0] = ld8(Vn + row_off[0]);
        return;
      }
    }
    floatx16 s[2], dp[2];
    bf16x8 da[2][2];
    float dsv[16];
    auto sdp_step = [&](int g) {
      const int blk = g / NF, st = g % NF;
      const int gx = g + 1;
      if (gx < 2 * NF) {
        rk2[gx % 2] = ld8(Ks + (gx / NF) * 32 * D + row_off[gx % NF]);
        rv2[gx % 2] = ld8(Vs + (gx / NF) * 32 * D + row_off[gx % NF]);
      }
      s[blk] = mfma_bf16(rk2[g % 2], qf[st], s[blk]);
      dp[blk] = mfma_bf16(rv2[g % 2], of[st], dp[blk]);
    };
    auto elem = [&](int blk, int i) {
      const bool dead = MASKED && kb0 + blk * 32 + 8 * (i >> 2) + 4 * h + (i & 3) > mytok;
      float r;
      const float w = pow2n<L2N>(weight_t(s[blk][i], b2, r), log2n);
      float ds = (w * r) * __builtin_fmaf(pz, dp[blk][i], nzd);
      if constexpr (MASKED) keep_here(ds);
      dsv[i] = dead ? 0.0f : ds;
      if (i & 1) {
        da[blk][i >> 3][(i & 7) - 1] = f2bf(dsv[i - 1]);
        da[blk][i >> 3][i & 7] = f2bf(dsv[i]);
      }
    };
    bf16x8 ft[2][2];
    auto dq_load = [&](int blk, int db, bf16x8 (&fr)[2]) {
      const bf16* kb = Ks + blk * 32 * D;
      // Formed here: held, four more addresses were spilled, and a reload waits for every copy
      // before it (307 us instead of 293).
      const int hi = eight_on(tk_lo[db]);
      fr[0] = tr_frag_at(kb, tk_lo[db], hi);
      fr[1] = tr_frag_at(kb + 16 * D, tk_lo[db], hi);
    };
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      s[b] = floatx16{};
      dp[b] = floatx16{};
    }
#pragma unroll
    for (int g = 0; g < NF; ++g) {
      sdp_step(g);
      if (g < PW) dma(Kn, Vn, gn, g);
      step_order<2, 0, 4, 0>();
    }
    constexpr int E2 = 16 / NF;
#pragma unroll
    for (int g = NF; g < 2 * NF; ++g) {
      sdp_step(g);
#pragma unroll
      for (int k = 0; k < E2; ++k) elem(0, E2 * (g - NF) + k);
      if (g == 2 * NF - 1) dq_load(0, 0, ft[0]);
      step_order<2, VE * E2, 4 + 4, 0>();
    }
    constexpr int E3 = 16 / NDB;
#pragma unroll
    for (int db = 0; db < NDB; ++db) {
      const int c = db & 1;
      if (db + 1 < NDB) dq_load(0, db + 1, ft[c ^ 1]);
      else dq_load(1, 0, ft[c ^ 1]);
      dqa[db] = mfma_bf16(ft[c][0], da[0][0], dqa[db]);
      dqa[db] = mfma_bf16(ft[c][1], da[0][1], dqa[db]);
#pragma unroll
      for (int k = 0; k < E3; ++k) elem(1, E3 * db + k);
      step_order<2, VE * E3, 4, 0>();
    }
#pragma unroll
    for (int db = 0; db < NDB; ++db) {
      const int c = (db + NDB) & 1;
      if (db + 1 < NDB) dq_load(1, db + 1, ft[c ^ 1]);
      dqa[db] = mfma_bf16(ft[c][0], da[1][0], dqa[db]);
      dqa[db] = mfma_bf16(ft[c][1], da[1][1], dqa[db]);
      step_order<2, 0, 4, 0>();
    }
    __builtin_amdgcn_s_waitcnt(VMCNT0);  // this wave's copies of the next tile have landed
    __syncthreads();                     // the next tile is complete; this buffer set is free
    rk2[0] = ld8(Kn + row_off[0]);
    rv2[0] = ld8(Vn + row_off[0]);
  };
  if (!careful) {
    // In pairs of tiles, as in the forward.
    const int full = kt0 + (max(min(nfull, kt1) - kt0, 0) & ~1);
    int kt = kt0;
    for (; kt < full; kt += 2) {
      tile(std::integral_constant<int, 0>{}, std::false_type{}, kt);
      tile(std::integral_constant<int, 1>{}, std::false_type{}, kt + 1);
    }
    for (; kt < kt1; kt += 2) {
      tile(std::integral_constant<int, 0>{}, std::true_type{}, kt);
      if (kt + 1 >= kt1) break;
      tile(std::integral_constant<int, 1>{}, std::true_type{}, kt + 1);
    }
  } else {
    // Key tile kt (past the sequence it reads as zeros), and S and dP of one of its blocks.
    auto load = [&](int kt) {
      __syncthreads();  // every wave is done with the tile before
      const KvGroup g = group(kt, posmax / BK + 1);
#pragma unroll
      for (int j = 0; j < PW; ++j) dma(Ks0, Vs0, g, j);
      __builtin_amdgcn_s_waitcnt(VMCNT0);
      __syncthreads();
    };
    auto scores = [&](int blk, floatx16& s, floatx16& dp) {
      s = floatx16{};
      dp = floatx16{};
#pragma unroll
      for (int st = 0; st < NF; ++st) {
        s = mfma_bf16(ld8(Ks0 + blk * 32 * D + row_off[st]), qf[st], s);
        dp = mfma_bf16(ld8(Vs0 + blk * 32 * D + row_off[st]), of[st], dp);
      }
    };
    // di = sum_j P dP over all of the row's keys, whatever range of them is this workgroup's.
    float dw = 0.0f;
    for (int kt = 0; kt <= posmax / BK; ++kt) {
      load(kt);
      for (int blk = 0; blk < 2; ++blk) {
        const int kb = kt * BK + 32 * blk;
        if (kb > wave_posmax) continue;
        floatx16 s, dp;
        scores(blk, s, dp);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const bool dead = kb + 8 * (i >> 2) + 4 * h + (i & 3) > mytok;
          float pw, ds;
          packed_elem<0, true>(s[i], dp[i], pz, b2, log2n, dead, pw, ds);
          dw += dead ? 0.0f : pw * dp[i];
        }
      }
    }
    dw += xor32(dw);
    if (mytok >= 0 && h == 0 && range == 0) p.ndi[packed_row<D>(p, f, kvh, again(r0 + wave * 32 + l32)).stat] = -dw;
    for (int kt = kt0; kt < kt1; ++kt) {
      load(kt);
      for (int blk = 0; blk < 2; ++blk) {
        const int kb = kt * BK + 32 * blk;
        if (kb > wave_posmax) continue;
        floatx16 s, dp;
        scores(blk, s, dp);
        bf16x8 da[2];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float pw, ds;
          packed_elem<0, true>(s[i], dp[i] - dw, pz, b2, log2n, kb + 8 * (i >> 2) + 4 * h + (i & 3) > mytok, pw, ds);
          da[i >> 3][i & 7] = f2bf(ds);
        }
        const bf16* kl = Ks0 + blk * 32 * D;
#pragma unroll
        for (int db = 0; db < NDB; ++db) {
          const int hi = eight_on(tk_lo[db]);
          dqa[db] = mfma_bf16(tr_frag_at(kl, tk_lo[db], hi), da[0], dqa[db]);
          dqa[db] = mfma_bf16(tr_frag_at(kl + 16 * D, tk_lo[db], hi), da[1], dqa[db]);
        }
      }
    }
  }

  if (mytok >= 0) {
    const size_t out = packed_row<D>(p, f, kvh, again(r0 + wave * 32 + l32)).out;
    if (p.dq_parts > 1) {
      float* DS = p.dq_sum + (size_t)range * p.N * p.H * D + out;
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          floatx4 v;
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = dqa[db][4 * g + e];
          *reinterpret_cast<floatx4*>(DS + db * 32 + 8 * g + 4 * h) = v;
        }
      return;
    }
    const float slope = (float)(1 << log2n) * p.sc.qmul;
    bf16* DQ = p.dq + out;
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        bf16x4 ob;
#pragma unroll
        for (int e = 0; e < 4; ++e) ob[e] = f2bf(dqa[db][4 * g + e] * slope);
        *reinterpret_cast<bf16x4*>(DQ + db * 32 + 8 * g + 4 * h) = ob;
      }
  }
}

// One head's sink gradient (a workgroup of packed_dkdv_kernel).
__device__ __forceinline__ void packed_sink_grad(const PackedBwdParams& p, int kvh, int g) {
  __shared__ float red[4];
  const int head = kvh * p.G + g;
  float r;
  const float t = weight_t_careful(sink_score(p, head), p.sc.b, r);
  const size_t base = (size_t)kvh * p.N * p.G + g;
  float sum = 0.0f;
#pragma unroll 8
  for (int i = threadIdx.x; i < p.N; i += 256) {
    const size_t at = base + (size_t)i * p.G;
    sum += pow2n<0>(t * __builtin_fabsf(p.stat[at]), p.sc.log2n) * p.ndi[at];
  }
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) sum += __shfl_xor(sum, m, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    const float d = (red[0] + red[1] + red[2] + red[3]) * (float)(1 << p.sc.log2n) * (r / p.sc.a) / p.c;
    if (p.dsink_bf16) static_cast<bf16*>(p.dsink)[head] = f2bf(d);
    else static_cast<float*>(p.dsink)[head] = d;
  }
}

template <int D>
constexpr int packed_dkdv_waves() { return D == 64 ? 3 : 2; }  // waves per SIMD
constexpr int PK_KEYS = 64;  // keys per dK/dV workgroup

// Whether a copy instruction's rows are whole tokens and tokens lie one behind another (ALIGNED, of a
// group that divides the 8 or 4 rows; host: packed_aligned): a lane's address is then the same in
// every tile but for a scalar, and rows past the sequence are past the descriptor's end
// (404 us at the size above; 424 with each lane's row divided by the group).
template <int D, int L2N, bool ALIGNED>
__global__ __launch_bounds__(256, packed_dkdv_waves<D>()) void packed_dkdv_kernel(PackedBwdParams p) {
  typedef Dkdv16Lay<D> Lay;
  constexpr int BQ = 64, CPR = D / 8, NS = D / 32, NDB = D / 16;
  constexpr int PF = 2;              // LDS fragments read PF steps ahead
  constexpr int RPI = 64 / CPR;      // tile rows per copy instruction
  constexpr int PW = BQ / RPI / 4;   // copy instruction pairs per wave and tile
  constexpr int EA = 4 / NS;         // weights per S/dP step (block b - 1)
  constexpr int CE = NDB / 4;        // dV/dK steps per weight of block 3
  __shared__ __attribute__((aligned(16))) bf16 Qs0[BQ * D];
  __shared__ __attribute__((aligned(16))) bf16 Qs1[BQ * D];
  __shared__ __attribute__((aligned(16))) bf16 dOs0[BQ * D];
  __shared__ __attribute__((aligned(16))) bf16 dOs1[BQ * D];
  __shared__ __attribute__((aligned(16))) float st0[BQ];
  __shared__ __attribute__((aligned(16))) float st1[BQ];
  __shared__ __attribute__((aligned(16))) float di0[BQ];
  __shared__ __attribute__((aligned(16))) float di1[BQ];

  const int kvh = blockIdx.x % p.Hkv, G = p.G;
  int item = blockIdx.x / p.Hkv;
  if (p.dsink) {
    if (item < G) {
      packed_sink_grad(p, kvh, item);
      return;
    }
    item -= G;
  }
  const int range = item % p.dkdv_parts;  // of the rows, in the order in which they are streamed
  item /= p.dkdv_parts;
  const int lane = threadIdx.x & 63, g = lane >> 4, l16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // wave-uniform
  // Keys: one row a token; the first keys of a sequence, which the most rows see, are its last tile.
  const PackedSeq f = packed_find_heavy(p.cu, p.N, p.S, 1, PK_KEYS, item, packed_slots(p.N, 1, p.S, PK_KEYS));
  const int k0 = ((f.len + PK_KEYS - 1) / PK_KEYS - 1 - f.tile) * PK_KEYS;
  if (f.tile < 0 || k0 < 0) return;
  const size_t dk_base = ((size_t)f.start * p.Hkv + kvh) * D;
  if (f.s == p.S) {  // tokens behind the last sequence
    const bf16x8 z = {};
    for (int i = threadIdx.x; range == 0 && i < min(PK_KEYS, f.len - k0) * CPR; i += 256) {
      const size_t at = dk_base + (size_t)(k0 + i / CPR) * p.Hkv * D + 8 * (i % CPR);
      *reinterpret_cast<bf16x8*>(p.dk + at) = z;
      *reinterpret_cast<bf16x8*>(p.dv + at) = z;
    }
    return;
  }
  const int key_in = wave * 16 + l16;  // this lane's key within the workgroup's
  const int mykey = k0 + key_in;
  const bool live = mykey < f.len;
  const int log2n = p.sc.log2n;
  const float b2 = p.sc.b;
  const int rows = (f.len - k0) * G;              // rows from the first key's token on
  const int nq = ceil_div(rows, BQ);
  const int nmask = min(ceil_div((PK_KEYS - 1) * G, BQ), nq);  // tiles with rows before the last key
  const int dead_below = key_in * G;              // rows before this lane's key
  int q0 = 0, q1 = nq;                            // this workgroup's row tiles, counted from the last rows
  if (p.dkdv_parts > 1) {
    const int per = ceil_div(nq, p.dkdv_parts);
    q0 = min(range * per, nq);
    q1 = min(q0 + per, nq);
  }

  // Copies of row tile j into LDS in this layout (lane l of an instruction writes 16 bytes at
  // base + 16 l). Row x of the tile is token tb + (rem + x) / G, head (rem + x) % G of the group;
  // rows past the sequence are kept off memory and land as zeros.
  const int inv_g = 65536 / G + 1;  // (y * inv_g) >> 16 = y / G for y G < 65536
  const bf16* qbase = p.q + (size_t)(f.start + k0) * p.q_ts + (size_t)kvh * G * p.q_hs;
  const bf16* dobase = p.dO + (size_t)(f.start + k0) * p.do_ts + (size_t)kvh * G * p.do_hs;
  const size_t sbase = (size_t)kvh * p.N * G + (size_t)(f.start + k0) * G;
  const int lrow = lane / CPR;
  const int chunkb = 16 * ((lane % CPR) ^ Lay::swz(lrow));
  const int q_row = (lrow / G * (int)p.q_ts + lrow % G * (int)p.q_hs) * 2;
  const int o_row = (lrow / G * (int)p.do_ts + lrow % G * (int)p.do_hs) * 2;
  struct Tile {
    const bf16 *q, *o;
    int rem, left;  // first row's head; rows left from the tile's first
  };
  // The tiles from the last rows to the first: workgroups of one sequence and head that run at the
  // same time then read the same rows, out of the L2, wherever their keys lie (packed documents of
  // 16384 tokens, 16 heads over 4, D = 128: 545 us from the first rows on, 418 us so then). The next
  // tile's first token and head are kept up without a division.
  const int step_t = BQ / G, step_h = BQ - step_t * G;
  int next_r = (nq - 1 - q0) * BQ, next_t = next_r / G, next_h = next_r - next_t * G;
  auto source = [&]() {
    const bool some = next_r >= 0;
    const size_t t = some ? next_t : 0;
    const Tile now{qbase + t * p.q_ts, dobase + t * p.do_ts, next_h, some ? rows - next_r : 0};
    next_r -= BQ;
    next_t -= step_t;
    next_h -= step_h;
    if (next_h < 0) {
      next_h += G;
      --next_t;
    }
    return now;
  };
  auto dma_part = [&](bf16* la, bf16* lb, const Tile& t, int j) {
    auto lla = LDS_PTR(bf16, la);
    auto llb = LDS_PTR(bf16, lb);
    asm volatile("" : "+s"(lla), "+s"(llb));
    const int J = wave * PW + j;
    const int col = chunkb ^ (16 * Lay::swz(RPI * j));  // 16 rows a wave: the swizzle's period
    int qo, oo, qn = 0x7ffffff0, on = 0x7ffffff0;
    if constexpr (ALIGNED) {
      const int tok = RPI * J / G, left = min(t.left, BQ) / G;  // whole tokens either way
      qo = q_row + col + tok * (int)p.q_ts * 2;
      oo = o_row + col + tok * (int)p.do_ts * 2;
      qn = left * (int)p.q_ts * 2;
      on = left * (int)p.do_ts * 2;
    } else {
      const int x = RPI * J + lrow, y = t.rem + x;
      const int dt = (y * inv_g) >> 16, gh = y - dt * G;
      const bool in = x < t.left;
      qo = in ? (dt * (int)p.q_ts + gh * (int)p.q_hs) * 2 + col : -16;
      oo = in ? (dt * (int)p.do_ts + gh * (int)p.do_hs) * 2 + col : -16;
    }
    const __amdgpu_buffer_rsrc_t rq = __builtin_amdgcn_make_buffer_rsrc((void*)t.q, (short)0, qn, BUF_RSRC_WORD3);
    const __amdgpu_buffer_rsrc_t ro = __builtin_amdgcn_make_buffer_rsrc((void*)t.o, (short)0, on, BUF_RSRC_WORD3);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rq, lla + J * 512, 16, qo, 0, 0, 0);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(ro, llb + J * 512, 16, oo, 0, 0, 0);
  };
  // Statistics of a row tile (stat by wave 0, di by wave 1); rows past the sequence are zeros.
  auto stat_dma = [&](float* ls, float* ld, const Tile& t) {
    const int left = min(max(t.left, 0), BQ);
    const size_t at = sbase + (left > 0 ? rows - t.left : 0);
    const __amdgpu_buffer_rsrc_t rst = __builtin_amdgcn_make_buffer_rsrc((void*)(p.stat + at), (short)0, left * 4, BUF_RSRC_WORD3);
    const __amdgpu_buffer_rsrc_t rdi = __builtin_amdgcn_make_buffer_rsrc((void*)(p.ndi + at), (short)0, left * 4, BUF_RSRC_WORD3);
    if (wave == 0) __builtin_amdgcn_raw_ptr_buffer_load_lds(rst, LDS_PTR(void, ls), 4, lane * 4, 0, 0, 0);
    if (wave == 1) __builtin_amdgcn_raw_ptr_buffer_load_lds(rdi, LDS_PTR(void, ld), 4, lane * 4, 0, 0, 0);
  };
  auto lds_at = [](int row, int col) { return row * D + (((col >> 3) ^ Lay::swz(row)) << 3) + (col & 7); };
  {
    const Tile t = source();
#pragma unroll
    for (int j = 0; j < PW; ++j) dma_part(Qs0, dOs0, t, j);
    stat_dma(st0, di0, t);
  }
  // K (scaled as the queries are in the forward: an exact power of two) and V fragments of this
  // wave's keys; keys past the sequence are zero.
  bf16x8 kf[NS], vf[NS];
  {
    const size_t key = (size_t)(f.start + min(mykey, f.len - 1));
    const bf16* K = p.k + key * p.k_ts + (size_t)kvh * p.k_hs;
    const bf16* V = p.v + key * p.v_ts + (size_t)kvh * p.v_hs;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      kf[s] = ld8(K + Lay::dcol(g, s));
      vf[s] = ld8(V + Lay::dcol(g, s));
    }
    keep_own_row<NS>(kf, live);
    keep_own_row<NS>(vf, live);
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) kf[s][j] = f2bf((float)kf[s][j] * p.sc.qmul);
  }
  floatx4 dk[NDB], dv[NDB];
#pragma unroll
  for (int db = 0; db < NDB; ++db) {
    dk[db] = floatx4{};
    dv[db] = floatx4{};
  }
  const int qoff = Lay::quad(g);
  int a_off[NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) a_off[s] = lds_at(Lay::arow(l16), Lay::dcol(g, s));
  int t_off[NDB];
#pragma unroll
  for (int db = 0; db < NDB; ++db) t_off[db] = lds_at(qoff + (l16 >> 2), 16 * db + 4 * (lane & 3));

  constexpr int RING = PF + 1;
  bf16x8 aq[RING], ao[RING];  // row fragments of Q / dO, PF steps ahead
  __builtin_amdgcn_s_waitcnt(VMCNT0);
  __syncthreads();
#pragma unroll
  for (int t = 0; t < PF; ++t) {
    aq[t] = ld8(Qs0 + (t / NS) * 16 * D + a_off[t % NS]);
    ao[t] = ld8(dOs0 + (t / NS) * 16 * D + a_off[t % NS]);
  }
  constexpr int VE = 14;  // VALU instructions per score (scheduling hint)

  auto tile = [&](auto bufc, auto maskc, int qt) {
    constexpr int BUF = decltype(bufc)::value;
    constexpr bool MASKED = decltype(maskc)::value;
    const bf16* Qs = BUF ? Qs1 : Qs0;
    const bf16* dOs = BUF ? dOs1 : dOs0;
    bf16* Qn = BUF ? Qs0 : Qs1;
    bf16* dOn = BUF ? dOs0 : dOs1;
    float* stn = BUF ? st0 : st1;
    float* din = BUF ? di0 : di1;
    const float* sts = BUF ? st1 : st0;
    const float* dis = BUF ? di1 : di0;
    const Tile next = source();
    const int row0 = (nq - 1 - qt) * BQ;  // the tile's first row
    floatx4 s[4], dp[4];
    floatx4 sv[2];  // statistics of a block's rows (slot = block & 1); dP's sum starts from - di
    bf16x8 pa[2], da[2];
    float pw[4], dsx[4];
    bf16x8 cf[RING][2];     // transposed dO / Q fragments of the dV/dK steps, PF steps ahead

    auto a_step = [&](int t) {
      const int b = t / NS, st = t % NS, tn = t + PF;
      if (tn < 4 * NS) {
        aq[tn % RING] = ld8(Qs + (tn / NS) * 16 * D + a_off[tn % NS]);
        ao[tn % RING] = ld8(dOs + (tn / NS) * 16 * D + a_off[tn % NS]);
      }
      s[b] = mfma16_bf16(aq[t % RING], kf[st], s[b]);
      dp[b] = mfma16_bf16(ao[t % RING], vf[st], dp[b]);
    };
    auto load_stats = [&](int b) {
      sv[b & 1] = *reinterpret_cast<const floatx4*>(sts + 16 * b + qoff);
      dp[b] = *reinterpret_cast<const floatx4*>(dis + 16 * b + qoff);
    };
    // P and dS of row 16 b + qoff + i of the tile.
    auto elem = [&](int b, int i) {
      const bool dead = MASKED && row0 + 16 * b + qoff + i < dead_below;
      packed_elem<L2N, false>(s[b][i], dp[b][i], sv[b & 1][i], b2, log2n, dead, pw[i], dsx[i]);
      const int c = b >> 1, j0 = 4 * (b & 1);
      if (i & 1) {
        pa[c][j0 + i - 1] = f2bf(pw[i - 1]);
        pa[c][j0 + i] = f2bf(pw[i]);
        da[c][j0 + i - 1] = f2bf(dsx[i - 1]);
        da[c][j0 + i] = f2bf(dsx[i]);
      }
    };
    auto c_load = [&](int u) {
      const int c = u / NDB, db = u % NDB;
      cf[u % RING][0] = tr_frag_at(dOs + 32 * c * D, t_off[db], t_off[db] + 16 * D);
      cf[u % RING][1] = tr_frag_at(Qs + 32 * c * D, t_off[db], t_off[db] + 16 * D);
    };
    auto c_step = [&](int u) {
      const int c = u / NDB, db = u % NDB;
      dv[db] = mfma16_bf16(pa[c], cf[u % RING][0], dv[db]);
      dk[db] = mfma16_bf16(da[c], cf[u % RING][1], dk[db]);
    };
#pragma unroll
    for (int b = 0; b < 4; ++b) s[b] = floatx4{};
    // S, dP steps: block b's carry the weights of block b - 1; block 0's the next tile's copy
    // (past the last tile nothing is read and zeros land in the unused buffer set).
    load_stats(0);
#pragma unroll
    for (int t = 0; t < 4 * NS; ++t) {
      const int b = t / NS, st = t % NS;
      if (st == 0 && b >= 1) load_stats(b);
      a_step(t);
      if (b == 0) {
        if (st < PW) dma_part(Qn, dOn, next, st);
        if (st == NS - 1) {
#pragma unroll
          for (int j = NS; j < PW; ++j) dma_part(Qn, dOn, next, j);
          stat_dma(stn, din, next);
        }
        step_order_r<2, 0>(t + PF < 4 * NS ? 2 : 0);
      } else {
#pragma unroll
        for (int e = 0; e < EA; ++e) elem(b - 1, EA * st + e);
        if (t >= 4 * NS - PF) c_load(t - (4 * NS - PF));
        step_order_r<2, VE * EA>((t + PF < 4 * NS ? 2 : 0) + (st == 0 ? 2 : 0) + (t >= 4 * NS - PF ? 4 : 0));
      }
    }
    // dV, dK steps: the first half (blocks 0, 1) under the weights of block 3.
#pragma unroll
    for (int u = 0; u < 2 * NDB; ++u) {
      if (u + PF < 2 * NDB) c_load(u + PF);
      c_step(u);
      if (u < NDB && u % CE == 0) {
        elem(3, u / CE);
        step_order_r<2, VE>(u + PF < 2 * NDB ? 4 : 0);
      } else {
        step_order_r<2, 0>(u + PF < 2 * NDB ? 4 : 0);
      }
    }
    __builtin_amdgcn_s_waitcnt(VMCNT0);  // this wave's copies of the next tile have landed
    __syncthreads();                     // the next buffer set is complete; this one is free
#pragma unroll
    for (int t = 0; t < PF; ++t) {
      aq[t] = ld8(Qn + (t / NS) * 16 * D + a_off[t % NS]);
      ao[t] = ld8(dOn + (t / NS) * 16 * D + a_off[t % NS]);
    }
  };
  // Whether a row of these tiles took the careful form.
  bool careful = false;
  {
    const int slot0 = f.start * G / PK_ROWS + f.s, last = (f.len * G - 1) / PK_ROWS;
    for (int i = k0 * G / PK_ROWS + lane; i <= last; i += 64) careful |= p.care[(size_t)(slot0 + i) * p.Hkv + kvh] != 0;
    careful = __any(careful);
  }
  if (!careful) {
    // In pairs of tiles, as in the forward.
    const int full = q0 + (max(min(nq - nmask, q1) - q0, 0) & ~1);
    int qt = q0;
    for (; qt < full; qt += 2) {
      tile(std::integral_constant<int, 0>{}, std::false_type{}, qt);
      tile(std::integral_constant<int, 1>{}, std::false_type{}, qt + 1);
    }
    for (; qt < q1; qt += 2) {
      tile(std::integral_constant<int, 0>{}, std::true_type{}, qt);
      if (qt + 1 >= q1) break;
      tile(std::integral_constant<int, 1>{}, std::true_type{}, qt + 1);
    }
  } else {
    next_r = (nq - 1 - q0) * BQ;
    next_t = next_r / G;
    next_h = next_r - next_t * G;
    for (int qt = q0; qt < q1; ++qt) {
      __syncthreads();  // every wave is done with the tile before
      const Tile now = source();
#pragma unroll
      for (int j = 0; j < PW; ++j) dma_part(Qs0, dOs0, now, j);
      stat_dma(st0, di0, now);
      __builtin_amdgcn_s_waitcnt(VMCNT0);
      __syncthreads();
      for (int c = 0; c < 2; ++c) {  // halves of 32 rows
        bf16x8 pa, da;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int b = 2 * c + u;
          floatx4 s = {}, dp = *reinterpret_cast<const floatx4*>(di0 + 16 * b + qoff);
#pragma unroll
          for (int st = 0; st < NS; ++st) {
            s = mfma16_bf16(ld8(Qs0 + b * 16 * D + a_off[st]), kf[st], s);
            dp = mfma16_bf16(ld8(dOs0 + b * 16 * D + a_off[st]), vf[st], dp);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int x = 16 * b + qoff + i;
            float pw, ds;
            packed_elem<0, true>(s[i], dp[i], st0[x], b2, log2n, (nq - 1 - qt) * BQ + x < dead_below, pw, ds);
            pa[4 * u + i] = f2bf(pw);
            da[4 * u + i] = f2bf(ds);
          }
        }
#pragma unroll
        for (int db = 0; db < NDB; ++db) {
          dv[db] = mfma16_bf16(pa, tr_frag_at(dOs0 + 32 * c * D, t_off[db], t_off[db] + 16 * D), dv[db]);
          dk[db] = mfma16_bf16(da, tr_frag_at(Qs0 + 32 * c * D, t_off[db], t_off[db] + 16 * D), dk[db]);
        }
      }
    }
  }

  // Register i of d block db holds key 16 wave + 4 g + i, column 16 db + l16.
  if (p.dkdv_parts > 1) {
    const size_t sum = (size_t)range * p.N * p.Hkv * D + dk_base;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int key = k0 + wave * 16 + 4 * g + i;
      if (key < f.len) {
#pragma unroll
        for (int db = 0; db < NDB; ++db) {
          const size_t o = sum + (size_t)key * p.Hkv * D + 16 * db + l16;
          p.dk_sum[o] = dk[db][i];
          p.dv_sum[o] = dv[db][i];
        }
      }
    }
    return;
  }
  const float slope = (float)(1 << log2n) * p.sc.qmul;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int key = k0 + wave * 16 + 4 * g + i;
    if (key < f.len) {
#pragma unroll
      for (int db = 0; db < NDB; ++db) {
        const size_t o = dk_base + (size_t)key * p.Hkv * D + 16 * db + l16;
        p.dk[o] = f2bf(dk[db][i] * slope);
        p.dv[o] = f2bf(dv[db][i]);
      }
    }
  }
}

// dQ, dK and dV whose keys or rows were split: the ranges' sums in their order, four columns a thread: dQ (dq_parts > 1), then dK and dV. The tokens
// behind the last sequence have their zeros already.
__global__ __launch_bounds__(256) void packed_join_kernel(PackedBwdParams p, int D) {
  const size_t nq = p.dq_parts > 1 ? (size_t)p.N * p.H * D : 0, nk = p.dkdv_parts > 1 ? (size_t)p.N * p.Hkv * D : 0;
  size_t i = ((size_t)blockIdx.x * 256 + threadIdx.x) * 4;
  const float* src = p.dq_sum;
  bf16* out = p.dq;
  size_t n = nq;
  int parts = p.dq_parts, heads = p.H;
  bool scaled = true;
  if (i >= nq) {
    i -= nq;
    scaled = i < nk;
    if (!scaled) i -= nk;
    if (i >= nk) return;
    src = scaled ? p.dk_sum : p.dv_sum;
    out = scaled ? p.dk : p.dv;
    n = nk;
    parts = p.dkdv_parts;
    heads = p.Hkv;
  }
  if ((int)(i / ((size_t)heads * D)) >= packed_start(p.cu, p.S, p.N)) return;
  floatx4 sum = *reinterpret_cast<const floatx4*>(src + i);
  for (int r = 1; r < parts; ++r) sum += *reinterpret_cast<const floatx4*>(src + r * n + i);
  if (scaled) sum *= (float)(1 << p.sc.log2n) * p.sc.qmul;
  bf16x4 b;
#pragma unroll
  for (int e = 0; e < 4; ++e) b[e] = f2bf(sum[e]);
  *reinterpret_cast<bf16x4*>(out + i) = b;
}

static bool packed_aligned(const PackedBwdParams& p, int D) {
  const int rows = 512 / D;  // of a copy instruction
  const auto behind = [&](long ts, long hs) { return (p.G - 1) * hs + D <= ts; };
  return rows % p.G == 0 && behind(p.q_ts, p.q_hs) && behind(p.do_ts, p.do_hs);
}

template <int D, int L2N>
static void launch_bwd(const PackedBwdParams& p, hipStream_t st) {
  {
    KTimer t("packed_dq", st);
    const dim3 grid(p.Hkv * p.dq_parts * packed_slots(p.N, p.G, p.S, PK_ROWS));
    hipLaunchKernelGGL((packed_dq_kernel<D, L2N>), grid, dim3(256), 0, st, p);
  }
  {
    KTimer t("packed_dkdv", st);
    const dim3 grid(p.Hkv * (p.dkdv_parts * packed_slots(p.N, 1, p.S, PK_KEYS) + (p.dsink ? p.G : 0)));
    if (packed_aligned(p, D)) hipLaunchKernelGGL((packed_dkdv_kernel<D, L2N, true>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((packed_dkdv_kernel<D, L2N, false>), grid, dim3(256), 0, st, p);
  }
  const size_t n = (size_t)p.N * D * ((p.dq_parts > 1 ? p.H : 0) + (p.dkdv_parts > 1 ? 2 * p.Hkv : 0));
  if (n == 0) return;
  KTimer t("packed_join", st);
  hipLaunchKernelGGL(packed_join_kernel, dim3((unsigned)((n / 4 + 255) / 256)), dim3(256), 0, st, p, D);
}

hipError_t launch_packed_bwd(const PackedBwdParams& p, int D, hipStream_t st) {
  if (D == 64) p.sc.log2n == 4 ? launch_bwd<64, 4>(p, st) : launch_bwd<64, 0>(p, st);
  else p.sc.log2n == 4 ? launch_bwd<128, 4>(p, st) : launch_bwd<128, 0>(p, st);
  return hipGetLastError();
}

}  // namespace alg
