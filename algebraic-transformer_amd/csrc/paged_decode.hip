// Attention of a few new tokens per sequence over a paged cache, bf16: a token's G queries at one
// key head (times the tokens, where there are several) make 16 or 32 rows, and the work is reading
// the held keys and values once.
//
// One workgroup = 4 waves = the rows of one sequence and key head over one range of its keys (the
// ranges are joined by packed_combine_kernel). Each wave takes every fourth block of 32 keys and
// keeps a state of its own, so that nothing synchronises until the waves' states are joined
// through LDS at the end:
//   S^T = K Q^T (16x16x32 MFMA; A = K straight from memory to registers: lane l holds 8 elements
//   of key l % 16), weights in registers, O^T += V^T P^T, where the 32 keys are numbered
//   (lane group g, slot j) -> 4 g + j % 4 + 16 (j / 4), the order in which S^T leaves the MFMA;
//   V comes through a private LDS tile (direct copies) and is read transposed.
// While a wave computes a block, the next one's 16 KB (D = 128) are under way: up to 128 KB a CU.
// (One workgroup of 16 waves for a whole short sequence, without a launch to join ranges, was slower
// than ranges: a CU alone reads about 50 GB/s, and 16 heads' 1024 keys took 23 us, 17 us in ranges.)
// A group of 16 keys lies in one page (pages hold a multiple of 16 keys): its page number is one
// scalar load, whose counter is not the vector loads', so that looking a page up never waits for
// the keys and values in flight.
// Bytes bound it, so that the weights' rounding to bf16 need not be: they go in as the sum of two bf16
// numbers (exact to 2^-17), twice the products of P V, at the same time to 1 % (64 requests over 200000
// keys: 149.1, 149.1 us).
// Measured: those 64 requests, 32 heads over 8 of 128, 820 MB: 150 us, 5.5 TB/s (a copy's 5.1 counts its
// writes); one over 131001 keys, 16 heads over 4, 268 MB, in 64 ranges: 45 us and 8 for joining them; four
// of 900 keys: 12 and 6, of which launches are about 5 each.
// Keys past the range read as zeros (buffer descriptors end there) and have no weight.
// The weights' two forms: packed_common.h; a wave whose rows need it goes over its blocks again in
// the careful form.
#include <type_traits>

#include "launchers.h"
#include "packed_common.h"

namespace alg {

template <int D, int RT, int L2N>
__global__ __launch_bounds__(256, 2) void paged_decode_kernel(PackedParams p) {
  static_assert(D == 64 || D == 128, "head_dim");
  constexpr int WAVES = 4;
  constexpr int NS = D / 32, NDB = D / 16, CPR = D / 8, RPI = 64 / CPR, PW = 16 / RPI;
  constexpr int LOADS = 2 * NS + 2 * PW;  // vector loads and copies of one block of 32 keys
  constexpr int ROWS = 16 * RT;
  constexpr int BLK = 32;
  __shared__ __attribute__((aligned(16))) bf16 Vs[WAVES * 2 * BLK * D];
  __shared__ float jT[WAVES][ROWS], jZ[WAVES][ROWS];
  static_assert(WAVES * ROWS * D * sizeof(float) <= sizeof(Vs), "the waves' sums fit the V tiles");

  const int lane = threadIdx.x & 63, g = lane >> 4, l16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Workgroups: key head, range of keys, item.
  const int kvh = blockIdx.x % p.Hkv, unit = blockIdx.x / p.Hkv, range = unit % p.nsplit;
  const PackedSeq f = packed_find<false>(p.cu, p.N, p.S, p.G, ROWS, unit / p.nsplit, gridDim.x / p.Hkv / p.nsplit);
  const int G = p.G, R = f.len * G, r0 = f.tile * ROWS;
  if (f.tile < 0 || r0 >= R) return;
  const int nrow = min(ROWS, R - r0);  // live rows of the tile
  if (f.s == p.S) {                    // tokens behind the last sequence
    if (range == 0)
      for (int i = threadIdx.x; i < nrow * (D / 8); i += 64 * WAVES) {
        const int r = r0 + i / (D / 8), tok = r / G, head = kvh * G + r - tok * G;
        const bf16x8 z = {};
        *reinterpret_cast<bf16x8*>(p.o + ((size_t)(f.start + tok) * p.H + head) * D + 8 * (i % (D / 8))) = z;
      }
    return;
  }
  const int held = max(p.kv_lens[f.s], 0), L = min(held, p.width * p.page);  // keys; those that the table reaches
  const int off = held - f.len;
  const int kend = min(max(off + (r0 + nrow - 1) / G + 1, 0), L);  // keys that some row sees: [0, kend)
  // This workgroup's blocks of 32 keys: an equal share, of at least DECODE_RANGE keys.
  int b0 = 0, b1 = ceil_div(kend, BLK);
  if (p.nsplit > 1) {
    const int per = max(ceil_div(b1, p.nsplit), DECODE_RANGE / BLK);
    b0 = min(range * per, b1);
    b1 = min(b0 + per, b1);
  }

  bf16x8 qf[RT][NS];
  int mypos[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = r0 + 16 * rt + l16;
    const bool live = r < R;
    const int rc = min(r, R - 1), tok = rc / G, head = kvh * G + rc - tok * G;
    mypos[rt] = live ? off + tok : -1;
    const bf16* Q = p.q + (size_t)(f.start + tok) * p.q_ts + (size_t)head * p.q_hs + 8 * g;
#pragma unroll
    for (int st = 0; st < NS; ++st) qf[rt][st] = ld8(Q + 32 * st);
    keep_own_row<NS>(qf[rt], live);
#pragma unroll
    for (int st = 0; st < NS; ++st)
#pragma unroll
      for (int j = 0; j < 8; ++j) qf[rt][st][j] = f2bf((float)qf[rt][st][j] * p.sc.qmul);
  }

  const int log2n = p.sc.log2n;
  const float b2 = p.sc.b;
  const auto* trow = (const __attribute__((address_space(4))) int*)(p.table + (size_t)f.s * p.width);
  const bf16* kbase = p.k + (size_t)kvh * p.k_hs;
  const bf16* vbase = p.v + (size_t)kvh * p.v_hs;
  bf16* vbuf = Vs + wave * 2 * BLK * D;
  const int lrow = lane / CPR;
  const int k_off = (l16 * (int)p.k_ts + 8 * g) * 2;
  const int v_off = lrow * (int)p.v_ts * 2;
  const int chunkb = 16 * ((lane % CPR) ^ swz_chunk<CPR>(lrow));
  int t_off[NDB];  // transposed V fragments: keys 4 g + (0..3), columns 16 db + (0..15)
#pragma unroll
  for (int db = 0; db < NDB; ++db) t_off[db] = swz_at<CPR>(4 * g + (l16 >> 2), 16 * db + 4 * (lane & 3));

  bool bad = false;
  typedef bf16x8 KBlock[2][NS];
  auto load = [&](int blk, KBlock& kf, bf16* vl) __attribute__((always_inline)) {
    auto ll = LDS_PTR(bf16, vl);
    asm volatile("" : "+s"(ll));
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int key = blk * BLK + 16 * u;
      int rows = blk < b1 ? min(max(kend - key, 0), 16) : 0;
      int id = 0, prow = 0;
      if (rows > 0) {
        const int pi = key / p.page;
        prow = key - pi * p.page;
        id = trow[pi];
        if ((unsigned)id >= (unsigned)p.pages) {  // never read; the rows' results become NaN
          bad = true;
          id = rows = 0;
        }
      }
      const bf16* K = kbase + (size_t)id * p.k_ps + (size_t)prow * p.k_ts;
      const bf16* V = vbase + (size_t)id * p.v_ps + (size_t)prow * p.v_ts;
      const int kn = rows > 0 ? ((rows - 1) * (int)p.k_ts + D) * 2 : 0, vn = rows > 0 ? ((rows - 1) * (int)p.v_ts + D) * 2 : 0;
      const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc((void*)K, (short)0, kn, BUF_RSRC_WORD3);
      const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc((void*)V, (short)0, vn, BUF_RSRC_WORD3);
#pragma unroll
      for (int st = 0; st < NS; ++st) {
        const auto v = __builtin_amdgcn_raw_buffer_load_b128(rk, k_off + 64 * st, 0, 0);
        const uint4 raw = make_uint4(v[0], v[1], v[2], v[3]);
        kf[u][st] = *reinterpret_cast<const bf16x8*>(&raw);
      }
#pragma unroll
      for (int j = 0; j < PW; ++j) {
        const int J = u * PW + j;
        const int col = chunkb ^ (16 * swz_chunk<CPR>(RPI * j));
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, ll + J * 512, 16, RPI * j * (int)p.v_ts * 2 + v_off + col, 0, 0, 0);
      }
    }
  };

  floatx4 oacc[RT][NDB];
  float lsum[RT], T[RT], shift[RT];  // weights (t shift)^n, T = 1 / shift (0: no key yet)
  int count[RT];                     // keys that the row saw
  auto reset = [&](float t) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      lsum[rt] = 0.0f;
      T[rt] = shift[rt] = t;
      count[rt] = 0;
#pragma unroll
      for (int db = 0; db < NDB; ++db) oacc[rt][db] = floatx4{};
    }
  };

  auto compute = [&](auto carec, int blk, const KBlock& kf, const bf16* vl) __attribute__((always_inline)) {
    constexpr bool CARE = decltype(carec)::value;
    bf16x8 pf[RT], pl[RT];  // the weights rounded, and what that left: with both, o has its own rounding alone
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      floatx4 s[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        s[u] = floatx4{};
#pragma unroll
        for (int st = 0; st < NS; ++st) s[u] = mfma16_bf16(kf[u][st], qf[rt][st], s[u]);
      }
      const int seen = mypos[rt] + 1 - blk * BLK;  // keys of the block up to the row's position
      count[rt] += min(max(seen, 0), BLK);
      float t[8], top = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int u = j >> 2, i = j & 3;
        float r;
        t[j] = CARE ? weight_t_careful(s[u][i], b2, r) : pow2n<L2N>(weight_t(s[u][i], b2, r), log2n);
        keep_here(t[j]);
        if (16 * u + 4 * g + i >= seen) t[j] = 0.0f;
        if (CARE) top = fmaxf(top, t[j]);
      }
      if constexpr (CARE) {
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        if (top > T[rt]) {
          const float fall = pow2n<0>(T[rt] / top, log2n);
          T[rt] = top;
          shift[rt] = 1.0f / top;
          lsum[rt] *= fall;
#pragma unroll
          for (int db = 0; db < NDB; ++db)
#pragma unroll
            for (int i = 0; i < 4; ++i) oacc[rt][db][i] *= fall;
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float w = CARE ? pow2n<0>(t[j] * shift[rt], log2n) : t[j];
        lsum[rt] += w;
        pf[rt][j] = f2bf(w);
        pl[rt][j] = f2bf(w - (float)pf[rt][j]);
      }
    }
#pragma unroll
    for (int db = 0; db < NDB; ++db) {
      const bf16x8 vf = tr_frag_at(vl, t_off[db], t_off[db] + 16 * D);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        oacc[rt][db] = mfma16_bf16(vf, pf[rt], oacc[rt][db]);
        oacc[rt][db] = mfma16_bf16(vf, pl[rt], oacc[rt][db]);
      }
    }
    // The block's V tile is read before the next copy into it is issued.
    __builtin_amdgcn_s_waitcnt(vmcnt_lgkm0_imm(63));
    __builtin_amdgcn_sched_barrier(0);
  };

  // Blocks b0 + wave, + WAVES, ...; a block past the range loads nothing (empty descriptors).
  KBlock ka, kb;
  auto sweep = [&](auto carec) __attribute__((always_inline)) {
    load(b0 + wave, ka, vbuf);
    for (int blk = b0 + wave; blk < b1; blk += 2 * WAVES) {
      load(blk + WAVES, kb, vbuf + BLK * D);
      __builtin_amdgcn_s_waitcnt(vmcnt_imm(LOADS));
      __builtin_amdgcn_sched_barrier(0);
      compute(carec, blk, ka, vbuf);
      load(blk + 2 * WAVES, ka, vbuf);
      __builtin_amdgcn_s_waitcnt(vmcnt_imm(LOADS));
      __builtin_amdgcn_sched_barrier(0);
      if (blk + WAVES < b1) compute(carec, blk + WAVES, kb, vbuf + BLK * D);
    }
    __builtin_amdgcn_s_waitcnt(VMCNT0);  // copies into the tiles that are written next
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {  // the row's sum over the lane groups
      lsum[rt] += __shfl_xor(lsum[rt], 16, 64);
      lsum[rt] += __shfl_xor(lsum[rt], 32, 64);
    }
  };
  bool careful = isinf(p.sc.low);
  reset(1.0f);
  if (!careful) {
    sweep(std::false_type{});
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) careful |= needs_care(lsum[rt], count[rt], p.sc.low);
    careful = __any(careful);
  }
  if (careful) {
    reset(0.0f);
    sweep(std::true_type{});
  }

  // The waves' states, joined in wave order.
  float* sO = reinterpret_cast<float*>(Vs);
  __syncthreads();
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    if (g == 0) {
      jT[wave][16 * rt + l16] = T[rt];
      // A position behind the table's end holds no key of its own.
      jZ[wave][16 * rt + l16] = bad || mypos[rt] >= L ? __builtin_nanf("") : lsum[rt];
    }
#pragma unroll
    for (int db = 0; db < NDB; ++db)
      *reinterpret_cast<floatx4*>(sO + ((wave * ROWS) + 16 * rt + l16) * D + 16 * db + 4 * g) = oacc[rt][db];
  }
  __syncthreads();
  constexpr int TPR = 64 * WAVES / ROWS, CPT = D / TPR;  // threads a row, columns a thread
  typedef float fvec __attribute__((ext_vector_type(CPT)));
  typedef bf16 bvec __attribute__((ext_vector_type(CPT)));
  const int row = threadIdx.x / TPR, c0 = (threadIdx.x % TPR) * CPT;
  const int r = r0 + row;
  if (r >= R) return;
  const int tok = r / G, head = kvh * G + r - tok * G;
  const bool sink = p.sink != nullptr && p.nsplit == 1;  // split: the sink joins in the combination
  float Tm = 0.0f, ts = 0.0f;
  if (sink) {
    float rr;
    Tm = ts = weight_t_careful(sink_score(p, head), b2, rr);
  }
#pragma unroll
  for (int w = 0; w < WAVES; ++w)
    if (jZ[w][row] != 0.0f) Tm = fmaxf(Tm, jT[w][row]);
  float Z = sink ? sink_weight(ts, Tm, log2n) : 0.0f;
  fvec acc = 0.0f;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    const float z = jZ[w][row];
    const float fw = z != 0.0f ? pow2n<0>(jT[w][row] / Tm, log2n) : 0.0f;
    Z += fw * z;
    acc += fw * *reinterpret_cast<const fvec*>(sO + (w * ROWS + row) * D + c0);  // zeros where z is
  }
  if (p.nsplit > 1) {
    const size_t part = (size_t)range * p.Hkv * p.N * G + (size_t)kvh * p.N * G + (size_t)f.start * G + r;
    if (c0 == 0) {
      p.part_zt[2 * part] = Z;
      p.part_zt[2 * part + 1] = Tm;
    }
    if (Z != 0.0f) *reinterpret_cast<fvec*>(p.part_o + part * D + c0) = acc;  // an empty range's is not read
    return;
  }
  const float inv = Z == 0.0f ? 0.0f : 1.0f / Z;
  bvec out;
#pragma unroll
  for (int e = 0; e < CPT; ++e) out[e] = f2bf(acc[e] * inv);
  *reinterpret_cast<bvec*>(p.o + ((size_t)(f.start + tok) * p.H + head) * D + c0) = out;
}

template <int D, int RT>
static void launch_decode(const PackedParams& p, hipStream_t st) {
  const dim3 grid(p.Hkv * p.nsplit * packed_slots(p.N, p.G, p.S, 16 * RT));
  if (p.sc.log2n == 4) hipLaunchKernelGGL((paged_decode_kernel<D, RT, 4>), grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL((paged_decode_kernel<D, RT, 0>), grid, dim3(256), 0, st, p);
}

hipError_t launch_paged_decode(const PackedParams& p, int D, int row_tiles, hipStream_t st) {
  {
    KTimer t("paged_decode", st);
    if (D == 64) row_tiles == 1 ? launch_decode<64, 1>(p, st) : launch_decode<64, 2>(p, st);
    else row_tiles == 1 ? launch_decode<128, 1>(p, st) : launch_decode<128, 2>(p, st);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.nsplit == 1) return e;
  return launch_packed_combine(p, D, st);
}

}  // namespace alg
