// Attention of a few new tokens per sequence over a paged cache of 8 bits: the work and its split over
// workgroups, waves and blocks of 32 keys are paged_decode.hip's, the weights' arithmetic
// packed_common.h's; the bytes are half. What differs is how they become operands:
//   * the stored values are bf16 numbers exactly (packed_common.h), so that the products and what they
//     round are those of a bf16 cache: o differs from the attention over the stored values by its
//     own rounding alone;
//   * K goes from memory to registers, 16 bytes a lane: lane group g holds elements 64 i + 16 g + (0..15)
//     of key l % 16, which feed two MFMA steps (the queries are laid out alike), converted with the
//     key's scale, one a lane;
//   * V comes through a private LDS tile and is read transposed in bytes (ds_read_b64_tr_b8: lane i
//     of a group of 16 receives element i % 8 of the 8 bytes that lane 2 e + i / 8 addresses, e < 8), eight
//     keys of a column, whose scales multiply the weights instead: a product by a power of two, which
//     rounds nothing.
// Memory bounds it where there are many keys: 64 requests of 200000 keys, 8 heads of 128: 91 us, 4.6 TB/s (VALU 38 %
// busy); one of 131001, 4 heads: 32 us and 5 for the join, 4.2 TB/s. 4 requests of 3600 keys, 4 heads: 20 us, a wave's
// blocks one after the other.
// V tile rows of D bytes, 16-byte chunk c of row r at c ^ f(r): the 16 rows that half a wave reads at one
// chunk lie in 16 different parts of the banks' 256 bytes.
#include <type_traits>

#include "launchers.h"
#include "packed_common.h"

namespace alg {

typedef int i32x2 __attribute__((ext_vector_type(2)));

template <int D>
__device__ __forceinline__ int swz8(int row) {
  if constexpr (D == 128) return ((row >> 1) & 3) | ((row >> 4) & 1) << 2;
  else return ((row >> 2) & 1) | ((row >> 4) & 1) << 1;
}

template <int D, int RT, int L2N>
__global__ __launch_bounds__(256, 2) void paged_decode_fp8_kernel(PackedParams p) {
  static_assert(D == 64 || D == 128, "head_dim");
  constexpr int WAVES = 4;
  constexpr int NK = D / 64, NDB = D / 16, CPR = D / 16, RPI = 64 / CPR, PW = 16 / RPI;
  constexpr int LOADS = 2 * (NK + PW + 2);  // vector loads and copies of one block of 32 keys
  constexpr int ROWS = 16 * RT;
  constexpr int BLK = 32;
  constexpr int TILE = BLK * D;  // bytes of a V tile
  constexpr int SUMS = WAVES * ROWS * D * 4, TILES = WAVES * 2 * TILE;
  __shared__ __attribute__((aligned(256))) uint8_t Vs[TILES > SUMS ? TILES : SUMS];
  __shared__ float jT[WAVES][ROWS], jZ[WAVES][ROWS];

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

  bf16x8 qf[RT][2 * NK];
  int mypos[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = r0 + 16 * rt + l16;
    const bool live = r < R;
    const int rc = min(r, R - 1), tok = rc / G, head = kvh * G + rc - tok * G;
    mypos[rt] = live ? off + tok : -1;
    const bf16* Q = p.q + (size_t)(f.start + tok) * p.q_ts + (size_t)head * p.q_hs + 16 * g;
#pragma unroll
    for (int st = 0; st < 2 * NK; ++st) qf[rt][st] = ld8(Q + 64 * (st >> 1) + 8 * (st & 1));
    keep_own_row<2 * NK>(qf[rt], live);
#pragma unroll
    for (int st = 0; st < 2 * NK; ++st)
#pragma unroll
      for (int j = 0; j < 8; ++j) qf[rt][st][j] = f2bf((float)qf[rt][st][j] * p.sc.qmul);
  }

  const int log2n = p.sc.log2n;
  const float b2 = p.sc.b;
  const auto* trow = (const __attribute__((address_space(4))) int*)(p.table + (size_t)f.s * p.width);
  const uint8_t* kbase = reinterpret_cast<const uint8_t*>(p.k) + (size_t)kvh * p.k_hs;
  const uint8_t* vbase = reinterpret_cast<const uint8_t*>(p.v) + (size_t)kvh * p.v_hs;
  const uint8_t* ksbase = p.ks + (size_t)kvh * p.ks_hs;
  const uint8_t* vsbase = p.vs + (size_t)kvh * p.vs_hs;
  uint8_t* vbuf = Vs + wave * 2 * TILE;
  const int k_off = l16 * (int)p.k_ts + 16 * g;
  const int v_off = (lane / CPR) * (int)p.v_ts;
  // Rows 8 J + lane / 8 (D = 128) or 16 J + lane / 4 of a copy: the swizzle's part that a lane has.
  const int chunkb = 16 * ((lane % CPR) ^ swz8<D>(lane / CPR));
  // Transposed V fragments: the lane's row (key slot e = l16 / 2), 8-byte half l16 % 2 of chunk db.
  const int e = l16 >> 1, trw = 4 * g + (e & 3) + 16 * (e >> 2);
  const int t_off = trw * D + 16 * swz8<D>(trw) + 8 * (l16 & 1);

  struct Block {
    u32x4 k[2][NK];
    unsigned ks[2], vs[2];  // the key l16's scale; those of keys 4 g + (0..3)
  };
  bool bad = false;
  auto load = [&](int blk, Block& b, uint8_t* vl) __attribute__((always_inline)) {
    auto ll = LDS_PTR(uint8_t, vl);
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
      const uint8_t* K = kbase + (size_t)id * p.k_ps + (size_t)prow * p.k_ts;
      const uint8_t* V = vbase + (size_t)id * p.v_ps + (size_t)prow * p.v_ts;
      const uint8_t* KS = ksbase + (size_t)id * p.ks_ps + prow;
      const uint8_t* VS = vsbase + (size_t)id * p.vs_ps + prow;
      const int kn = rows > 0 ? (rows - 1) * (int)p.k_ts + D : 0, vn = rows > 0 ? (rows - 1) * (int)p.v_ts + D : 0;
      const int sn = rows > 0 ? 16 : 0;  // a page holds all 16 places
      const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc((void*)K, (short)0, kn, BUF_RSRC_WORD3);
      const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc((void*)V, (short)0, vn, BUF_RSRC_WORD3);
      const __amdgpu_buffer_rsrc_t rks = __builtin_amdgcn_make_buffer_rsrc((void*)KS, (short)0, sn, BUF_RSRC_WORD3);
      const __amdgpu_buffer_rsrc_t rvs = __builtin_amdgcn_make_buffer_rsrc((void*)VS, (short)0, sn, BUF_RSRC_WORD3);
#pragma unroll
      for (int i = 0; i < NK; ++i) b.k[u][i] = __builtin_amdgcn_raw_buffer_load_b128(rk, k_off + 64 * i, 0, 0);
      b.ks[u] = __builtin_amdgcn_raw_buffer_load_b8(rks, l16, 0, 0);
      b.vs[u] = __builtin_amdgcn_raw_buffer_load_b32(rvs, 4 * g, 0, 0);
#pragma unroll
      for (int j = 0; j < PW; ++j) {
        const int J = u * PW + j;
        const int col = chunkb ^ (16 * swz8<D>(RPI * J));
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, ll + J * 1024, 16, RPI * j * (int)p.v_ts + v_off + col, 0, 0, 0);
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

  auto compute = [&](auto carec, int blk, const Block& b, const uint8_t* vl) __attribute__((always_inline)) {
    constexpr bool CARE = decltype(carec)::value;
    floatx4 s[RT][2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) s[rt][u] = floatx4{};
      const float unit = scale_value(b.ks[u]);
#pragma unroll
      for (int st = 0; st < 2 * NK; ++st) {
        const bf16x8 kf = values8(b.k[u][st >> 1][2 * (st & 1)], b.k[u][st >> 1][2 * (st & 1) + 1], unit);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) s[rt][u] = mfma16_bf16(kf, qf[rt][st], s[rt][u]);
      }
    }
    float vunit[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) vunit[j] = scale_value((b.vs[j >> 2] >> (8 * (j & 3))) & 255);
    bf16x8 pf[RT], pl[RT];  // the weights (times V's scale) rounded, and what that left
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int seen = mypos[rt] + 1 - blk * BLK;  // keys of the block up to the row's position
      count[rt] += min(max(seen, 0), BLK);
      float t[8], top = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int u = j >> 2, i = j & 3;
        float r;
        t[j] = CARE ? weight_t_careful(s[rt][u][i], b2, r) : pow2n<L2N>(weight_t(s[rt][u][i], b2, r), log2n);
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
        float wv = w * vunit[j];
        keep_here(wv);
        // A scale of 255 (a row that was not finite) reaches the rows that see it and no other.
        if (16 * (j >> 2) + 4 * g + (j & 3) >= seen) wv = 0.0f;
        pf[rt][j] = f2bf(wv);
        pl[rt][j] = f2bf(wv - (float)pf[rt][j]);
      }
    }
#pragma unroll
    for (int db = 0; db < NDB; ++db) {
      const i32x2 raw = __builtin_amdgcn_ds_read_tr8_b64_v2i32(LDS_PTR(i32x2, vl + (t_off ^ (16 * db))));
      const bf16x8 vf = values8(raw[0], raw[1], 1.0f);
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
  Block ba, bb;
  auto sweep = [&](auto carec) __attribute__((always_inline)) {
    load(b0 + wave, ba, vbuf);
    for (int blk = b0 + wave; blk < b1; blk += 2 * WAVES) {
      load(blk + WAVES, bb, vbuf + TILE);
      __builtin_amdgcn_s_waitcnt(vmcnt_imm(LOADS));
      __builtin_amdgcn_sched_barrier(0);
      compute(carec, blk, ba, vbuf);
      load(blk + 2 * WAVES, ba, vbuf);
      __builtin_amdgcn_s_waitcnt(vmcnt_imm(LOADS));
      __builtin_amdgcn_sched_barrier(0);
      if (blk + WAVES < b1) compute(carec, blk + WAVES, bb, vbuf + TILE);
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
  for (int i = 0; i < CPT; ++i) out[i] = f2bf(acc[i] * inv);
  *reinterpret_cast<bvec*>(p.o + ((size_t)(f.start + tok) * p.H + head) * D + c0) = out;
}

template <int D, int RT>
static void launch_decode(const PackedParams& p, hipStream_t st) {
  const dim3 grid(p.Hkv * p.nsplit * packed_slots(p.N, p.G, p.S, 16 * RT));
  if (p.sc.log2n == 4) hipLaunchKernelGGL((paged_decode_fp8_kernel<D, RT, 4>), grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL((paged_decode_fp8_kernel<D, RT, 0>), grid, dim3(256), 0, st, p);
}

hipError_t launch_paged_decode_fp8(const PackedParams& p, int D, int row_tiles, hipStream_t st) {
  {
    KTimer t("paged_decode_fp8", st);
    if (D == 64) row_tiles == 1 ? launch_decode<64, 1>(p, st) : launch_decode<64, 2>(p, st);
    else row_tiles == 1 ? launch_decode<128, 1>(p, st) : launch_decode<128, 2>(p, st);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.nsplit == 1) return e;
  return launch_packed_combine(p, D, st);
}

}  // namespace alg
