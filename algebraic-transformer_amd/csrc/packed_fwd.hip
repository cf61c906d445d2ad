// Causal algebraic attention over packed sequences of different lengths, or of new tokens over a
// paged cache, with grouped heads, bf16: the forward pass for many rows (packed_common.h has the
// arithmetic, the row order and the mapping of workgroups; paged_decode.hip the few rows of single
// tokens).
//
// One workgroup = 4 waves = 128 rows (token, head of the group) of one sequence and key head; a
// wave owns 32 rows and streams K and V through LDS in 64-key tiles, as the (B, H, T, D) forward
// does: S^T = K Q^T (32x32x16 MFMA, lane = row), t^n in registers, O^T += V^T P^T with V^T read
// transposed from LDS, two buffer sets, each filled by direct global -> LDS copies while the other
// is consumed. What differs:
//   * a wave copies 16 consecutive keys of a tile, through a buffer descriptor made for those keys:
//     they start anywhere (packed rows: a 64-bit base per tile, so no length passes an offset's 32
//     bits; pages: one table entry, since a page holds a multiple of 16 keys), and keys past the
//     sequence read as zeros, whatever memory holds there;
//   * the rows of a tile end at different positions, so the number of masked tiles is not fixed;
//   * nothing is known of the scores' range in advance: see the two forms in packed_common.h.
// With nsplit > 1 the keys of a row are split over workgroups, whose sums are joined by
// packed_combine_kernel. The weights are rounded to bf16 for the second product (2^-8 of each, random),
// sums and O in f32; o is rounded once.
//
// What bounds it: a weight takes 8.5 full-rate VALU instructions and one at a quarter of the rate, 50
// cycles for a wave's 64 scores, of which the two products take 32 (D = 128) or 16 (D = 64) on the matrix
// cores beside them. 16384 tokens in 3 sequences, 32 heads over 8, D = 128: 850 us, 0.93 PFLOP/s (VALU busy
// 70 % of cycles, matrix cores 50 %, no LDS bank conflict); nine documents of 16384 tokens, 16 heads over 4:
// 203 us, 0.79 PFLOP/s (65, 43: more of their tiles are at the diagonal); 13 documents, 8161 tokens, 16
// heads, D = 64: 38 us (73, 22). Over a cache, 701 tokens each of 3 requests over 24000 keys, 16 heads over 4: 172 us,
// 0.77 PFLOP/s, and 12 for joining two ranges.
// Over a cache of 8 bits the same takes 186 and 10 for the join (VALU busy 65 %, matrix cores 39 %; the first twenty of
// a process 212).
// A key head's workgroups are neighbours in steps of Hkv: with 2, 4, 8 key heads each XCD's L2 holds the
// keys of one, or of the same few, and K and V leave memory about once.
#include <type_traits>

#include "launchers.h"
#include "packed_common.h"

namespace alg {

template <int D, int L2N, bool PAGED, bool KV8 = false>
__global__ __launch_bounds__(256, 2) void packed_fwd_kernel(PackedParams p) {
  static_assert(D == 64 || D == 128, "head_dim");
  constexpr int BK = PK_BK, CPR = D / 8, NDB = D / 32, NF = D / 16;
  constexpr int RPI = 64 / CPR;       // keys per copy instruction
  constexpr int PW = 16 / RPI;        // copy instruction pairs per wave and tile: 16 keys
  __shared__ __attribute__((aligned(16))) bf16 Ks0[BK * D];
  __shared__ __attribute__((aligned(16))) bf16 Ks1[BK * D];
  __shared__ __attribute__((aligned(16))) bf16 Vs0[BK * D];
  __shared__ __attribute__((aligned(16))) bf16 Vs1[BK * D];
  __shared__ int bad_page;

  const int lane = threadIdx.x & 63, h = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // wave-uniform
  // Workgroups: key head, range of keys, item; a sequence's longest rows first (over a
  // cache the longest sequence's).
  const int kvh = blockIdx.x % p.Hkv, unit = blockIdx.x / p.Hkv, range = unit % p.nsplit;
  const PackedSeq f = packed_find<true>(p.cu, p.N, p.S, p.G, PK_ROWS, unit / p.nsplit, gridDim.x / p.Hkv / p.nsplit,
                                        PAGED ? p.kv_lens : nullptr);
  const int G = p.G;
  const int R = f.len * G;           // rows of the sequence
  const int r0 = f.tile * PK_ROWS;   // this workgroup's first row
  if (f.tile < 0 || r0 >= R) return;
  const int myr = r0 + wave * 32 + l32;
  const bool live = myr < R;
  const PackedRow at = packed_row<D>(p, f, kvh, min(myr, R - 1));

  if (f.s == p.S) {  // tokens behind the last sequence
    if (live && range == 0) {
      const bf16x8 z = {};
      for (int d = 8 * h; d < D; d += 16) *reinterpret_cast<bf16x8*>(p.o + at.out + d) = z;
      if (p.stat && h == 0) p.stat[at.stat] = 0.0f;
    }
    return;
  }

  // Keys of the sequence, those that the table reaches, and the position of its first token among them.
  const int held = PAGED ? max(p.kv_lens[f.s], 0) : f.len;
  const int L = PAGED ? min(held, p.width * p.page) : held;
  const int off = held - f.len;
  const int mypos = live ? off + at.tok : -1;
  const int rlast = min(r0 + PK_ROWS, R) - 1;
  const int posmin = off + r0 / G, posmax = off + rlast / G;
  const int wave_posmax = off + min(r0 + wave * 32 + 31, R - 1) / G;
  int kt0 = 0, kt1 = posmax < 0 ? 0 : min(posmax, L - 1) / BK + 1;  // this workgroup's key tiles
  if (p.nsplit > 1) {  // an equal share, of at least DECODE_RANGE keys
    const int per = max(ceil_div(kt1, p.nsplit), DECODE_RANGE / BK);
    kt0 = min(range * per, kt1);
    kt1 = min(kt0 + per, kt1);
    if (kt0 == kt1) {  // no key: only that is written
      if (live && h == 0) {
        const size_t part = (size_t)range * p.Hkv * p.N * G + at.stat;
        p.part_zt[2 * part] = 0.0f;
        p.part_zt[2 * part + 1] = 1.0f;
      }
      return;
    }
  }
  const int nfull = posmin < 0 ? 0 : (posmin + 1) / BK;  // tiles before every row's position

  // The 16 keys of tile kt that this wave copies. Pages: one table entry, read a tile ahead.
  typedef std::conditional_t<KV8, uint8_t, bf16> Stored;
  const Stored* kbase = reinterpret_cast<const Stored*>(p.k) + (size_t)kvh * p.k_hs + (PAGED ? 0 : (size_t)f.start * p.k_ts);
  const Stored* vbase = reinterpret_cast<const Stored*>(p.v) + (size_t)kvh * p.v_hs + (PAGED ? 0 : (size_t)f.start * p.v_ts);
  int pidx = 0, prow = 0;  // page of the group within the sequence, and row in the page
  if constexpr (PAGED) {
    const int key = kt0 * BK + 16 * wave;
    pidx = key / p.page;
    prow = key - pidx * p.page;
  }
  // Constant address space: a scalar load, which does not wait in the order of the copies.
  const auto* trow = (const __attribute__((address_space(4))) int*)(PAGED ? p.table + (size_t)f.s * p.width : nullptr);
  int next_id = PAGED && pidx < p.width && kt0 < kt1 ? trow[pidx] : 0;
  bool bad = false;
  auto group = [&](int kt) {
    KvGroupOf<Stored> g;
    const int key = kt * BK + 16 * wave;
    g.rows = kt < kt1 ? min(max(L - key, 0), 16) : 0;
    if constexpr (PAGED) {
      int id = __builtin_amdgcn_readfirstlane(next_id);
      if (g.rows > 0 && (unsigned)id >= (unsigned)p.pages) {  // never read; the rows' results become NaN
        bad = true;
        g.rows = 0;
      }
      id = g.rows > 0 ? id : 0;
      g.k = kbase + (size_t)id * p.k_ps + (size_t)prow * p.k_ts;
      g.v = vbase + (size_t)id * p.v_ps + (size_t)prow * p.v_ts;
      if constexpr (KV8) {
        g.ks = p.ks + (size_t)kvh * p.ks_hs + (size_t)id * p.ks_ps + prow;
        g.vs = p.vs + (size_t)kvh * p.vs_hs + (size_t)id * p.vs_ps + prow;
      }
      prow += BK;
      while (prow >= p.page) {
        prow -= p.page;
        ++pidx;
      }
      next_id = pidx < p.width && kt + 1 < kt1 ? trow[pidx] : 0;
    } else {
      const int k = g.rows > 0 ? key : 0;
      g.k = kbase + (size_t)k * p.k_ts;
      g.v = vbase + (size_t)k * p.v_ts;
    }
    return g;
  };
  // Instruction pair j of a copy: a lane's row and swizzled chunk, the same for every tile; the rest
  // of the address is scalar.
  const int lrow = lane / CPR;
  const int k_row = lrow * (int)p.k_ts * 2, v_row = lrow * (int)p.v_ts * 2;
  const int chunkb = 16 * ((lane % CPR) ^ swz_chunk<CPR>(lrow));
  auto dma = [&](bf16* la, bf16* lb, const KvGroupOf<Stored>& g, int j) {
    if constexpr (!KV8) {
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
    }
  };
  // A cache of 8 bits goes through registers: a lane a quarter of a key's row, D / 4 bytes each of K and V, fetched
  // while a tile is computed, made bf16 (exactly, packed_common.h) and written into the tiles one 16-byte
  // chunk after the other, beside the last products, which leave the VALU free. 16 neighbouring lanes hold 16
  // rows, whose chunks the swizzle keeps in 16 parts of the banks (four rows of four lanes each: 217 us, 200
  // so). Descriptors and byte scales stay scalar and unshifted until used: a wait for them here would be one
  // for the whole fetch.
  constexpr int NC = D / 32;  // chunks a lane
  struct Fetched {
    int k[D / 16], v[D / 16];
    int ks, vs;  // bytes; from mark() on the scales' bits
  };
  Fetched next8;
  auto fetch = [&](const KvGroupOf<Stored>& g) {
    if constexpr (KV8) {
      const int l = again(lane), row = l & 15, col = (l >> 4) * (D / 4);
      const int kn = g.rows > 0 ? (g.rows - 1) * (int)p.k_ts + D : 0, vn = g.rows > 0 ? (g.rows - 1) * (int)p.v_ts + D : 0;
      const int sn = g.rows > 0 ? 16 : 0;  // a page holds all 16 places
      const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc((void*)g.k, (short)0, kn, BUF_RSRC_WORD3);
      const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc((void*)g.v, (short)0, vn, BUF_RSRC_WORD3);
      const __amdgpu_buffer_rsrc_t rks = __builtin_amdgcn_make_buffer_rsrc((void*)g.ks, (short)0, sn, BUF_RSRC_WORD3);
      const __amdgpu_buffer_rsrc_t rvs = __builtin_amdgcn_make_buffer_rsrc((void*)g.vs, (short)0, sn, BUF_RSRC_WORD3);
      const int ko = __umul24(row, (int)p.k_ts) + col, vo = __umul24(row, (int)p.v_ts) + col;  // strides are under 2^24
#pragma unroll
      for (int i = 0; i < D / 64; ++i) {
        const auto a = __builtin_amdgcn_raw_buffer_load_b128(rk, ko, 16 * i, 0);
        const auto b = __builtin_amdgcn_raw_buffer_load_b128(rv, vo, 16 * i, 0);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          next8.k[4 * i + e] = a[e];
          next8.v[4 * i + e] = b[e];
        }
      }
      next8.ks = __builtin_amdgcn_raw_buffer_load_b8(rks, row, 0, 0);
      next8.vs = __builtin_amdgcn_raw_buffer_load_b8(rvs, row, 0, 0);
    }
  };
  // A key whose value was not finite (its bytes are zeros, its scale 255) becomes a NaN key: the rows that
  // see it are NaN, and the others do not meet it as a factor of their zero weights.
  auto mark = [&]() {
    int at = 0;  // where the lane's first chunk goes
    if constexpr (KV8) {
      next8.k[0] |= next8.vs == 255 ? 0x7F7F7F7F : 0;  // one element is enough
      next8.vs = min(next8.vs, 254) << 23;
      next8.ks <<= 23;
      const int l = again(lane), row = 16 * wave + (l & 15);
      at = row * D + (((NC * (l >> 4)) ^ swz_chunk<CPR>(row)) << 3);
    }
    return at;
  };
  auto put = [&](bf16* la, bf16* lb, int at, int c) {
    if constexpr (KV8) {
      *reinterpret_cast<bf16x8*>(la + (at ^ (8 * c))) = values8(next8.k[2 * c], next8.k[2 * c + 1], __builtin_bit_cast(float, next8.ks));
      *reinterpret_cast<bf16x8*>(lb + (at ^ (8 * c))) = values8(next8.v[2 * c], next8.v[2 * c + 1], __builtin_bit_cast(float, next8.vs));
    }
  };
  auto put_all = [&](bf16* la, bf16* lb) {
    if constexpr (KV8) {
      const int at = mark();
#pragma unroll
      for (int c = 0; c < NC; ++c) put(la, lb, at, c);
    }
  };

  if constexpr (PAGED) {
    if (threadIdx.x == 0) bad_page = 0;
  }
  {
    const KvGroupOf<Stored> g = group(kt0);
    fetch(g);
#pragma unroll
    for (int j = 0; j < PW; ++j) dma(Ks0, Vs0, g, j);
    put_all(Ks0, Vs0);
  }
  // Query fragments (B operand of S^T = K Q^T), held for the whole kernel; dead rows are zero.
  bf16x8 qf[NF];
  {
    const bf16* Q = p.q + (size_t)(f.start + at.tok) * p.q_ts + (size_t)at.head * p.q_hs;
#pragma unroll
    for (int s = 0; s < NF; ++s) qf[s] = ld8(Q + 16 * s + 8 * h);
    keep_own_row<NF>(qf, live);
#pragma unroll
    for (int s = 0; s < NF; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) qf[s][j] = f2bf((float)qf[s][j] * p.sc.qmul);
  }
  const int log2n = p.sc.log2n;
  const float b2 = p.sc.b;
  floatx16 oacc[NDB];
#pragma unroll
  for (int db = 0; db < NDB; ++db) oacc[db] = floatx16{};
  float lsum = 0.0f;

  const int tr = (lane & 15) >> 2;
  int row_off[NF];  // row fragments of K: row l32, k chunk 2 st + h
#pragma unroll
  for (int st = 0; st < NF; ++st) row_off[st] = swz_at<CPR>(l32, 16 * st + 8 * h);
  int tv_lo[NDB], tv_hi[NDB];  // transposed V fragments: rows 4h + (0..3), 4h + 8 + (0..3)
#pragma unroll
  for (int db = 0; db < NDB; ++db) {
    tv_lo[db] = swz_at<CPR>(4 * h + tr, tr_col(db * 32, lane));
    tv_hi[db] = swz_at<CPR>(4 * h + 8 + tr, tr_col(db * 32, lane));
  }

  bf16x8 rk3[3];  // row fragments of K, two steps ahead
  __builtin_amdgcn_s_waitcnt(VMCNT0);
  __syncthreads();
  rk3[0] = ld8(Ks0 + row_off[0]);
  rk3[1] = ld8(Ks0 + row_off[1]);
  constexpr int VE = 10;  // VALU instructions per weight (scheduling hint)

  // One key tile in the plain form, software-pipelined over its two 32-key blocks:
  //   R1 S^T of keys 0..31 | the next tile's copy    R2 S^T of 32..63 | weights of 0..31
  //   R3 O^T over 0..31 | weights of 32..63          R4 O^T over 32..63
  auto tile = [&](auto bufc, auto maskc, int kt) {
    constexpr int BUF = decltype(bufc)::value;
    constexpr bool MASKED = decltype(maskc)::value;
    const bf16* Ks = BUF ? Ks1 : Ks0;
    const bf16* Vs = BUF ? Vs1 : Vs0;
    bf16* Kn = BUF ? Ks0 : Ks1;
    bf16* Vn = BUF ? Vs0 : Vs1;
    const int kb0 = kt * BK;
    const KvGroupOf<Stored> gn = group(kt + 1);
    fetch(gn);
    if constexpr (MASKED) {
      if (kb0 > wave_posmax) {  // every key lies after this wave's rows
#pragma unroll
        for (int j = 0; j < PW; ++j) dma(Kn, Vn, gn, j);
        put_all(Kn, Vn);
        __builtin_amdgcn_s_waitcnt(VMCNT0);
        __syncthreads();
        rk3[0] = ld8(Kn + row_off[0]);
        rk3[1] = ld8(Kn + row_off[1]);
        return;
      }
    }
    floatx16 s[2];
    bf16x8 pf[2][2];
    float w[16];
    auto s_step = [&](int g) {
      const int blk = g / NF, st = g % NF;
      const int gx = g + 2;
      if (gx < 2 * NF) rk3[gx % 3] = ld8(Ks + (gx / NF) * 32 * D + row_off[gx % NF]);
      s[blk] = mfma_bf16(rk3[g % 3], qf[st], s[blk]);
    };
    auto elem = [&](int blk, int i) {
      const bool dead = MASKED && kb0 + blk * 32 + 8 * (i >> 2) + 4 * h + (i & 3) > mypos;
      float r;
      float wi = pow2n<L2N>(weight_t(s[blk][i], b2, r), log2n);
      if constexpr (MASKED) keep_here(wi);
      if (dead) wi = 0.0f;
      lsum += wi;
      w[i] = wi;
      if (i & 1) {
        pf[blk][i >> 3][(i & 7) - 1] = f2bf(w[i - 1]);
        pf[blk][i >> 3][i & 7] = f2bf(w[i]);
      }
    };
    bf16x8 ft[2][2];
    auto pv_load = [&](int blk, int db, bf16x8 (&fr)[2]) {
      const bf16* vb = Vs + blk * 32 * D;
      fr[0] = tr_frag_at(vb, tv_lo[db], tv_hi[db]);
      fr[1] = tr_frag_at(vb + 16 * D, tv_lo[db], tv_hi[db]);
    };
    s[0] = floatx16{};
    s[1] = floatx16{};
#pragma unroll
    for (int g = 0; g < NF; ++g) {
      s_step(g);
      if (g < PW) dma(Kn, Vn, gn, g);
      step_order<1, 0, 2, 0>();
    }
    constexpr int E2 = 16 / NF;
#pragma unroll
    for (int g = NF; g < 2 * NF; ++g) {
      s_step(g);
#pragma unroll
      for (int k = 0; k < E2; ++k) elem(0, E2 * (g - NF) + k);
      if (g == 2 * NF - 1) pv_load(0, 0, ft[0]);
      step_order<1, VE * E2, 2, 0>();
    }
    constexpr int E3 = 16 / NDB;
#pragma unroll
    for (int db = 0; db < NDB; ++db) {
      const int c = db & 1;
      if (db + 1 < NDB) pv_load(0, db + 1, ft[c ^ 1]);
      else pv_load(1, 0, ft[c ^ 1]);
      oacc[db] = mfma_bf16(ft[c][0], pf[0][0], oacc[db]);
      oacc[db] = mfma_bf16(ft[c][1], pf[0][1], oacc[db]);
#pragma unroll
      for (int k = 0; k < E3; ++k) elem(1, E3 * db + k);
      step_order<2, VE * E3, 4, 0>();
    }
    const int put_at = mark();
#pragma unroll
    for (int db = 0; db < NDB; ++db) {
      const int c = (db + NDB) & 1;
      if (db + 1 < NDB) pv_load(1, db + 1, ft[c ^ 1]);
      oacc[db] = mfma_bf16(ft[c][0], pf[1][0], oacc[db]);
      oacc[db] = mfma_bf16(ft[c][1], pf[1][1], oacc[db]);
      put(Kn, Vn, put_at, db);
      if constexpr (KV8) step_order<2, 8, 4, 2>();
      else step_order<2, 0, 4, 0>();
    }
    __builtin_amdgcn_s_waitcnt(VMCNT0);  // this wave's copies of the next tile have landed
    __syncthreads();                     // the next tile is complete; this buffer set is free
    rk3[0] = ld8(Kn + row_off[0]);
    rk3[1] = ld8(Kn + row_off[1]);
  };

  const bool has_sink = p.sink != nullptr && p.nsplit == 1;  // split: the sink joins in the combination
  const float ss = has_sink ? sink_score(p, at.head) : 0.0f;
  bool careful = isinf(p.sc.low);
  if (!careful) {
    // The tiles in pairs (buffer sets 0 and 1); the last pair may be half one, and a pair counts as
    // masked when one of its tiles does. No branch chooses a buffer set inside the loops: the
    // accumulators' registers stay put.
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
    const int count = min(mypos + 1, kt1 * BK) - kt0 * BK;  // the row's keys in this range
    float sink_w = 1.0f;
    if (has_sink) {
      float r;
      sink_w = pow2n<L2N>(weight_t_careful(ss, b2, r), log2n);
    }
    careful = __syncthreads_or(live && (needs_care(lsum + xor32(lsum), count, p.sc.low) || !(sink_w <= 0x1p30f))) != 0;
  }

  float shift = 1.0f, tmax = 1.0f;  // the row's weights are (t shift)^n; tmax = 1 / shift
  if (careful) {
    // The rows again, with a running maximum of the scores per row (the sink a first key).
    float m = has_sink ? ss : -INFINITY;
    lsum = has_sink && h == 0 ? 1.0f : 0.0f;
    {
      float r;
      tmax = has_sink ? weight_t_careful(ss, b2, r) : 0.0f;
      shift = has_sink ? 1.0f / tmax : 0.0f;
    }
#pragma unroll
    for (int db = 0; db < NDB; ++db) oacc[db] = floatx16{};
    if constexpr (PAGED) {
      const int key = kt0 * BK + 16 * wave;
      pidx = key / p.page;
      prow = key - pidx * p.page;
      next_id = pidx < p.width && kt0 < kt1 ? trow[pidx] : 0;
    }
    for (int kt = kt0; kt < kt1; ++kt) {
      __syncthreads();  // every wave is done with the tile before
      const KvGroupOf<Stored> g = group(kt);
      fetch(g);
#pragma unroll
      for (int j = 0; j < PW; ++j) dma(Ks0, Vs0, g, j);
      put_all(Ks0, Vs0);
      __builtin_amdgcn_s_waitcnt(VMCNT0);
      __syncthreads();
      for (int blk = 0; blk < 2; ++blk) {
        const int kb = kt * BK + 32 * blk;
        if (kb > wave_posmax) continue;
        floatx16 s = {};
#pragma unroll
        for (int st = 0; st < NF; ++st) s = mfma_bf16(ld8(Ks0 + blk * 32 * D + row_off[st]), qf[st], s);
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (kb + 8 * (i >> 2) + 4 * h + (i & 3) <= mypos) top = fmaxf(top, s[i]);
        top = fmaxf(top, xor32(top));
        if (top > m) {
          float r;
          const float t = weight_t_careful(top, b2, r);
          const float fall = m == -INFINITY ? 0.0f : pow2n<0>(tmax / t, log2n);
          m = top;
          tmax = t;
          shift = 1.0f / t;
          lsum *= fall;
#pragma unroll
          for (int db = 0; db < NDB; ++db)
#pragma unroll
            for (int i = 0; i < 16; ++i) oacc[db][i] *= fall;
        }
        bf16x8 pf[2];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const bool dead = kb + 8 * (i >> 2) + 4 * h + (i & 3) > mypos;
          float r;
          float w = pow2n<0>(weight_t_careful(dead ? 0.0f : s[i], b2, r) * shift, log2n);
          keep_here(w);
          if (dead) w = 0.0f;
          lsum += w;
          pf[i >> 3][i & 7] = f2bf(w);
        }
        const bf16* vb = Vs0 + blk * 32 * D;
#pragma unroll
        for (int db = 0; db < NDB; ++db) {
          oacc[db] = mfma_bf16(tr_frag_at(vb, tv_lo[db], tv_hi[db]), pf[0], oacc[db]);
          oacc[db] = mfma_bf16(tr_frag_at(vb + 16 * D, tv_lo[db], tv_hi[db]), pf[1], oacc[db]);
        }
      }
    }
  }

  float Z = lsum + xor32(lsum);
  if constexpr (PAGED) {
    if (bad) bad_page = 1;
    __syncthreads();
    if (bad_page || mypos >= L) Z = __builtin_nanf("");  // a position behind the table's end holds no key of its own
  }
  if (!live) return;
  const PackedRow my = packed_row<D>(p, f, kvh, again(r0 + wave * 32 + l32));
  if (p.nsplit > 1) {
    const size_t part = (size_t)range * p.Hkv * p.N * G + my.stat;
    float* O = p.part_o + part * D;
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        floatx4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = oacc[db][4 * g + e];
        *reinterpret_cast<floatx4*>(O + db * 32 + 8 * g + 4 * h) = v;
      }
    if (h == 0) {
      p.part_zt[2 * part] = Z;
      p.part_zt[2 * part + 1] = careful ? -tmax : tmax;
    }
    return;
  }
  if (!careful && has_sink) {
    float r;
    Z += pow2n<L2N>(weight_t_careful(ss, b2, r), log2n);
  }
  const float inv = Z == 0.0f ? 0.0f : 1.0f / Z;  // a row without keys and sink is zero
  bf16* O = p.o + my.out;
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      bf16x4 ob;
#pragma unroll
      for (int e = 0; e < 4; ++e) ob[e] = f2bf(oacc[db][4 * g + e] * inv);
      *reinterpret_cast<bf16x4*>(O + db * 32 + 8 * g + 4 * h) = ob;
    }
  if (p.stat && h == 0) {
    const float rs = Z == 0.0f ? 0.0f : shift * inv_root(Z, 1 << log2n);
    p.stat[my.stat] = careful ? -rs : rs;
  }
}

// Rows whose keys were split: o = sum_i f_i O_i / (sum_i f_i Z_i + sink), f_i = (T_i / T)^n with
// T_i the range's shift and T the largest of them and the sink's; a range without keys for the row
// has Z_i = 0 and counts for nothing (its sums are not read: they may not be written). The order of
// the sums is fixed. Every load that can be is issued before a result is waited for.
struct CombineRow {
  size_t out, stat;
  int head;
  bool held;  // in a sequence: the tokens behind the last one are the first range's workgroups' to write
};
__device__ __forceinline__ CombineRow combine_row(const PackedParams& p, int row) {
  const int tok = row / p.H, head = row - tok * p.H, kvh = head / p.G;
  return CombineRow{(size_t)row, (size_t)kvh * p.N * p.G + (size_t)tok * p.G + (head - kvh * p.G), head,
                    tok < packed_start(p.cu, p.S, p.N)};
}
__device__ __forceinline__ void combine_stat(const PackedParams& p, size_t at, float Z, float T, bool careful) {
  const float rs = Z == 0.0f ? 0.0f : inv_root(Z, 1 << p.sc.log2n) / T;
  p.stat[at] = careful ? -rs : rs;
}

// Up to RANGES ranges: D / 4 lanes a row, four columns each, every lane all of the ranges' factors.
// Bytes bound it: 33648 rows of 128 in two ranges, 43 MB, 7 us beside the
// launch's 5 (16 by a wave a row, whose loads are 8 bytes a lane).
template <int D, int RANGES>
__global__ __launch_bounds__(256) void packed_combine_kernel(PackedParams p) {
  constexpr int LPR = D / 4;
  const int row = blockIdx.x * (256 / LPR) + threadIdx.x / LPR, col = threadIdx.x % LPR * 4;
  if (row >= p.N * p.H) return;
  const CombineRow at = combine_row(p, row);
  if (!at.held) return;
  const size_t rows = (size_t)p.Hkv * p.N * p.G;
  const float* O = p.part_o + at.stat * D + col;
  const int log2n = p.sc.log2n;
  float2 zt[RANGES];
  floatx4 o[RANGES];
#pragma unroll
  for (int i = 0; i < RANGES; ++i) {
    const size_t skip = (size_t)min(i, p.nsplit - 1) * rows;
    zt[i] = *reinterpret_cast<const float2*>(p.part_zt + 2 * (skip + at.stat));
    o[i] = *reinterpret_cast<const floatx4*>(O + skip * D);
  }
  float T = 0.0f, ts = 0.0f;
  if (p.sink) {
    float r;
    T = ts = weight_t_careful(sink_score(p, at.head), p.sc.b, r);
  }
  bool careful = false;  // whether a range took that form
#pragma unroll
  for (int i = 0; i < RANGES; ++i) {
    if (i >= p.nsplit) zt[i].x = 0.0f;
    if (zt[i].x != 0.0f) {
      T = fmaxf(T, __builtin_fabsf(zt[i].y));
      careful |= zt[i].y < 0.0f;
    }
  }
  float Z = 0.0f;
  floatx4 acc = {};
#pragma unroll
  for (int i = 0; i < RANGES; ++i)
    if (zt[i].x != 0.0f) {
      const float f = pow2n<0>(__builtin_fabsf(zt[i].y) / T, log2n);
      Z += f * zt[i].x;
      acc += f * o[i];
    }
  if (p.sink) Z += sink_weight(ts, T, log2n);
  if (p.stat && col == 0) combine_stat(p, at.stat, Z, T, careful);
  const float inv = Z == 0.0f ? 0.0f : 1.0f / Z;
  bf16x4 out;
#pragma unroll
  for (int e = 0; e < 4; ++e) out[e] = f2bf(acc[e] * inv);
  *reinterpret_cast<bf16x4*>(p.o + at.out * D + col) = out;
}

// Over 16 ranges, few rows: latency is all of it. A workgroup a row, thread i range i, its waves a
// quarter of the ranges' sums each (16 rows of 64 ranges: 12.7 us by one wave a row, of which launches
// are about 5).
template <int D>
__global__ __launch_bounds__(256) void packed_combine_wide_kernel(PackedParams p) {
  constexpr int E = D / 64;  // columns a lane
  typedef float fvec __attribute__((ext_vector_type(E)));
  __shared__ float fs[MAX_RANGES], red[2][4];
  __shared__ fvec part[4][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const CombineRow at = combine_row(p, blockIdx.x);
  if (!at.held) return;
  const size_t rows = (size_t)p.Hkv * p.N * p.G;
  const float* O = p.part_o + at.stat * D + lane * E;
  const int log2n = p.sc.log2n;
  float T = 0.0f, ts = 0.0f;
  if (p.sink) {
    float r;
    T = ts = weight_t_careful(sink_score(p, at.head), p.sc.b, r);
  }
  const bool mine = (int)threadIdx.x < p.nsplit;
  const float2 zt = mine ? *reinterpret_cast<const float2*>(p.part_zt + 2 * (threadIdx.x * rows + at.stat)) : make_float2(0.0f, 0.0f);
  if (zt.x != 0.0f) T = fmaxf(T, __builtin_fabsf(zt.y));
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) T = fmaxf(T, __shfl_xor(T, m, 64));
  if (lane == 0) red[0][wave] = T;
  const bool careful = __syncthreads_or(zt.x != 0.0f && zt.y < 0.0f) != 0;
  T = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  const float f = zt.x != 0.0f ? pow2n<0>(__builtin_fabsf(zt.y) / T, log2n) : 0.0f;
  fs[threadIdx.x] = f;
  float Z = f * zt.x;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) Z += __shfl_xor(Z, m, 64);
  if (lane == 0) red[1][wave] = Z;
  __syncthreads();
  Z = red[1][0] + red[1][1] + red[1][2] + red[1][3];
  fvec acc = 0.0f;
  for (int i0 = wave; i0 < p.nsplit; i0 += 32) {  // eight ranges' loads in flight
    fvec o[8];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      o[k] = *reinterpret_cast<const fvec*>(O + min(i0 + 4 * k, p.nsplit - 1) * rows * D);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float fi = i0 + 4 * k < p.nsplit ? fs[i0 + 4 * k] : 0.0f;
      if (fi != 0.0f) acc += fi * o[k];
    }
  }
  part[wave][lane] = acc;
  __syncthreads();
  if (wave != 0) return;
  acc = part[0][lane] + part[1][lane] + part[2][lane] + part[3][lane];
  if (p.sink) Z += sink_weight(ts, T, log2n);
  if (p.stat && lane == 0) combine_stat(p, at.stat, Z, T, careful);
  const float inv = Z == 0.0f ? 0.0f : 1.0f / Z;
  bf16* out = p.o + at.out * D + lane * E;
  if constexpr (E == 2) *reinterpret_cast<unsigned*>(out) = pack_bf16x2(acc[0] * inv, acc[1] * inv);
  else out[0] = f2bf(acc[0] * inv);
}

template <int D, bool PAGED, bool KV8 = false>
static void launch_fwd(const PackedParams& p, dim3 grid, hipStream_t st) {
  if (p.sc.log2n == 4) hipLaunchKernelGGL((packed_fwd_kernel<D, 4, PAGED, KV8>), grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL((packed_fwd_kernel<D, 0, PAGED, KV8>), grid, dim3(256), 0, st, p);
}

template <int D>
static void launch_combine(const PackedParams& p, hipStream_t st) {
  const long rows = (long)p.N * p.H, each = 256 / (D / 4);
  const dim3 grid((unsigned)((rows + each - 1) / each));
  if (p.nsplit > 16) hipLaunchKernelGGL(packed_combine_wide_kernel<D>, dim3((unsigned)rows), dim3(256), 0, st, p);
  else if (p.nsplit > 8) hipLaunchKernelGGL((packed_combine_kernel<D, 16>), grid, dim3(256), 0, st, p);
  else if (p.nsplit > 2) hipLaunchKernelGGL((packed_combine_kernel<D, 8>), grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL((packed_combine_kernel<D, 2>), grid, dim3(256), 0, st, p);
}

hipError_t launch_packed_combine(const PackedParams& p, int D, hipStream_t st) {
  KTimer t("packed_combine", st);
  if (D == 64) launch_combine<64>(p, st);
  else launch_combine<128>(p, st);
  return hipGetLastError();
}

hipError_t launch_packed_fwd(const PackedParams& p, int D, bool paged, hipStream_t st) {
  const dim3 grid(p.Hkv * p.nsplit * packed_slots(p.N, p.G, p.S, PK_ROWS));
  {
    KTimer t(p.ks ? "paged_fwd_fp8" : paged ? "paged_fwd" : "packed_fwd", st);
    if (p.ks) D == 64 ? launch_fwd<64, true, true>(p, grid, st) : launch_fwd<128, true, true>(p, grid, st);
    else if (D == 64) paged ? launch_fwd<64, true>(p, grid, st) : launch_fwd<64, false>(p, grid, st);
    else paged ? launch_fwd<128, true>(p, grid, st) : launch_fwd<128, false>(p, grid, st);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.nsplit == 1) return e;
  return launch_packed_combine(p, D, st);
}

}  // namespace alg
