// Attention of one sequence over another, backward.  With P = exp2(logit - the row's numbers of the forward), dP = dO V^T and
// delta = rowsum(dO O) = rowsum(P dP):   dS = P (dP - delta),  dV = P^T dO,  dK = scale dS^T Q,  dQ = scale dS K,
// dtable[bucket] = sum of dS over the bucket's diagonals.
//
// Two passes, each recomputing S and dP (7 products instead of 5) rather than adding to one of the gradients with atomics: results do
// not depend on the order of workgroups.
//   * dQ pass: the forward's walk (128 rows, key tiles of 64).  S^T and dP^T have the softmax rows as columns, so the row's log-sum
//     and delta are one register each, and dS^T is at once the B operand of dQ^T = K^T dS^T.  delta = dO O comes from the lane's own
//     operand of dO and the stored O, whose two roundings (P's and its own) it inherits; exact arithmetic makes a row of dS sum to
//     zero, so the row sum that is left, taken in fp32, is what delta lacks: delta + that sum goes to the second pass.
//   * dK, dV pass: 128 keys per workgroup, K^T and V^T operands in registers, query tiles of 64 of all heads of the group in LDS:
//     the sum over shared heads is the accumulator's.  The bias gradient (an fp32 result) is formed here, from fp32 dS with the
//     corrected delta.
// Bias gradient: 32 x 32 blocks beyond the last border add to one register per side.  A nearer block goes through LDS: rows of dS at a
// pitch of 64 whose other half stays zero, so that lane t reads the 32 entries of diagonal t - 31 without a test, and adds its sum to
// the wave's histogram over distances: 16 writes, 32 reads and 32 additions per block, in a fixed order.  (LDS float atomics on the
// histogram itself: 234 cycles per instruction of 64 lanes, the pass 110 us instead of 44 at 4 x 8 x 1001^2.)
#include "seq_attn.h"
#include "seq_dtable.h"
#include <math.h>

#define SA_DIAG (32 + 32 * 64)         // floats of a wave's block of dS, a margin in front

struct SaBwdParams {
  const char *q, *k, *v, *o, *d_o;
  char *dq, *dk, *dv;
  const float* lse;
  float *delta, *ws_q, *ws_k, *ws_t, *dtable;
  const uint8_t* key_mask;
  const int32_t* kv_lens;
  long q_sb, q_sl, q_sh, k_sb, k_sl, k_sh, v_sb, v_sl, v_sh, o_sb, o_sl, o_sh, do_sb, do_sl, do_sh, mask_sb;
  int B, Lq, Lk, H, Hkv, D, splits_q, splits_k, nrb, num_buckets;
  float scale, sl2;
  SaRel rel;
};

// logits x log2 e minus the row's log-sum (lse, and base where wide: see SA_WIDE) of a block whose columns are softmax rows (rows: keys
// d0 + 8 (r / 4) + r % 4).  A wide row's logits are rounded as in the forward before its reference goes.
template <bool REL>
__device__ __forceinline__ void sa_logits(f32x16& s, float sl2, float lse, float base, bool wide, const float* myb, int W, int far, float farv, int d0) {
  if constexpr (REL) {
    auto near = [&](int r) { return myb[min(max(d0 + 8 * (r >> 2) + (r & 3), -W), W)]; };
    if (__builtin_expect(wide, 0)) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = (__builtin_fmaf(s[r], sl2, far ? farv : near(r)) - base) - lse;
    } else if (far) {
      const float c = farv - lse;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = __builtin_fmaf(s[r], sl2, c);
    } else {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = __builtin_fmaf(s[r], sl2, near(r) - lse);
    }
  } else {
    float mult = sl2;
    if (__builtin_expect(wide, 0)) {
      mult = 1.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = sa_exponent(s[r], sl2, base);
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = __builtin_fmaf(s[r], mult, -lse);
  }
}

// A block of dS that f16 cannot hold, though the products' sums may well be within it (dS is nobody's gradient): every column beyond the type
// is scaled by a power of two to just below its largest value, and the accumulators' same column with it for the length of `products`.
// Both lane halves of a column agree on the factor; columns within the type keep theirs, bit for bit.  f16 pays a maximum per block for
// it (bf16 holds every finite dS).
template <int DT, int N, typename F>
__device__ __forceinline__ void sa_within(f32x16& ds, f32x16(&acc)[N], F products) {
  bool beyond = false;
  int e = 0;
  if constexpr (DT == DFOLD_DT_F16) {
    float mx = 0.f;
#pragma unroll
    for (int r = 0; r < 16; r += 2) mx = fmaxf(fmaxf(mx, fabsf(ds[r])), fabsf(ds[r + 1]));
    beyond = __ballot(mx > 65504.f) != 0;
    if (__builtin_expect(beyond, 0)) {
      mx = sa_xmax(mx);
      e = mx > 65504.f && mx < INFINITY ? __builtin_amdgcn_frexp_expf(mx) - 15 : 0;      // mx < 2^(15 + e)
      const float down = ldexpf(1.f, -e);
#pragma unroll
      for (int r = 0; r < 16; ++r) ds[r] *= down;
#pragma unroll
      for (int i = 0; i < N; ++i) acc[i] *= down;
    }
  }
  products();
  if (__builtin_expect(beyond, 0)) {
    const float up = ldexpf(1.f, e);
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] *= up;
  }
}

// PAIR: as in the forward, two waves for the same 32 rows, one per half of a key tile
template <int DT, int DP, bool REL, bool PAIR>
__global__ __launch_bounds__((PAIR ? 2 : 1) * 64 * SA_WAVES, 2) void seq_attn_dq_kernel(const SaBwdParams p) {
  using T = SaTile<DP>;
  constexpr int KS = T::KS, NT = T::NT, NW = PAIR ? 2 * SA_WAVES : SA_WAVES, NB = PAIR ? 1 : 2;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  using C = SaKvCfg<DP, PAIR>;
  float* const ldsB = (float*)(smem + C::LDS);
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l31 = lane & 31, h = lane >> 5;
  unsigned id = sa_work_id();
  const int rb = id % p.nrb; id /= p.nrb;
  const int sp = id % p.splits_q; id /= p.splits_q;
  const int head = id % p.H, b = id / p.H, hkv = head / (p.H / p.Hkv);
  const int wr = w & (SA_WAVES - 1), half = PAIR ? w / SA_WAVES : 0;
  const int row_w = rb * SA_ROWS + wr * 32, row = row_w + l31;
  const bool wave_on = row_w < p.Lq, on = row < p.Lq;
  const int qi = min(row, p.Lq - 1);

  int kv_end = p.Lk;
  if (p.kv_lens) kv_end = min(max(p.kv_lens[b], 0), p.Lk);
  const int nt = (kv_end + SA_KT - 1) / SA_KT, per = (nt + p.splits_q - 1) / p.splits_q;
  const int t0 = sp * per, t1 = min(nt, t0 + per);

  int qpos = 0, qlo = 0, qhi = 0;
  float bL = 0.f, bR = 0.f;
  const float* myb = ldsB + p.rel.W;
  if constexpr (REL) {
    sa_fill_bias<NW>(ldsB, p.rel, head, 1, tid);
    const int off = sa_q_offset(p.rel, b);
    qpos = qi + off;
    qlo = row_w + off;
    qhi = min(row_w + 31, p.Lq - 1) + off;
    __syncthreads();
    bL = myb[-p.rel.W];
    bR = myb[p.rel.W];
  }

  sa_u32x4 qf[KS], of[KS];
  float dl = 0.f;
  {
    const char* sq = p.q + ((long)b * p.q_sb + (long)qi * p.q_sl + (long)head * p.q_sh) * 2;
    const char* sg = p.d_o + ((long)b * p.do_sb + (long)qi * p.do_sl + (long)head * p.do_sh) * 2;
    const char* so = p.o + ((long)b * p.o_sb + (long)qi * p.o_sl + (long)head * p.o_sh) * 2;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int d = ks * 16 + h * 8;
      qf[ks] = of[ks] = (sa_u32x4){0u, 0u, 0u, 0u};
      if (d < p.D) {
        qf[ks] = *(const sa_u32x4*)(sq + d * 2);
        of[ks] = *(const sa_u32x4*)(sg + d * 2);
        const sa_u32x4 o = *(const sa_u32x4*)(so + d * 2);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          dl = __builtin_fmaf(sa_lo<DT>(of[ks][e]), sa_lo<DT>(o[e]), dl);
          dl = __builtin_fmaf(sa_hi<DT>(of[ks][e]), sa_hi<DT>(o[e]), dl);
        }
      }
    }
  }
  dl = sa_xsum(dl);
  const long rowi = ((long)b * p.H + head) * p.Lq + qi;
  const float lse = on ? p.lse[rowi] : INFINITY, base = on ? p.lse[(long)p.B * p.H * p.Lq + rowi] : 0.f;
  const bool wide = __ballot(base != 0.f) != 0;

  const char* const kb_ = p.k + ((long)b * p.k_sb + (long)hkv * p.k_sh) * 2;
  const char* const vb_ = p.v + ((long)b * p.v_sb + (long)hkv * p.v_sh) * 2;
  const uint8_t* const mb_ = p.key_mask ? p.key_mask + (long)b * p.mask_sb : nullptr;
  f32x16 dq[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) dq[i][r] = 0.f;

  float left = 0.f;          // row sum of dS
  const SaAddr<DP> ad(lane, half * 32);
  const SaKvTiles<DP, PAIR> kv(kb_, p.k_sl, vb_, p.v_sl, p.D, tid, w);
  const SaLive<NW> keys{mb_, kv_end, t0, t1, w, lane, (unsigned long*)(smem + C::TILES)};
  auto fetch = [&](int t, int stage) { kv.load(t * SA_KT, kv_end, smem + stage * 2 * T::BYTES); };
  auto step = [&](int t, auto stage) {
    char* const lk = smem + decltype(stage)::value * 2 * T::BYTES;
    char* const lv = lk + T::BYTES;
    const unsigned long live = keys.tile(t);
    if (live != ~0ul) {
      if (live == 0) return;
      kv.zero(live, lk);
      sa_lds_barrier();
    }
    if (!wave_on) return;
#pragma unroll
    for (int kb = 0; kb < NB; ++kb) {
      f32x16 s, dp;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = dp[r] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        s = sa_mfma<DT>(ad.rows(lk, kb * 32, ks), qf[ks], s);
        dp = sa_mfma<DT>(ad.rows(lv, kb * 32, ks), of[ks], dp);
      }
      const int k0 = t * SA_KT + (half + kb) * 32;
      const int far = !REL ? 0 : k0 - qhi >= p.rel.W ? 1 : k0 + 31 - qlo <= -p.rel.W ? -1 : 0;
      sa_logits<REL>(s, p.sl2, lse, base, wide, myb, p.rel.W, far, far > 0 ? bR : bL, k0 + 4 * h - qpos);
      if (live != ~0ul) {
        const unsigned bits = (unsigned)(live >> ((half + kb) * 32)) >> (4 * h);
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (!((bits >> (8 * (r >> 2) + (r & 3))) & 1)) s[r] = -INFINITY;
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[r] = sa_exp2(s[r]) * (dp[r] - dl);
        left += s[r];
      }
      sa_within<DT>(s, dq, [&] {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          sa_u32x4 df;      // dS in the operand type: relative error up to 2^-8 (bf16) / 2^-11 (f16) of each term of dQ's sum
#pragma unroll
          for (int e = 0; e < 4; ++e) df[e] = sa_pack2<DT>(s[8 * c + 2 * e], s[8 * c + 2 * e + 1]);
#pragma unroll
          for (int i = 0; i < NT; ++i) dq[i] = sa_mfma<DT>(ad.cols(lk, kb * 32 + c * 16, i), df, dq[i]);
        }
      });
    }
  };
  kv.zero_columns(p.D, smem);
  sa_walk(t0, t1, fetch, step);

  left = sa_xsum(left);
  if constexpr (PAIR) {
    float* const ls = (float*)(smem + C::TILES + SA_MASKS * 8) + wr * 64 + lane;
    f32x16* const acc = (f32x16*)smem + wr * NT * 64 + lane;
    __syncthreads();
    if (half) {
      *ls = left;
#pragma unroll
      for (int i = 0; i < NT; ++i) acc[i * 64] = dq[i];
    }
    __syncthreads();
    if (half) return;
    left += *ls;
#pragma unroll
    for (int i = 0; i < NT; ++i) dq[i] += acc[i * 64];
  }
  if (on && h == 0) {
    // parts of the key axis: plane 0 holds delta, plane 1 + part the part's row sum (seq_attn_delta_kernel adds them up)
    if (p.splits_q == 1) p.delta[rowi] = dl + left;
    else {
      if (sp == 0) p.delta[rowi] = dl;
      p.delta[(long)(1 + sp) * p.B * p.H * p.Lq + rowi] = left;
    }
  }
  if (on) {
    const long r1 = ((long)b * p.Lq + qi) * p.H + head;
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d = i * 32 + g * 8 + h * 4;
        if (d >= p.D) continue;
        float o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = dq[i][g * 4 + e] * p.scale;
        if (p.splits_q == 1)
          *(uint2*)(p.dq + (r1 * p.D + d) * 2) = (uint2){sa_pack2<DT>(o[0], o[1]), sa_pack2<DT>(o[2], o[3])};
        else
          *(f32x4*)(p.ws_q + ((long)sp * p.B * p.Lq * p.H + r1) * p.D + d) = (f32x4){o[0], o[1], o[2], o[3]};
      }
  }
}

// Four waves of 32 keys each, K^T and V^T operands in registers; PAIR: eight waves, two for the same 32 keys, one per 32-query half of
// a tile; the two sums meet in LDS at the end.  Small launches then have two waves per SIMD.  At D = 128 the four-wave form needs more
// than 256 registers, one wave per SIMD, and nothing runs under its products: always PAIR there, with V^T operands from LDS (417 -> 303
// us) -- except with a bias, where eight waves' blocks of dS of 32 rows do not fit LDS beside the tiles (blocks of 16 rows would: not built).
template <int DP, bool REL, bool PAIR>
struct SaDkvCfg {
  static constexpr bool VLDS = PAIR && DP == 128;
  static constexpr int WAVES = PAIR ? 2 * SA_WAVES : SA_WAVES;
  static constexpr int TILES = 4 * SaTile<DP>::BYTES, ROWS = 6 * SA_KT * 4;      // two stages of two tiles; log-sums and deltas of their rows
  static constexpr int LDS = TILES + ROWS + (VLDS ? SA_ROWS * SaTile<DP>::PITCH : 0);
  static int bytes(int W) { return LDS + (REL ? (2 * W + 1 + WAVES * (2 * (W + SA_REACH) + 1 + SA_DIAG)) * 4 : 0); }
};
template <int DT, int DP, bool REL, bool PAIR>
__global__ __launch_bounds__((PAIR ? 2 : 1) * 64 * SA_WAVES, (DP == 128 && REL ? 1 : 2)) void seq_attn_dkv_kernel(const SaBwdParams p) {
  using T = SaTile<DP>;
  constexpr int KS = T::KS, NT = T::NT;
  constexpr bool VLDS = SaDkvCfg<DP, REL, PAIR>::VLDS;
  constexpr int NW = SaDkvCfg<DP, REL, PAIR>::WAVES;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  using C = SaDkvCfg<DP, REL, PAIR>;
  float* const ldsL = (float*)(smem + C::TILES);                // [stage][log-sum | delta | its wide part][SA_KT]
  char* const ldsV = smem + C::TILES + C::ROWS;
  float* const ldsB = (float*)(smem + C::LDS);
  float* const ldsH = ldsB + (REL ? 2 * p.rel.W + 1 : 0);       // [wave][distance]
  const int hn = REL ? 2 * (p.rel.W + SA_REACH) + 1 : 0;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l31 = lane & 31, h = lane >> 5;
  unsigned id = sa_work_id();
  const int nkb = (p.Lk + SA_ROWS - 1) / SA_ROWS, G = p.H / p.Hkv;
  const int kbk = id % nkb; id /= nkb;
  const int sp = id % p.splits_k; id /= p.splits_k;
  const int hkv = id % p.Hkv, b = id / p.Hkv;
  const int wk = w & (SA_WAVES - 1), half = PAIR ? w / SA_WAVES : 0;
  const int key_w = kbk * SA_ROWS + wk * 32, key = key_w + l31;

  int kv_end = p.Lk;
  if (p.kv_lens) kv_end = min(max(p.kv_lens[b], 0), p.Lk);
  const bool wg_on = kbk * SA_ROWS < kv_end, wave_on = key_w < kv_end;
  bool key_on = key < kv_end;
  if (key_on && p.key_mask) key_on = p.key_mask[(long)b * p.mask_sb + key] != 0;

  // units of work: (head of the group, query tile), this part's share
  const int nqt = (p.Lq + SA_KT - 1) / SA_KT, nu = G * nqt, per = (nu + p.splits_k - 1) / p.splits_k;
  const int u0 = sp * per, u1 = wg_on ? min(nu, u0 + per) : 0;

  sa_u32x4 kf[KS], vf[VLDS ? 1 : KS];
  {
    const char* sk = p.k + ((long)b * p.k_sb + (long)key * p.k_sl + (long)hkv * p.k_sh) * 2;
    const char* sv = p.v + ((long)b * p.v_sb + (long)key * p.v_sl + (long)hkv * p.v_sh) * 2;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int d = ks * 16 + h * 8;
      kf[ks] = (sa_u32x4){0u, 0u, 0u, 0u};
      if (key_on && d < p.D) kf[ks] = *(const sa_u32x4*)(sk + d * 2);
      if constexpr (!VLDS) {
        vf[ks] = (sa_u32x4){0u, 0u, 0u, 0u};
        if (key_on && d < p.D) vf[ks] = *(const sa_u32x4*)(sv + d * 2);
      }
    }
  }
  if constexpr (VLDS)
    if (u0 < u1) {
      const SaDma<DP, NW, SA_ROWS> ldv(p.v_sl, p.D, tid);
      ldv.load(p.v + ((long)b * p.v_sb + (long)hkv * p.v_sh) * 2, kbk * SA_ROWS, kv_end, ldsV, w);
      ldv.zero_columns(ldsV, tid);
    }
  f32x16 dk[NT], dv[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) dk[i][r] = dv[i][r] = 0.f;

  int off = 0, head_in = -1;
  const float* myb = ldsB + p.rel.W;
  float* const myh = ldsH + w * hn + p.rel.W + SA_REACH;
  float* const diag = ldsH + NW * hn + w * SA_DIAG + 32;   // 32 rows of 64 behind a margin of 32; columns 32 .. 63 and the margin are zero
  float accL = 0.f, accR = 0.f;
  auto table_part = [&](int head) { return p.ws_t + ((((long)b * p.H + head) * p.splits_k + sp) * nkb + kbk) * p.num_buckets; };
  // a head's histogram over distances -> its buckets; the far sums belong to the last bucket of their side
  auto flush = [&](int head) {
    accL = wave_sum(accL);
    accR = wave_sum(accR);
    if (lane == 0) {           // (entries -W and W carry their buckets)
      myh[-p.rel.W] += accL;
      myh[p.rel.W] += accR;
    }
    accL = accR = 0.f;
    __syncthreads();
    for (int i = tid; i < hn; i += 64 * NW) {
      float a = 0.f;
#pragma unroll
      for (int c = 0; c < NW; ++c) a += ldsH[c * hn + i];
      ldsH[i] = a;             // (entry i of every copy is this thread's)
    }
    __syncthreads();
    sa_bucket_sums<NW>(p.rel, ldsH, p.rel.W + SA_REACH, p.num_buckets, table_part(head), w, lane);
    __syncthreads();
  };
  if constexpr (REL) {
    off = sa_q_offset(p.rel, b);
    for (int i = lane; i < SA_DIAG; i += 64) diag[i - 32] = 0.f;
    for (int g = 0; g < G; ++g)          // heads this part does not touch
      if (max(u0, g * nqt) >= min(u1, (g + 1) * nqt))
        for (int j = tid; j < p.num_buckets; j += 64 * NW) table_part(hkv * G + g)[j] = 0.f;
  }

  const SaAddr<DP> ad(lane, half * 32);
  const SaKvTiles<DP, PAIR> qg(p.q, p.q_sl, p.d_o, p.do_sl, p.D, tid, w);
  const char* const lv = ldsV + (wk - half) * 32 * T::PITCH;
  // position in the walk of the unit that is fetched next, and of the one that is worked on
  int fg = u0 / nqt, fq = (u0 - fg * nqt) * SA_KT, wg = fg, wq = fq;
  auto fetch = [&](int, int stage) {
    const int head = hkv * G + fg;
    const long oq = ((long)b * p.q_sb + (long)head * p.q_sh) * 2, og = ((long)b * p.do_sb + (long)head * p.do_sh) * 2;
    qg.load(qg.a + (half ? og : oq), qg.b + og, fq, p.Lq, smem + stage * 2 * T::BYTES);
    // the rows' log-sums and deltas, a lane each
    const long r = ((long)b * p.H + head) * p.Lq + min(fq + lane, p.Lq - 1);
    float* const ll = ldsL + stage * 3 * SA_KT;
    if (w == 0) __builtin_amdgcn_global_load_lds((const void*)(p.lse + r), (sa_lds_ptr)ll, 4, 0, 0);
    if (w == 1) __builtin_amdgcn_global_load_lds((const void*)(p.delta + r), (sa_lds_ptr)(ll + SA_KT), 4, 0, 0);
    if (w == 2) __builtin_amdgcn_global_load_lds((const void*)(p.lse + (long)p.B * p.H * p.Lq + r), (sa_lds_ptr)(ll + 2 * SA_KT), 4, 0, 0);
    if ((fq += SA_KT) >= p.Lq) { fq = 0; ++fg; }
  };
  auto step = [&](int, auto stage) {
    char* const lq = smem + decltype(stage)::value * 2 * T::BYTES;
    char* const lg = lq + T::BYTES;
    float* const ll = ldsL + decltype(stage)::value * 3 * SA_KT;
    const int q0 = wq;
    if constexpr (REL) {
      const int head = hkv * G + wg;
      if (head != head_in) {       // (uniform)
        if (head_in >= 0) flush(head_in);      // (ends in a barrier: nobody reads the previous head's rows any more)
        for (int i = tid; i < NW * hn; i += 64 * NW) ldsH[i] = 0.f;
        sa_fill_bias<NW>(ldsB, p.rel, head, 1, tid);
        head_in = head;
        sa_lds_barrier();
      }
    }
    if ((wq += SA_KT) >= p.Lq) { wq = 0; ++wg; }
    if (q0 + SA_KT > p.Lq) {       // rows past the end repeat the last one: P = 0 for them
      if (tid < SA_KT && q0 + tid >= p.Lq) ll[tid] = INFINITY;
      sa_lds_barrier();
    }
    if (!wave_on) return;
    const bool wide = __ballot(ll[2 * SA_KT + lane] != 0.f) != 0;
#pragma unroll
    for (int qb = 0; qb < (PAIR ? 1 : 2); ++qb) {
      const int qs = (PAIR ? half : qb) * 32;
      if (q0 + qs >= p.Lq) continue;
      f32x16 s, dp;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = dp[r] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        s = sa_mfma<DT>(ad.rows(lq, qb * 32, ks), kf[ks], s);
        dp = sa_mfma<DT>(ad.rows(lg, qb * 32, ks), VLDS ? ad.rows(lv, 0, ks) : vf[VLDS ? 0 : ks], dp);
      }
      const int qlo = q0 + qs + off, qhi = qlo + 31;
      const int far = !REL ? 0 : key_w - qhi >= p.rel.W ? 1 : key_w + 31 - qlo <= -p.rel.W ? -1 : 0;
      if constexpr (REL) {
        if (far) {
          const float c = myb[far > 0 ? p.rel.W : -p.rel.W];
#pragma unroll
          for (int r = 0; r < 16; ++r) s[r] = __builtin_fmaf(s[r], p.sl2, c);
        } else {
          const int d0 = key - qlo - 4 * h;
#pragma unroll
          for (int r = 0; r < 16; ++r) s[r] = __builtin_fmaf(s[r], p.sl2, myb[min(max(d0 - 8 * (r >> 2) - (r & 3), -p.rel.W), p.rel.W)]);
        }
      }
      float mult = p.sl2;
      if (__builtin_expect(wide, 0)) {
        mult = 1.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float base = ll[2 * SA_KT + qs + 8 * (r >> 2) + 4 * h + (r & 3)];
          s[r] = REL ? s[r] - base : sa_exponent(s[r], p.sl2, base);
        }
      }
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 rl = *(const f32x4*)(ll + qs + g * 8 + h * 4);
        const f32x4 rd = *(const f32x4*)(ll + SA_KT + qs + g * 8 + h * 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = g * 4 + e;
          // a masked key's column holds products with zeros: whatever comes of them stays in that column, which is not stored (only the
          // bias gradient sums over columns)
          const float x = sa_exp2(REL ? s[r] - rl[e] : __builtin_fmaf(s[r], mult, -rl[e]));
          s[r] = REL ? (key_on ? x : 0.f) : x;
          dp[r] = s[r] * (dp[r] - rd[e]);
        }
      }
      if constexpr (REL) {
        if (far) {
          float a = 0.f;
#pragma unroll
          for (int r = 0; r < 16; ++r) a += dp[r];
          if (far > 0) accR += a; else accL += a;
        } else {
          // row = query; diagonal of distance key - query = (key_w - qlo) + (column - row)
#pragma unroll
          for (int r = 0; r < 16; ++r) diag[(8 * (r >> 2) + 4 * h + (r & 3)) * 64 + l31] = dp[r];
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          __builtin_amdgcn_wave_barrier();
          float a = 0.f, c = 0.f;
#pragma unroll
          for (int k = 0; k < 32; k += 2) {      // column k + lane - 31 of row k
            a += diag[k * 65 + lane - 31];
            c += diag[(k + 1) * 65 + lane - 31];
          }
          if (lane < 63) myh[key_w - qlo + lane - 31] += a + c;
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          __builtin_amdgcn_wave_barrier();
        }
      }
      sa_within<DT>(dp, dk, [&] {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          sa_u32x4 pf, df;      // P and dS in the operand type: relative error up to 2^-8 (bf16) / 2^-11 (f16) of each term
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            pf[e] = sa_pack2<DT>(s[8 * c + 2 * e], s[8 * c + 2 * e + 1]);
            df[e] = sa_pack2<DT>(dp[8 * c + 2 * e], dp[8 * c + 2 * e + 1]);
          }
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            dv[i] = sa_mfma<DT>(ad.cols(lg, qb * 32 + c * 16, i), pf, dv[i]);
            dk[i] = sa_mfma<DT>(ad.cols(lq, qb * 32 + c * 16, i), df, dk[i]);
          }
        }
      });
    }
  };
  qg.zero_columns(p.D, smem);
  sa_walk(u0, u1, fetch, step);

  if constexpr (REL)
    if (head_in >= 0) flush(head_in);
  if constexpr (PAIR) {
    // the second wave of a pair hands its sums over, 64 KB at a time through the tiles' memory
    f32x16* const acc = (f32x16*)smem + (wk * NT) * 64 + lane;
    auto join = [&](f32x16(&x)[NT]) {
      __syncthreads();
      if (half)
#pragma unroll
        for (int i = 0; i < NT; ++i) acc[i * 64] = x[i];
      __syncthreads();
      if (!half)
#pragma unroll
        for (int i = 0; i < NT; ++i) x[i] += acc[i * 64];
    };
    join(dk);
    join(dv);
    if (half) return;
  }
  if (key >= p.Lk) return;
  const long r1 = ((long)b * p.Lk + key) * p.Hkv + hkv, n = (long)p.B * p.Lk * p.Hkv;
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = i * 32 + g * 8 + h * 4;
      if (d >= p.D) continue;
      f32x4 a, c;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        a[e] = key_on ? dk[i][g * 4 + e] * p.scale : 0.f;
        c[e] = key_on ? dv[i][g * 4 + e] : 0.f;
      }
      if (p.splits_k == 1) {
        *(uint2*)(p.dk + (r1 * p.D + d) * 2) = (uint2){sa_pack2<DT>(a[0], a[1]), sa_pack2<DT>(a[2], a[3])};
        *(uint2*)(p.dv + (r1 * p.D + d) * 2) = (uint2){sa_pack2<DT>(c[0], c[1]), sa_pack2<DT>(c[2], c[3])};
      } else {
        *(f32x4*)(p.ws_k + ((long)(2 * sp) * n + r1) * p.D + d) = a;
        *(f32x4*)(p.ws_k + ((long)(2 * sp + 1) * n + r1) * p.D + d) = c;
      }
    }
}

// out[i] = sum of the parts in order, 8 elements per thread; part s at ws + s * stride
template <int DT>
__global__ __launch_bounds__(256) void seq_attn_sum_kernel(const float* __restrict__ ws, long stride, int parts, char* __restrict__ out, long n8) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= n8) return;
  f32x4 a = (f32x4){0.f, 0.f, 0.f, 0.f}, b = a;
  for (int s = 0; s < parts; ++s) {
    a += *(const f32x4*)(ws + s * stride + i * 8);
    b += *(const f32x4*)(ws + s * stride + i * 8 + 4);
  }
  *(sa_u32x4*)(out + i * 16) = (sa_u32x4){sa_pack2<DT>(a[0], a[1]), sa_pack2<DT>(a[2], a[3]), sa_pack2<DT>(b[0], b[1]), sa_pack2<DT>(b[2], b[3])};
}

// delta + the parts' row sums, in order
__global__ __launch_bounds__(256) void seq_attn_delta_kernel(float* __restrict__ delta, int parts, long n) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  float a = delta[n + i];
  for (int s = 2; s <= parts; ++s) a += delta[s * n + i];
  delta[i] += a;
}

template <typename F, typename K>
static int sa_launch_bwd(K kernel, const SaBwdParams& p, long nwg, int waves, int lds, hipStream_t st) {
  if (lds > SA_MAX_LDS) return DFOLD_EINVAL;
  if (!sa_raise_lds<F>(kernel, lds)) return DFOLD_ELAUNCH;
  DFOLD_LAUNCH(kernel, dim3((unsigned)nwg), dim3(64 * waves), lds, st, p);
  return dfold_check_launch();
}
template <int DT, int DP, bool REL, bool PAIR>
static int sa_dq(const SaBwdParams& p, hipStream_t st) {
  struct Mine;
  const int lds = SaKvCfg<DP, PAIR>::LDS + (REL ? (2 * p.rel.W + 1) * 4 : 0);
  return sa_launch_bwd<Mine>(seq_attn_dq_kernel<DT, DP, REL, PAIR>, p, (long)p.nrb * p.splits_q * p.H * p.B, PAIR ? 2 * SA_WAVES : SA_WAVES, lds, st);
}
template <int DT, int DP, bool REL, bool PAIR>
static int sa_dkv(const SaBwdParams& p, hipStream_t st) {
  struct Mine;
  const long nkb = (p.Lk + SA_ROWS - 1) / SA_ROWS;
  using C = SaDkvCfg<DP, REL, PAIR>;
  return sa_launch_bwd<Mine>(seq_attn_dkv_kernel<DT, DP, REL, PAIR>, p, nkb * p.splits_k * p.Hkv * p.B, C::WAVES, C::bytes(p.rel.W), st);
}
template <int DT, int DP, bool REL>
static int sa_bwd_dp(const SaBwdParams& p, bool pair_q, bool pair_k, hipStream_t st) {
  int rc = pair_q ? sa_dq<DT, DP, REL, true>(p, st) : sa_dq<DT, DP, REL, false>(p, st);
  if (rc != DFOLD_OK) return rc;
  if (p.splits_q > 1) {
    const long n8 = (long)p.B * p.Lq * p.H * p.D / 8;
    DFOLD_LAUNCH(seq_attn_sum_kernel<DT>, dim3((unsigned)((n8 + 255) / 256)), dim3(256), 0, st, (const float*)p.ws_q, n8 * 8, p.splits_q, p.dq, n8);
    if ((rc = dfold_check_launch()) != DFOLD_OK) return rc;
    const long nd = (long)p.B * p.H * p.Lq;
    DFOLD_LAUNCH(seq_attn_delta_kernel, dim3((unsigned)((nd + 255) / 256)), dim3(256), 0, st, p.delta, p.splits_q, nd);
    if ((rc = dfold_check_launch()) != DFOLD_OK) return rc;
  }
  const long nkb = (p.Lk + SA_ROWS - 1) / SA_ROWS;
  if constexpr (DP == 128) rc = sa_dkv<DT, DP, REL, !REL>(p, st);
  else if (pair_k && SaDkvCfg<DP, REL, true>::bytes(p.rel.W) <= SA_MAX_LDS) rc = sa_dkv<DT, DP, REL, true>(p, st);
  else rc = sa_dkv<DT, DP, REL, false>(p, st);
  if (rc != DFOLD_OK) return rc;
  if (REL) {
    DFOLD_LAUNCH(seq_dtable_kernel, dim3(p.H, (p.num_buckets + 63) / 64), dim3(1024), 0, st, (const float*)p.ws_t, p.dtable, p.num_buckets,
                 p.B, p.H, (int)nkb * p.splits_k);
    if ((rc = dfold_check_launch()) != DFOLD_OK) return rc;
  }
  if (p.splits_k == 1) return DFOLD_OK;
  const long n = (long)p.B * p.Lk * p.Hkv * p.D, n8 = n / 8;
  for (int i = 0; i < 2; ++i) {
    DFOLD_LAUNCH(seq_attn_sum_kernel<DT>, dim3((unsigned)((n8 + 255) / 256)), dim3(256), 0, st, (const float*)(p.ws_k + i * n), 2 * n, p.splits_k,
                 i ? p.dv : p.dk, n8);
    if ((rc = dfold_check_launch()) != DFOLD_OK) return rc;
  }
  return DFOLD_OK;
}
template <int DT>
static int sa_bwd(const SaBwdParams& p, bool rel, bool pq, bool pk, hipStream_t st) {
  if (p.D <= 32) return rel ? sa_bwd_dp<DT, 32, true>(p, pq, pk, st) : sa_bwd_dp<DT, 32, false>(p, pq, pk, st);
  if (p.D <= 64) return rel ? sa_bwd_dp<DT, 64, true>(p, pq, pk, st) : sa_bwd_dp<DT, 64, false>(p, pq, pk, st);
  return rel ? sa_bwd_dp<DT, 128, true>(p, pq, pk, st) : sa_bwd_dp<DT, 128, false>(p, pq, pk, st);
}

extern "C" int dfold_seq_attn_bwd(const dfold_seq_attn_desc* d, const dfold_seq_attn_grad* g, void* stream) {
  SaBwdParams p;
  if (!sa_desc_ok(d) || d->Lk == 0 || !g || !d->lse || !g->d_o || !g->dq || !g->delta || !g->dk || !g->dv) return DFOLD_EINVAL;
  if (g->splits_q < 1 || g->splits_q > 4096 || g->splits_k < 1 || g->splits_k > 4096) return DFOLD_EINVAL;
  if (((uintptr_t)g->d_o | (uintptr_t)g->dq | (uintptr_t)g->dk | (uintptr_t)g->dv | (uintptr_t)g->ws) & 15) return DFOLD_EINVAL;
  if ((g->do_sb | g->do_sl | g->do_sh) % 8 || g->do_sl >= SA_MAX_ROW || g->do_sb < 0 || g->do_sl < 0 || g->do_sh < 0) return DFOLD_EINVAL;
  const bool rel = d->rel.table != nullptr;
  if (rel && (!g->dtable || !sa_make_rel(&d->rel, d->H, &p.rel))) return DFOLD_EINVAL;
  if ((rel || g->splits_q > 1 || g->splits_k > 1) && !g->ws) return DFOLD_EINVAL;
  if (!rel) p.rel.W = 0;
  p.q = (const char*)d->q; p.k = (const char*)d->k; p.v = (const char*)d->v; p.o = (const char*)d->o;
  p.d_o = (const char*)g->d_o; p.dq = (char*)g->dq; p.dk = (char*)g->dk; p.dv = (char*)g->dv;
  p.lse = d->lse; p.delta = g->delta; p.dtable = g->dtable; p.key_mask = d->key_mask; p.kv_lens = d->kv_lens;
  p.q_sb = d->q_sb; p.q_sl = d->q_sl; p.q_sh = d->q_sh; p.k_sb = d->k_sb; p.k_sl = d->k_sl; p.k_sh = d->k_sh;
  p.v_sb = d->v_sb; p.v_sl = d->v_sl; p.v_sh = d->v_sh; p.o_sb = d->o_sb; p.o_sl = d->o_sl; p.o_sh = d->o_sh;
  p.do_sb = g->do_sb; p.do_sl = g->do_sl; p.do_sh = g->do_sh; p.mask_sb = d->mask_sb;
  p.B = d->B; p.Lq = d->Lq; p.Lk = d->Lk; p.H = d->H; p.Hkv = d->Hkv; p.D = d->D;
  p.splits_q = g->splits_q; p.splits_k = g->splits_k; p.num_buckets = rel ? d->rel.num_buckets : 0;
  p.scale = d->scale; p.sl2 = d->scale * SA_LOG2E;
  p.nrb = (d->Lq + SA_ROWS - 1) / SA_ROWS;
  const long nq = (long)d->B * d->Lq * d->H * d->D, nk = (long)d->B * d->Lk * d->Hkv * d->D, lim = 0x7fffffffL;
  if ((long)p.nrb * p.splits_q * p.H * p.B > lim || (((long)d->Lk + SA_ROWS - 1) / SA_ROWS) * p.splits_k * p.Hkv * p.B > lim ||
      nq / 2048 > lim - 1 || nk / 2048 > lim - 1 || d->H > 0x7fffffff / 64)
    return DFOLD_EINVAL;
  auto up4 = [](long x) { return (x + 3) & ~3L; };
  p.ws_q = g->ws;
  p.ws_k = g->ws + (p.splits_q > 1 ? up4(p.splits_q * nq) : 0);
  p.ws_t = p.ws_k + (p.splits_k > 1 ? up4(2 * p.splits_k * nk) : 0);
  const bool pq = g->pair_q != 0, pk = g->pair_k != 0;
  return d->dtype == DFOLD_DT_BF16 ? sa_bwd<DFOLD_DT_BF16>(p, rel, pq, pk, (hipStream_t)stream) : sa_bwd<DFOLD_DT_F16>(p, rel, pq, pk, (hipStream_t)stream);
}
