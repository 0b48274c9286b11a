// Attention of one sequence over another, forward:  o = softmax(scale q k^T + bias) v  per head, one pass over the keys with the
// running maximum and sum of the softmax.
//
// Parts of the keys and pairs of waves meet by their references and sums: weights exp2(mu_part - mu) l_part.
//
// A workgroup owns 128 softmax rows of one key head (4 waves x 32 rows; with pack > 1 the rows of the query heads of a group are
// interleaved, head fastest, so that one token of a grouped layer fills its tile), walks its part of the keys in tiles of 64 and
// keeps S, P and O in registers; K and V tiles go to LDS by DMA ahead of the arithmetic, one barrier per tile.  Key masks are one
// word per tile: an empty tile is skipped, a full one takes no mask arithmetic, K / V rows of masked keys are
// zeroed in LDS behind one more barrier (0 * NaN would not stay 0).
// Few rows and many keys: the key axis is cut over workgroups (splits), partial results meet in seq_attn_combine_kernel in split
// order (deterministic).
#include "seq_attn.h"
#include <math.h>

struct SaFwdParams {
  const char *q, *k, *v;
  char* o;
  float *lse, *ws;
  const uint8_t* key_mask;
  const int32_t* kv_lens;
  long q_sb, q_sl, q_sh, k_sb, k_sl, k_sh, v_sb, v_sl, v_sh, o_sb, o_sl, o_sh, mask_sb;
  int B, Lq, Lk, H, Hkv, D, splits, pack, nrb;
  float sl2;
  SaRel rel;
};

// Rescaling the accumulators costs as much as the rest of the softmax: the reference value of the exponents follows the running
// maximum only when it has grown by more than this (P stays <= 2^8: exact in fp32 sums, harmless in 16-bit operands)
#define SA_LAZY 8.f
#define SA_MAX_SPLITS 1024

// a row for the backward, planes of lse: P = exp2(logit - plane 1 - plane 0).  any: the row has keys
__device__ __forceinline__ void sa_row_stat(const SaFwdParams& p, int b, int head, int qi, bool any, float mu, float l) {
  float* const st = p.lse + ((long)b * p.H + head) * p.Lq + qi;
  const bool wide = any && fabsf(mu) >= SA_WIDE;
  st[0] = any ? (wide ? 0.f : mu) + __log2f(l) : INFINITY;
  st[(long)p.B * p.H * p.Lq] = wide ? mu : 0.f;
}

// PAIR: eight waves, two for the same 32 rows, one per half of a key tile, joined in LDS at the end: a launch of at most one workgroup
// per CU has two waves per SIMD instead of one.
template <int DT, int DP, bool REL, bool PAIR>
__global__ __launch_bounds__((PAIR ? 2 : 1) * 64 * SA_WAVES, 2) void seq_attn_fwd_kernel(const SaFwdParams p) {
  using T = SaTile<DP>;
  constexpr int KS = T::KS, NT = T::NT, NW = PAIR ? 2 * SA_WAVES : SA_WAVES, NB = PAIR ? 1 : 2;      // NB: 32-key blocks of a wave
  extern __shared__ __attribute__((aligned(16))) char smem[];
  using C = SaKvCfg<DP, PAIR>;
  float* const ldsB = (float*)(smem + C::LDS);
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l31 = lane & 31, h = lane >> 5;
  unsigned id = sa_work_id();
  const int rb = id % p.nrb; id /= p.nrb;
  const int sp = id % p.splits; id /= p.splits;
  const int hgs = p.H / p.pack, hg = id % hgs, b = id / hgs;
  const int head0 = hg * p.pack, hkv = head0 / (p.H / p.Hkv);
  const int rows = p.Lq * p.pack;
  const int wr = w & (SA_WAVES - 1), half = PAIR ? w / SA_WAVES : 0;
  const int row_w = rb * SA_ROWS + wr * 32, row = row_w + l31;
  const bool wave_on = row_w < rows, on = row < rows;
  const int rowc = min(row, rows - 1), qi = rowc / p.pack, hl = rowc - qi * p.pack;

  // keys of this part, in tiles
  int kv_end = p.Lk;
  if (p.kv_lens) kv_end = min(max(p.kv_lens[b], 0), p.Lk);
  const int nt = (kv_end + SA_KT - 1) / SA_KT, per = (nt + p.splits - 1) / p.splits;
  const int t0 = sp * per, t1 = min(nt, t0 + per);

  int qpos = 0, qlo = 0, qhi = 0;
  const float* myb = nullptr;
  float bL = 0.f, bR = 0.f;
  if constexpr (REL) {
    sa_fill_bias<NW>(ldsB, p.rel, head0, p.pack, tid);
    const int off = sa_q_offset(p.rel, b);
    qpos = qi + off;
    qlo = row_w / p.pack + off;
    qhi = min(row_w + 31, rows - 1) / p.pack + off;
    myb = ldsB + hl * (2 * p.rel.W + 1) + p.rel.W;
    __syncthreads();
    bL = myb[-p.rel.W];
    bR = myb[p.rel.W];
  }

  // Q^T operand of the lane's row; a negative scale turns its sign, so that the softmax can take its maximum over unscaled products
  sa_u32x4 qf[KS];
  {
    const char* src = p.q + ((long)b * p.q_sb + (long)qi * p.q_sl + (long)(head0 + hl) * p.q_sh) * 2;
    const unsigned flip = p.sl2 < 0.f ? 0x80008000u : 0u;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int d = ks * 16 + h * 8;
      qf[ks] = (sa_u32x4){0u, 0u, 0u, 0u};
      if (d < p.D) qf[ks] = *(const sa_u32x4*)(src + d * 2);
#pragma unroll
      for (int e = 0; e < 4; ++e) qf[ks][e] ^= flip;
    }
  }
  const float sl2 = fabsf(p.sl2);
  const float us = REL ? 1.f : sl2, lazy = SA_LAZY / us;       // units of the logits below: log2 with a bias, else unscaled products
  const char* const kb_ = p.k + ((long)b * p.k_sb + (long)hkv * p.k_sh) * 2;
  const char* const vb_ = p.v + ((long)b * p.v_sb + (long)hkv * p.v_sh) * 2;
  const uint8_t* const mb_ = p.key_mask ? p.key_mask + (long)b * p.mask_sb : nullptr;

  f32x16 O[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) O[i][r] = 0.f;
  float m = -INFINITY, l = 0.f;

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

    // S^T: keys x rows
    f32x16 s[NB];
#pragma unroll
    for (int kb = 0; kb < NB; ++kb) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[kb][r] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) s[kb] = sa_mfma<DT>(ad.rows(lk, kb * 32, ks), qf[ks], s[kb]);
    }
    if constexpr (REL) {
#pragma unroll
      for (int kb = 0; kb < NB; ++kb) {
        const int k0 = t * SA_KT + (half + kb) * 32;
        if (k0 - qhi >= p.rel.W || k0 + 31 - qlo <= -p.rel.W) {       // the whole block lies in the last bucket of a side
          const float c = k0 - qhi >= p.rel.W ? bR : bL;
#pragma unroll
          for (int r = 0; r < 16; ++r) s[kb][r] = __builtin_fmaf(s[kb][r], sl2, c);
        } else {
          const int d0 = k0 + 4 * h - qpos;
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int d = d0 + 8 * (r >> 2) + (r & 3);
            s[kb][r] = __builtin_fmaf(s[kb][r], sl2, myb[min(max(d, -p.rel.W), p.rel.W)]);
          }
        }
      }
    }
    if (live != ~0ul) {
#pragma unroll
      for (int kb = 0; kb < NB; ++kb) {
        const unsigned bits = (unsigned)(live >> ((half + kb) * 32)) >> (4 * h);
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (!((bits >> (8 * (r >> 2) + (r & 3))) & 1)) s[kb][r] = -INFINITY;
      }
    }
    float mt = -INFINITY;
#pragma unroll
    for (int kb = 0; kb < NB; ++kb)
#pragma unroll
      for (int r = 0; r < 16; r += 2) mt = fmaxf(fmaxf(mt, s[kb][r]), s[kb][r + 1]);
    mt = sa_xmax(mt);
    if (__ballot(mt > m + lazy)) {
      // (the difference of the references as they are subtracted below; m == mn also for rows without keys so far)
      const float mn = fmaxf(m, mt), a = m == mn ? 1.f : sa_exp2(m * us - mn * us);
      m = mn;
      l *= a;
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) O[i][r] *= a;
    }
    const float nm = m == -INFINITY ? 0.f : -m * us;
    float mult = sl2;
    if (!REL && __builtin_expect(__ballot(fabsf(nm) >= SA_HUGE) != 0, 0)) {
      mult = 1.f;
#pragma unroll
      for (int kb = 0; kb < NB; ++kb) s[kb] *= sl2;
    }
    sa_u32x4 pf[2 * NB];
#pragma unroll
    for (int kb = 0; kb < NB; ++kb) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[kb][r] = sa_exp2(REL ? s[kb][r] + nm : __builtin_fmaf(s[kb][r], mult, nm));
        l += s[kb][r];
      }
#pragma unroll
      for (int c = 0; c < 2; ++c)      // P in the operand type: relative error up to 2^-8 (bf16) / 2^-11 (f16) of each term of O's sum
#pragma unroll
        for (int e = 0; e < 4; ++e) pf[kb * 2 + c][e] = sa_pack2<DT>(s[kb][8 * c + 2 * e], s[kb][8 * c + 2 * e + 1]);
    }
#pragma unroll
    for (int c = 0; c < 2 * NB; ++c)
#pragma unroll
      for (int i = 0; i < NT; ++i) O[i] = sa_mfma<DT>(ad.cols(lv, c * 16, i), pf[c], O[i]);
  };
  kv.zero_columns(p.D, smem);
  sa_walk(t0, t1, fetch, step);

  l = sa_xsum(l);
  if constexpr (PAIR) {
    // the second wave of a pair hands its maximum, sum and O over through the tiles' memory
    float* const ml = (float*)(smem + C::TILES + SA_MASKS * 8) + (wr * 64 + lane) * 2;
    f32x16* const acc = (f32x16*)smem + wr * NT * 64 + lane;
    __syncthreads();
    if (half) {
      ml[0] = m;
      ml[1] = l;
#pragma unroll
      for (int i = 0; i < NT; ++i) acc[i * 64] = O[i];
    }
    __syncthreads();
    if (half) return;
    const float m1 = ml[0], mn = fmaxf(m, m1);
    const float a0 = m == mn ? 1.f : sa_exp2(m * us - mn * us), a1 = m1 == mn ? 1.f : sa_exp2(m1 * us - mn * us);
    m = mn;
    l = l * a0 + ml[1] * a1;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const f32x16 o1 = acc[i * 64];
#pragma unroll
      for (int r = 0; r < 16; ++r) O[i][r] = O[i][r] * a0 + o1[r] * a1;
    }
  }
  if (!wave_on) return;
  const bool any = l > 0.f || l != l;
  const float inv = any ? 1.f / l : 0.f;
  if (!on) return;
  const int head = head0 + hl;
  if (p.splits == 1) {
    if (p.lse && h == 0) sa_row_stat(p, b, head, qi, any, m * us, l);
    char* const dst = p.o + ((long)b * p.o_sb + (long)qi * p.o_sl + (long)head * p.o_sh) * 2;
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d = i * 32 + g * 8 + h * 4;
        if (d >= p.D) continue;
        *(uint2*)(dst + d * 2) = (uint2){sa_pack2<DT>(O[i][g * 4] * inv, O[i][g * 4 + 1] * inv), sa_pack2<DT>(O[i][g * 4 + 2] * inv, O[i][g * 4 + 3] * inv)};
      }
  } else {
    // partial result: normalised O [split][b][query][head][D], then the part's reference (-inf: no keys) and its sum [2][split][b][query][head]
    const long r1 = ((long)b * p.Lq + qi) * p.H + head, nr = (long)p.B * p.Lq * p.H;
    float* const dst = p.ws + ((long)sp * nr + r1) * p.D;
    if (h == 0) {
      float* const st = p.ws + p.splits * nr * p.D + sp * nr + r1;
      st[0] = any ? m * us : -INFINITY;
      st[p.splits * nr] = l;
    }
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d = i * 32 + g * 8 + h * 4;
        if (d < p.D) *(f32x4*)(dst + d) = (f32x4){O[i][g * 4] * inv, O[i][g * 4 + 1] * inv, O[i][g * 4 + 2] * inv, O[i][g * 4 + 3] * inv};
      }
  }
}

// o = sum_s w_s o_s / sum_s w_s, w_s = 2^(mu_s - max mu) l_s, splits in order.  One 8-element chunk of a row per thread.
template <int DT>
__global__ __launch_bounds__(256) void seq_attn_combine_kernel(const SaFwdParams p) {
  const int cpr = p.D / 8;
  const long nr = (long)p.B * p.Lq * p.H, idx = (long)blockIdx.x * 256 + threadIdx.x;
  if (idx >= nr * cpr) return;
  const long r = idx / cpr;
  const int c = (int)(idx - r * cpr);
  const float *const ls = p.ws + p.splits * nr * p.D + r, *const sums = ls + p.splits * nr;
  float m = -INFINITY;
  for (int s = 0; s < p.splits; ++s) m = fmaxf(m, ls[s * nr]);
  const float mu = m == -INFINITY ? 0.f : m;
  float l = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < p.splits; ++s) {
    const float wgt = sa_exp2(ls[s * nr] - mu) * sums[s * nr];
    const float* const src = p.ws + (s * nr + r) * p.D + c * 8;
    const f32x4 a = *(const f32x4*)src, bb = *(const f32x4*)(src + 4);
    l += wgt;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      o[e] = __builtin_fmaf(wgt, a[e], o[e]);
      o[4 + e] = __builtin_fmaf(wgt, bb[e], o[4 + e]);
    }
  }
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
  const int head = (int)(r % p.H);
  const long bq = r / p.H;
  const int qi = (int)(bq % p.Lq), b = (int)(bq / p.Lq);
  if (p.lse && c == 0) sa_row_stat(p, b, head, qi, l > 0.f || l != l, m, l);
  sa_u32x4 u;
#pragma unroll
  for (int e = 0; e < 4; ++e) u[e] = sa_pack2<DT>(o[2 * e] * inv, o[2 * e + 1] * inv);
  *(sa_u32x4*)(p.o + ((long)b * p.o_sb + (long)qi * p.o_sl + (long)head * p.o_sh + c * 8) * 2) = u;
}

// The same for many parts (a token over a long cache): one row per workgroup, its parts shared out over 256 / (D / 4) groups of lanes.
// With one thread per chunk the loop over the parts is a chain of loads: 26 us for 47 parts of 544 rows, D = 64; here 5.
template <int DT>
__global__ __launch_bounds__(256) void seq_attn_combine_row_kernel(const SaFwdParams p) {
  __shared__ float wgt[SA_MAX_SPLITS];
  __shared__ f32x4 part[256];
  const int tid = threadIdx.x, lane = tid & 63;
  const long nr = (long)p.B * p.Lq * p.H, r = blockIdx.x;
  const float *const ls = p.ws + p.splits * nr * p.D + r, *const sums = ls + p.splits * nr;
  // (every wave forms the maximum and the sum for itself)
  float m = -INFINITY, l = 0.f;
  for (int s = lane; s < p.splits; s += 64) m = fmaxf(m, ls[s * nr]);
  m = wave_max(m);
  const float mu = m == -INFINITY ? 0.f : m;
  for (int s = lane; s < p.splits; s += 64) {
    const float x = sa_exp2(ls[s * nr] - mu) * sums[s * nr];
    if (tid < 64) wgt[s] = x;
    l += x;
  }
  l = wave_sum(l);
  __syncthreads();
  const int nc = p.D / 4, groups = 256 / nc, c = tid % nc, g = tid / nc;
  f32x4 o = (f32x4){0.f, 0.f, 0.f, 0.f};
  if (g < groups) {
#pragma unroll 4
    for (int s = g; s < p.splits; s += groups) {
      const f32x4 a = *(const f32x4*)(p.ws + (s * nr + r) * p.D + c * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(wgt[s], a[e], o[e]);
    }
    part[tid] = o;
  }
  __syncthreads();
  if (tid >= nc) return;
  for (int k = 1; k < groups; ++k) o += part[k * nc + tid];
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
  const int head = (int)(r % p.H);
  const long bq = r / p.H;
  const int qi = (int)(bq % p.Lq), b = (int)(bq / p.Lq);
  if (p.lse && tid == 0) sa_row_stat(p, b, head, qi, l > 0.f || l != l, m, l);
  *(uint2*)(p.o + ((long)b * p.o_sb + (long)qi * p.o_sl + (long)head * p.o_sh + tid * 4) * 2) =
      (uint2){sa_pack2<DT>(o[0] * inv, o[1] * inv), sa_pack2<DT>(o[2] * inv, o[3] * inv)};
}

template <int DT, int DP, bool REL, bool PAIR>
static int sa_launch_fwd(const SaFwdParams& p, unsigned nwg, hipStream_t st) {
  struct Mine;
  const int lds = SaKvCfg<DP, PAIR>::LDS + (REL ? p.pack * (2 * p.rel.W + 1) * 4 : 0);
  if (lds > SA_MAX_LDS) return DFOLD_EINVAL;
  if (!sa_raise_lds<Mine>(seq_attn_fwd_kernel<DT, DP, REL, PAIR>, lds)) return DFOLD_ELAUNCH;
  DFOLD_LAUNCH((seq_attn_fwd_kernel<DT, DP, REL, PAIR>), dim3(nwg), dim3((PAIR ? 2 : 1) * 64 * SA_WAVES), lds, st, p);
  return dfold_check_launch();
}
template <int DT, int DP>
static int sa_fwd_dp(const SaFwdParams& p, bool rel, bool pair, unsigned nwg, hipStream_t st) {
  if (rel) return pair ? sa_launch_fwd<DT, DP, true, true>(p, nwg, st) : sa_launch_fwd<DT, DP, true, false>(p, nwg, st);
  return pair ? sa_launch_fwd<DT, DP, false, true>(p, nwg, st) : sa_launch_fwd<DT, DP, false, false>(p, nwg, st);
}
template <int DT>
static int sa_fwd(const SaFwdParams& p, bool rel, bool pair, unsigned nwg, hipStream_t st) {
  const int rc = p.D <= 32 ? sa_fwd_dp<DT, 32>(p, rel, pair, nwg, st) : p.D <= 64 ? sa_fwd_dp<DT, 64>(p, rel, pair, nwg, st) : sa_fwd_dp<DT, 128>(p, rel, pair, nwg, st);
  if (rc != DFOLD_OK || p.splits == 1) return rc;
  const long rows = (long)p.B * p.Lq * p.H, n = rows * (p.D / 8);
  if (p.splits >= 8 && rows <= 65536) {
    DFOLD_LAUNCH(seq_attn_combine_row_kernel<DT>, dim3((unsigned)rows), dim3(256), 0, st, p);
    return dfold_check_launch();
  }
  DFOLD_LAUNCH(seq_attn_combine_kernel<DT>, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, p);
  return dfold_check_launch();
}

extern "C" int dfold_seq_attn_fwd(const dfold_seq_attn_desc* d, void* stream) {
  SaFwdParams p;
  if (!sa_desc_ok(d) || d->splits < 1 || d->splits > SA_MAX_SPLITS || (d->splits > 1 && !d->ws)) return DFOLD_EINVAL;
  if (d->pack != 1 && d->pack != d->H / d->Hkv) return DFOLD_EINVAL;
  if (d->rel.table && !sa_make_rel(&d->rel, d->H, &p.rel)) return DFOLD_EINVAL;
  if (d->rel.table && (long)d->pack * (2 * p.rel.W + 1) * 4 > 32768) return DFOLD_EINVAL;
  p.q = (const char*)d->q; p.k = (const char*)d->k; p.v = (const char*)d->v; p.o = (char*)d->o;
  p.lse = d->lse; p.ws = d->ws; p.key_mask = d->key_mask; p.kv_lens = d->kv_lens;
  p.q_sb = d->q_sb; p.q_sl = d->q_sl; p.q_sh = d->q_sh; p.k_sb = d->k_sb; p.k_sl = d->k_sl; p.k_sh = d->k_sh;
  p.v_sb = d->v_sb; p.v_sl = d->v_sl; p.v_sh = d->v_sh; p.o_sb = d->o_sb; p.o_sl = d->o_sl; p.o_sh = d->o_sh; p.mask_sb = d->mask_sb;
  p.B = d->B; p.Lq = d->Lq; p.Lk = d->Lk; p.H = d->H; p.Hkv = d->Hkv; p.D = d->D; p.splits = d->splits; p.pack = d->pack;
  p.sl2 = d->scale * SA_LOG2E;
  const long rows = (long)d->Lq * d->pack, nrb = (rows + SA_ROWS - 1) / SA_ROWS;
  const long nwg = nrb * d->splits * (d->H / d->pack) * d->B, n = (long)d->B * d->Lq * d->H * (d->D / 8);
  if (rows > 0x7fffff00L || nwg > 0x7fffffffL || n / 256 > 0x7ffffff0L) return DFOLD_EINVAL;
  p.nrb = (int)nrb;
  return d->dtype == DFOLD_DT_BF16 ? sa_fwd<DFOLD_DT_BF16>(p, d->rel.table != nullptr, d->pair != 0, (unsigned)nwg, (hipStream_t)stream)
                                   : sa_fwd<DFOLD_DT_F16>(p, d->rel.table != nullptr, d->pair != 0, (unsigned)nwg, (hipStream_t)stream);
}
