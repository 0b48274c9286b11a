// Norm of query and key heads with the position rotation in the same pass:  y = R(position) (x * rsqrt(mean x^2 + eps) * w).
// Backward, with xh = x * rstd and g' = R^T g:   dw = sum over rows of g' xh,   dx = rstd (w g' - xh mean(w g' xh)).
//
// Bound by memory: forward x in, y out; backward x, g in, dx out (rstd is formed again from x, nothing is kept in between).  A row
// (token, head) is held by 2^lpr lanes of 16 bytes each; a row slot keeps ONE token and walks several heads of it, so that the
// angles -- an fp64 product, a subtraction of whole turns and one sincos per rotated pair -- are formed once per token and slot.
// q and k go in one launch: the first blocks are q's, the rest k's.
#include "seq_attn.h"
#include <math.h>

#define NR_MAX_D 256
#define NR_BWD_BLOCKS 1024

struct NrPart {
  const char *x, *g;
  char* y;
  const float* w;
  float *dw, *ws;
  const int64_t* pos;
  long x_sb, x_sl, x_sh, g_sb, g_sl, g_sh, pos_sb, items;   // items: (token, first head) slots of work
  int L, H, spt, blocks;                                    // spt: slots per token; a slot's heads are first, first + spt, ...
};
struct NrParams {
  NrPart part[2];
  int D, rd, inter, lpr;         // 2^lpr lanes per row
  float eps;
  double turns[NR_MAX_D / 2];    // base^(-2 i / rd) / (2 pi)
};

template <int DT> struct NrVec { static constexpr int V = DT == DFOLD_DT_F32 ? 4 : 8; };
template <int DT>
__device__ __forceinline__ void nr_load(const char* p, float (&v)[NrVec<DT>::V]) {
  if constexpr (DT == DFOLD_DT_F32) {
    const f32x4 x = *(const f32x4*)p;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = x[e];
  } else {
    const sa_u32x4 x = *(const sa_u32x4*)p;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[2 * e] = sa_lo<DT>(x[e]);
      v[2 * e + 1] = sa_hi<DT>(x[e]);
    }
  }
}
template <int DT>
__device__ __forceinline__ void nr_store(char* p, const float (&v)[NrVec<DT>::V]) {
  if constexpr (DT == DFOLD_DT_F32) *(f32x4*)p = (f32x4){v[0], v[1], v[2], v[3]};
  else *(sa_u32x4*)p = (sa_u32x4){sa_pack2<DT>(v[0], v[1]), sa_pack2<DT>(v[2], v[3]), sa_pack2<DT>(v[4], v[5]), sa_pack2<DT>(v[6], v[7])};
}
// cosine and signed sine of the lane's dimensions: y = x cos + partner(x) sin
template <int DT>
__device__ __forceinline__ void nr_angles(const NrParams& p, double pos, int d0, float (&c)[NrVec<DT>::V], float (&s)[NrVec<DT>::V]) {
  constexpr int V = NrVec<DT>::V;
  auto sc = [&](int i, float& sn, float& cs) {
    double t = pos * p.turns[i];
    // whole turns drop out in fp64.  The factor's and the product's roundings: below 2^-24 rad up to positions of 2^28, doubling with the
    // position from there (a second word of the factor: right to 2^34, but 141 -> 155 us of the forward at 4 x 8192, 32 + 8 heads x 128)
    t -= rint(t);
    sincospif(2.f * (float)t, &sn, &cs);
  };
  if (p.inter) {
#pragma unroll
    for (int e = 0; e < V; e += 2) {
      float sn, cs;
      sc((d0 + e) >> 1, sn, cs);
      c[e] = c[e + 1] = cs;
      s[e] = -sn;
      s[e + 1] = sn;
    }
  } else {
    const int half = p.rd >> 1;
    const bool second = d0 >= half;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float sn, cs;
      sc(d0 + e - (second ? half : 0), sn, cs);
      c[e] = cs;
      s[e] = second ? sn : -sn;
    }
  }
}
// r = x cos + sgn partner(x) sin for the rotated lanes (every lane of the wave takes part in the exchange)
template <int DT>
__device__ __forceinline__ void nr_rotate(const NrParams& p, bool rot, int partner, float sgn, const float (&c)[NrVec<DT>::V], const float (&s)[NrVec<DT>::V],
                                          float (&v)[NrVec<DT>::V]) {
  constexpr int V = NrVec<DT>::V;
  float o[V];
  if (p.inter) {
#pragma unroll
    for (int e = 0; e < V; ++e) o[e] = v[e ^ 1];
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) o[e] = __shfl(v[e], partner, 64);
  }
  if (rot)
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = __builtin_fmaf(o[e], sgn * s[e], v[e] * c[e]);
}

template <int DT, bool BWD>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(const NrParams p) {
  constexpr int V = NrVec<DT>::V, ES = DT == DFOLD_DT_F32 ? 4 : 2;
  __shared__ float red[BWD ? 256 * V : 1];
  const int tid = threadIdx.x, lane = tid & 63;
  const bool second = (int)blockIdx.x >= p.part[0].blocks;
  const NrPart& q = p.part[second ? 1 : 0];
  const int blk = blockIdx.x - (second ? p.part[0].blocks : 0);
  const int lanes = 1 << p.lpr, slots = 256 >> p.lpr, li = tid & (lanes - 1), d0 = li * V;
  const bool on = d0 < p.D, rot = d0 < p.rd;
  // partner lane of the half-split rotation: +- rd / 2 dimensions
  const int hl = (p.rd >> 1) / V;
  const int partner = rot ? (d0 < (p.rd >> 1) ? lane + hl : lane - hl) : lane;
  float w[V], acc[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    w[e] = on ? (q.w ? q.w[d0 + e] : 1.f) : 0.f;
    acc[e] = 0.f;
  }
  const float invD = 1.f / (float)p.D;
  const long step = (long)q.blocks * slots;
  // (all lanes of a wave walk together: lanes whose slot has no item left repeat the last one and store nothing)
  for (long it0 = (long)blk * slots; it0 < q.items; it0 += step) {
    const long item_r = it0 + (tid >> p.lpr), item = min(item_r, q.items - 1);
    const bool live = on && item_r < q.items;
    const long tok = item / q.spt;
    const int h0 = (int)(item - tok * q.spt);
    const int b = (int)(tok / q.L), l = (int)(tok - (long)b * q.L);
    float c[V], s[V];
    if (rot) nr_angles<DT>(p, q.pos ? (double)q.pos[(long)b * q.pos_sb + l] : (double)l, d0, c, s);
    const char* const xb = q.x + ((long)b * q.x_sb + (long)l * q.x_sl + d0) * ES;
    char* const yb = q.y + (tok * q.H * p.D + d0) * ES;
    const char* const gb = BWD ? q.g + ((long)b * q.g_sb + (long)l * q.g_sl + d0) * ES : nullptr;
    for (int hh = 0; hh < q.H; hh += q.spt) {          // (same number of turns in every slot)
      const int h = h0 + hh;
      const bool use = live && h < q.H;
      float x[V], g[V];
#pragma unroll
      for (int e = 0; e < V; ++e) x[e] = g[e] = 0.f;
      if (use) {
        nr_load<DT>(xb + (long)h * q.x_sh * ES, x);
        if constexpr (BWD) nr_load<DT>(gb + (long)h * q.g_sh * ES, g);
      }
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < V; ++e) ss = __builtin_fmaf(x[e], x[e], ss);
      for (int o = 1; o < lanes; o <<= 1) ss += __shfl_xor(ss, o, 64);
      // (lanes without a row would divide by 0 where eps is 0: 0 * inf in dw's sum.  Chosen before the root: no branch around it)
      const float rstd = 1.f / sqrtf(use ? __builtin_fmaf(ss, invD, p.eps) : 1.f);
      if constexpr (!BWD) {
#pragma unroll
        for (int e = 0; e < V; ++e) x[e] = x[e] * rstd * w[e];
        nr_rotate<DT>(p, rot, partner, 1.f, c, s, x);
        if (use) nr_store<DT>(yb + (long)h * p.D * ES, x);
      } else {
        nr_rotate<DT>(p, rot, partner, -1.f, c, s, g);
        float dot = 0.f;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          x[e] *= rstd;
          acc[e] = __builtin_fmaf(g[e], x[e], acc[e]);
          g[e] *= w[e];
          dot = __builtin_fmaf(g[e], x[e], dot);
        }
        for (int o = 1; o < lanes; o <<= 1) dot += __shfl_xor(dot, o, 64);
        dot *= invD;
#pragma unroll
        for (int e = 0; e < V; ++e) x[e] = rstd * (g[e] - x[e] * dot);
        if (use) nr_store<DT>(yb + (long)h * p.D * ES, x);
      }
    }
  }
  if constexpr (BWD) {
    if (!q.dw) return;
    // the block's sum over its row slots, in slot order
#pragma unroll
    for (int e = 0; e < V; ++e) red[tid * V + e] = acc[e];
    __syncthreads();
    const int width = lanes * V;
    for (int d = tid; d < p.D; d += 256) {
      float a = 0.f;
      for (int k = 0; k < slots; ++k) a += red[k * width + d];
      q.ws[(long)blk * p.D + d] = a;
    }
  }
}

// dw[d] = sum of the blocks' sums, in a fixed order: 16 dimensions x 64 strided parts per workgroup
__global__ __launch_bounds__(1024) void qk_norm_rope_dw_kernel(const NrParams p) {
  __shared__ double part[64][16];
  const NrPart& q = p.part[blockIdx.y];
  if (!q.dw) return;
  const int d = blockIdx.x * 16 + (threadIdx.x & 15), w = threadIdx.x >> 4;
  double a = 0.;
  if (d < p.D)
#pragma unroll 8
    for (int i = w; i < q.blocks; i += 64) a += (double)q.ws[(long)i * p.D + d];
  part[w][threadIdx.x & 15] = a;
  __syncthreads();
  if (w == 0 && d < p.D) {
#pragma unroll
    for (int k = 1; k < 64; ++k) a += part[k][threadIdx.x];
    q.dw[d] = (float)a;
  }
}

extern "C" int dfold_qk_norm_rope_ws(void) { return 2 * NR_BWD_BLOCKS * NR_MAX_D; }

static int nr_run(const dfold_norm_rope_desc* d, bool bwd, void* stream) {
  NrParams p;
  if (!d || d->dtype < DFOLD_DT_BF16 || d->dtype > DFOLD_DT_F32 || d->B <= 0) return DFOLD_EINVAL;
  if (d->D <= 0 || d->D > NR_MAX_D || d->D % 8 || d->rotary_dim < 0 || d->rotary_dim > d->D || d->rotary_dim % 16) return DFOLD_EINVAL;
  if (!(d->eps >= 0.f) || !(d->base > 0.)) return DFOLD_EINVAL;
  const int V = d->dtype == DFOLD_DT_F32 ? 4 : 8;
  p.D = d->D; p.rd = d->rotary_dim; p.inter = d->interleaved != 0; p.eps = d->eps;
  p.lpr = 0;
  while ((V << p.lpr) < d->D) ++p.lpr;
  const int slots = 256 >> p.lpr;
  for (int i = 0; i < p.rd / 2; ++i) p.turns[i] = pow(d->base, -2.0 * i / p.rd) / (2.0 * M_PI);
  long blocks = 0;
  bool dw = false;
  for (int k = 0; k < 2; ++k) {
    const dfold_norm_rope_part* s = &d->part[k];
    NrPart* q = &p.part[k];
    *q = NrPart();
    if (!s->x) continue;
    if (!s->y || (bwd && !s->g) || s->L <= 0 || s->H <= 0) return DFOLD_EINVAL;
    if (((uintptr_t)s->x | (uintptr_t)s->y | (uintptr_t)(bwd ? s->g : nullptr)) & 15) return DFOLD_EINVAL;
    const int64_t st[6] = {s->x_sb, s->x_sl, s->x_sh, bwd ? s->g_sb : 0, bwd ? s->g_sl : 0, bwd ? s->g_sh : 0};
    for (int i = 0; i < 6; ++i)
      if (st[i] % V || st[i] < 0) return DFOLD_EINVAL;
    if (s->pos && s->pos_sb < 0) return DFOLD_EINVAL;
    q->x = (const char*)s->x; q->g = (const char*)s->g; q->y = (char*)s->y; q->w = s->w; q->pos = s->pos;
    q->x_sb = s->x_sb; q->x_sl = s->x_sl; q->x_sh = s->x_sh; q->g_sb = s->g_sb; q->g_sl = s->g_sl; q->g_sh = s->g_sh; q->pos_sb = s->pos_sb;
    q->L = s->L; q->H = s->H;
    const long tokens = (long)d->B * s->L, rows = tokens * s->H;
    // heads per slot: as many as leave the chip 4 workgroups per CU, up to 8 (the angles then cost an eighth); few rows: 1
    int hps = 1;
    while (hps < 8 && hps < s->H && rows / (2 * hps) >= 1024L * slots) hps *= 2;
    q->spt = (s->H + hps - 1) / hps;
    q->items = tokens * q->spt;
    long nb = (q->items + slots - 1) / slots;
    if (bwd) {
      if (nb > NR_BWD_BLOCKS) nb = NR_BWD_BLOCKS;
      if (s->dw) {
        if (!d->ws) return DFOLD_EINVAL;
        q->dw = s->dw;
        q->ws = d->ws + (long)k * NR_BWD_BLOCKS * NR_MAX_D;
        dw = true;
      }
    } else if (nb > 65536) nb = 65536;
    q->blocks = (int)nb;
    blocks += nb;
  }
  if (blocks == 0) return DFOLD_EINVAL;
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)blocks);
#define NR_LAUNCH(DT)                                                                              \
  do {                                                                                             \
    if (bwd) DFOLD_LAUNCH((qk_norm_rope_kernel<DT, true>), grid, dim3(256), 0, st, p);             \
    else DFOLD_LAUNCH((qk_norm_rope_kernel<DT, false>), grid, dim3(256), 0, st, p);                \
  } while (0)
  if (d->dtype == DFOLD_DT_BF16) NR_LAUNCH(DFOLD_DT_BF16);
  else if (d->dtype == DFOLD_DT_F16) NR_LAUNCH(DFOLD_DT_F16);
  else NR_LAUNCH(DFOLD_DT_F32);
  const int rc = dfold_check_launch();
  if (rc != DFOLD_OK || !dw) return rc;
  DFOLD_LAUNCH(qk_norm_rope_dw_kernel, dim3((p.D + 15) / 16, 2), dim3(1024), 0, st, p);
  return dfold_check_launch();
}
extern "C" int dfold_qk_norm_rope_fwd(const dfold_norm_rope_desc* d, void* stream) { return nr_run(d, false, stream); }
extern "C" int dfold_qk_norm_rope_bwd(const dfold_norm_rope_desc* d, void* stream) { return nr_run(d, true, stream); }
