// Learned relative position bias as a matrix: out[h][i][j] = table[bucket(j - i - offset)][h], and the table's gradient.
//
// Bound by the one write (forward) or read (backward) of the matrix.  Forward: a workgroup holds its head's bias over the distances
// -W .. W in LDS (beyond W it is constant) and writes 16-byte chunks of the head's matrix taken as one line; most chunks of a long
// matrix are one constant.  Backward: a workgroup reads a run of whole rows; what lies beyond W goes into two registers, in 16-byte
// chunks, a row per wave, eight chunks in flight per lane; the band in between is read along its diagonals, one distance per thread, so
// that no two threads add to the same number: no atomics, and an order that does not change.
#include "seq_attn.h"
#include "seq_dtable.h"

struct SaMatParams {
  void* out;
  const void* g;
  float* ws;
  int H, Lq, Lk, nb, nblk, rows;
  SaRel rel;
};

template <int DT> struct SaElem { typedef uint16_t type; static constexpr int VEC = 8; };
template <> struct SaElem<DFOLD_DT_F32> { typedef float type; static constexpr int VEC = 4; };
template <int DT>
__device__ __forceinline__ float sa_to_f32(typename SaElem<DT>::type v) {
  if constexpr (DT == DFOLD_DT_F32) return v;
  else return sa_lo<DT>((uint32_t)v);
}

#define SA_MAT_ITERS 8
template <int DT>
__global__ __launch_bounds__(256) void relpos_fwd_kernel(const SaMatParams p) {
  using E = typename SaElem<DT>::type;
  constexpr int V = SaElem<DT>::VEC;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  float* const bias = (float*)smem;
  const int tid = threadIdx.x, head = blockIdx.y, W = p.rel.W;
  const int off = p.rel.q_offset;
  for (int i = tid; i < 2 * W + 1; i += 256) bias[i] = p.rel.table[(long)sa_bucket(p.rel, i - W) * p.H + head];
  __syncthreads();
  const long n = (long)p.Lq * p.Lk, a = (head * n) % V;     // a: elements between the last 16-byte border and the head's matrix
  E* const dst = (E*)p.out + head * n;
  const float* const mid = bias + W;
  const float bL = mid[-W], bR = mid[W];
  long e0 = ((long)blockIdx.x * SA_MAT_ITERS * 256 + tid) * V - a;
  long i = e0 > 0 ? e0 / p.Lk : 0;
  long j = e0 - i * p.Lk;                                    // (negative in the first chunk of a head that starts off a border)
  const long si = 256L * V / p.Lk, sj = 256L * V - si * p.Lk;
  for (int it = 0; it < SA_MAT_ITERS && e0 < n; ++it) {
    float v[V];
    const long d0 = j - i - off;
    if (j >= 0 && j + V <= p.Lk && (d0 >= W || d0 + V - 1 <= -W)) {
      const float c = d0 >= W ? bR : bL;
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = c;
    } else {
      long jj = j, ii = i;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const long d = jj - ii - off;
        v[e] = mid[(int)min(max(d, (long)-W), (long)W)];
        if (++jj == p.Lk) { jj = 0; ++ii; }
      }
    }
    if constexpr (DT == DFOLD_DT_F32) {
      if (e0 >= 0 && e0 + V <= n) *(f32x4*)(dst + e0) = (f32x4){v[0], v[1], v[2], v[3]};
      else
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (e0 + e >= 0 && e0 + e < n) dst[e0 + e] = v[e];
    } else {
      sa_u32x4 u;
#pragma unroll
      for (int e = 0; e < 4; ++e) u[e] = sa_pack2<DT>(v[2 * e], v[2 * e + 1]);
      if (e0 >= 0 && e0 + V <= n) *(sa_u32x4*)(dst + e0) = u;
      else
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (e0 + e >= 0 && e0 + e < n) dst[e0 + e] = (uint16_t)(u[e / 2] >> (16 * (e & 1)));
    }
    e0 += 256L * V;
    i += si;
    j += sj;
    if (j >= p.Lk) { j -= p.Lk; ++i; }
    if (j < 0) { i = e0 / p.Lk; j = e0 - i * p.Lk; }
  }
}

template <int DT>
__global__ __launch_bounds__(256, 5) void relpos_bwd_kernel(const SaMatParams p) {
  using E = typename SaElem<DT>::type;
  constexpr int V = SaElem<DT>::VEC;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  float* const hist = (float*)smem;                 // [2 W + 1]
  __shared__ float side[2][4];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), head = blockIdx.y, W = p.rel.W, off = p.rel.q_offset;
  const long n = (long)p.Lq * p.Lk;
  const int i0 = blockIdx.x * p.rows, i1 = min(p.Lq, i0 + p.rows);
  const E* const g = (const E*)p.g + head * n;
  float aL = 0.f, aR = 0.f;
  if (i0 < i1) {
    // far distances: columns [0, jl) and [jr, Lk) of a row, as the aligned chunks that hold them -- a lane's loads are all issued before the
    // first sum; a chunk over a border counts by element.  (The loads go through a buffer descriptor that ends with the tensor's last
    // whole chunk: nothing to test.  Single elements in front of the first and behind the last border, each loaded under a test, cost an
    // L2 round trip each; only what lies behind the tensor's last whole chunk is read that way.)
    const long whole = (long)p.H * n / V * V;
    for (int i = i0 + w; i < i1; i += 4) {
      const long at = (long)i + off;
      const int jl = (int)min(max(at - W + 1, 0L), (long)p.Lk), jr = (int)min(max(at + W, (long)jl), (long)p.Lk);
      const long row = head * n + (long)i * p.Lk, base = row / V * V;
      const int shift = (int)(row - base);
      const unsigned bytes = (unsigned)min(max(whole - base, 0L) * (long)sizeof(E), 0x7ffffff0L);
      const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)((const E*)p.g + base), 0, bytes, 0x00020000);
      const int nl = jl > 0 ? (jl + shift + V - 1) / V : 0;                                  // chunks on the left: 0 .. nl
      const int r0 = (jr + shift) / V, nr = jr < p.Lk ? (p.Lk + shift + V - 1) / V - r0 : 0;  // and on the right: r0 .. r0 + nr
      for (int k0 = lane; k0 < nl + nr; k0 += 512) {
        sa_u32x4 x[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const int k = k0 + 64 * u, c = k < nl ? k : r0 + k - nl;
          x[u] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, k < nl + nr ? c * 16 : (int)0x80000000, 0, 0);
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const int k = k0 + 64 * u;
          const bool left = k < nl;
          const int j0 = (left ? k : r0 + k - nl) * V - shift, lo = left ? 0 : jr, hi = left ? jl : p.Lk;
          float v[V], a = 0.f;
          if constexpr (DT == DFOLD_DT_F32) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = __uint_as_float(x[u][e]);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              v[2 * e] = sa_lo<DT>(x[u][e]);
              v[2 * e + 1] = sa_hi<DT>(x[u][e]);
            }
          }
          if (k < nl + nr) {
            if (j0 >= lo && j0 + V <= hi) {
#pragma unroll
              for (int e = 0; e < V; ++e) a += v[e];
            } else {
#pragma unroll
              for (int e = 0; e < V; ++e) a += j0 + e >= lo && j0 + e < hi ? v[e] : 0.f;
            }
            if (left) aL += a; else aR += a;
          }
        }
      }
      if (row + p.Lk > whole) {          // (the last rows of the last head)
        const long e = whole + lane, j = e - row;
        if (lane < V && j >= 0 && j < p.Lk && (j < jl || j >= jr)) {
          const float x = sa_to_f32<DT>(((const E*)p.g)[e]);
          if (j < jl) aL += x; else aR += x;
        }
      }
    }
    // the band: distance d of every row of the run
    for (int d = tid - (W - 1); d <= W - 1; d += 256) {
      // j = i + off + d in [0, Lk)
      const long s = (long)off + d;
      const int ilo = (int)min(max((long)i0, -s), (long)i1), ihi = (int)max(min((long)i1, p.Lk - s), (long)ilo);
      float acc = 0.f;
#pragma unroll 16
      for (int i = ilo; i < ihi; ++i) acc += sa_to_f32<DT>(g[(long)i * p.Lk + i + s]);
      hist[W + d] = acc;
    }
  } else {
    for (int d = tid; d < 2 * W + 1; d += 256) hist[d] = 0.f;
  }
  aL = wave_sum(aL);
  aR = wave_sum(aR);
  if (lane == 0) { side[0][w] = aL; side[1][w] = aR; }
  __syncthreads();
  if (tid < 2) hist[tid ? 2 * W : 0] = (side[tid][0] + side[tid][1]) + (side[tid][2] + side[tid][3]);
  __syncthreads();
  sa_bucket_sums<4>(p.rel, hist, W, p.nb, p.ws + ((long)head * p.nblk + blockIdx.x) * p.nb, w, lane);
}

// row blocks of the backward: five workgroups per CU, one round of what fits (2048 of them: a second round of three, 170 -> 167 us at
// 16 x 4097 x 4100, 12.0 -> 8.2 at 8 x 256 x 256)
static inline int sa_mat_blocks(int H, int Lq) {
  const int want = 1280 / H > 1 ? 1280 / H : 1;
  return Lq < want ? Lq : want;
}
extern "C" int dfold_relpos_ws(int32_t H, int32_t Lq, int32_t num_buckets) {
  if (H <= 0 || Lq <= 0 || num_buckets <= 0) return DFOLD_EINVAL;
  const long f = (long)H * sa_mat_blocks(H, Lq) * num_buckets;
  return f > 0x7fffffffL ? DFOLD_EINVAL : (int)f;
}
static bool sa_mat_params(const dfold_rel_bias* rel, int dtype, int H, int Lq, int Lk, SaMatParams* p) {
  if (!rel || dtype < DFOLD_DT_BF16 || dtype > DFOLD_DT_F32 || H <= 0 || H > 65535 || Lq <= 0 || Lk <= 0 || Lq > (1 << 30) || Lk > (1 << 28)) return false;
  if (!sa_make_rel(rel, H, &p->rel)) return false;
  if (rel->q_offset > (1 << 29) || rel->q_offset < -(1 << 29)) return false;
  p->H = H; p->Lq = Lq; p->Lk = Lk; p->nb = rel->num_buckets;
  return true;
}

extern "C" int dfold_relpos_fwd(const dfold_rel_bias* rel, void* out, int32_t dtype, int32_t H, int32_t Lq, int32_t Lk, void* stream) {
  SaMatParams p;
  if (!out || ((uintptr_t)out & 15) || !sa_mat_params(rel, dtype, H, Lq, Lk, &p)) return DFOLD_EINVAL;
  p.out = out;
  const int V = dtype == DFOLD_DT_F32 ? 4 : 8;
  const long n = (long)Lq * Lk, chunks = (n + V - 1) / V + 1, nx = (chunks + 256 * SA_MAT_ITERS - 1) / (256 * SA_MAT_ITERS);
  if (nx > 0x7fffffffL) return DFOLD_EINVAL;
  const dim3 grid((unsigned)nx, H);
  const int lds = (2 * p.rel.W + 1) * 4;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == DFOLD_DT_BF16) DFOLD_LAUNCH(relpos_fwd_kernel<DFOLD_DT_BF16>, grid, dim3(256), lds, st, p);
  else if (dtype == DFOLD_DT_F16) DFOLD_LAUNCH(relpos_fwd_kernel<DFOLD_DT_F16>, grid, dim3(256), lds, st, p);
  else DFOLD_LAUNCH(relpos_fwd_kernel<DFOLD_DT_F32>, grid, dim3(256), lds, st, p);
  return dfold_check_launch();
}

extern "C" int dfold_relpos_bwd(const dfold_rel_bias* rel, const void* g, int32_t dtype, int32_t H, int32_t Lq, int32_t Lk, float* dtable, float* ws,
                                void* stream) {
  SaMatParams p;
  if (!g || ((uintptr_t)g & 15) || !dtable || !ws || !sa_mat_params(rel, dtype, H, Lq, Lk, &p)) return DFOLD_EINVAL;
  p.g = g;
  p.ws = ws;
  p.nblk = sa_mat_blocks(H, Lq);
  p.rows = (Lq + p.nblk - 1) / p.nblk;
  const dim3 grid(p.nblk, H);
  const int lds = (2 * p.rel.W + 1) * 4;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == DFOLD_DT_BF16) DFOLD_LAUNCH(relpos_bwd_kernel<DFOLD_DT_BF16>, grid, dim3(256), lds, st, p);
  else if (dtype == DFOLD_DT_F16) DFOLD_LAUNCH(relpos_bwd_kernel<DFOLD_DT_F16>, grid, dim3(256), lds, st, p);
  else DFOLD_LAUNCH(relpos_bwd_kernel<DFOLD_DT_F32>, grid, dim3(256), lds, st, p);
  const int rc = dfold_check_launch();
  if (rc != DFOLD_OK) return rc;
  DFOLD_LAUNCH(seq_dtable_kernel, dim3(H, (p.nb + 63) / 64), dim3(1024), 0, st, (const float*)ws, dtable, p.nb, 1, H, p.nblk);
  return dfold_check_launch();
}
