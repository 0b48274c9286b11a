// Attention of one sequence over another (seq_attn_fwd.hip, seq_attn_bwd.hip): tile images, operand fragments and the bucketed
// relative position bias that the forward and the backward kernels share.
//
// Everything runs on v_mfma_f32_32x32x16 (bf16 / f16 operands, fp32 accumulators).  Its accumulator holds column lane & 31 and rows
// 8 (r / 4) + 4 (lane / 32) + r % 4, r = 0 .. 15, so a product whose COLUMNS are the softmax rows (S^T = K Q^T) leaves every lane
// with scores of one row only: maxima and sums are a register tree and one exchange between the two lane halves, and eight
// consecutive accumulator registers ARE a B operand of the next product once its A operand counts the reduction index in the same
// order: slot s of half h of 16-block c <-> index 16 c + 8 (s / 4) + 4 h + s % 4.  A operands of that order come out of LDS by the
// transpose read (4 rows x 16 columns per 16 lanes); P and dS never touch LDS.
#pragma once
#include "dfold_common.h"
#include "../../include/dfold_hip.h"
#include <atomic>

#define SA_LOG2E 1.44269504088896341f
#define SA_KT 64                       // rows of an LDS tile
#define SA_MAX_LDS (160 * 1024)
#define SA_WAVES 4
#define SA_REACH 64                    // distances a 32 x 32 block can lie beyond W and still not be uniform
#define SA_ROWS (32 * SA_WAVES)        // softmax rows (forward, dQ) or keys (dK, dV) of a workgroup

typedef __attribute__((ext_vector_type(4))) unsigned sa_u32x4;
typedef __attribute__((ext_vector_type(4))) short sa_s16x4;
typedef __attribute__((ext_vector_type(8))) short sa_s16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 sa_f16x8;
typedef __attribute__((ext_vector_type(2))) _Float16 sa_f16x2;
typedef __attribute__((address_space(3))) char sa_lchar;
typedef __attribute__((address_space(3))) sa_s16x4 sa_ls16x4;

template <int DT>
__device__ __forceinline__ f32x16 sa_mfma(const sa_u32x4 a, const sa_u32x4 b, const f32x16 c) {
  if constexpr (DT == DFOLD_DT_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(sa_f16x8, a), __builtin_bit_cast(sa_f16x8, b), c, 0, 0, 0);
}
// two fp32 values rounded to nearest even in the operand type
template <int DT>
__device__ __forceinline__ uint32_t sa_pack2(float lo, float hi) {
  if constexpr (DT == DFOLD_DT_BF16) return pack2bf_hw(lo, hi);
  const dfold_f32x2 v = {lo, hi};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, sa_f16x2));
}
template <int DT>
__device__ __forceinline__ float sa_lo(uint32_t pair) {
  if constexpr (DT == DFOLD_DT_BF16) return bf_lo(pair);
  return (float)__builtin_bit_cast(sa_f16x2, pair)[0];
}
template <int DT>
__device__ __forceinline__ float sa_hi(uint32_t pair) {
  if constexpr (DT == DFOLD_DT_BF16) return bf_hi(pair);
  return (float)__builtin_bit_cast(sa_f16x2, pair)[1];
}
// combine the two lane halves (lane, lane ^ 32) of a value
__device__ __forceinline__ float sa_xmax(float v) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float sa_xsum(float v) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}
__device__ __forceinline__ float sa_exp2(float v) { return __builtin_amdgcn_exp2f(v); }

// A row's softmax is two numbers: the reference mu of its exponents (log2 units, as rounded where it is subtracted) and the sum l of exp2(logit - mu).
// One fp32, mu + log2(l), would lose l where |mu| is large (rows of nothing but keys whose bias is -1e9).  Up to SA_WIDE the sum of the two is right to
// 2^-16, and the backward subtracts it at once; beyond, it subtracts one after the other.
#define SA_WIDE 256.f
// Without a bias the exponent is fma(s, sl2, -mu) for mu = m sl2 as rounded.  The exact product differs from a rounded one by up to half a step of mu: a
// factor common to the row, but a step is 2 from 2^24 on, and the factor leaves fp32 at 2^31 (f16 P at 2^28).  Rows beyond 2^24 round the product as
// the reference was, forward and backward alike.
#define SA_HUGE 0x1p24f
__device__ __forceinline__ float sa_exponent(float s, float sl2, float mu) {
  return fabsf(mu) >= SA_HUGE ? s * sl2 - mu : __builtin_fmaf(s, sl2, -mu);
}

// workgroup id -> work id: blockIdx round-robins over the 8 XCDs, consecutive work ids (which share K and V) stay on one of them
__device__ __forceinline__ unsigned sa_work_id() {
  const unsigned nwg = gridDim.x, bid = blockIdx.x;
  const unsigned q = nwg >> 3, r = nwg & 7, xcd = bid & 7, idx = bid >> 3;
  return (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + idx;
}

// ---- LDS tiles: SA_KT rows of DP 16-bit values, 16-byte chunks XOR-permuted within a row.  The key makes both kinds of read
//      conflict-free: 16 consecutive rows at one chunk (operand rows) and 4 consecutive rows at 4 consecutive chunks (transpose
//      reads; rows 0 .. 3 of a quadruple must land in different 64-byte groups of the 256-byte bank line).  It depends on row % 16
//      only, so every address is one of a lane's few offsets plus a constant that fits the instruction ----
template <int DP>
struct SaTile {
  static constexpr int CPR = DP / 8;                       // chunks per row: 4, 8, 16
  static constexpr int PITCH = DP * 2;
  static constexpr int BYTES = SA_KT * PITCH;
  static constexpr int KS = DP / 16, NT = DP / 32;         // 16-deep steps, 32-wide column tiles
  static __device__ __forceinline__ int key(int row) {
    if constexpr (CPR == 16) return ((row & 3) << 2) | ((row >> 2) & 3);
    if constexpr (CPR == 8) return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
    return (row >> 2) & 3;
  }
  static __device__ __forceinline__ int off(int row, int chunk) { return row * PITCH + ((chunk ^ key(row)) << 4); }
};

// A lane's offsets into a tile.  rows(r0, ks): lane holds row r0 + (lane & 31), elements 16 ks + 8 h .. + 8.  cols(r0, dt): lane holds
// column 32 dt + (lane & 31), rows r0 + 4 h + 0 .. 3 and r0 + 8 + 4 h + 0 .. 3.  r0 a multiple of 16, a constant at every use.
template <int DP>
struct SaAddr {
  using T = SaTile<DP>;
  int row[T::KS], col[T::NT][2];
  // shift: rows added to every r0 (a multiple of 16, the same for the wave)
  __device__ __forceinline__ SaAddr(int lane, int shift = 0) {
    const int h = lane >> 5, i = lane & 15;
#pragma unroll
    for (int ks = 0; ks < T::KS; ++ks) row[ks] = T::off(lane & 31, 2 * ks + h) + shift * T::PITCH;
#pragma unroll
    for (int dt = 0; dt < T::NT; ++dt)
#pragma unroll
      for (int x = 0; x < 2; ++x)
        col[dt][x] = T::off(8 * x + 4 * h + (i >> 2), 4 * dt + 2 * ((lane >> 4) & 1) + ((i & 3) >> 1)) + (i & 1) * 8 + shift * T::PITCH;
  }
  __device__ __forceinline__ sa_u32x4 rows(const char* t, int r0, int ks) const { return *(const sa_u32x4*)(t + row[ks] + r0 * T::PITCH); }
  __device__ __forceinline__ sa_u32x4 cols(const char* t, int r0, int dt) const {
    sa_lchar* b = (sa_lchar*)t;
    const sa_s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((sa_ls16x4*)(b + col[dt][0] + r0 * T::PITCH));
    const sa_s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((sa_ls16x4*)(b + col[dt][1] + r0 * T::PITCH));
    return __builtin_bit_cast(sa_u32x4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  }
};

// SA_KT (or ROWS) rows of a [rows][D] matrix with row stride `rs` elements (< SA_MAX_ROW) into an LDS tile, by LDS-DMA: no registers and
// no LDS write instructions.  A wave's instruction fills 1 KB of the tile in lane order, so the chunk permutation is applied to the
// source.  Rows past the last one repeat it (never out of range; their content is masked by the caller).  Lanes whose chunk lies past D load
// nothing: zero_columns() clears their places once, and they stay zeros under every tile that follows.
#define SA_MAX_ROW (1 << 24)
typedef __attribute__((address_space(3))) void* sa_lds_ptr;
template <int DP, int NW = SA_WAVES, int ROWS = SA_KT>
struct SaDma {
  using T = SaTile<DP>;
  static constexpr int NCH = ROWS * T::CPR / (64 * NW);    // instructions per wave
  static constexpr int STEP = 64 * NW / T::CPR;            // rows between a lane's chunks (a multiple of 16: one permutation key)
  static_assert(NCH >= 1 && STEP % 16 == 0, "whole instructions, one key per lane");
  int row, col, plain;     // plain: rows from which a tile is loaded without a test
  bool in;                 // the lane's columns are below D
  unsigned rs2, voff;      // bytes of a row, of this lane's first chunk
  __device__ __forceinline__ SaDma(long rs, int D, int tid) {
    row = tid / T::CPR;
    const int cc = (tid % T::CPR) ^ T::key(row);
    in = cc * 8 < D;
    col = cc * 16;
    plain = D == DP ? ROWS : INT32_MAX;
    rs2 = (unsigned)rs * 2u;
    voff = row * rs2 + col;
  }
  // rows row0 .. of a matrix of `end` > row0 rows -> tile; w: the wave's number in the workgroup
  __device__ __forceinline__ void load(const char* base, int row0, int end, char* tile, int w) const {
    const char* const src = base + (long)row0 * rs2;
    const int last = end - 1 - row0;
    if (last + 1 >= plain) {
#pragma unroll
      for (int i = 0; i < NCH; ++i)
        __builtin_amdgcn_global_load_lds((const void*)(src + (long)(i * STEP) * rs2 + voff), (sa_lds_ptr)(tile + (i * NW + w) * 1024), 16, 0, 0);
    } else if (in) {
#pragma unroll
      for (int i = 0; i < NCH; ++i)
        __builtin_amdgcn_global_load_lds((const void*)(src + (min(row + i * STEP, last) * rs2 + col)), (sa_lds_ptr)(tile + (i * NW + w) * 1024), 16, 0, 0);
    }
  }
  // columns past D of this lane's share of a tile become zeros (before the first load's barrier)
  __device__ __forceinline__ void zero_columns(char* tile, int tid) const {
    if (in) return;
#pragma unroll
    for (int i = 0; i < NCH; ++i) *(sa_u32x4*)(tile + (i * 64 * NW + tid) * 16) = (sa_u32x4){0u, 0u, 0u, 0u};
  }
  // rows whose bit is 0 become zeros (this thread's share; between two barriers)
  __device__ __forceinline__ void zero(unsigned long live, char* tile, int tid) const {
#pragma unroll
    for (int i = 0; i < NCH; ++i)
      if (!((live >> (row + i * STEP)) & 1)) *(sa_u32x4*)(tile + (i * 64 * NW + tid) * 16) = (sa_u32x4){0u, 0u, 0u, 0u};
  }
};
#define SA_MASKS 64                    // tiles whose key masks wait in LDS
// LDS of the K, V walk: two stages of two tiles, mask words, what pairs exchange; then the bias
template <int DP, bool PAIR>
struct SaKvCfg {
  static constexpr int TILES = 4 * SaTile<DP>::BYTES;
  static constexpr int LDS = TILES + SA_MASKS * 8 + (PAIR ? SA_WAVES * 64 * 8 : 0);
};
// The two tiles of a step side by side in LDS (K and V, or Q and dO).  One group of four waves: each loads its share of both; two
// groups: the first loads one, the second the other.
template <int DP, bool PAIR>
struct SaKvTiles {
  using T = SaTile<DP>;
  const char *a, *b;
  SaDma<DP> la, lb;
  int tid, w, half;
  __device__ __forceinline__ SaKvTiles(const char* pa, long rsa, const char* pb, long rsb, int D, int t, int wave)
      : a(PAIR && wave >= SA_WAVES ? pb : pa), b(pb), la(PAIR && wave >= SA_WAVES ? rsb : rsa, D, t & (64 * SA_WAVES - 1)), lb(rsb, D, t & (64 * SA_WAVES - 1)),
        tid(t & (64 * SA_WAVES - 1)), w(wave & (SA_WAVES - 1)), half(wave / SA_WAVES) {}
  __device__ __forceinline__ void load(int row0, int end, char* tile) const { load(a, b, row0, end, tile); }
  // the same from other bases (sa, sb: this wave's first, and for one group its second matrix)
  __device__ __forceinline__ void load(const char* sa, const char* sb, int row0, int end, char* tile) const {
    la.load(sa, row0, end, tile + (PAIR ? half * T::BYTES : 0), w);
    if constexpr (!PAIR) lb.load(sb, row0, end, tile + T::BYTES, w);
  }
  // columns past D of both stages at `tiles`
  __device__ __forceinline__ void zero_columns(int D, char* tiles) const {
    if (D == DP) return;
#pragma unroll
    for (int stage = 0; stage < 2; ++stage) {
      la.zero_columns(tiles + (2 * stage + (PAIR ? half : 0)) * T::BYTES, tid);
      if constexpr (!PAIR) lb.zero_columns(tiles + (2 * stage + 1) * T::BYTES, tid);
    }
  }
  __device__ __forceinline__ void zero(unsigned long live, char* tile) const {
    la.zero(live, tile + (PAIR ? half * T::BYTES : 0), tid);
    if constexpr (!PAIR) lb.zero(live, tile + T::BYTES, tid);
  }
};
// every DMA of this wave has landed and its LDS accesses are done, then everybody's
__device__ __forceinline__ void sa_landed() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
// a barrier for LDS accesses only
__device__ __forceinline__ void sa_lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
template <int I>
struct SaInt {
  static constexpr int value = I;
};
// The walk over tiles n0 .. n1 through two stages of LDS, one tile ahead: load(n, stage) requests tile n, work(n, stage) runs when it has
// landed for everybody, its stage a constant.  (Three and four stages, also for a single workgroup per CU: no gain at any size.)
template <typename L, typename W>
__device__ __forceinline__ void sa_walk(int n0, int n1, L load, W work) {
  if (n0 < n1) load(n0, 0);
  auto one = [&](int n, auto stage) {
    sa_landed();
    if (n + 1 < n1) load(n + 1, 1 - decltype(stage)::value);      // into the stage of tile n - 1: everybody is done with it
    work(n, stage);
  };
  for (int n = n0; n < n1; n += 2) {
    one(n, SaInt<0>());
    if (n + 1 < n1) one(n + 1, SaInt<1>());
  }
}
// Which keys of a tile exist, one bit per key.  Without a key mask that is arithmetic; with one, the words of SA_MASKS tiles at a time are
// formed by all waves (a byte per lane, a ballot per tile) and wait in LDS.
template <int NW>
struct SaLive {
  const uint8_t* mask;
  int end, t0, t1, w, lane;
  unsigned long* lds;
  // (every wave calls it for every tile in order, behind the tile's barrier)
  __device__ __forceinline__ unsigned long tile(int t) const {
    if (!mask) {
      const int n = end - t * SA_KT;
      return n >= SA_KT ? ~0ul : (1ul << n) - 1;
    }
    const int i = (t - t0) & (SA_MASKS - 1);
    if (i == 0) {
      for (int k = w; k < SA_MASKS && t + k < t1; k += NW) {
        const int key = (t + k) * SA_KT + lane;
        const unsigned long live = __ballot(key < end && mask[min(key, end - 1)] != 0);
        if (lane == 0) lds[k] = live;
      }
      sa_lds_barrier();
    }
    const unsigned long v = lds[i];
    return ((unsigned long)(unsigned)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32) | (unsigned)__builtin_amdgcn_readfirstlane((int)v);
  }
};

// ---- bucketed relative position bias ----
struct SaRel {
  const float* table;      // [num_buckets][H]
  const int32_t* q_offsets;  // [B] or null: position of query 0 minus position of key 0
  int q_offset, H, half, exact, nfar, W, both;   // W: every |distance| >= W is in the last bucket of its side
  int16_t far[DFOLD_REL_FAR];                    // far[k]: first distance of bucket exact + 1 + k
};
// first distance of one-sided bucket j
__device__ __forceinline__ int sa_bucket_lo(const SaRel& r, int j) { return j <= r.exact ? j : r.far[j - r.exact - 1]; }
__device__ __forceinline__ int sa_bucket(const SaRel& r, int delta) {
  const int n = r.both ? abs(delta) : max(-delta, 0);
  const int base = r.both && delta > 0 ? r.half : 0;
  if (n < r.exact) return base + n;
  int lo = 0, hi = r.nfar;              // number of borders <= n
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (r.far[mid] <= n) lo = mid + 1; else hi = mid;
  }
  return base + r.exact + lo;
}
// bias x log2(e).  A finite entry stays finite: entries near the type's lowest value act as a mask that still orders (a row of
// nothing but such entries is an ordinary softmax), only a true -inf removes a key.
__device__ __forceinline__ float sa_bias_log2(float b) {
  const float v = b * SA_LOG2E;
  return __builtin_isfinite(b) ? fminf(fmaxf(v, -3.3e38f), 3.3e38f) : v;
}
// position of query 0 of batch item b; far beyond every sequence it only saturates (no 32-bit wrap in key - query)
__device__ __forceinline__ int sa_q_offset(const SaRel& r, int b) {
  return min(max(r.q_offsets ? r.q_offsets[b] : r.q_offset, -(1 << 29)), 1 << 29);
}
// LDS rows of 2 W + 1 values per head: entry W + delta, delta = key position - query position in [-W, W]
template <int NW>
__device__ __forceinline__ void sa_fill_bias(float* lds, const SaRel& r, int head0, int nheads, int tid) {
  const int n = 2 * r.W + 1;
  for (int i = tid; i < n * nheads; i += 64 * NW) {
    const int h = i / n, d = i - h * n - r.W;
    lds[i] = sa_bias_log2(r.table[(long)sa_bucket(r, d) * r.H + head0 + h]);
  }
}

// one wave's share of a workgroup: the histogram over distances (hist[reach + delta], |delta| <= reach) summed into buckets j = w,
// w + waves, ...; out[j].  A bucket is a run of distances on one side.
template <int NW>
__device__ __forceinline__ void sa_bucket_sums(const SaRel& r, const float* hist, int reach, int num_buckets, float* out, int w, int lane) {
  for (int j = w; j < num_buckets; j += NW) {
    const bool pos = r.both && j >= r.half;
    const int jj = pos ? j - r.half : j;
    const int nlo = max(sa_bucket_lo(r, jj), pos ? 1 : 0);
    const int nhi = jj == r.half - 1 ? reach : min(sa_bucket_lo(r, jj + 1) - 1, reach);
    float a = 0.f;
    for (int n = nlo + lane; n <= nhi; n += 64) a += hist[reach + (pos ? n : -n)];
    if (!r.both && jj == 0)              // keys behind the query all count as distance 0
      for (int n = 1 + lane; n <= reach; n += 64) a += hist[reach + n];
    a = wave_sum(a);
    if (lane == 0) out[j] = a;
  }
}
// host side: validates the bias part of a descriptor and fills SaRel; false: rejected
static inline bool sa_make_rel(const dfold_rel_bias* d, int H, SaRel* r) {
  if (!d->table || d->num_buckets < 2 || d->num_buckets > 2 * DFOLD_REL_FAR) return false;
  const bool both = d->bidirectional != 0;
  if (both && (d->num_buckets & 1)) return false;
  const int half = both ? d->num_buckets / 2 : d->num_buckets, exact = half / 2, nfar = half - exact - 1;
  if (exact < 1 || nfar < 0 || nfar > DFOLD_REL_FAR) return false;
  r->table = d->table; r->q_offsets = d->q_offsets; r->q_offset = d->q_offset;
  r->H = H; r->half = half; r->exact = exact; r->nfar = nfar; r->both = both;
  int prev = exact;
  for (int i = 0; i < nfar; ++i) {
    if (d->far_border[i] < prev || d->far_border[i] > DFOLD_REL_MAX_DISTANCE) return false;
    r->far[i] = (int16_t)(prev = d->far_border[i]);
  }
  r->W = nfar ? prev : exact;
  return true;
}

// Launches with more than 64 KB of dynamic LDS need the kernel's limit raised, once per device and kernel (F: a type of the caller's own
// per kernel, so that each has its flags; setting it twice does no harm).
template <typename F, typename K>
static inline bool sa_raise_lds(K kernel, int lds) {
  static std::atomic<bool> done[64];
  int dev = 0;
  if (lds <= 65536) return true;
  if (hipGetDevice(&dev) != hipSuccess) return false;
  if (dev < 64 && done[dev].load(std::memory_order_relaxed)) return true;
  if (hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, SA_MAX_LDS) != hipSuccess) return false;
  if (dev < 64) done[dev].store(true, std::memory_order_relaxed);
  return true;
}

// what both directions require of the forward descriptor (an empty key axis is allowed: k, v may then be null)
static inline bool sa_desc_ok(const dfold_seq_attn_desc* d) {
  if (!d || !d->q || !d->o || (d->Lk > 0 && (!d->k || !d->v))) return false;
  if (d->dtype != DFOLD_DT_BF16 && d->dtype != DFOLD_DT_F16) return false;
  if (d->B <= 0 || d->Lq <= 0 || d->Lk < 0 || d->H <= 0 || d->Hkv <= 0 || d->H % d->Hkv) return false;
  if (d->D <= 0 || d->D > 128 || d->D % 8 || d->Lq > (1 << 30) || d->Lk > (1 << 30)) return false;
  if (((uintptr_t)d->q | (uintptr_t)d->k | (uintptr_t)d->v | (uintptr_t)d->o | (uintptr_t)d->ws) & 15) return false;
  const int64_t st[12] = {d->q_sb, d->q_sl, d->q_sh, d->k_sb, d->k_sl, d->k_sh, d->v_sb, d->v_sl, d->v_sh, d->o_sb, d->o_sl, d->o_sh};
  for (int i = 0; i < 12; ++i)
    if (st[i] % 8 || st[i] < 0) return false;
  if (d->q_sl >= SA_MAX_ROW || d->k_sl >= SA_MAX_ROW || d->v_sl >= SA_MAX_ROW) return false;
  // scale, scale x log2 e and the forward's threshold 8 / (scale x log2 e) are normal fp32 numbers
  const float sc = d->scale < 0.f ? -d->scale : d->scale;
  if (!(sc >= 0x1p-120f && sc <= 0x1p120f)) return false;
  return d->mask_sb >= 0;
}
