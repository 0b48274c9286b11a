// Last step of the bias table's gradient (seq_attn_bwd.hip, seq_relpos.hip).
#pragma once
#include "dfold_common.h"

// dtable[bucket][head] = sum over the batch and the parts, in a fixed order: grid (H, buckets / 64), ws [B][H][per][nb]
static __global__ __launch_bounds__(1024) void seq_dtable_kernel(const float* __restrict__ ws, float* __restrict__ dtable, int nb, int B, int H,
                                                                 int per) {
  __shared__ float part[16][64];
  const int head = blockIdx.x, j = blockIdx.y * 64 + (threadIdx.x & 63), w = threadIdx.x >> 6;
  float a = 0.f;
  if (j < nb)
    for (long i = w; i < (long)B * per; i += 16) {
      const long b = i / per, r = i - b * per;
      a += ws[((b * H + head) * per + r) * nb + j];
    }
  part[w][threadIdx.x & 63] = a;
  __syncthreads();
  if (w == 0 && j < nb) {
    for (int k = 1; k < 16; ++k) a += part[k][threadIdx.x];
    dtable[(long)j * H + head] = a;
  }
}
