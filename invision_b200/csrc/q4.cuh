// q4.cuh -- linears over 4-bit weights: y[m][n] = sum_k x[m][k] (c[n][k] - z[n][k / g]) s[n][k / g].
//
// Device layout.  The weight is cut into blocks of 16 rows x 128 columns, a row tile's blocks one
// after another along K (rows and columns past the weight's end hold c = z = 8, s = 0).  A block is
//   codes [2][32 lanes][4 words] | scales [128 / g][16] fp32 | zeros [128 / g][16] bytes
// where lane (r, t) = 4 r + t holds row r (first half) and r + 8 (second), and its word w the 8
// columns 32 w + 8 t + j, nibble j: the A fragments of m16n8k16 without a shuffle, 512 contiguous
// bytes for each load of a warp.  A gate/up weight puts gate rows 8 i .. 8 i + 7 in rows 0..7 of
// tile i and the matching up rows in 8..15, so that both halves of a pair meet in one thread.
#pragma once
#include <cuda_fp16.h>
#include <stdint.h>

#include "ptx.cuh"

namespace envg {

constexpr int Q4_ROWS = 16, Q4_COLS = 128;
constexpr int SITE_Q4_ZERO = 1004;  // status[1]: a zero point above 15
__host__ __device__ constexpr int q4_block_bytes(int group) { return 1024 + 80 * (Q4_COLS / group); }

struct Q4View {
  const uint8_t* base;
  int tiles, kblocks;  // row tiles, blocks along K
  int group, gate_up;
  int64_t N, K;        // logical rows and columns
};

// Row of the caller's weight that row r of tile i holds, or -1.
ENVG_DEV int64_t q4_src_row(const Q4View& w, int64_t tile, int r) {
  if (w.gate_up) {
    const int64_t half = w.N / 2, j = tile * 8 + (r & 7);
    return j < half ? (r < 8 ? j : half + j) : -1;
  }
  const int64_t n = tile * 16 + r;
  return n < w.N ? n : -1;
}

// Lays out codes [N][ceil(K / 2)] (low nibble = even column), scales and zeros [N][ceil(K / g)].
// One CTA of 256 threads per block; thread i makes word i of the codes.
__global__ void __launch_bounds__(256) k_q4_pack(const Q4View w, uint8_t* out, const uint8_t* codes, const float* scales,
                                                 const uint8_t* zeros, int* status) {
  const int64_t blk = blockIdx.x, tile = blk / w.kblocks, kb = blk % w.kblocks;
  const int bytes = q4_block_bytes(w.group), per = Q4_COLS / w.group;
  uint8_t* dst = out + blk * bytes;
  const int64_t ldc = (w.K + 1) / 2, ngroups = (w.K + w.group - 1) / w.group;
  {
    const int i = threadIdx.x, hi = i >> 7, lane = (i >> 2) & 31, word = i & 3;
    const int64_t n = q4_src_row(w, tile, (lane >> 2) + 8 * hi);
    const int64_t k0 = kb * Q4_COLS + 32 * word + 8 * (lane & 3);
    uint32_t v = 0;
    for (int j = 0; j < 8; ++j) {
      const int64_t k = k0 + j;
      uint32_t c = 8;
      if (n >= 0 && k < w.K) {
        const uint8_t byte = codes[n * ldc + (k >> 1)];
        c = (k & 1) ? byte >> 4 : byte & 15;
      }
      v |= c << (4 * j);
    }
    reinterpret_cast<uint32_t*>(dst)[i] = v;
  }
  for (int i = threadIdx.x; i < 16 * per; i += 256) {
    const int64_t n = q4_src_row(w, tile, i & 15);
    const int64_t gi = kb * per + i / 16;
    const bool in = n >= 0 && gi < ngroups;
    reinterpret_cast<float*>(dst + 1024)[i] = in ? scales[n * ngroups + gi] : 0.0f;
    const uint8_t z = in && zeros ? zeros[n * ngroups + gi] : 8;
    if (z > 15) {
      atomicExch(status, -1);  // ENVG_ERR_ARG
      atomicExch(status + 1, SITE_Q4_ZERO);
    }
    dst[1024 + 64 * per + i] = z & 15;
  }
}

// Epilogues (ENVG_EPI_*): y + bias, silu(gate) * up, or dst + g (y + bias).
struct Q4Args {
  Q4View w;
  const float* x;
  float* dst;
  int64_t ldx, ldd;
  int M, mode;
  const float *bias, *gate;
};
constexpr int Q4_PLAIN = 0, Q4_SILU_GATE = 1, Q4_GATED_RES = 2;

// Stores output column n of row m; v0 and v1 are rows r and r + 8 of the tile (SiLU gate: the pair).
ENVG_DEV void q4_store(const Q4Args& a, int64_t tile, int r, int m, float v0, float v1) {
  float* row = a.dst + (int64_t)m * a.ldd;
  if (a.mode == Q4_SILU_GATE) {
    const int64_t half = a.w.N / 2, j = tile * 8 + r;
    if (j >= half) return;
    if (a.bias) v0 += a.bias[j], v1 += a.bias[half + j];
    row[j] = v0 / (1.0f + expf(-v0)) * v1;
    return;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t n = tile * 16 + r + 8 * i;
    if (n >= a.w.N) continue;
    float v = i ? v1 : v0;
    if (a.bias) v += a.bias[n];
    row[n] = a.mode == Q4_GATED_RES ? fmaf(a.gate[n], v, row[n]) : v;
  }
}

// One warp per (tile, row m), one lane per (r, t): plain fp32 products in the layout's order.
__global__ void __launch_bounds__(128) k_q4_simple(const Q4Args a) {
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
  const int64_t tile = (int64_t)blockIdx.x * 4 + threadIdx.x / 32;
  const int m = blockIdx.y;
  if (tile >= a.w.tiles) return;
  const int bytes = q4_block_bytes(a.w.group), per = Q4_COLS / a.w.group;
  float acc[2] = {};
  for (int kb = 0; kb < a.w.kblocks; ++kb) {
    const uint8_t* blk = a.w.base + (tile * a.w.kblocks + kb) * bytes;
    for (int i = 0; i < 2; ++i)
      for (int w = 0; w < 4; ++w) {
        const uint32_t v = reinterpret_cast<const uint32_t*>(blk)[i * 128 + lane * 4 + w];
        const int gi = 32 * w / a.w.group;
        const float s = reinterpret_cast<const float*>(blk + 1024)[gi * 16 + r + 8 * i];
        const int z = blk[1024 + 64 * per + gi * 16 + r + 8 * i];
        float part = 0.0f;
        for (int j = 0; j < 8; ++j) {
          const int64_t k = (int64_t)kb * Q4_COLS + 32 * w + 8 * t + j;
          if (k < a.w.K) part = fmaf(a.x[(int64_t)m * a.ldx + k], (float)((int)((v >> (4 * j)) & 15u) - z), part);
        }
        acc[i] = fmaf(part, s, acc[i]);
      }
  }
  for (int o = 1; o < 4; o <<= 1)
    for (int i = 0; i < 2; ++i) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], o);
  if (t == 0) q4_store(a, tile, r, m, acc[0], acc[1]);
}

}  // namespace envg
