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

#include "mma16.cuh"
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

// k_q4: y = x . W^T over the 4-bit blocks, 4 NT rows of x per launch row.
//
// Mathematics.  Of a block, group gi adds s[n][gi] sum_k (c[n][k] - z[n][gi]) x[m][k].  The products
// run on the tensor cores as m16n8k16: c - z, exact as an fp16, is the 16-row operand (c or 16 c is
// put into the mantissa of 1024, then one subtraction or multiply-add.  A bare c would be a
// subnormal, which the cores align by its nominal exponent and so lose up to ten low bits of x);
// x is the 8-column one, each row of it in two fp16 parts in adjacent columns, scaled by a power of
// two per (row, block) so that its largest value is in [2^14, 2^15).  Each group's fp32 sum starts
// from zero, gets both parts added and is then multiplied by its scale: nothing is rounded to 16
// bits, and the cores' cutting off of low bits stays within one group.
//
// Split.  A cluster of CTAs (one CTA of 16 warps per SM) takes a run of row tiles, each CTA a range
// of K, as many CTAs as fill the GPU when there are few tiles.  Up to R tiles at a time, the CTA's
// (tile, block) pairs are cut evenly among its warps, each of which streams its run of blocks
// through a ring of its own (a lane copies the codes that it will read itself) and leaves one sum
// per tile it touched in shared memory; the sums are added in warp order and, in a cluster, handed
// to the tile's owner and added in rank order.  Weights do not depend on the previous kernel: the
// ring starts before waiting for it.
constexpr int Q4_WARPS = 16, Q4_THREADS = 32 * Q4_WARPS;
constexpr int Q4_SMEM = 227 * 1024;

struct Q4Plan {
  int splits;         // CTAs of a cluster: K ranges
  int clusters;       // runs of tiles
  int kb_per;         // blocks of K per CTA
  int stages;         // ring depth: 6, 4 or 3
  int vec;            // rows of x are 16-byte aligned
};
template <int NT>
struct Q4Smem {
  static constexpr int R = NT == 4 ? 16 : 32;   // tiles at a time
  static constexpr int SUMS = NT * 2 * 32 * 4;  // bytes of one tile's sums
  static constexpr int SLOTS = (R + Q4_WARPS) * SUMS;
  static constexpr int RECV = R * SUMS;       // [ranks][tiles of the owner], used by clusters
  static constexpr int X_ROW = 4 * Q4_COLS;   // bytes of x's parts per (row, block)
  static constexpr int FIXED = SLOTS + RECV;
  __host__ __device__ static int x_bytes(int kb) { return kb * 4 * NT * (X_ROW + 4); }
  __host__ __device__ static int total(int kb, int stages, int group) {
    return FIXED + x_bytes(kb) + Q4_WARPS * stages * q4_block_bytes(group);
  }
};

ENVG_DEV void st_cluster_f2(uint32_t addr, float x, float y) {
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(addr), "f"(x), "f"(y) : "memory");
}

template <int NT, int GROUP>
__global__ void __launch_bounds__(Q4_THREADS, 1) k_q4(const Q4Args a, const Q4Plan p) {
  using S = Q4Smem<NT>;
  constexpr int R = S::R, BLOCK = q4_block_bytes(GROUP), PER = Q4_COLS / GROUP, MC = 4 * NT;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  float* slots = reinterpret_cast<float*>(smem);
  float* recv = reinterpret_cast<float*>(smem + S::SLOTS);
  uint8_t* xf = smem + S::FIXED;                                         // [kb][word][row][part][t] 16 bytes
  float* xs = reinterpret_cast<float*>(xf + p.kb_per * MC * S::X_ROW);  // [kb][row] 2^-e
  uint8_t* ring = xf + S::x_bytes(p.kb_per) + warp * p.stages * BLOCK;

  const int rank = p.splits > 1 ? (int)cluster_ctarank() : 0, cl = blockIdx.x / p.splits;
  const int kb0 = rank * p.kb_per, kbn = max(0, min(p.kb_per, a.w.kblocks - kb0));
  const int tile0 = (int)((int64_t)a.w.tiles * cl / p.clusters), tile1 = (int)((int64_t)a.w.tiles * (cl + 1) / p.clusters);
  const int m0 = blockIdx.y * MC, mn = min(MC, a.M - m0);

  // the warp's blocks: of each round (R tiles), an even share of its (tile, block) pairs
  auto share = [&](int r0, int w) { return min(R, tile1 - r0) * kbn * w / Q4_WARPS; };
  const int stage_end = p.stages * BLOCK;
  const uint32_t ring_s = smem_u32(ring) + lane * 16;
  int fr = tile0, left = 0, run = 0;  // fetching: the round, its blocks left, those up to the end of their row
  const uint8_t* next = nullptr;      // the lane's piece of the next one
  auto fetch_round = [&]() {
    const int i = share(fr, warp), j = kbn > 0 ? i / kbn : 0;
    left = share(fr, warp + 1) - i;
    run = min(left, (j + 1) * kbn - i);
    next = a.w.base + ((int64_t)(fr + j) * a.w.kblocks + kb0 + i - j * kbn) * BLOCK + lane * 16;
  };
  fetch_round();
  auto fetch = [&](int at) {  // one group of copies to ring offset `at`, empty past the warp's last block
    if (run == 0) {
      if (left > 0) {
        run = min(left, kbn);
        next += (int64_t)(a.w.kblocks - kbn) * BLOCK;
      } else {
        while (left == 0 && fr + R < tile1) fr += R, fetch_round();
      }
    }
    if (run > 0) {
      copy16_async(ring_s + at, next);
      copy16_async(ring_s + at + 512, next + 512);
      if (lane < 5 * PER) copy16_async(ring_s + at + 1024, next + 1024);
      --left, --run;
      next += BLOCK;
    }
    copy_group_end();
  };
  for (int i = 0; i < p.stages; ++i) fetch(i * BLOCK);
  griddep_wait();
  griddep_launch_dependents();

  // x of this K range as operand parts: a warp takes 128 columns of a row at a time
  constexpr int AHEAD = 8;  // loads of a warp under way at a time
  for (int i0 = warp; i0 < kbn * MC; i0 += AHEAD * Q4_WARPS) {
    float4 in[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int i = i0 + u * Q4_WARPS, kb = i / MC, m = i % MC, k = (kb0 + kb) * Q4_COLS + 4 * lane;
      in[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (kb < kbn && m < mn) {
        const float* src = a.x + (int64_t)(m0 + m) * a.ldx + k;
        if (k + 3 < a.w.K) {
          in[u] = ld_f4(src, p.vec != 0);
        } else {
          if (k < a.w.K) in[u].x = src[0];
          if (k + 1 < a.w.K) in[u].y = src[1];
          if (k + 2 < a.w.K) in[u].z = src[2];
        }
      }
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int i = i0 + u * Q4_WARPS, kb = i / MC, m = i % MC;
      if (kb >= kbn) break;
      float4 v = in[u];
      float top = fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w)));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const int e = scale_exp(top);
      const float up = pow2(e);
      v.x *= up, v.y *= up, v.z *= up, v.w *= up;
      const __half2 h0 = __floats2half2_rn(v.x, v.y), h1 = __floats2half2_rn(v.z, v.w);
      const float2 b0 = __half22float2(h0), b1 = __half22float2(h1);
      const uint32_t l0 = h2_bits(__floats2half2_rn(v.x - b0.x, v.y - b0.y)), l1 = h2_bits(__floats2half2_rn(v.z - b1.x, v.w - b1.y));
      // lanes 2 i and 2 i + 1 hold nibbles 0..3 and 4..7 of a word: the even lane collects the high
      // parts, the odd one the low parts, as the pairs (0, 4), (1, 5), (2, 6), (3, 7)
      const bool odd = lane & 1;
      const uint32_t s0 = __shfl_xor_sync(0xffffffffu, odd ? h2_bits(h0) : l0, 1), s1 = __shfl_xor_sync(0xffffffffu, odd ? h2_bits(h1) : l1, 1);
      const uint32_t a0 = odd ? s0 : h2_bits(h0), a1 = odd ? s1 : h2_bits(h1), c0 = odd ? l0 : s0, c1 = odd ? l1 : s1;
      uint4 out;
      out.x = __byte_perm(a0, c0, 0x5410), out.y = __byte_perm(a0, c0, 0x7632);
      out.z = __byte_perm(a1, c1, 0x5410), out.w = __byte_perm(a1, c1, 0x7632);
      const int word = lane >> 3, tt = (lane >> 1) & 3;
      *reinterpret_cast<uint4*>(xf + ((((kb * 4 + word) * MC + m) * 2 + (odd ? 1 : 0)) * 4 + tt) * 16) = out;
      if (lane == 0) xs[kb * MC + m] = pow2(-e);
    }
  }
  if (p.splits > 1) cluster_sync();  // every CTA of the cluster is there to be written to
  else __syncthreads();

  const uint32_t mask0 = in_register(0x000F000Fu), mask1 = in_register(0x00F000F0u), magic = in_register(0x64006400u);
  const __half2 c16 = __float2half2_rn(0.0625f);
  int at = 0;  // ring offset
  for (int r0 = tile0; r0 < tile1; r0 += R) {
    const int tiles = min(R, tile1 - r0), nb = tiles * kbn;
    int i = share(r0, warp), j = kbn > 0 ? i / kbn : 0;
    int more = share(r0, warp + 1) - i;              // blocks of the round left
    int row = min(more, (j + 1) * kbn - i);          // of them in this tile
    const uint8_t* xk = xf + (i - j * kbn) * (MC * S::X_ROW) + g * 64 + t * 16;
    const float* xsk = xs + (i - j * kbn) * MC + t;
    float acc[NT][2] = {};
    for (; more > 0; --more) {
      if (p.stages == 6) copy_groups_wait<5>();
      else if (p.stages == 4) copy_groups_wait<3>();
      else copy_groups_wait<2>();
      __syncwarp();  // the scales were copied by other lanes
      const uint8_t* blk = ring + at;
      const uint4 q0 = *reinterpret_cast<const uint4*>(blk + lane * 16), q1 = *reinterpret_cast<const uint4*>(blk + 512 + lane * 16);
      const uint32_t w0[4] = {q0.x, q0.y, q0.z, q0.w}, w1[4] = {q1.x, q1.y, q1.z, q1.w};
      float sum[NT][2] = {};
#pragma unroll
      for (int gi = 0; gi < PER; ++gi) {
        const float s0 = *reinterpret_cast<const float*>(blk + 1024 + (gi * 16 + g) * 4), s1 = *reinterpret_cast<const float*>(blk + 1024 + (gi * 16 + g + 8) * 4);
        const uint32_t z0 = blk[1024 + 64 * PER + gi * 16 + g], z1 = blk[1024 + 64 * PER + gi * 16 + g + 8];
        // 1024 + z, and -(64 + z) for 16 times the code
        const __half2 zl0 = bits_h2(z0 * 0x00010001u + magic), zh0 = bits_h2(z0 * 0x00100010u + 0xD400D400u);
        const __half2 zl1 = bits_h2(z1 * 0x00010001u + magic), zh1 = bits_h2(z1 * 0x00100010u + 0xD400D400u);
        float d[2][NT][4];  // two chains of products where a group has more than one word
#pragma unroll
        for (int wi = 0; wi < 4 / PER; ++wi) {
          const int w = gi * (4 / PER) + wi;
          uint4 xw[NT];  // the word's eight columns of x, for both of its products
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) xw[nt] = *reinterpret_cast<const uint4*>(xk + (w * MC + 4 * nt) * 128);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t u0 = h ? w0[w] >> 8 : w0[w], u1 = h ? w1[w] >> 8 : w1[w];
            const uint32_t A0 = h2_bits(__hsub2(bits_h2(and_or(u0, mask0, magic)), zl0));
            const uint32_t A1 = h2_bits(__hsub2(bits_h2(and_or(u1, mask0, magic)), zl1));
            const uint32_t A2 = h2_bits(__hfma2(bits_h2(and_or(u0, mask1, magic)), c16, zh0));
            const uint32_t A3 = h2_bits(__hfma2(bits_h2(and_or(u1, mask1, magic)), c16, zh1));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              const uint32_t bb[2] = {h ? xw[nt].z : xw[nt].x, h ? xw[nt].w : xw[nt].y};
              if (wi < 2 && h == 0) mma_f16_zero(d[wi & 1][nt], A0, A1, A2, A3, bb);
              else mma_f16(d[wi & 1][nt], A0, A1, A2, A3, bb);
            }
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i2 = 0; i2 < 2; ++i2) {
            float v = d[0][nt][2 * i2] + d[0][nt][2 * i2 + 1];
            if (PER < 4) v += d[1][nt][2 * i2] + d[1][nt][2 * i2 + 1];
            sum[nt][i2] = fmaf(v, i2 ? s1 : s0, sum[nt][i2]);
          }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float xsc = xsk[4 * nt];
        acc[nt][0] = fmaf(sum[nt][0], xsc, acc[nt][0]);
        acc[nt][1] = fmaf(sum[nt][1], xsc, acc[nt][1]);
      }
      __syncwarp();  // every lane has read the stage
      fetch(at);
      at += BLOCK;
      if (at == stage_end) at = 0;
      xk += MC * S::X_ROW, xsk += MC;
      if (--row == 0) {  // the warp leaves the tile
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          *reinterpret_cast<float2*>(slots + ((j + warp) * NT + nt) * 64 + 2 * lane) = make_float2(acc[nt][0], acc[nt][1]);
          acc[nt][0] = acc[nt][1] = 0.0f;
        }
        ++j;
        row = min(more - 1, kbn);
        xk = xf + g * 64 + t * 16, xsk = xs + t;
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < tiles * NT * 32; i += Q4_THREADS) {
      const int j = i / (NT * 32), nt = (i / 32) % NT, ln = i & 31;
      float2 v = make_float2(0.0f, 0.0f);
      if (kbn > 0) {
        // warp of block b: the last w whose share starts at or before b
        const int wa = (int)(((int64_t)j * kbn + 1) * Q4_WARPS - 1) / nb, wb = (int)(((int64_t)(j + 1) * kbn) * Q4_WARPS - 1) / nb;
        for (int w = wa; w <= wb; ++w) {
          if (nb * w / Q4_WARPS == nb * (w + 1) / Q4_WARPS) continue;  // a warp without a block
          const float2 s = *reinterpret_cast<const float2*>(slots + ((j + w) * NT + nt) * 64 + 2 * ln);
          v.x += s.x, v.y += s.y;
        }
      }
      if (p.splits == 1) {
        const int m = 4 * nt + (ln & 3);
        if (m < mn) q4_store(a, r0 + j, ln >> 2, m0 + m, v.x, v.y);
      } else {
        const int owner = j % p.splits, at = rank * (R / p.splits) + j / p.splits;
        st_cluster_f2(mapa_shared(smem_u32(recv + (at * NT + nt) * 64 + 2 * ln), owner), v.x, v.y);
      }
    }
    if (p.splits == 1) {
      __syncthreads();
      continue;
    }
    cluster_sync();
    const int each = R / p.splits;
    for (int i = threadIdx.x; i < each * NT * 32; i += Q4_THREADS) {
      const int jj = i / (NT * 32), j = jj * p.splits + rank, nt = (i / 32) % NT, ln = i & 31, m = 4 * nt + (ln & 3);
      if (j >= tiles || m >= mn) continue;
      float2 v = make_float2(0.0f, 0.0f);
      for (int q = 0; q < p.splits; ++q) {
        const float2 s = *reinterpret_cast<const float2*>(recv + ((q * each + jj) * NT + nt) * 64 + 2 * ln);
        v.x += s.x, v.y += s.y;
      }
      q4_store(a, r0 + j, ln >> 2, m0 + m, v.x, v.y);
    }
    if (r0 + R < tile1) cluster_sync();  // the next round's sums may come when all have read these
  }
}

}  // namespace envg
