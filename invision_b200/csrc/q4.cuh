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

// k_q4: y = x . W^T over the 4-bit blocks, MC rows of x per launch row.
//
// Mathematics.  Of a block, group gi adds s[n][gi] sum_k (c[n][k] - z[n][gi]) x[m][k].  The codes are
// the 16-row operand of the tensor cores' products, x the 8-column one, in as many parts as fp32
// accuracy takes; a group's sum starts from zero and is multiplied by its scale in fp32.  Two forms:
//   integers (HALF false): codes as unsigned bytes (two logic operations unpack four), x per (row,
//     scale group) as a 31-bit fixed-point number in four signed digits to the base 256, a row's digits
//     in four adjacent columns, two rows to a product.  The 32-bit sums are exact; a thread joins its
//     two digits, takes off z sum(x) in integers, converts once; a row's two threads are added when the
//     tile is left.
//   halves (HALF true): c - z exact as an fp16 (put into the mantissa of 1024, then one subtraction
//     or multiply-add; a bare c would be a subnormal, which the cores align by its nominal exponent
//     and so lose up to ten low bits of x), x in two fp16 parts in adjacent columns, scaled by a power
//     of two per (row, block), four rows to a product.  The low part is held 2^11 larger: values down to
//     2^-28 of the block's largest keep their 22 bits, down to 2^-17 without it.
// The integer form unpacks a block in 24 operations against 72, the other form spends 4 per group on
// four rows against 22; the kernel is bound by its warps' own steps (16 warps an SM, issue slots 54%
// busy, DRAM 40%), so few rows take integers and many rows halves.  Measured, us (integers / halves):
// 1 x 2560 x 19456, groups of 64: 7.9 / 13.7; 4 x 4096 x 36864, groups of 128: 20.4 / 28.1 (4.0 TB/s);
// 4 x 9728 x 2560, groups of 32: 9.9 / 10.2; 16 x 9728 x 2560, groups of 32: 21.8 / 14.4.  These
// weights stay in L2 from call to call; from HBM the first takes 1.2 us more, the second 1.0.
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
  int splits, log_splits;  // CTAs of a cluster, a power of two: K ranges
  int clusters;       // runs of tiles
  int kb_per;         // blocks of K per CTA
  int stages;         // ring depth: 6, 4 or 3
  int vec;            // rows of x are 16-byte aligned
  int each, rest;     // tiles per cluster; the first `rest` clusters take one more
};
template <int NT, bool HALF>
struct Q4Smem {
  static constexpr int RT = HALF ? 4 : 2;       // rows of x to a product
  static constexpr int MC = RT * NT;
  static constexpr int R = 32;                  // tiles at a time
  static constexpr int SUMS = MC * 64;          // bytes of one tile's sums
  static constexpr int SLOTS = (R + Q4_WARPS) * SUMS;
  static constexpr int RECV = R * SUMS;         // [ranks][tiles of the owner], used by clusters
  static constexpr int FIXED = SLOTS + RECV + R * 8;  // and each tile's first and last warp
  static constexpr int X_ROW = 4 * Q4_COLS;     // bytes of x's parts per (row, block)
  // parts and their weight, or digits with their sum and weight per scale group and pair of digits
  __host__ __device__ static int x_bytes(int kb, int group) {
    return (int)((kb * MC * (X_ROW + (HALF ? 4 : 16 * (Q4_COLS / group))) + 15) & ~15);
  }
  __host__ __device__ static int total(int kb, int stages, int group) {
    return FIXED + x_bytes(kb, group) + Q4_WARPS * stages * q4_block_bytes(group);
  }
};

ENVG_DEV void st_cluster_f2(uint32_t addr, float x, float y) {
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(addr), "f"(x), "f"(y) : "memory");
}

template <int NT, int GROUP, bool HALF>
__global__ void __launch_bounds__(Q4_THREADS, 1) k_q4(const Q4Args a, const Q4Plan p) {
  using S = Q4Smem<NT, HALF>;
  constexpr int R = S::R, RT = S::RT, BLOCK = q4_block_bytes(GROUP), PER = Q4_COLS / GROUP, MC = S::MC;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  float* slots = reinterpret_cast<float*>(smem);
  float* recv = reinterpret_cast<float*>(smem + S::SLOTS);
  int2* ends = reinterpret_cast<int2*>(smem + S::SLOTS + S::RECV);
  // integers: [kb][word pair][row][digit][t][word] 8 bytes; halves: [kb][word][row][part][t] 16 bytes
  uint8_t* xf = smem + S::FIXED;
  float* xs = reinterpret_cast<float*>(xf + p.kb_per * MC * S::X_ROW);  // halves: weights [kb][row]
  int2* xt = reinterpret_cast<int2*>(xs);  // integers: (sum of digits, weight as a float) [kb][group][row][digit pair]
  uint8_t* ring = xf + S::x_bytes(p.kb_per, GROUP) + warp * p.stages * BLOCK;

  const int rank = p.splits > 1 ? (int)cluster_ctarank() : 0, cl = blockIdx.x >> p.log_splits;
  const int kb0 = rank * p.kb_per, kbn = max(0, min(p.kb_per, a.w.kblocks - kb0));
  const int tile0 = cl * p.each + min(cl, p.rest), tile1 = tile0 + p.each + (cl < p.rest ? 1 : 0);
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

  // x of this K range in parts: a warp takes 128 columns of a row at a time.  A single row goes without
  // its product's second one, which keeps what shared memory holds: a row's columns of the products are
  // its own, and those are never stored.
  constexpr int AHEAD = 10;  // loads of a warp under way at a time
  const bool one = MC == 2 && mn == 1;
  for (int i0 = warp; i0 < (one ? kbn : kbn * MC); i0 += AHEAD * Q4_WARPS) {
    float4 in[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int i = i0 + u * Q4_WARPS, kb = one ? i : i / MC, m = one ? 0 : i % MC, k = (kb0 + kb) * Q4_COLS + 4 * lane;
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
      const int i = i0 + u * Q4_WARPS, kb = one ? i : i / MC, m = one ? 0 : i % MC;
      if (kb >= kbn) break;
      float4 v = in[u];
      // magnitudes as integers order as floats do, and keep a NaN on top
      uint32_t top = max(max(__float_as_uint(v.x) & 0x7fffffffu, __float_as_uint(v.y) & 0x7fffffffu),
                         max(__float_as_uint(v.z) & 0x7fffffffu, __float_as_uint(v.w) & 0x7fffffffu));
      // integers: the largest of the scale group, whose sums the digits end in; halves: of the block
      if (HALF || GROUP == 128) {
        top = __reduce_max_sync(0xffffffffu, top);
      } else if (GROUP == 32) {
#pragma unroll
        for (int o = 1; o < GROUP / 4; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      } else {
        uint32_t all = 0;
#pragma unroll
        for (int gi = 0; gi < PER; ++gi) {
          const bool here = lane / (GROUP / 4) == gi;
          const uint32_t largest = __reduce_max_sync(0xffffffffu, here ? top : 0u);
          if (here) all = largest;
        }
        top = all;
      }
      const bool odd = lane & 1;
      const int word = lane >> 3, tt = (lane >> 1) & 3;
      const float nan = __int_as_float(0x7fc00000);  // an infinity or a NaN makes its row's outputs NaN
      if (HALF) {
        const int e = scale_exp(__uint_as_float(top));
        const float up = pow2(e), y0 = v.x * up, y1 = v.y * up, y2 = v.z * up, y3 = v.w * up;
        const __half2 h0 = __floats2half2_rn(y0, y1), h1 = __floats2half2_rn(y2, y3);
        const float2 b0 = __half22float2(h0), b1 = __half22float2(h1);
        const uint32_t l0 = h2_bits(__floats2half2_rn((y0 - b0.x) * 2048.0f, (y1 - b0.y) * 2048.0f));
        const uint32_t l1 = h2_bits(__floats2half2_rn((y2 - b1.x) * 2048.0f, (y3 - b1.y) * 2048.0f));
        // lanes 2 i and 2 i + 1 hold nibbles 0..3 and 4..7 of a word: the even lane collects the high
        // parts, the odd one the low parts, as the pairs (0, 4), (1, 5), (2, 6), (3, 7)
        const uint32_t r0 = __shfl_xor_sync(0xffffffffu, odd ? h2_bits(h0) : l0, 1), r1 = __shfl_xor_sync(0xffffffffu, odd ? h2_bits(h1) : l1, 1);
        const uint32_t a0 = odd ? r0 : h2_bits(h0), a1 = odd ? r1 : h2_bits(h1), c0 = odd ? l0 : r0, c1 = odd ? l1 : r1;
        *reinterpret_cast<uint4*>(xf + ((((kb * 4 + word) * MC + m) * 2 + (odd ? 1 : 0)) * 4 + tt) * 16) =
            make_uint4(__byte_perm(a0, c0, 0x5410), __byte_perm(a0, c0, 0x7632), __byte_perm(a1, c1, 0x5410), __byte_perm(a1, c1, 0x7632));
        if (lane == 0) xs[kb * MC + m] = top >= 0x7f800000u ? nan : pow2(-e);
      } else {
        const int e = fixed_exp(__uint_as_float(top));
        float up = pow2(e), wt = pow2(-e);
        if (e > 126) {  // a row near fp32's end: in two exact steps, and its unit may be a denormal
          up = pow2(e - 23), wt = fixed_unit(e);
          v = make_float4(v.x * 8388608.0f, v.y * 8388608.0f, v.z * 8388608.0f, v.w * 8388608.0f);
        }
        const uint32_t x0 = digits256(__float2int_rn(v.x * up)), x1 = digits256(__float2int_rn(v.y * up));
        const uint32_t x2 = digits256(__float2int_rn(v.z * up)), x3 = digits256(__float2int_rn(v.w * up));
        // A word's columns go in as (0, 2, 4, 6) and (1, 3, 5, 7); lanes 2 i and 2 i + 1 hold columns
        // 0..3 and 4..7.  The even lane collects digits 0 and 1, the odd one digits 2 and 3.
        const uint32_t l0 = __byte_perm(x0, x2, 0x5140), l1 = __byte_perm(x1, x3, 0x5140);  // digits 0, 1
        const uint32_t h0 = __byte_perm(x0, x2, 0x7362), h1 = __byte_perm(x1, x3, 0x7362);  // digits 2, 3
        const uint32_t r0 = __shfl_xor_sync(0xffffffffu, odd ? l0 : h0, 1), r1 = __shfl_xor_sync(0xffffffffu, odd ? l1 : h1, 1);
        const uint32_t lo0 = odd ? r0 : l0, lo1 = odd ? r1 : l1, hi0 = odd ? h0 : r0, hi1 = odd ? h1 : r1;
        uint2* out = reinterpret_cast<uint2*>(xf + (((((kb * 2 + (word >> 1)) * MC + m) * 4 + (odd ? 2 : 0)) * 4 + tt) * 2 + (word & 1)) * 8);
        out[0] = make_uint2(__byte_perm(lo0, hi0, 0x5410), __byte_perm(lo1, hi1, 0x5410));
        out[8] = make_uint2(__byte_perm(lo0, hi0, 0x7632), __byte_perm(lo1, hi1, 0x7632));
        const int gi = lane / (GROUP / 4), pair = lane % (GROUP / 4);
        if (pair < 2) xt[((kb * PER + gi) * MC + m) * 2 + pair].y = __float_as_int((top >= 0x7f800000u ? nan : wt) * (pair ? 65536.0f : 1.0f));
      }
    }
  }
  if (p.splits > 1) cluster_sync();  // every CTA of the cluster is there to be written to
  else __syncthreads();
  if (!HALF) {
    // sums of x's digits per group, by products with codes of one
    for (int kb = warp; kb < kbn; kb += Q4_WARPS)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        int d[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint2 b = *reinterpret_cast<const uint2*>(xf + ((((kb * 2 + (w >> 1)) * MC + 2 * nt) * 4 + g) * 8 + t * 2 + (w & 1)) * 8);
          if (w % (4 / PER) == 0) mma_u8s8<true>(d, 0x01010101u, 0x01010101u, 0x01010101u, 0x01010101u, b.x, b.y);
          else mma_u8s8<false>(d, 0x01010101u, 0x01010101u, 0x01010101u, 0x01010101u, b.x, b.y);
          if (w % (4 / PER) == 4 / PER - 1 && g == 0) xt[((kb * PER + w / (4 / PER)) * MC + 2 * nt) * 2 + t].x = d[1] * 256 + d[0];
        }
      }
    __syncthreads();
  }

  const uint32_t nib = in_register(0x0F0F0F0Fu), mask0 = in_register(0x000F000Fu), mask1 = in_register(0x00F000F0u), magic = in_register(0x64006400u);
  const __half2 c16 = __float2half2_rn(0.0625f);
  int at = 0;  // ring offset
  for (int r0 = tile0; r0 < tile1; r0 += R) {
    const int tiles = min(R, tile1 - r0), nb = tiles * kbn;
    if (threadIdx.x < tiles && kbn > 0) {  // warp of block b: the last w whose share starts at or before b
      const int b = threadIdx.x * kbn;
      ends[threadIdx.x] = make_int2(((b + 1) * Q4_WARPS - 1) / nb, ((b + kbn) * Q4_WARPS - 1) / nb);
    }
    const int i = share(r0, warp);
    int j = kbn > 0 ? i / kbn : 0;
    int more = share(r0, warp + 1) - i;      // blocks of the round left
    int row = min(more, (j + 1) * kbn - i);  // of them in this tile
    int kb = i - j * kbn;
    const uint8_t* xk = xf + kb * (MC * S::X_ROW) + lane * 16;
    const int2* xtk = xt + kb * (PER * MC * 2) + t;
    const float* xsk = xs + kb * MC + t;
    float acc[NT][2] = {};
    for (; more > 0; --more) {
      if (p.stages == 6) copy_groups_wait<5>();
      else if (p.stages == 4) copy_groups_wait<3>();
      else copy_groups_wait<2>();
      __syncwarp();  // the scales were copied by other lanes
      const uint8_t* blk = ring + at;
      const uint4 q0 = *reinterpret_cast<const uint4*>(blk + lane * 16), q1 = *reinterpret_cast<const uint4*>(blk + 512 + lane * 16);
      const uint32_t w0[4] = {q0.x, q0.y, q0.z, q0.w}, w1[4] = {q1.x, q1.y, q1.z, q1.w};
      if constexpr (HALF) {
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
              const uint32_t a0 = h2_bits(__hsub2(bits_h2(and_or(u0, mask0, magic)), zl0));
              const uint32_t a1 = h2_bits(__hsub2(bits_h2(and_or(u1, mask0, magic)), zl1));
              const uint32_t a2 = h2_bits(__hfma2(bits_h2(and_or(u0, mask1, magic)), c16, zh0));
              const uint32_t a3 = h2_bits(__hfma2(bits_h2(and_or(u1, mask1, magic)), c16, zh1));
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                const uint32_t bb[2] = {h ? xw[nt].z : xw[nt].x, h ? xw[nt].w : xw[nt].y};
                if (wi < 2 && h == 0) mma_f16_zero(d[wi & 1][nt], a0, a1, a2, a3, bb);
                else mma_f16(d[wi & 1][nt], a0, a1, a2, a3, bb);
              }
            }
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i2 = 0; i2 < 2; ++i2) {
              float high = d[0][nt][2 * i2], low = d[0][nt][2 * i2 + 1];
              if (PER < 4) high += d[1][nt][2 * i2], low += d[1][nt][2 * i2 + 1];
              sum[nt][i2] = fmaf(fmaf(low, 1.0f / 2048.0f, high), i2 ? s1 : s0, sum[nt][i2]);
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float wt = xsk[4 * nt];
          acc[nt][0] = fmaf(sum[nt][0], wt, acc[nt][0]);
          acc[nt][1] = fmaf(sum[nt][1], wt, acc[nt][1]);
        }
      } else {
        int d[NT][4];
        uint4 xw[NT];  // x's digits for two words
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int gi = w / (4 / PER);
          if (w % 2 == 0)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) xw[nt] = *reinterpret_cast<const uint4*>(xk + ((w >> 1) * MC + 2 * nt) * 256);
          const uint32_t a0 = w0[w] & nib, a1 = w1[w] & nib, a2 = (w0[w] >> 4) & nib, a3 = (w1[w] >> 4) & nib;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const uint32_t b0 = w % 2 ? xw[nt].z : xw[nt].x, b1 = w % 2 ? xw[nt].w : xw[nt].y;
            if (w % (4 / PER) == 0) mma_u8s8<true>(d[nt], a0, a1, a2, a3, b0, b1);
            else mma_u8s8<false>(d[nt], a0, a1, a2, a3, b0, b1);
          }
          if (w % (4 / PER) == 4 / PER - 1) {
            const float s0 = *reinterpret_cast<const float*>(blk + 1024 + (gi * 16 + g) * 4), s1 = *reinterpret_cast<const float*>(blk + 1024 + (gi * 16 + g + 8) * 4);
            const int z0 = blk[1024 + 64 * PER + gi * 16 + g], z1 = blk[1024 + 64 * PER + gi * 16 + g + 8];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              const int2 xw = xtk[(gi * MC + 2 * nt) * 2];
              const float wt = __int_as_float(xw.y);
              acc[nt][0] = fmaf((float)(d[nt][1] * 256 + d[nt][0] - z0 * xw.x) * s0, wt, acc[nt][0]);
              acc[nt][1] = fmaf((float)(d[nt][3] * 256 + d[nt][2] - z1 * xw.x) * s1, wt, acc[nt][1]);
            }
          }
        }
      }
      __syncwarp();  // every lane has read the stage
      fetch(at);
      at += BLOCK;
      if (at == stage_end) at = 0;
      xk += MC * S::X_ROW, xtk += PER * MC * 2, xsk += MC;
      if (--row == 0) {  // the warp leaves the tile
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float* slot = slots + (j + warp) * (MC * 16) + nt * (RT * 16);
          if (HALF) {
            *reinterpret_cast<float2*>(slot + 2 * lane) = make_float2(acc[nt][0], acc[nt][1]);
          } else {
            const float y0 = acc[nt][0] + __shfl_xor_sync(0xffffffffu, acc[nt][0], 1);
            const float y1 = acc[nt][1] + __shfl_xor_sync(0xffffffffu, acc[nt][1], 1);
            if (!(t & 1)) *reinterpret_cast<float2*>(slot + lane) = make_float2(y0, y1);
          }
          acc[nt][0] = acc[nt][1] = 0.0f;
        }
        ++j;
        row = min(more - 1, kbn);
        xk = xf + lane * 16, xtk = xt + t, xsk = xs + t;
      }
    }
    __syncthreads();
    // item: (tile, product's rows of x, row g of the tile and row of x), as the slots hold them
    constexpr int ITEMS = MC * 8;  // of a tile
    for (int it = threadIdx.x; it < tiles * ITEMS; it += Q4_THREADS) {
      const int jt = it / ITEMS, q = it % ITEMS;
      float2 v = make_float2(0.0f, 0.0f);
      if (kbn > 0) {
        const int2 e = ends[jt];
        for (int w = e.x; w <= e.y; ++w) {
          if (nb * w / Q4_WARPS == nb * (w + 1) / Q4_WARPS) continue;  // a warp without a block
          const float2 s = *reinterpret_cast<const float2*>(slots + (jt + w) * (MC * 16) + 2 * q);
          v.x += s.x, v.y += s.y;
        }
      }
      if (p.splits == 1) {
        const int m = q / (8 * RT) * RT + q % RT;
        if (m < mn) q4_store(a, r0 + jt, q % (8 * RT) / RT, m0 + m, v.x, v.y);
      } else {
        const int owner = jt & (p.splits - 1), to = rank * (R >> p.log_splits) + (jt >> p.log_splits);
        st_cluster_f2(mapa_shared(smem_u32(recv + to * (MC * 16) + 2 * q), owner), v.x, v.y);
      }
    }
    if (p.splits == 1) {
      __syncthreads();
      continue;
    }
    cluster_sync();
    const int each = R >> p.log_splits;
    for (int it = threadIdx.x; it < each * ITEMS; it += Q4_THREADS) {
      const int jj = it / ITEMS, jt = (jj << p.log_splits) + rank, q = it % ITEMS, m = q / (8 * RT) * RT + q % RT;
      if (jt >= tiles || m >= mn) continue;
      float2 v = make_float2(0.0f, 0.0f);
      for (int r = 0; r < p.splits; ++r) {
        const float2 s = *reinterpret_cast<const float2*>(recv + (r * each + jj) * (MC * 16) + 2 * q);
        v.x += s.x, v.y += s.y;
      }
      q4_store(a, r0 + jt, q % (8 * RT) / RT, m0 + m, v.x, v.y);
    }
    if (r0 + R < tile1) cluster_sync();  // the next round's sums may come when all have read these
  }
}

}  // namespace envg
